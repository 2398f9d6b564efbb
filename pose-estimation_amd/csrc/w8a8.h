// 8-bit products (w8a8.hip): shared declarations of the kernels and of their callers.
#pragma once
#include "../../include/posehip.h"
#include "common.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Rows of a tensor in up to three nested dimensions: row m -> element offset.  The inner sizes are n1, n2; a tensor whose
// rows are evenly spaced (flat) needs no division.
struct PhRowMap {
  unsigned n1, n2;
  int flat;
  int64_t s0, s1, s2;   // element strides
};

__host__ __device__ static inline int64_t ph_row_off(const PhRowMap& r, unsigned m) {
  if (r.flat) return (int64_t)m * r.s2;
  const unsigned t = m / r.n2, i2 = m - t * r.n2;
  const unsigned i0 = t / r.n1, i1 = t - i0 * r.n1;
  return (int64_t)i0 * r.s0 + (int64_t)i1 * r.s1 + (int64_t)i2 * r.s2;
}

// A launch holds fewer than 2^32 threads: a call of more rows than that is refused.
static inline bool ph_w8_fits_launch(int64_t blocks, int64_t threads) {
  return blocks * threads <= 0xff000000ll;   // (counts rounded up to whole blocks still fit)
}
static inline int ph_w8_launchable(int64_t blocks, int64_t threads) {
  if (ph_w8_fits_launch(blocks, threads)) return 0;
  ph_set_error("8-bit layer: %lld blocks of %lld threads are more than a launch holds: take the rows in parts",
               (long long)blocks, (long long)threads);
  return -1;
}

struct PhW8Params {
  const int8_t* q;       // 8-bit rows, K contiguous values each (rows 16-byte aligned, unless loose)
  PhRowMap qr;
  const float* qs;       // scale of each row [M]
  const int8_t* w;       // packed weight fragments [N16/16][K128/64][1024]
  const float* ws;       // scale of each channel [N16]
  const float* bias;     // [N16] or NULL
  const float* slope;    // [N16] or NULL
  int act;
  int stream;            // store past the caches
  int loose;             // rows start anywhere (ph_w8_choose_loose())
  unsigned M;
  int N, K, nkb, nnb;    // nkb = K128 / 64 fragments along K (even), nnb = N16 / 16 along N
  void* out;
  PhRowMap outr;
  int* parts;            // split along K: sums [part][M][N16]
};

// How a product is done: which kernel, in how many parts along K, and what that is expected to take.
struct PhW8Choice {
  int kernel, parts;
  float us;
};
PhW8Choice ph_w8_choose(int64_t M, int N, int nkb);
PhW8Choice ph_w8_choose_loose(int64_t M, int K, int N);   // kernel < 0: none takes them
int64_t ph_w8_parts_bytes(const PhW8Choice& c, int64_t M, int N);
int ph_launch_w8_product(const PhW8Params& p, const PhW8Choice& c, int out_type, hipStream_t st);

// Float rows that a product's blocks quantise themselves (p.q, p.qr and p.qs are not used).
struct FloatRows {
  const void* x;
  PhRowMap r;
};
bool ph_w8_few_float(int64_t M, int K);
int ph_launch_w8_few_float(const PhW8Params& p, const FloatRows& f, int x_type, int out_type, hipStream_t st);

#define PAIR_MAX 512   // widest rows of the kernels that quantise them themselves, and widest inner rows
bool ph_w8_rows_fit(int64_t M, int K, int N);
int ph_launch_w8_rows(const PhW8Params& p, const FloatRows& f, int x_type, int out_type, hipStream_t st);

struct PhW8Out {
  void* p;
  PhRowMap r;
  int64_t step;          // elements from a channel to the next (1, or a plane of f32 maps)
  int type;
};
struct PhW8Pair {
  const void* x;
  PhRowMap xr;
  unsigned M;
  int K, H, N, nkb1, nnb1, nkb2, nnb2, act1, act2;
  const int8_t *w1, *w2;
  const float *ws1, *bias1, *slope1, *ws2, *bias2, *slope2;
  int n_out;             // the result goes to each of these
  PhW8Out out[PH_MAX_DST + 1];
};
bool ph_w8_pair_fits(int K, int H, int N);
int ph_launch_w8_pair(const PhW8Pair& p, int x_type, hipStream_t st);
