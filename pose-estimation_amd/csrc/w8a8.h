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

struct PhW8Params {
  const int8_t* q;       // 8-bit rows, K contiguous values each (rows 16-byte aligned)
  PhRowMap qr;
  const float* qs;       // scale of each row [M]
  const int8_t* w;       // packed weight fragments [N16/16][K128/64][1024]
  const float* ws;       // scale of each channel [N16]
  const float* bias;     // [N16] or NULL
  const float* slope;    // [N16] or NULL
  int act;
  int stream;            // store past the caches
  unsigned M;
  int N, K, nkb, nnb;    // nkb = K128 / 64 fragments along K (even), nnb = N16 / 16 along N
  void* out;
  PhRowMap outr;
  int* parts;            // split along K: sums [part][M][N16]
};
