// Matrix products of 8-bit integers with a scale for each token (row) and each output channel, gfx950.
//
//   s[m]    = max(f32(max_k |x[m,k]| / 127), 2^-126)
//   q[m,k]  = round_half_even(x[m,k] / s[m])                              of the exact quotient, |q| <= 127
//   acc     = sum_k q[m,k] w[n,k]                                         int32, exact: K <= 131071
//   y[m,n]  = act((f32(acc) * ws[n]) * s[m] + bias[n])                    each operation rounded to f32, then one
//                                                                         rounding to the output's type
// The product of the two scales is never formed: acc * ws * s overflows or underflows only where the result does
// (acc = 0 with two huge scales would give 0 * inf).  A row that holds a NaN or an infinity gets the scale NaN and
// zeros, so that its whole output row is NaN and no other row is touched.
#include "w8a8.h"

// ---- quantisation of rows ------------------------------------------------------------------------------------------

// Running maximum of magnitudes that a NaN stays in (fmaxf would drop it).
__device__ __forceinline__ float max_abs(float m, float v) { return __builtin_elementwise_maximum(m, fabsf(v)); }
// Over groups of G lanes side by side (G = 8 .. 64); all get it.
template <int CTRL>
__device__ __forceinline__ float max_dpp(float m) {
  return __builtin_elementwise_maximum(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), CTRL, 0xf, 0xf, true)));
}
__device__ __forceinline__ float max_16(float m) {   // lanes 16 apart
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float max_32(float m) {   // lanes 32 apart
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
template <int G>
__device__ __forceinline__ float max_group(float m) {
  m = max_dpp<0xb1>(m);    // lanes 1 apart
  m = max_dpp<0x4e>(m);    // 2 apart
  m = max_dpp<0x141>(m);   // 4: a half row mirrored, its quads being alike
  if (G > 8) m = max_dpp<0x140>(m);   // 8: a row mirrored
  if (G > 16) m = max_16(m);
  if (G > 32) m = max_32(m);
  return m;
}

struct RowScale {
  float s, inv, half;   // scale, 1 / scale, scale / 2
  bool finite;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.finite = amax < __builtin_inff();
  r.s = r.finite ? fmaxf(amax / 127.f, 0x1p-126f) : 1.f;
  r.inv = 1.f / r.s;
  r.half = 0.5f * r.s;
  return r;
}
__device__ __forceinline__ float scale_out(const RowScale& r) { return r.finite ? r.s : __builtin_nanf(""); }

// round_half_even(x / s), N values to N bytes.  Adding 1.5 * 2^23 rounds to a whole number, which then stands in the low
// bits of the sum.  x * (1/s) is within 127 * 2^-23 of the quotient, so that number is the wanted one or its neighbour;
// the remainder x - q s is exact in one fused operation and tells which.  Where no remainder reaches half a step, as
// almost always, all stand.
template <int N>
__device__ __forceinline__ void quantize_n(const float (&x)[N], const RowScale& r, unsigned (&out)[N / 4]) {
  constexpr float MAGIC = 12582912.f;
  float t[N], worst = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) {
    t[i] = __builtin_fmaf(x[i], r.inv, MAGIC);
    worst = fmaxf(worst, fabsf(__builtin_fmaf(-(t[i] - MAGIC), r.s, x[i])));
  }
  if (worst >= r.half) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float rem = __builtin_fmaf(-(t[i] - MAGIC), r.s, x[i]), a = fabsf(rem);
      const bool odd = __float_as_uint(t[i]) & 1;
      const float far = odd ? a : __uint_as_float(__float_as_uint(a) - (a > 0.f));   // a tie moves an odd number only
      t[i] += far >= r.half ? __builtin_copysignf(1.f, rem) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < N / 4; i++) {
    const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 1]), __float_as_uint(t[4 * i]), 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 3]), __float_as_uint(t[4 * i + 2]), 0x04000c0cu);
    out[i] = r.finite ? lo | hi : 0;
  }
}

// Eight values of a row from k on; rows start at any multiple of their element.  Where fewer are left, the row's last
// eight: a value seen twice does not change a maximum, and the bytes move to their place by `shift` bits.
template <typename T>
struct Eight {
  T v __attribute__((ext_vector_type(8)));
  typedef T t8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  __device__ __forceinline__ void load_long(const T* row, int k, int K) { v = *(const t8*)(row + min(k, K - 8)); }   // K >= 8
  __device__ __forceinline__ void load(const T* row, int k, int K) {
    if (K >= 8) {
      load_long(row, k, K);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = i < K ? row[i] : (T)0.f;
    }
  }
  static __device__ __forceinline__ int shift(int k, int K) { return 8 * max(0, k - max(K - 8, 0)); }   // k < K
  __device__ __forceinline__ float max_with(float m) const {
#pragma unroll
    for (int i = 0; i < 8; i++) m = max_abs(m, (float)v[i]);
    return m;
  }
  __device__ __forceinline__ uint64_t quantize(const RowScale& r) const {
    float x[8];
    unsigned o[2];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)v[i];
    quantize_n(x, r, o);
    return (uint64_t)o[1] << 32 | o[0];
  }
};

// G lanes own a row (G <= 64: several rows a wave; more: a block of G threads), with up to CH chunks of 8 values a lane
// kept in registers between the two passes; what a longer row has beyond is read again.
template <typename T, int G, int CH>
__global__ __launch_bounds__(G <= 64 ? 256 : G) void quantize_rows_kernel(const T* __restrict__ x, PhRowMap xr, unsigned M, int K,
                                                                         int8_t* __restrict__ q, int64_t q_pitch,
                                                                         float* __restrict__ scale) {
  constexpr int STEP = G * 8;
  const int lane = threadIdx.x % G;
  constexpr int PER = G <= 64 ? 256 / G : 1;   // rows of a block
  const unsigned m = blockIdx.x * PER + threadIdx.x / G;
  if (m >= M) return;   // (G > 64: never)
  const T* row = x + ph_row_off(xr, m);
  Eight<T> v[CH];
  float am = 0.f;
#pragma unroll
  for (int c = 0; c < CH; c++)
    if (c * STEP < K) v[c].load(row, c * STEP + lane * 8, K);
#pragma unroll
  for (int c = 0; c < CH; c++)
    if (c * STEP < K) am = v[c].max_with(am);
  for (int k = CH * STEP + lane * 8; k < K; k += STEP) {
    Eight<T> t;
    t.load(row, k, K);
    am = t.max_with(am);
  }
  am = max_group<(G < 64 ? G : 64)>(am);
  if constexpr (G > 64) {
    __shared__ float s_am[G / 64];
    if ((lane & 63) == 0) s_am[lane >> 6] = am;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < G / 64; w++) am = max_abs(am, s_am[w]);
  }
  const RowScale r = row_scale(am);
  if (lane == 0) scale[m] = scale_out(r);
  int8_t* const qrow = q + (int64_t)m * q_pitch;   // (pitch and base are multiples of 16: whole chunks, also the last)
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int k = c * STEP + lane * 8;
    if (k < K) *(uint64_t*)(qrow + k) = v[c].quantize(r) >> Eight<T>::shift(k, K);
  }
  for (int k = CH * STEP + lane * 8; k < K; k += STEP) {
    Eight<T> t;
    t.load(row, k, K);
    *(uint64_t*)(qrow + k) = t.quantize(r) >> Eight<T>::shift(k, K);
  }
}

// As few lanes own a row as hold it in 4 chunks each (120704 rows of 384 bf16: 28 us = 5.0 TB/s with 16 lanes a row, 47 with
// 64 -- four rows of a wave are on their way at once, and no lane idles), but more of them where there are few rows (3772
// rows: 5.2 us with 16, 3.8 with 64).
template <typename T>
static int launch_quantize_t(const T* x, const PhRowMap& xr, unsigned M, int K, int8_t* q, int64_t pitch, float* scale,
                             hipStream_t st) {
  static const int groups[] = {8, 16, 32, 64, 256, 1024};
  int g = 0;
  while (g < 5 && groups[g] * 32 < K) g++;
  while (g < 5 && groups[g] * 8 < K && (int64_t)M * groups[g] < 64 * 4096) g++;
#define PH_Q(G)                                                                                                            \
  hipLaunchKernelGGL((quantize_rows_kernel<T, G, 4>), dim3(G <= 64 ? (M - 1) / (G <= 64 ? 256 / G : 1) + 1 : M),              \
                     dim3(G <= 64 ? 256 : G), 0, st, x, xr, M, K, q, pitch, scale);                                         \
  break
  switch (g) {
    case 0: PH_Q(8);
    case 1: PH_Q(16);
    case 2: PH_Q(32);
    case 3: PH_Q(64);
    case 4: PH_Q(256);
    default: PH_Q(1024);
  }
#undef PH_Q
  PH_CHECK(hipGetLastError());
  return 0;
}

// ---- weights ---------------------------------------------------------------------------------------------------------

// int8 [N][K] -> fragments of the 16 x 64 operand of the matrix instruction, [N16/16][K128/64][lane][16]: lane l of a
// fragment holds channel l % 16, k = (l / 16) * 16 .. + 15.  Rows and columns beyond N, K are zero: whatever stands
// behind a token's last value is multiplied by zero.
__global__ void pack_weight_kernel(const int8_t* __restrict__ w, int64_t row_stride, int N, int K, int nkb, int nnb,
                                   int8_t* __restrict__ out) {
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;   // one 16-byte piece
  if (t >= (int64_t)nnb * nkb * 64) return;
  const int lane = (int)(t & 63);
  const int64_t f = t >> 6;
  const int kb = (int)(f % nkb), nb = (int)(f / nkb);
  const int n = nb * 16 + (lane & 15), k = kb * 64 + (lane >> 4) * 16;
  union { int8_t b[16]; u32x4 v; } p;
#pragma unroll
  for (int i = 0; i < 16; i++) p.b[i] = (n < N && k + i < K) ? w[(int64_t)n * row_stride + k + i] : (int8_t)0;
  *(u32x4*)(out + t * 16) = p.v;
}

// rows of any alignment -> rows of `pitch` bytes, 16-byte aligned
__global__ void repitch_kernel(const int8_t* __restrict__ q, PhRowMap qr, unsigned M, int K, int8_t* __restrict__ out,
                               int64_t pitch) {
  const int64_t ppr = pitch >> 4;
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= (int64_t)M * ppr) return;
  const unsigned m = (unsigned)(t / ppr);
  const int k = (int)(t - m * ppr) * 16;
  const int8_t* row = q + ph_row_off(qr, m);
  union { int8_t b[16]; u32x4 v; } p;
#pragma unroll
  for (int i = 0; i < 16; i++) p.b[i] = k + i < K ? row[k + i] : (int8_t)0;
  *(u32x4*)(out + (int64_t)m * pitch + k) = p.v;
}

// ---- epilogue ----------------------------------------------------------------------------------------------------------

template <int ACT>
__device__ __forceinline__ float w8_value(int acc, float ws, float s, float bias, float slope) {
  const float v = ((float)acc * ws) * s + bias;
  if (ACT == PH_ACT_RELU) return v < 0.f ? 0.f : v;
  if (ACT == PH_ACT_PRELU) return v < 0.f ? v * slope : v;
  return v;
}
// four consecutive channels of a token, rounded to the output's type; only the first `have` of them exist
template <typename O>
__device__ __forceinline__ void w8_store4(O* o, const f32x4 v, int have) {
  typedef O o4 __attribute__((ext_vector_type(4), aligned(sizeof(O))));
  if (have >= 4) {
    o4 w;
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = (O)v[e];
    *(o4*)o = w;
  } else {
#pragma unroll
    for (int e = 0; e < 3; e++)
      if (e < have) o[e] = (O)v[e];
  }
}
struct Channels {   // of four consecutive channels
  f32x4 ws, bias, slope;
};
__device__ __forceinline__ Channels w8_channels(const PhW8Params& p, int n) {   // n: a multiple of 4 below N16
  Channels c;
  c.ws = *(const f32x4*)(p.ws + n);
  c.bias = p.bias ? *(const f32x4*)(p.bias + n) : f32x4{0.f, 0.f, 0.f, 0.f};
  c.slope = p.slope ? *(const f32x4*)(p.slope + n) : f32x4{0.f, 0.f, 0.f, 0.f};
  return c;
}
template <int ACT>
__device__ __forceinline__ f32x4 w8_values(const i32x4 acc, const Channels& c, float s) {
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = w8_value<ACT>(acc[e], c.ws[e], s, c.bias[e], c.slope[e]);
  return v;
}

// one sum of four channels -> out
template <typename O>
__device__ __forceinline__ void w8_finish4(const PhW8Params& p, const i32x4 a, const Channels& c, unsigned m, int n, float s) {
  f32x4 v;
  if (p.act == PH_ACT_RELU) v = w8_values<PH_ACT_RELU>(a, c, s);
  else if (p.act == PH_ACT_PRELU) v = w8_values<PH_ACT_PRELU>(a, c, s);
  else v = w8_values<PH_ACT_NONE>(a, c, s);
  w8_store4<O>((O*)p.out + ph_row_off(p.outr, m) + n, v, p.N - n);
}

// A wave's TM x TN fragments -> out, tokens m0 + .., channels n0 + ...  In a fragment the 16 lanes side by side hold 16
// tokens (rows of out) and 4 channels each: stored like that, every 8-byte piece is a request of its own (13 us for a
// 256 x 256 tile of bf16).  So two fragments' tokens at a time go through the wave's own LDS piece and leave as whole
// rows of its channels, 16 bytes a lane.
template <int TM, int TN, typename O>
struct WaveOut {
  static constexpr int ROW = TN * 16 * (int)sizeof(O);
  static constexpr int PITCH = ROW + 16;
  static constexpr int STEP = TM < 2 ? 1 : 2;
  static constexpr int BYTES = STEP * 16 * PITCH;
  typedef O oe __attribute__((ext_vector_type(16 / sizeof(O)), aligned(sizeof(O))));
  typedef O o4 __attribute__((ext_vector_type(4)));

  template <int ACT, bool STREAM>
  static __device__ __forceinline__ void put(const PhW8Params& p, const i32x4 (&acc)[TN][TM], unsigned m0, int n0, char* buf,
                                             int lane) {
    const int fr = lane & 15, fq = lane >> 4;
    Channels c[TN];
    float s[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) s[i] = p.qs[min(m0 + i * 16 + fr, p.M - 1)];
    const int last = p.nnb * 16 - 4;
#pragma unroll
    for (int j = 0; j < TN; j++) c[j] = w8_channels(p, min(n0 + j * 16 + fq * 4, last));
    constexpr int PER = 16 / (int)sizeof(O);          // values of a 16-byte unit
    constexpr int UNITS = STEP * 16 * (ROW / 16);     // units of a pass
#pragma unroll
    for (int i0 = 0; i0 < TM; i0 += STEP) {
#pragma unroll
      for (int i = 0; i < STEP; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) {
          const f32x4 v = w8_values<ACT>(acc[j][i0 + i], c[j], s[i0 + i]);
          o4 w;
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = (O)v[e];
          *(o4*)(buf + (i * 16 + fr) * PITCH + (j * 16 + fq * 4) * (int)sizeof(O)) = w;
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // a wave's own pass: no other wave touches this piece
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int u0 = 0; u0 < UNITS; u0 += 64) {
        const int u = u0 + lane, t = u / (ROW / 16), col = (u - t * (ROW / 16)) * PER;
        const unsigned m = m0 + i0 * 16 + t;
        const int n = n0 + col;
        if ((UNITS % 64 == 0 || u < UNITS) && m < p.M && n < p.N) {
          const oe w = *(const oe __attribute__((aligned(16)))*)(buf + t * PITCH + col * (int)sizeof(O));
          O* const o = (O*)p.out + ph_row_off(p.outr, m) + n;
          if (n + PER <= p.N) {
            if constexpr (STREAM) __builtin_nontemporal_store(w, (oe*)o);
            else *(oe*)o = w;
          }
          else {
#pragma unroll
            for (int e = 0; e < PER - 1; e++)
              if (n + e < p.N) o[e] = w[e];
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
  }
  static __device__ __forceinline__ void store(const PhW8Params& p, const i32x4 (&acc)[TN][TM], unsigned m0, int n0, char* buf,
                                               int lane) {
    if (p.stream) store_act<true>(p, acc, m0, n0, buf, lane);
    else store_act<false>(p, acc, m0, n0, buf, lane);
  }
  template <bool STREAM>
  static __device__ __forceinline__ void store_act(const PhW8Params& p, const i32x4 (&acc)[TN][TM], unsigned m0, int n0, char* buf,
                                                   int lane) {
    if (p.act == PH_ACT_RELU) put<PH_ACT_RELU, STREAM>(p, acc, m0, n0, buf, lane);
    else if (p.act == PH_ACT_PRELU) put<PH_ACT_PRELU, STREAM>(p, acc, m0, n0, buf, lane);
    else put<PH_ACT_NONE, STREAM>(p, acc, m0, n0, buf, lane);
  }
};

// ---- product: tiles through LDS ------------------------------------------------------------------------------------------

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void glb_void;

// Blocks go round the 8 dies in turn: each die gets a run of consecutive tiles, and a run walks 8 tiles of tokens for
// each tile of channels, so that the tiles in flight on a die share rows and weights in its L2.
__device__ __forceinline__ void tile_of_block(unsigned bid, unsigned mt, unsigned nt, unsigned& tm, unsigned& tn) {
  const unsigned total = mt * nt, per = total >> 3, more = total & 7, die = bid & 7;
  const unsigned t = die * per + min(die, more) + (bid >> 3);
  const unsigned group = 8 * nt, g = t / group, r = t - g * group;
  const unsigned rows = min(8u, mt - g * 8);
  tn = r / rows;
  tm = g * 8 + (r - tn * rows);
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// BM tokens x BN channels per block, WM x WN waves, a step is 128 k (two fragments), NST steps' operands in LDS.
// Fragments are read one half step ahead of their products: while the first half's run, the second half's are read;
// then the block meets, the slot just left is filled again, and the next step's first half is read while the second
// half's products run.
template <int BM, int BN, int WM, int WN, int NST, bool SPLIT, typename O>
__global__ __launch_bounds__(64 * WM * WN) void w8_tile_kernel(const PhW8Params p, unsigned mt, unsigned nt) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int XP = BM / 8, WP = BN / 8;               // 1-KiB pieces of a step
  constexpr int XL = XP / WAVES, WL = WP / WAVES;       // pieces a wave fetches
  static_assert(XL * WAVES == XP && WL * WAVES == WP, "pieces divide among the waves");
  constexpr int STAGE = (XP + WP) * 1024;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int fr = lane & 15, fq = lane >> 4;
  unsigned tm, tn;
  tile_of_block(blockIdx.x, mt, nt, tm, tn);
  const unsigned m0 = tm * BM;
  const int nb0 = tn * (BN / 16);

  const int all = p.nkb >> 1, first = SPLIT ? (int)((int64_t)all * blockIdx.y / gridDim.y) : 0;
  const int steps = SPLIT ? (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y) - first : all;   // (at least one)
  // a piece of rows: 16 rows x 64 bytes, four lanes a row; the 16-byte unit a lane fetches is swapped in rows 4..7 and
  // 12..15 of the piece, so that reading a fragment (16 rows, one unit each) does not hit a bank twice
  const int unit = (lane & 3) ^ (((lane >> 4) & 1) << 1);
  const int8_t* xsrc[XL];
  int xk[XL];
#pragma unroll
  for (int u = 0; u < XL; u++) {
    const int piece = wave + u * WAVES;
    xsrc[u] = p.q + ph_row_off(p.qr, min(m0 + (piece >> 1) * 16 + (lane >> 2), p.M - 1));
    xk[u] = (piece & 1) * 64 + unit * 16;
  }
  const int8_t* wsrc[WL];
#pragma unroll
  for (int u = 0; u < WL; u++) {
    const int piece = wave + u * WAVES, nb = min(nb0 + (piece >> 1), p.nnb - 1);
    wsrc[u] = p.w + ((int64_t)nb * p.nkb + (piece & 1)) * 1024 + lane * 16;
  }
  auto fetch = [&](int g, int slot) {
    char* const st = lds + slot * STAGE;
#pragma unroll
    for (int u = 0; u < XL; u++) {
      int k = (first + g) * 128 + xk[u];
      k = k < p.K ? k : 0;   // units behind the row's end meet zero weights
      __builtin_amdgcn_global_load_lds((glb_void*)(xsrc[u] + k), (lds_void*)(st + (wave + u * WAVES) * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < WL; u++)
      __builtin_amdgcn_global_load_lds((glb_void*)(wsrc[u] + (int64_t)(first + g) * 2048),
                                       (lds_void*)(st + (XP + wave + u * WAVES) * 1024), 16, 0, 0);
  };
  const int xrd = wm * TM * 2048 + fr * 64 + ((fq * 16) ^ ((fr & 4) << 3));
  const int wrd = XP * 1024 + wn * TN * 2048 + lane * 16;
  auto read = [&](i32x4 (&xf)[TM], i32x4 (&wf)[TN], int slot, int kb) {
    const char* const st = lds + slot * STAGE + kb * 1024;
#pragma unroll
    for (int j = 0; j < TN; j++) wf[j] = *(const i32x4*)(st + wrd + j * 2048);
#pragma unroll
    for (int i = 0; i < TM; i++) xf[i] = *(const i32x4*)(st + xrd + i * 2048);
  };
  i32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < TM; i++) acc[j][i] = i32x4{0, 0, 0, 0};
  auto multiply = [&](const i32x4 (&xf)[TM], const i32x4 (&wf)[TN]) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[j][i], 0, 0, 0);
  };

#pragma unroll
  for (int g = 0; g < NST; g++)
    if (g < steps) fetch(g, g);
  if (NST <= steps) wait_loads<(NST - 1) * (XL + WL)>();
  else wait_loads<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  i32x4 xa[TM], wa[TN], xb[TM], wb[TN];
  read(xa, wa, 0, 0);
  int slot = 0;
  for (int g = 0; g < steps; g++) {
    read(xb, wb, slot, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(xa, wa);
    __builtin_amdgcn_sched_barrier(0);
    if (g + 1 < steps) {
      if (g + NST <= steps) wait_loads<(NST - 2) * (XL + WL)>();
      else wait_loads<0>();
      __builtin_amdgcn_s_barrier();   // step g + 1 is in LDS, and everybody has read all of step g
      asm volatile("" ::: "memory");
      const int old = slot;
      slot = slot + 1 == NST ? 0 : slot + 1;
      read(xa, wa, slot, 0);
      if (g + NST < steps) fetch(g + NST, old);
    }
    __builtin_amdgcn_sched_barrier(0);
    multiply(xb, wb);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (SPLIT) {   // sums of a part of K, joined by w8_join_kernel
    int* const part = p.parts + (int64_t)blockIdx.y * p.M * (p.nnb * 16);
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int n = (nb0 + wn * TN + j) * 16 + fq * 4;
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const unsigned m = m0 + (wm * TM + i) * 16 + fr;
        if (m < p.M && n < p.N) *(i32x4*)(part + (int64_t)m * (p.nnb * 16) + n) = acc[j][i];
      }
    }
    return;
  }
  __builtin_amdgcn_s_barrier();   // everybody has read the last step: LDS is free
  asm volatile("" ::: "memory");
  WaveOut<TM, TN, O>::store(p, acc, m0 + wm * TM * 16, (nb0 + wn * TN) * 16, lds + wave * WaveOut<TM, TN, O>::BYTES, lane);
}

template <int BM, int BN, int WM, int WN, int NST, bool SPLIT, typename O>
static int launch_tile(const PhW8Params& p, int parts, hipStream_t st) {
  constexpr int ring = NST * (BM + BN) * 128, tile = WM * WN * WaveOut<BM / WM / 16, BN / WN / 16, O>::BYTES;
  constexpr int lds = ring > tile ? ring : tile;
  static int granted[PH_MAX_DEVICES];
  const void* fn = (const void*)w8_tile_kernel<BM, BN, WM, WN, NST, SPLIT, O>;
  if (lds > 64 * 1024 && ph_ensure_lds(fn, lds, granted)) return -1;
  const unsigned mt = (p.M + BM - 1) / BM, nt = (p.N + BN - 1) / BN;
  hipLaunchKernelGGL((w8_tile_kernel<BM, BN, WM, WN, NST, SPLIT, O>), dim3(mt * nt, SPLIT ? parts : 1), dim3(64 * WM * WN), lds, st, p, mt, nt);
  PH_CHECK(hipGetLastError());
  return 0;
}

// ---- product: few tokens -------------------------------------------------------------------------------------------------
//
// Up to 64 tokens: the weights are read once, each fragment by one wave straight into registers (a fragment is 1 KiB in
// one piece), and the rows, which every block needs, come from cache.  A block has 16 channels; its waves take fragments
// along K in turn and their sums meet in LDS.
//
// T is int8_t, or the type of float rows that the block quantises itself, into LDS, while its first weights are on their
// way: for one to a few tokens that costs less than a launch of its own before this one (see launch_few_float).
struct FloatRows {
  const void* x;
  PhRowMap r;
};

// M <= 8 rows -> int8 rows of `pitch` bytes and their scales in LDS; W waves, W / (M rounded up to a power of two) a row
template <int W, typename T>
__device__ __forceinline__ void quantize_block(const FloatRows& f, unsigned M, int K, char* q, int pitch, float* scale,
                                               float* amax, int wave, int lane) {
  const T* const x = (const T*)f.x;
  const unsigned per = M > 4 ? 1 : M > 2 ? 2 : M > 1 ? 4 : 8;   // waves of a row (W = 8)
  static_assert(W == 8, "waves are dealt to rows for 8");
  const unsigned row = wave / per;
  const bool has = row < M;
  const T* const xr = x + ph_row_off(f.r, has ? row : 0);
  const int k0 = ((wave % per) * 64 + lane) * 8, step = per * 512;
  Eight<T> first;
  float am = 0.f;
  if (has) {
    first.load(xr, k0, K);
    am = first.max_with(am);
    for (int k = k0 + step; k < K; k += step) {
      Eight<T> v;
      v.load(xr, k, K);
      am = v.max_with(am);
    }
  }
  am = max_group<64>(am);
  if (lane == 0) amax[wave] = am;
  __syncthreads();
  if (has) {
    am = 0.f;
    for (unsigned w = 0; w < per; w++) am = max_abs(am, amax[row * per + w]);
    const RowScale r = row_scale(am);
    if (lane == 0 && wave % per == 0) scale[row] = scale_out(r);
    if (k0 < K) *(uint64_t*)(q + (int)row * pitch + k0) = first.quantize(r) >> Eight<T>::shift(k0, K);
    for (int k = k0 + step; k < K; k += step) {
      Eight<T> v;
      v.load(xr, k, K);
      *(uint64_t*)(q + (int)row * pitch + k) = v.quantize(r) >> Eight<T>::shift(k, K);
    }
  }
  __syncthreads();
}

template <int TM, int W, bool SPLIT, typename T, typename O>
__global__ __launch_bounds__(64 * W) void w8_few_kernel(const PhW8Params p, const FloatRows f) {
  constexpr bool FLOAT = !__is_same(T, int8_t);
  constexpr int DEPTH = 4;   // fragments of weights in flight per wave
  __shared__ __attribute__((aligned(16))) int red[W][TM][256];
  extern __shared__ __attribute__((aligned(16))) char s_q[];   // FLOAT: the rows in 8 bits
  __shared__ float s_scale[8];
  __shared__ float s_amax[W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int nb = blockIdx.x;
  const int kb0 = SPLIT ? (int)((int64_t)p.nkb * blockIdx.y / gridDim.y) : 0;
  const int kb1 = SPLIT ? (int)((int64_t)p.nkb * (blockIdx.y + 1) / gridDim.y) : p.nkb;
  const int8_t* const wp = p.w + (int64_t)nb * p.nkb * 1024 + lane * 16;
  i32x4 wf[DEPTH];
  auto weights = [&](int kb) {
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
      if (kb + d * W < kb1) wf[d] = __builtin_nontemporal_load((const i32x4*)(wp + (int64_t)(kb + d * W) * 1024));
  };
  weights(kb0 + wave);
  const int pitch = p.nkb * 64 + 16;   // (16 rows at one multiple of 64 bytes would share their banks)
  if constexpr (FLOAT) quantize_block<W, T>(f, p.M, p.K, s_q, pitch, s_scale, s_amax, wave, lane);
  const int8_t* xp[TM];   // (FLOAT: one fragment of tokens, in LDS)
  const char* const xq = s_q + min((unsigned)fr, p.M - 1) * pitch;
#pragma unroll
  for (int i = 0; i < TM; i++) xp[i] = FLOAT ? nullptr : p.q + ph_row_off(p.qr, min((unsigned)(i * 16 + fr), p.M - 1));
  i32x4 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; i++) acc[i] = i32x4{0, 0, 0, 0};
  for (int kb = kb0 + wave; kb < kb1; kb += W * DEPTH) {
    i32x4 xf[DEPTH][TM], w[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      int k = (kb + d * W) * 64 + fq * 16;
      k = k < p.K ? k : 0;   // units behind the row's end meet zero weights
#pragma unroll
      for (int i = 0; i < TM; i++) {
        if constexpr (FLOAT) xf[d][i] = *(const i32x4*)(xq + k);
        else xf[d][i] = *(const i32x4*)(xp[i] + k);
      }
      w[d] = wf[d];
    }
    weights(kb + W * DEPTH);
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
      if (kb + d * W < kb1)
#pragma unroll
        for (int i = 0; i < TM; i++) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d], xf[d][i], acc[i], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < TM; i++) *(i32x4*)&red[wave][i][lane * 4] = acc[i];
  __syncthreads();
  if (wave < TM) {
    i32x4 a = *(const i32x4*)&red[0][wave][lane * 4];
#pragma unroll
    for (int w = 1; w < W; w++) a += *(const i32x4*)&red[w][wave][lane * 4];
    const unsigned m = wave * 16 + fr;
    const int n = nb * 16 + fq * 4;
    if (m >= p.M || n >= p.N) return;
    if (SPLIT) *(i32x4*)(p.parts + ((int64_t)blockIdx.y * p.M + m) * (p.nnb * 16) + n) = a;
    else w8_finish4<O>(p, a, w8_channels(p, n), m, n, FLOAT ? s_scale[m & 7] : p.qs[m]);
  }
}

// sums of the parts of K -> out; integers, so that their order does not matter
template <typename O>
__global__ __launch_bounds__(256) void w8_join_kernel(const PhW8Params p, int parts) {
  const int q4 = (p.N + 3) / 4;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= (int64_t)p.M * q4) return;
  const unsigned m = (unsigned)(t / q4);
  const int n = (int)(t - (int64_t)m * q4) * 4;
  const int64_t pitch = (int64_t)p.M * (p.nnb * 16);
  const int* at = p.parts + (int64_t)m * (p.nnb * 16) + n;
  i32x4 a = i32x4{0, 0, 0, 0};
  for (int s0 = 0; s0 < parts; s0 += 8) {   // eight at a time on their way
    i32x4 b[8];
#pragma unroll
    for (int s = 0; s < 8; s++) b[s] = s0 + s < parts ? *(const i32x4*)(at + (s0 + s) * pitch) : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 8; s++) a += b[s];
  }
  w8_finish4<O>(p, a, w8_channels(p, n), m, n, p.qs[m]);
}

template <int TM, bool SPLIT, typename O>
static int launch_few(const PhW8Params& p, int parts, hipStream_t st) {
  hipLaunchKernelGGL((w8_few_kernel<TM, 8, SPLIT, int8_t, O>), dim3(p.nnb, SPLIT ? parts : 1), dim3(512), 0, st, p, FloatRows{});
  PH_CHECK(hipGetLastError());
  return 0;
}

// What a product costs by each kernel, in us, as measured: a block's step of 128 k alone on its CU (`alone`) and with
// the CU full (`full`), what a round of blocks costs beside its steps (`fixed`), blocks that fit a CU (`fit`).
//   4096^3, us: 256x256 60, 128x128 69 (three slots: 84), 128x64 84, 64x64 99
//   1024 x 4096 x 4096: 128x128 24 (three slots: 22), 128x64 23, 64x64 29;  512: 128x64 21, 64x64 16
//   61 x 32500 x 187: 64x64 in one piece 50, in 4 parts 22, in 16 parts 11
struct Kernel {
  int bm, bn, fit;
  float alone, full, fixed;
};
enum { K_256, K_128, K_128_3, K_128x64, K_64, K_FEW, N_KERNELS = K_FEW };
static const Kernel kernels[N_KERNELS] = {
    {256, 256, 1, 1.72f, 1.72f, 6.f}, {128, 128, 2, 0.64f, 0.50f, 3.5f}, {128, 128, 1, 0.56f, 0.56f, 3.5f},
    {128, 64, 3, 0.55f, 0.32f, 2.6f}, {64, 64, 3, 0.32f, 0.20f, 2.2f}};

struct Choice {
  int kernel, parts;
};
// Splitting K pays where there are far fewer blocks than CUs: the parts' sums (4 bytes each) are written, read and
// joined by a second launch.
static Choice choose(int64_t M, int N, int nkb) {
  const int steps = nkb / 2;
  const int64_t n16 = (N + 15) / 16 * 16;
  const float wire = (float)n16 * nkb * 64 / 5.5e6f;   // the weights, once, from memory
  auto join = [&](int parts) { return parts > 1 ? 3.3f + (float)M * n16 * 4e-6f * parts / 2.f : 0.f; };   // (2 TB/s)
  Choice best = {K_64, 1};
  float least = 1e30f;
  const int64_t small = (M + 63) / 64 * ((N + 63) / 64);   // blocks of the smallest tile: two rounds of them need no parts
  for (int parts = 1; parts <= 32 && parts <= steps; parts *= 2) {
    if (parts > 1 && (small >= 1024 || (float)M * n16 * parts > (float)(1 << 24))) break;
    const int s = (steps + parts - 1) / parts;
    for (int k = 0; k < N_KERNELS; k++) {
      const Kernel& c = kernels[k];
      const int64_t blocks = (M + c.bm - 1) / c.bm * ((N + c.bn - 1) / c.bn) * parts;
      const int64_t each = (blocks + 255) / 256, rounds = (each + c.fit - 1) / c.fit;
      const float run = (float)s * (each * c.full > rounds * c.alone ? each * c.full : rounds * c.alone);
      const float t = (run > wire ? run : wire) + rounds * c.fixed + join(parts);
      if (t < least) least = t, best = {k, parts};
    }
    if (M <= 64) {   // a wave's step is one fragment of 64 k; blocks' loads share the memory's rate
      const int tm = (int)(M + 15) / 16;
      const int64_t blocks = n16 / 16 * parts, rounds = (blocks + 511) / 512;
      const float run = (s * 2 + 31) / 32 * rounds * (0.35f + 0.45f * tm), w = wire * (0.8f + 0.2f * tm);
      const float t = 1.f + 0.5f * tm + (run > w ? run : w) + join(parts);
      if (t < least) least = t, best = {K_FEW, parts};
    }
  }
  return best;
}

static int64_t parts_bytes(const Choice& c, int64_t M, int N) {
  return c.parts > 1 ? (int64_t)c.parts * M * ((N + 15) / 16 * 16) * 4 : 0;
}

template <bool SPLIT, typename O>
static int launch_kernel(const PhW8Params& p, const Choice& c, hipStream_t st) {
  switch (c.kernel) {
    case K_256: return launch_tile<256, 256, 2, 4, 2, SPLIT, O>(p, c.parts, st);
    case K_128: return launch_tile<128, 128, 2, 4, 2, SPLIT, O>(p, c.parts, st);
    case K_128_3: return launch_tile<128, 128, 2, 4, 3, SPLIT, O>(p, c.parts, st);
    case K_128x64: return launch_tile<128, 64, 4, 2, 2, SPLIT, O>(p, c.parts, st);
    case K_64: return launch_tile<64, 64, 2, 2, 3, SPLIT, O>(p, c.parts, st);
    default:
      if (p.M <= 16) return launch_few<1, SPLIT, O>(p, c.parts, st);
      if (p.M <= 32) return launch_few<2, SPLIT, O>(p, c.parts, st);
      if (p.M <= 48) return launch_few<3, SPLIT, O>(p, c.parts, st);
      return launch_few<4, SPLIT, O>(p, c.parts, st);
  }
}

// parts_bytes() of workspace at p.parts
template <typename O>
static int launch_product_t(const PhW8Params& p, const Choice& c, hipStream_t st) {
  if (c.parts == 1) return launch_kernel<false, O>(p, c, st);
  if (launch_kernel<true, O>(p, c, st)) return -1;
  const int64_t pieces = (int64_t)p.M * ((p.N + 3) / 4);
  hipLaunchKernelGGL((w8_join_kernel<O>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, st, p, c.parts);
  PH_CHECK(hipGetLastError());
  return 0;
}

// Up to 8 tokens of up to 32 K values in all: the product's blocks quantise the rows themselves.
static bool few_float(int64_t M, int K) { return M <= 8 && M * K <= 32768; }

template <typename T, typename O>
static int launch_few_float_t(const PhW8Params& p, const FloatRows& f, hipStream_t st) {
  const int lds = (int)p.M * (p.nkb * 64 + 16);   // at most 34 KB
  hipLaunchKernelGGL((w8_few_kernel<1, 8, false, T, O>), dim3(p.nnb), dim3(512), lds, st, p, f);
  PH_CHECK(hipGetLastError());
  return 0;
}
template <typename O>
static int launch_few_float(const PhW8Params& p, int x_type, const FloatRows& f, hipStream_t st) {
  switch (x_type) {
    case PH_F32: return launch_few_float_t<float, O>(p, f, st);
    case PH_F16: return launch_few_float_t<_Float16, O>(p, f, st);
    default: return launch_few_float_t<bf16, O>(p, f, st);
  }
}

// Long rows of a large output go past the caches: 120704 x 512 bf16 of K = 384 69 -> 55 us, 16384 x 4096 of K = 4096 263 ->
// 247 us.  Rows that end inside a line lose by it (N = 52: 17.5 -> 18.7 us).
static int launch_product(PhW8Params p, const Choice& c, int out_type, hipStream_t st) {
  const int64_t row = (int64_t)p.N * (out_type == PH_F32 ? 4 : 2);
  p.stream = row >= 512 && row * p.M >= (4 << 20);
  switch (out_type) {
    case PH_F32: return launch_product_t<float>(p, c, st);
    case PH_F16: return launch_product_t<_Float16>(p, c, st);
    default: return launch_product_t<bf16>(p, c, st);
  }
}

// ---- two layers --------------------------------------------------------------------------------------------------------
//
// x [.., 8 <= K <= 512] -> H <= 512 -> N <= 64 in one kernel: the inner rows never leave the CU.  A block owns 16 TF tokens at a
// time and all H inner channels, 64 to a wave: their sums fill its registers, so the maximum of an inner row, which the
// second quantisation needs, is known before anything is rounded.  Per tile: the rows are quantised into LDS; first product
// (weights straight from cache, each fragment read by one wave and used for TF products); inner values and their maxima;
// inner rows in 8 bits into the same LDS; second product, its weights in LDS for good.  Two blocks share a CU, so that one's
// rounding (12 vector operations per inner value) runs under the other's products.
#define PAIR_MAX 512   // widest input and widest inner row
struct PhW8Pair {
  const void* x;
  PhRowMap xr;
  unsigned M;
  int K, H, N, nkb1, nnb1, nkb2, nnb2, act1, act2;
  const int8_t *w1, *w2;
  const float *ws1, *bias1, *slope1, *ws2, *bias2, *slope2;
  void* out;
  PhRowMap outr;
  int out_type;
};

template <int TF, int ACT, typename T>
__global__ __launch_bounds__(512, 4) void w8_pair_kernel(const PhW8Pair p) {
  constexpr int BT = 16 * TF, RP = BT / 32, CH = 4;   // 16 lanes a row, 32 rows at a time, 4 chunks of 128 values
  constexpr int PITCH = PAIR_MAX + 16;                // of a row in LDS: 16 rows' units lie in different banks
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* const q = lds;                                // the rows in 8 bits, then the inner rows
  float* const s1 = (float*)(q + BT * PITCH);
  float* const s2 = s1 + BT;
  float* const red = s2 + BT;                         // [8][BT]
  float* const par = red + 8 * BT;                    // scale, bias, slope of the inner channels [3][PAIR_MAX]
  char* const w2 = (char*)(par + 3 * PAIR_MAX);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const unsigned m0 = blockIdx.x * BT;
  const int K = p.K;
  {   // rows -> q, s1
    Eight<T> raw[RP][CH];
#pragma unroll
    for (int r = 0; r < RP; r++) {
      const T* row = (const T*)p.x + ph_row_off(p.xr, min(m0 + r * 32 + (tid >> 4), p.M - 1));
#pragma unroll
      for (int c = 0; c < CH; c++)
        if (c * 128 < K) raw[r][c].load_long(row, c * 128 + (tid & 15) * 8, K);
    }
    for (int n = tid; n < PAIR_MAX; n += 512) {   // (channels that do not exist: zeros)
      const bool is = n < p.nnb1 * 16;
      par[n] = is ? p.ws1[n] : 0.f;
      par[PAIR_MAX + n] = is && p.bias1 ? p.bias1[n] : 0.f;
      par[2 * PAIR_MAX + n] = is && p.slope1 ? p.slope1[n] : 0.f;
    }
    for (int f = wave; f < p.nnb2 * p.nkb2; f += 8)
      __builtin_amdgcn_global_load_lds((glb_void*)(p.w2 + f * 1024 + lane * 16), (lds_void*)(w2 + f * 1024), 16, 0, 0);
#pragma unroll
    for (int r = 0; r < RP; r++) {
      float am = 0.f;
#pragma unroll
      for (int c = 0; c < CH; c++)
        if (c * 128 < K) am = raw[r][c].max_with(am);
      const RowScale sc = row_scale(max_group<16>(am));
      const int t = r * 32 + (tid >> 4);
      if ((tid & 15) == 0) s1[t] = scale_out(sc);
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const int k = c * 128 + (tid & 15) * 8;
        if (k < K) *(uint64_t*)(q + t * PITCH + k) = raw[r][c].quantize(sc) >> Eight<T>::shift(k, K);
      }
    }
  }
  const int8_t* wp[4];
#pragma unroll
  for (int j = 0; j < 4; j++) wp[j] = p.w1 + (int64_t)min(wave * 4 + j, p.nnb1 - 1) * p.nkb1 * 1024 + lane * 16;
  i32x4 wa[4], wb[4];
#pragma unroll
  for (int j = 0; j < 4; j++) wa[j] = *(const i32x4*)wp[j];
  __syncthreads();
  i32x4 acc[4][TF];
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int i = 0; i < TF; i++) acc[j][i] = i32x4{0, 0, 0, 0};
  const char* const xq = q + fr * PITCH + fq * 16;
  for (int kb = 0; kb < p.nkb1; kb += 2) {
#pragma unroll
    for (int j = 0; j < 4; j++) wb[j] = *(const i32x4*)(wp[j] + (kb + 1) * 1024);
#pragma unroll
    for (int i = 0; i < TF; i++) {
      const i32x4 xf = *(const i32x4*)(xq + i * 16 * PITCH + kb * 64);
#pragma unroll
      for (int j = 0; j < 4; j++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa[j], xf, acc[j][i], 0, 0, 0);
    }
    const int nx = min(kb + 2, p.nkb1 - 1);
#pragma unroll
    for (int j = 0; j < 4; j++) wa[j] = *(const i32x4*)(wp[j] + nx * 1024);
#pragma unroll
    for (int i = 0; i < TF; i++) {
      const i32x4 xf = *(const i32x4*)(xq + i * 16 * PITCH + kb * 64 + 64);
#pragma unroll
      for (int j = 0; j < 4; j++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wb[j], xf, acc[j][i], 0, 0, 0);
    }
  }
  // inner values, in place of their sums, and each row's maximum
  float am[TF], sc[TF];
#pragma unroll
  for (int i = 0; i < TF; i++) am[i] = 0.f, sc[i] = s1[i * 16 + fr];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int n = (wave * 4 + j) * 16 + fq * 4;
    Channels c;
    c.ws = *(const f32x4*)(par + n);
    c.bias = *(const f32x4*)(par + PAIR_MAX + n);
    c.slope = *(const f32x4*)(par + 2 * PAIR_MAX + n);
#pragma unroll
    for (int i = 0; i < TF; i++) {
      const f32x4 v = w8_values<ACT>(acc[j][i], c, sc[i]);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        acc[j][i][e] = (int)__float_as_uint(v[e]);
        am[i] = max_abs(am[i], v[e]);
      }
      __builtin_amdgcn_sched_barrier(0);   // (all at once they would not fit the registers)
    }
  }
#pragma unroll
  for (int i = 0; i < TF; i++) {
    am[i] = max_32(max_16(am[i]));
    if (fq == 0) red[wave * BT + i * 16 + fr] = am[i];
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the second layer's weights are in LDS
  __syncthreads();   // the first product is done everywhere: q is free
#pragma unroll
  for (int i = 0; i < TF; i++) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) a = max_abs(a, red[w * BT + i * 16 + fr]);
    const RowScale r = row_scale(a);
    if (wave == 0 && fq == 0) s2[i * 16 + fr] = scale_out(r);
    float v[16];
    unsigned o[4];
#pragma unroll
    for (int e = 0; e < 16; e++) v[e] = __uint_as_float((unsigned)acc[e >> 2][i][e & 3]);
    quantize_n(v, r, o);
#pragma unroll
    for (int j = 0; j < 4; j++) *(unsigned*)(q + (i * 16 + fr) * PITCH + (wave * 4 + j) * 16 + fq * 4) = o[j];
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  // second product: a wave has one fragment of channels and every dt-th fragment of tokens
  const int div = p.nnb2 > 2 ? 4 : p.nnb2, nb2 = wave % div, t0 = wave / div, dt = 8 / div;
  constexpr int U = TF / 2;
  i32x4 z[U];
#pragma unroll
  for (int u = 0; u < U; u++) z[u] = i32x4{0, 0, 0, 0};
  const int n = nb2 * 16 + fq * 4;
  PhW8Params o;
  o.ws = p.ws2, o.bias = p.bias2, o.slope = p.slope2, o.act = p.act2, o.N = p.N, o.out = p.out, o.outr = p.outr;
  const Channels c2 = w8_channels(o, min(n, p.nnb2 * 16 - 4));
  const char* const wq = w2 + min(nb2, p.nnb2 - 1) * p.nkb2 * 1024 + lane * 16;
  for (int kb = 0; kb < p.nkb2; kb++) {
    const i32x4 w = *(const i32x4*)(wq + kb * 1024);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = t0 + u * dt;
      if (i < TF) z[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, *(const i32x4*)(xq + i * 16 * PITCH + kb * 64), z[u], 0, 0, 0);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int i = t0 + u * dt;
    const unsigned m = m0 + i * 16 + fr;
    if (i < TF && m < p.M && n < p.N && nb2 < p.nnb2) {
      const float s = s2[i * 16 + fr];
      if (p.out_type == PH_F32) w8_finish4<float>(o, z[u], c2, m, n, s);
      else if (p.out_type == PH_F16) w8_finish4<_Float16>(o, z[u], c2, m, n, s);
      else w8_finish4<bf16>(o, z[u], c2, m, n, s);
    }
  }
}

static bool pair_fits(int K, int H, int N) { return K >= 8 && K <= PAIR_MAX && H <= PAIR_MAX && N <= 64; }

template <int TF, int ACT, typename T>
static int launch_pair_f(const PhW8Pair& p, hipStream_t st) {
  constexpr int BT = 16 * TF;
  const int lds = BT * (PAIR_MAX + 16) + 10 * BT * 4 + 12 * PAIR_MAX + p.nnb2 * p.nkb2 * 1024;   // <= 74 KB: two blocks a CU
  static int granted[PH_MAX_DEVICES];
  if (lds > 64 * 1024 && ph_ensure_lds((const void*)w8_pair_kernel<TF, ACT, T>, lds, granted)) return -1;
  hipLaunchKernelGGL((w8_pair_kernel<TF, ACT, T>), dim3((p.M - 1) / BT + 1), dim3(512), lds, st, p);
  PH_CHECK(hipGetLastError());
  return 0;
}
template <int ACT, typename T>
static int launch_pair_t(const PhW8Pair& p, hipStream_t st) {
  // 32 tokens a block fill the chip earlier (15088 tokens of 384 -> 512 -> 26: 13.6 against 14.5 us), 64 read the first
  // weights half as often (30176: 22.4 against 24.0, 120704: 80 against 91)
  return p.M <= 20000 ? launch_pair_f<2, ACT, T>(p, st) : launch_pair_f<4, ACT, T>(p, st);
}
template <int ACT>
static int launch_pair_a(const PhW8Pair& p, int x_type, hipStream_t st) {
  switch (x_type) {
    case PH_F32: return launch_pair_t<ACT, float>(p, st);
    case PH_F16: return launch_pair_t<ACT, _Float16>(p, st);
    default: return launch_pair_t<ACT, bf16>(p, st);
  }
}
static int launch_pair(const PhW8Pair& p, int x_type, hipStream_t st) {
  switch (p.act1) {
    case PH_ACT_RELU: return launch_pair_a<PH_ACT_RELU>(p, x_type, st);
    case PH_ACT_PRELU: return launch_pair_a<PH_ACT_PRELU>(p, x_type, st);
    default: return launch_pair_a<PH_ACT_NONE>(p, x_type, st);
  }
}

// ---- entry points --------------------------------------------------------------------------------------------------------

#define W8_MAX_K 131071      // 128 * 128 * K < 2^31
#define W8_MAX_N (1 << 20)

namespace {

// the call's device is current inside, the caller's again afterwards
struct DeviceScope {
  int prev = -1;
  bool ok = false;
  explicit DeviceScope(int device) {
    if (hipGetDevice(&prev) != hipSuccess) return;
    if (prev == device) prev = -1, ok = true;
    else ok = hipSetDevice(device) == hipSuccess;
  }
  ~DeviceScope() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};
#define W8_DEVICE(device)                                       \
  DeviceScope scope_(device);                                   \
  if (!scope_.ok) {                                             \
    ph_set_error("%s: no device %d", __func__, device);         \
    return -1;                                                  \
  }

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t q_pitch_of(int64_t K) { return up(K, 16); }
int nkb_of(int k) { return (int)(up(k, 128) / 64); }

PhRowMap row_map(const ph_rows& r) {
  PhRowMap m;
  const int64_t s0 = r.n[0] > 1 ? r.stride[0] : 0, s1 = r.n[1] > 1 ? r.stride[1] : 0, s2 = r.n[2] > 1 ? r.stride[2] : 0;
  m.n1 = (unsigned)r.n[1];
  m.n2 = (unsigned)r.n[2];
  m.s0 = s0, m.s1 = s1, m.s2 = s2;
  // evenly spaced: a dimension of one row is passed over
  int64_t step = 0, rows = 1;
  bool flat = true;
  for (int d = 2; d >= 0; d--) {
    if (r.n[d] == 1) continue;
    if (rows == 1) step = r.stride[d];
    else if (r.stride[d] != rows * step) flat = false;
    rows *= r.n[d];
  }
  m.flat = flat;
  if (flat) m.s0 = m.s1 = 0, m.s2 = step;
  return m;
}

bool rows_ok(const char* who, const ph_rows* r, int64_t& M) {
  if (!r || r->n[0] < 0 || r->n[1] < 0 || r->n[2] < 0) {
    ph_set_error("%s: bad row counts", who);
    return false;
  }
  const int64_t lim = 0x7fffffff;
  M = 0;
  if (r->n[0] == 0 || r->n[1] == 0 || r->n[2] == 0) return true;
  if (r->n[0] > lim || r->n[1] > lim || r->n[2] > lim || r->n[0] * r->n[1] > lim || r->n[0] * r->n[1] * r->n[2] > lim) {
    ph_set_error("%s: more than 2^31 - 1 rows", who);
    return false;
  }
  M = r->n[0] * r->n[1] * r->n[2];
  return true;
}

bool layer_ok(const char* who, const ph_w8_layer* l) {
  if (!l || !l->packed || !l->scale || l->n < 1 || l->n > W8_MAX_N || l->k < 1 || l->k > W8_MAX_K ||
      l->act < PH_ACT_NONE || l->act > PH_ACT_PRELU || (l->act == PH_ACT_PRELU && !l->slope)) {
    ph_set_error("%s: bad layer (1 <= n <= %d, 1 <= k <= %d, PReLU needs slopes)", who, W8_MAX_N, W8_MAX_K);
    return false;
  }
  return true;
}
bool type_ok(const char* who, int t) {
  if (t == PH_F32 || t == PH_F16 || t == PH_BF16) return true;
  ph_set_error("%s: unknown element type %d", who, t);
  return false;
}
bool some(const char* who, const void* a, const void* b) {
  if (a && b) return true;
  ph_set_error("%s: null pointer", who);
  return false;
}

bool aligned16(const void* p, const PhRowMap& r) {   // rows of bytes
  return ((uintptr_t)p & 15) == 0 && (r.s0 | r.s1 | r.s2) % 16 == 0;
}

int quantize(const void* x, int type, const PhRowMap& xr, unsigned M, int K, int8_t* q, int64_t pitch, float* scale,
             hipStream_t st) {
  switch (type) {
    case PH_F32: return launch_quantize_t((const float*)x, xr, M, K, q, pitch, scale, st);
    case PH_F16: return launch_quantize_t((const _Float16*)x, xr, M, K, q, pitch, scale, st);
    default: return launch_quantize_t((const bf16*)x, xr, M, K, q, pitch, scale, st);
  }
}

PhW8Params product_params(const int8_t* q, const PhRowMap& qr, const float* qs, unsigned M, const ph_w8_layer& l, void* out,
                          const PhRowMap& outr, int* parts) {
  PhW8Params p;
  p.q = q, p.qr = qr, p.qs = qs, p.w = l.packed, p.ws = l.scale, p.bias = l.bias, p.slope = l.slope, p.act = l.act;
  p.parts = parts;
  p.stream = 0;
  p.M = M, p.N = l.n, p.K = l.k, p.nkb = nkb_of(l.k), p.nnb = (l.n + 15) / 16, p.out = out, p.outr = outr;
  return p;
}

PhRowMap even_rows(int64_t pitch) {
  PhRowMap r = {1, 1, 1, 0, 0, pitch};
  return r;
}

// pieces of a workspace, each 256-byte aligned
struct Pieces {
  char* base;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = (T*)(base + used);
    used += up(n * (int64_t)sizeof(T), 256);
    return p;
  }
};

// The workspace of one product: its parts' sums, 8-bit rows and their scales, as far as the call needs them.
struct RowsSpace {
  Pieces w;
  Choice choice;
  int* parts;
  int8_t* q = nullptr;
  float* s = nullptr;
  RowsSpace(void* ws, int64_t M, int K, int N, bool rows, bool scales) : w{(char*)ws}, choice(choose(M, N, nkb_of(K))) {
    parts = (int*)w.take<char>(parts_bytes(choice, M, N));
    if (rows) q = w.take<int8_t>(M * q_pitch_of(K));
    if (scales) s = w.take<float>(M);
  }
  int64_t used() const { return w.used; }
};
// Of two layers: the inner rows in f32, and the larger of the two products' spaces, one after the other in one place.
struct PairSpace {
  float* h;
  RowsSpace a, b;
  int64_t hbytes;
  PairSpace(void* ws, int64_t M, int K, int H, int N)
      : h((float*)ws), a((char*)ws + up(M * up(H, 4) * 4, 256), M, K, H, true, true),
        b((char*)ws + up(M * up(H, 4) * 4, 256), M, H, N, true, true), hbytes(up(M * up(H, 4) * 4, 256)) {}
  int64_t used() const { return hbytes + (a.used() > b.used() ? a.used() : b.used()); }
};

}  // namespace

extern "C" {

int64_t ph_w8_packed_bytes(int n, int k) {
  if (n < 1 || n > W8_MAX_N || k < 1 || k > W8_MAX_K) {
    ph_set_error("ph_w8_packed_bytes: 1 <= n <= %d and 1 <= k <= %d, got %d and %d", W8_MAX_N, W8_MAX_K, n, k);
    return -1;
  }
  return up(n, 16) * up(k, 128);
}

int ph_w8_pack(int device, void* stream, const int8_t* w, int64_t row_stride, int n, int k, int8_t* packed) {
  if (ph_w8_packed_bytes(n, k) < 0 || !some("ph_w8_pack", w, packed)) return -1;
  if ((uintptr_t)packed & 15) {
    ph_set_error("ph_w8_pack: packed weights need 16-byte alignment");
    return -1;
  }
  W8_DEVICE(device);
  const int nkb = nkb_of(k), nnb = (n + 15) / 16;
  const int64_t pieces = (int64_t)nkb * nnb * 64;
  hipLaunchKernelGGL(pack_weight_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream, w,
                     row_stride, n, k, nkb, nnb, packed);
  PH_CHECK(hipGetLastError());
  return 0;
}

int ph_w8_quantize_rows(int device, void* stream, const void* x, int x_type, const ph_rows* rows, int k, int8_t* q,
                        int64_t q_pitch, float* scale) {
  int64_t M;
  if (!rows_ok("ph_w8_quantize_rows", rows, M) || !type_ok("ph_w8_quantize_rows", x_type)) return -1;
  if (k < 1 || q_pitch < q_pitch_of(k) || q_pitch % 16 || ((uintptr_t)q & 15)) {
    ph_set_error("ph_w8_quantize_rows: k %d, q_pitch %lld: rows of 8-bit values are 16-byte aligned and hold k rounded up to 16",
                 k, (long long)q_pitch);
    return -1;
  }
  if (M == 0) return 0;
  if (!some("ph_w8_quantize_rows", x, q) || !some("ph_w8_quantize_rows", x, scale)) return -1;
  W8_DEVICE(device);
  return quantize(x, x_type, row_map(*rows), (unsigned)M, k, q, q_pitch, scale, (hipStream_t)stream);
}

int64_t ph_w8_workspace(int op, int64_t m, int k, int h, int n) {
  if (m < 0 || m > 0x7fffffff || k < 1 || k > W8_MAX_K || h < 0 || h > W8_MAX_K || n < 1 || n > W8_MAX_N) {
    ph_set_error("ph_w8_workspace: bad sizes");
    return -1;
  }
  if (m == 0) return 0;
  switch (op) {
    case PH_W8_MATMUL: return RowsSpace(nullptr, m, k, n, false, false).used();
    case PH_W8_MATMUL_ANY: return RowsSpace(nullptr, m, k, n, true, false).used();
    case PH_W8_LINEAR: return few_float(m, k) ? 0 : RowsSpace(nullptr, m, k, n, true, true).used();
    case PH_W8_FEED_FORWARD:
      if (h < 1) {
        ph_set_error("ph_w8_workspace: a feed-forward's inner width is 1 or more");
        return -1;
      }
      return pair_fits(k, h, n) ? 0 : PairSpace(nullptr, m, k, h, n).used();
    default:
      ph_set_error("ph_w8_workspace: unknown operator %d", op);
      return -1;
  }
}

static bool ws_ok(const char* who, const void* ws, int64_t have, int64_t need) {
  if (need == 0 || (ws && have >= need && ((uintptr_t)ws & 255) == 0)) return true;
  ph_set_error("%s: needs a 256-byte aligned workspace of %lld bytes, got %lld", who, (long long)need, (long long)have);
  return false;
}

int ph_w8_matmul(int device, void* stream, const int8_t* q, const ph_rows* rows, const float* scale, const ph_w8_layer* layer,
                 void* out, int out_type, const int64_t* out_stride, void* ws, int64_t ws_bytes) {
  const char* who = "ph_w8_matmul";
  int64_t M;
  if (!rows_ok(who, rows, M) || !layer_ok(who, layer) || !type_ok(who, out_type)) return -1;
  if (M == 0) return 0;
  if (!some(who, q, scale) || !some(who, out, out_stride)) return -1;
  ph_rows orow = *rows;
  for (int d = 0; d < 3; d++) orow.stride[d] = out_stride[d];
  PhRowMap qr = row_map(*rows);
  const bool direct = aligned16(q, qr);
  const RowsSpace w(ws, M, layer->k, layer->n, !direct, false);
  if (!ws_ok(who, ws, ws_bytes, w.used())) return -3;
  W8_DEVICE(device);
  if (!direct) {
    const int64_t pitch = q_pitch_of(layer->k), pieces = M * (pitch / 16);
    hipLaunchKernelGGL(repitch_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream, q, qr,
                       (unsigned)M, layer->k, w.q, pitch);
    PH_CHECK(hipGetLastError());
    q = w.q;
    qr = even_rows(pitch);
  }
  return launch_product(product_params(q, qr, scale, (unsigned)M, *layer, out, row_map(orow), w.parts), w.choice, out_type,
                        (hipStream_t)stream);
}

int ph_w8_linear(int device, void* stream, const void* x, int x_type, const ph_rows* rows, const ph_w8_layer* layer, void* out,
                 int out_type, const int64_t* out_stride, void* ws, int64_t ws_bytes) {
  const char* who = "ph_w8_linear";
  int64_t M;
  if (!rows_ok(who, rows, M) || !layer_ok(who, layer) || !type_ok(who, x_type) || !type_ok(who, out_type)) return -1;
  if (M == 0) return 0;
  if (!some(who, x, out) || !some(who, out, out_stride)) return -1;
  ph_rows orow = *rows;
  for (int d = 0; d < 3; d++) orow.stride[d] = out_stride[d];
  hipStream_t st = (hipStream_t)stream;
  const PhRowMap xr = row_map(*rows), outr = row_map(orow);
  if (few_float(M, layer->k)) {
    W8_DEVICE(device);
    const FloatRows f = {x, xr};
    const PhW8Params p = product_params(nullptr, xr, nullptr, (unsigned)M, *layer, out, outr, nullptr);
    switch (out_type) {
      case PH_F32: return launch_few_float<float>(p, x_type, f, st);
      case PH_F16: return launch_few_float<_Float16>(p, x_type, f, st);
      default: return launch_few_float<bf16>(p, x_type, f, st);
    }
  }
  const int64_t pitch = q_pitch_of(layer->k);
  const RowsSpace w(ws, M, layer->k, layer->n, true, true);
  if (!ws_ok(who, ws, ws_bytes, w.used())) return -3;
  W8_DEVICE(device);
  if (quantize(x, x_type, xr, (unsigned)M, layer->k, w.q, pitch, w.s, st)) return -1;
  return launch_product(product_params(w.q, even_rows(pitch), w.s, (unsigned)M, *layer, out, outr, w.parts), w.choice, out_type, st);
}

int ph_w8_feed_forward(int device, void* stream, const void* x, int x_type, const ph_rows* rows, const ph_w8_layer* layer1,
                       const ph_w8_layer* layer2, void* out, int out_type, const int64_t* out_stride, void* ws,
                       int64_t ws_bytes) {
  const char* who = "ph_w8_feed_forward";
  int64_t M;
  if (!rows_ok(who, rows, M) || !layer_ok(who, layer1) || !layer_ok(who, layer2) || !type_ok(who, x_type) || !type_ok(who, out_type)) return -1;
  if (layer2->k != layer1->n) {
    ph_set_error("%s: the first layer has %d outputs, the second %d inputs", who, layer1->n, layer2->k);
    return -1;
  }
  if (M == 0) return 0;
  if (!some(who, x, out) || !some(who, out, out_stride)) return -1;
  const int K = layer1->k, H = layer1->n;
  ph_rows orow = *rows;
  for (int d = 0; d < 3; d++) orow.stride[d] = out_stride[d];
  hipStream_t st = (hipStream_t)stream;
  if (pair_fits(K, H, layer2->n)) {
    W8_DEVICE(device);
    const ph_w8_layer &a = *layer1, &b = *layer2;
    const PhW8Pair p = {x, row_map(*rows), (unsigned)M, K, H, b.n, nkb_of(K), (H + 15) / 16, nkb_of(H), (b.n + 15) / 16, a.act, b.act,
                        a.packed, b.packed, a.scale, a.bias, a.slope, b.scale, b.bias, b.slope, out, row_map(orow), out_type};
    return launch_pair(p, x_type, st);
  }
  const PairSpace w(ws, M, K, H, layer2->n);
  if (!ws_ok(who, ws, ws_bytes, w.used())) return -3;
  W8_DEVICE(device);
  const int64_t pitch = q_pitch_of(K), hpitch = up(H, 4), pitch2 = q_pitch_of(H);
  if (quantize(x, x_type, row_map(*rows), (unsigned)M, K, w.a.q, pitch, w.a.s, st)) return -1;
  if (launch_product(product_params(w.a.q, even_rows(pitch), w.a.s, (unsigned)M, *layer1, w.h, even_rows(hpitch), w.a.parts),
                     w.a.choice, PH_F32, st)) return -1;
  if (quantize(w.h, PH_F32, even_rows(hpitch), (unsigned)M, H, w.b.q, pitch2, w.b.s, st)) return -1;
  return launch_product(product_params(w.b.q, even_rows(pitch2), w.b.s, (unsigned)M, *layer2, out, row_map(orow), w.b.parts),
                        w.b.choice, out_type, st);
}

}  // extern "C"
