// 8-bit layers from float rows in one kernel (formulas: w8a8.hip).
#include "w8a8_dev.h"

constexpr int PITCH = PAIR_MAX + 16;   // of an 8-bit row in LDS: 16 rows' units lie in different banks

// rows m0 .. of 8 <= K <= 512 values -> 8 bits and scales in LDS; 16 lanes a row, 32 rows at a time, 4 chunks of 128 values.
template <int TF, typename T, typename Between>
__device__ __forceinline__ void rows_to_lds(const void* rows, const PhRowMap& xr, unsigned M, int K, unsigned m0, char* q, float* s,
                                            int tid, Between between) {
  constexpr int RP = TF / 2, CH = 4;
  Eight<T> raw[RP][CH];
#pragma unroll
  for (int r = 0; r < RP; r++) {
    const T* row = (const T*)rows + ph_row_off(xr, min(m0 + r * 32 + (tid >> 4), M - 1));
#pragma unroll
    for (int c = 0; c < CH; c++)
      if (c * 128 < K) raw[r][c].load_long(row, c * 128 + (tid & 15) * 8, K);
  }
  between();
  float x[RP][CH][8];
  RowScale sc[RP];
#pragma unroll
  for (int r = 0; r < RP; r++) {
    float am = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++)
      if (c * 128 < K) {
        raw[r][c].to_floats(x[r][c]);
#pragma unroll
        for (int i = 0; i < 8; i++) am = max_abs(am, x[r][c][i]);
      }
    sc[r] = row_scale(max_group<16>(am));
  }
#pragma unroll
  for (int r = 0; r < RP; r++) {
    const int t = r * 32 + (tid >> 4);
    if ((tid & 15) == 0) s[t] = scale_out(sc[r]);
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const int k = c * 128 + (tid & 15) * 8;
      if (k < K) *(uint64_t*)(q + t * PITCH + k) = quantize_8(x[r][c], sc[r]) >> Eight<T>::shift(k, K);
    }
  }
}

// TF token fragments in LDS (xq: this lane's unit of the first) x 4 channel fragments straight from cache, one read ahead;
// nkb is even
template <int TF>
__device__ __forceinline__ void rows_product(const char* xq, const int8_t* const (&wp)[4], i32x4 (&wa)[4], int nkb,
                                             i32x4 (&acc)[4][TF]) {
  i32x4 wb[4];
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int i = 0; i < TF; i++) acc[j][i] = i32x4{0, 0, 0, 0};
  for (int kb = 0; kb < nkb; kb += 2) {
#pragma unroll
    for (int j = 0; j < 4; j++) wb[j] = *(const i32x4*)(wp[j] + (kb + 1) * 1024);
#pragma unroll
    for (int i = 0; i < TF; i++) {
      const i32x4 xf = *(const i32x4*)(xq + i * 16 * PITCH + kb * 64);
#pragma unroll
      for (int j = 0; j < 4; j++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa[j], xf, acc[j][i], 0, 0, 0);
    }
    const int nx = min(kb + 2, nkb - 1);
#pragma unroll
    for (int j = 0; j < 4; j++) wa[j] = *(const i32x4*)(wp[j] + nx * 1024);
#pragma unroll
    for (int i = 0; i < TF; i++) {
      const i32x4 xf = *(const i32x4*)(xq + i * 16 * PITCH + kb * 64 + 64);
#pragma unroll
      for (int j = 0; j < 4; j++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wb[j], xf, acc[j][i], 0, 0, 0);
    }
  }
}

// ---- one layer -------------------------------------------------------------------------------------------------------
//
// Float rows of 8 <= K <= 512 values x layer: a block quantises its 16 TF tokens into LDS and multiplies them with 64 WN
// channels, the rows' 8-bit form never in memory.
template <int TF, int WN, typename T, typename O>
__global__ __launch_bounds__(512, 4) void w8_rows_kernel(const PhW8Params p, const FloatRows f) {
  constexpr int BT = 16 * TF, WM = 8 / WN, TFW = TF / WM;
  static_assert(TFW * WM == TF, "token fragments divide among the waves");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* const s1 = (float*)lds;
  float* const par = s1 + BT;   // scale, bias, slope of the block's channels [3][64 WN]
  char* const q = (char*)(par + 3 * 64 * WN);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4, wn = wave % WN, wm = wave / WN;
  const unsigned m0 = blockIdx.x * BT;
  const int nb0 = (blockIdx.y * WN + wn) * 4;
  const int8_t* wp[4];
  i32x4 wa[4];
#pragma unroll
  for (int j = 0; j < 4; j++) wp[j] = p.w + (int64_t)min(nb0 + j, p.nnb - 1) * p.nkb * 1024 + lane * 16;
  rows_to_lds<TF, T>(f.x, f.r, p.M, p.K, m0, q, s1, tid, [&] {
#pragma unroll
    for (int j = 0; j < 4; j++) wa[j] = *(const i32x4*)wp[j];
    for (int n = tid; n < 64 * WN; n += 512) {
      const int at = blockIdx.y * (64 * WN) + n;
      const bool is = at < p.nnb * 16;
      par[n] = is ? p.ws[at] : 0.f;
      par[64 * WN + n] = is && p.bias ? p.bias[at] : 0.f;
      par[128 * WN + n] = is && p.slope ? p.slope[at] : 0.f;
    }
  });
  __syncthreads();
  i32x4 acc[4][TFW];
  rows_product<TFW>(q + (wm * TFW * 16 + fr) * PITCH + fq * 16, wp, wa, p.nkb, acc);
  float s[TFW];
#pragma unroll
  for (int i = 0; i < TFW; i++) s[i] = s1[(wm * TFW + i) * 16 + fr];
  __syncthreads();   // the rows have been read everywhere: their place is free
  if (nb0 < p.nnb) WaveOut<TFW, 4, O>::store(p, acc, s, m0 + wm * TFW * 16, nb0 * 16, q + wave * WaveOut<TFW, 4, O>::BYTES, lane,
                                                [&](int j) {
                                                  __builtin_amdgcn_sched_barrier(0);   // (one column's at a time: registers)
                                                  const float* c = par + (wn * 4 + j) * 16 + fq * 4;
                                                  return Channels{*(const f32x4*)c, *(const f32x4*)(c + 64 * WN), *(const f32x4*)(c + 128 * WN)};
                                                });
}

template <int TF, int WN, typename T, typename O>
static int launch_rows_f(const PhW8Params& p, const FloatRows& f, hipStream_t st) {
  constexpr int BT = 16 * TF, rows = BT * PITCH, tile = 8 * WaveOut<TF * WN / 8, 4, O>::BYTES;
  constexpr int lds = BT * 4 + 12 * 64 * WN + (rows > tile ? rows : tile);   // <= 76 KB: two blocks a CU
  static int granted[PH_MAX_DEVICES];
  if (lds > 64 * 1024 && ph_ensure_lds((const void*)w8_rows_kernel<TF, WN, T, O>, lds, granted)) return -1;
  if (ph_w8_launchable((int64_t)((p.M - 1) / BT + 1) * ((p.N - 1) / (64 * WN) + 1), 512)) return -1;
  hipLaunchKernelGGL((w8_rows_kernel<TF, WN, T, O>), dim3((p.M - 1) / BT + 1, (p.N - 1) / (64 * WN) + 1), dim3(512), lds, st, p, f);
  PH_CHECK(hipGetLastError());
  return 0;
}
// us for bf16 -> bf16, beside quantisation and product in two launches:
//   32 tokens x 256 channels: 3772 x 288 -> 256 6.4 (two launches 7.8), 3772 x 512 -> 26 7.1 (8.3), 1000 x 200 -> 4000 7.3 (8.4)
//   64 x 512: 120704 x 384 -> 512 57 (75), 30176 x 384 -> 1024 28 (38), 30176 x 512 -> 2048 63 (69)
//   64 x 256: 120704 x 288 -> 256 40 (47);  64 x 128: 120704 x 512 -> 52 47 (50), 120704 x 384 -> 128 40 (47)
bool ph_w8_rows_fit(int64_t M, int K, int N) { return K >= 8 && K <= PAIR_MAX && N <= (M <= 8192 ? 4096 : 2048); }

template <typename T, typename O>
static int launch_rows_t(const PhW8Params& p, const FloatRows& f, hipStream_t st) {
  if (p.M <= 8192) return launch_rows_f<2, 4, T, O>(p, f, st);
  if (p.N > 256) return launch_rows_f<4, 8, T, O>(p, f, st);
  if (p.N > 128) return launch_rows_f<4, 4, T, O>(p, f, st);
  return launch_rows_f<4, 2, T, O>(p, f, st);
}
template <typename T>
static int launch_rows_x(const PhW8Params& p, const FloatRows& f, int out_type, hipStream_t st) {
  switch (out_type) {
    case PH_F32: return launch_rows_t<T, float>(p, f, st);
    case PH_F16: return launch_rows_t<T, _Float16>(p, f, st);
    default: return launch_rows_t<T, bf16>(p, f, st);
  }
}

int ph_launch_w8_rows(const PhW8Params& p, const FloatRows& f, int x_type, int out_type, hipStream_t st) {
  switch (x_type) {
    case PH_F32: return launch_rows_x<float>(p, f, out_type, st);
    case PH_F16: return launch_rows_x<_Float16>(p, f, out_type, st);
    default: return launch_rows_x<bf16>(p, f, out_type, st);
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
// 120704 x 384 -> 512 -> 52 bf16: 59 .. 64 us (its bytes 22, its products 22 at 2.4 POP/s).  Per SIMD 24.8 k vector instructions
// (43 us at 4 cycles each, less as fma, add, mul take 2) and 1650 matrix instructions (11 us); a wave waits for memory, LDS or
// its block 43 % of its time and for another wave's instruction 24 %.
constexpr int AHEAD = 512;   // blocks that run at a time: two on each of 256 CUs

template <int TF, int ACT, typename T>
__global__ __launch_bounds__(512, 4) void w8_pair_kernel(const PhW8Pair p) {
  constexpr int BT = 16 * TF;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* const q = lds;                                // the rows in 8 bits, then the inner rows
  float* const s1 = (float*)(q + BT * PITCH);
  float* const s2 = s1 + BT;
  float* const red = s2 + BT;                         // [8][BT]
  float* const par = red + 8 * BT;                    // scale, bias, slope of the inner channels [3][PAIR_MAX]
  float* const par2 = par + 3 * PAIR_MAX;             // of the outputs [3][64]
  char* const w2 = (char*)(par2 + 3 * 64);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const unsigned m0 = blockIdx.x * BT;
  const int8_t* wp[4];
  i32x4 wa[4];
#pragma unroll
  for (int j = 0; j < 4; j++) wp[j] = p.w1 + (int64_t)min(wave * 4 + j, p.nnb1 - 1) * p.nkb1 * 1024 + lane * 16;
  // (from cache, so here before the rows, which loads that return in order would hold up otherwise)
  for (int f = wave; f < p.nnb2 * p.nkb2; f += 8)
    __builtin_amdgcn_global_load_lds((glb_void*)(p.w2 + f * 1024 + lane * 16), (lds_void*)(w2 + f * 1024), 16, 0, 0);
  const bool is = tid < p.nnb1 * 16;
  float out_par = 0.f;
  if (tid < 3 * 64 && (tid & 63) < p.nnb2 * 16) {
    const float* const from = tid < 64 ? p.ws2 : tid < 128 ? p.bias2 : p.slope2;
    if (from) out_par = from[tid & 63];
  }
  const float par0_ = is ? p.ws1[tid] : 0.f, par1_ = is && p.bias1 ? p.bias1[tid] : 0.f, par2_ = is && p.slope1 ? p.slope1[tid] : 0.f;
#pragma unroll
  for (int j = 0; j < 4; j++) wa[j] = *(const i32x4*)wp[j];
  rows_to_lds<TF, T>(p.x, p.xr, p.M, p.K, m0, q, s1, tid, [&] {});
  const bool exists = tid < p.H;   // channels that do not: zeros, whatever stands in their places, as all enter the rows' maxima
  par[tid] = exists ? par0_ : 0.f, par[PAIR_MAX + tid] = exists ? par1_ : 0.f, par[2 * PAIR_MAX + tid] = exists ? par2_ : 0.f;
  if (tid < 3 * 64) par2[tid] = out_par;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the second layer's weights are in LDS (as the rows, requested after them)
  __syncthreads();
  const char* const xq = q + fr * PITCH + fq * 16;
  i32x4 acc[4][TF];
  rows_product<TF>(xq, wp, wa, p.nkb1, acc);
  // A line of each 128 bytes of the rows that the block after the next on this CU will read: its loads find them in L2
  // (120704 x 384 -> 512 -> 52 74 -> 72.5 us).
  T ahead = T(0.f);
  if (TF == 4) {
    const int64_t m = (int64_t)m0 + AHEAD * BT + (tid >> 3);
    const int k = (tid & 7) * (128 / (int)sizeof(T));
    ahead = ((const T*)p.x)[ph_row_off(p.xr, m < p.M ? (unsigned)m : p.M - 1) + min(k, p.K - 1)];
  }
  __builtin_amdgcn_sched_barrier(0);
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
    quantize_n<false>(v, r, o);
#pragma unroll
    for (int j = 0; j < 4; j++) *(unsigned*)(q + (i * 16 + fr) * PITCH + (wave * 4 + j) * 16 + fq * 4) = o[j];
    __builtin_amdgcn_sched_barrier(0);
  }
  // (read here, under the rounding: one after the other behind the last product they take 0.5 us)
  PhW8Out o = p.out[0];
  const int act2 = p.act2, n_out = p.n_out, nnb2 = p.nnb2, nkb2 = p.nkb2;
  asm volatile("" ::"s"(o.p), "s"(o.step), "s"(o.type), "s"(o.r.flat), "s"(o.r.s2), "s"(act2), "s"(n_out), "s"(nnb2), "s"(nkb2));
  __syncthreads();
  // second product: a wave has one fragment of channels and every dt-th fragment of tokens
  const int div = nnb2 > 2 ? 4 : nnb2, nb2 = wave % div, t0 = wave / div, dt = 8 / div;
  constexpr int U = TF / 2;
  i32x4 z[U];
#pragma unroll
  for (int u = 0; u < U; u++) z[u] = i32x4{0, 0, 0, 0};
  const int n = nb2 * 16 + fq * 4;
  const Channels c2 = {*(const f32x4*)(par2 + n), *(const f32x4*)(par2 + 64 + n), *(const f32x4*)(par2 + 128 + n)};
  const char* const wq = w2 + min(nb2, nnb2 - 1) * nkb2 * 1024 + lane * 16;
  for (int kb = 0; kb < nkb2; kb += 4) {
    i32x4 w[4], xf[4][U];
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int at = min(kb + b, nkb2 - 1);
      w[b] = *(const i32x4*)(wq + at * 1024);
#pragma unroll
      for (int u = 0; u < U; u++) xf[b][u] = *(const i32x4*)(xq + min(t0 + u * dt, TF - 1) * 16 * PITCH + at * 64);
    }
#pragma unroll
    for (int b = 0; b < 4; b++)
      if (kb + b < nkb2)
#pragma unroll
        for (int u = 0; u < U; u++) z[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[b], xf[b][u], z[u], 0, 0, 0);
  }
  f32x4 v[U];
#pragma unroll
  for (int u = 0; u < U; u++) v[u] = w8_values_of(z[u], c2, s2[min(t0 + u * dt, TF - 1) * 16 + fr], act2);
  for (int d = 0; d < n_out; d++) {
    if (d) o = p.out[d];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = t0 + u * dt;
      const unsigned m = m0 + i * 16 + fr;
      if (i >= TF || m >= p.M || n >= p.N || nb2 >= nnb2) continue;
      const int64_t off = ph_row_off(o.r, m) + n * o.step;
      if (o.step != 1) {   // planes of f32
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (n + e < p.N) ((float*)o.p)[off + e * o.step] = v[u][e];
      } else if (o.type == PH_F32) {
        w8_store4<float>((float*)o.p + off, v[u], p.N - n);
      } else if (o.type == PH_F16) {
        w8_store4<_Float16>((_Float16*)o.p + off, v[u], p.N - n);
      } else {
        w8_store4<bf16>((bf16*)o.p + off, v[u], p.N - n);
      }
    }
  }
  if (TF == 4) asm volatile("" ::"v"(ahead));
}

bool ph_w8_pair_fits(int K, int H, int N) { return K >= 8 && K <= PAIR_MAX && H <= PAIR_MAX && N <= 64; }

template <int TF, int ACT, typename T>
static int launch_pair_f(const PhW8Pair& p, hipStream_t st) {
  constexpr int BT = 16 * TF;
  const int lds = BT * PITCH + 10 * BT * 4 + 12 * PAIR_MAX + 12 * 64 + p.nnb2 * p.nkb2 * 1024;   // <= 74 KB: two blocks a CU
  static int granted[PH_MAX_DEVICES];
  if (lds > 64 * 1024 && ph_ensure_lds((const void*)w8_pair_kernel<TF, ACT, T>, lds, granted)) return -1;
  if (ph_w8_launchable((p.M - 1) / BT + 1, 512)) return -1;
  hipLaunchKernelGGL((w8_pair_kernel<TF, ACT, T>), dim3((p.M - 1) / BT + 1), dim3(512), lds, st, p);
  PH_CHECK(hipGetLastError());
  return 0;
}
template <int ACT, typename T>
static int launch_pair_t(const PhW8Pair& p, hipStream_t st) {
  // 32 tokens a block fill the chip earlier (3772 tokens of 384 -> 512 -> 26: 7.7 against 11.3 us, 15088: 11.1 against 12.2), 64 read
  // the first weights half as often (30176: 16.5 against 18.6, 120704 -> 52: 59 against 69); 20000: 15.6 and 16.0
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
int ph_launch_w8_pair(const PhW8Pair& p, int x_type, hipStream_t st) {
  switch (p.act1) {
    case PH_ACT_RELU: return launch_pair_a<PH_ACT_RELU>(p, x_type, st);
    case PH_ACT_PRELU: return launch_pair_a<PH_ACT_PRELU>(p, x_type, st);
    default: return launch_pair_a<PH_ACT_NONE>(p, x_type, st);
  }
}
