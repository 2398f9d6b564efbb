// Products of 8-bit rows with packed weights (formulas: w8a8.hip): tiles through LDS, few tokens, parts of K, and the
// choice among them.
#include "w8a8_dev.h"

// ---- product: tiles through LDS ------------------------------------------------------------------------------------------

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
  float s[TM];
#pragma unroll
  for (int i = 0; i < TM; i++) s[i] = p.qs[min(m0 + (wm * TM + i) * 16 + fr, p.M - 1)];
  const int n0 = (nb0 + wn * TN) * 16;
  Channels c[TN];
#pragma unroll
  for (int j = 0; j < TN; j++) c[j] = w8_channels(p, min(n0 + j * 16 + fq * 4, p.nnb * 16 - 4));
  WaveOut<TM, TN, O>::store(p, acc, s, m0 + wm * TM * 16, n0, lds + wave * WaveOut<TM, TN, O>::BYTES, lane, [&](int j) { return c[j]; });
}

template <int BM, int BN, int WM, int WN, int NST, bool SPLIT, typename O>
static int launch_tile(const PhW8Params& p, int parts, hipStream_t st) {
  constexpr int ring = NST * (BM + BN) * 128, tile = WM * WN * WaveOut<BM / WM / 16, BN / WN / 16, O>::BYTES;
  constexpr int lds = ring > tile ? ring : tile;
  static int granted[PH_MAX_DEVICES];
  const void* fn = (const void*)w8_tile_kernel<BM, BN, WM, WN, NST, SPLIT, O>;
  if (lds > 64 * 1024 && ph_ensure_lds(fn, lds, granted)) return -1;
  const unsigned mt = (p.M - 1) / BM + 1, nt = (p.N - 1) / BN + 1;
  if (ph_w8_launchable((int64_t)mt * nt * parts, 64 * WM * WN)) return -1;
  hipLaunchKernelGGL((w8_tile_kernel<BM, BN, WM, WN, NST, SPLIT, O>), dim3(mt * nt, SPLIT ? parts : 1), dim3(64 * WM * WN), lds, st, p, mt, nt);
  PH_CHECK(hipGetLastError());
  return 0;
}

// ---- product: few tokens -------------------------------------------------------------------------------------------------
//
// Up to 64 tokens (and more, 64 to a block, where rows of any alignment would have to be laid out anew first): the weights
// are read once, each fragment by one wave straight into registers (a fragment is 1 KiB in
// one piece), and the rows, which every block needs, come from cache.  A block has 16 channels; its waves take fragments
// along K in turn and their sums meet in LDS.
//
// T is int8_t, or the type of float rows that the block quantises itself, into LDS, while its first weights are on their
// way: for few tokens that costs less than a launch of its own before this one (ph_w8_few_float).

// up to 64 rows -> int8 rows of `pitch` bytes and their scales in LDS, all rows at once: 512 / (their number rounded up to a
// power of two) lanes a row
template <int W, typename T>
__device__ __forceinline__ void quantize_block(const FloatRows& f, unsigned M, int K, char* q, int pitch, float* scale,
                                               float* amax, int tid) {
  static_assert(W == 8, "512 threads");
  const int lg = M <= 1 ? 9 : 9 - (32 - __builtin_clz(M - 1));   // log2 of the lanes of a row, 3 .. 9
  const int G = 1 << lg, lane = tid & (G - 1), step = G * 8;
  const unsigned row = tid >> lg;
  const bool has = row < M;
  const T* const xr = (const T*)f.x + ph_row_off(f.r, has ? row : 0);
  constexpr int D = 4;   // chunks on their way at once
  Eight<T> v[D];
  float am = 0.f;
  auto load = [&](int k0) {
#pragma unroll
    for (int d = 0; d < D; d++)
      if (k0 + d * step < K) v[d].load(xr, k0 + d * step + lane * 8, K);   // (lanes beyond the end: the row's last eight)
  };
  for (int k0 = 0; k0 < K; k0 += D * step) {
    load(k0);
#pragma unroll
    for (int d = 0; d < D; d++)
      if (k0 + d * step < K) am = v[d].max_with(am);
  }
  am = max_group<8>(am);
  if (G > 8) am = max_dpp<0x140>(am);
  if (G > 16) am = max_16(am);
  if (G > 32) am = max_32(am);
  if (G > 64) {
    if ((tid & 63) == 0) amax[tid >> 6] = am;
    __syncthreads();
    const int w0 = (int)(row << lg) >> 6;
    for (int w = 0; w < G / 64; w++) am = max_abs(am, amax[w0 + w]);
  }
  const RowScale r = row_scale(am);
  if (has && lane == 0) scale[row] = scale_out(r);
  for (int k0 = 0; k0 < K; k0 += D * step) {
    if (K > D * step) load(k0);   // (else they are here)
#pragma unroll
    for (int d = 0; d < D; d++) {
      const int k = k0 + d * step + lane * 8;
      if (has && k < K) *(uint64_t*)(q + (int)row * pitch + k) = v[d].quantize(r) >> Eight<T>::shift(k, K);
    }
  }
  __syncthreads();
}

// A row's last 16 bytes -> those from k on (k + 16 - K = `over` > 0; the shift is the same in every lane that has one, and what
// moves in meets zero weights)
__device__ __forceinline__ i32x4 tail_16(i32x4 v, int K) {
  const int b = 16 - (K & 15), bs = b & 3;
  if (b & 8) v = i32x4{v[2], v[3], 0, 0};
  if (b & 4) v = i32x4{v[1], v[2], v[3], 0};
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = (int)__builtin_amdgcn_alignbyte(i < 3 ? (unsigned)v[i + 1] : 0u, (unsigned)v[i], bs);
  return v;
}

// Blocks of 64 tokens stand along z, which ends at 65535 of them; with more tokens along y too (folded into x they need a division
// in every block: 2000000 x 31 -> 16 113 -> 118 us).
constexpr unsigned FEW_Z = 64 * 65535;

template <int TM, int W, bool SPLIT, typename T, typename O>
__global__ __launch_bounds__(64 * W) void w8_few_kernel(const PhW8Params p, const FloatRows f) {
  constexpr bool FLOAT = !__is_same(T, int8_t);
  constexpr int DEPTH = 4;   // fragments of weights in flight per wave
  __shared__ __attribute__((aligned(16))) int red[W][TM][256];
  extern __shared__ __attribute__((aligned(16))) char s_q[];   // FLOAT: the rows in 8 bits
  __shared__ float s_scale[FLOAT ? 16 * TM : 1];
  __shared__ float s_amax[W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int nb = blockIdx.x;
  unsigned t = blockIdx.z;
  if (TM == 4 && !SPLIT && !FLOAT && p.M > FEW_Z) t = t * gridDim.y + blockIdx.y;
  const unsigned m0 = t * (16 * TM);
  const int nk = (p.K + 63) >> 6;   // (a fragment of zeros that the weights may end with is left out)
  const int kb0 = SPLIT ? (int)((int64_t)nk * blockIdx.y / gridDim.y) : 0;
  const int kb1 = SPLIT ? (int)((int64_t)nk * (blockIdx.y + 1) / gridDim.y) : nk;
  const int8_t* const wp = p.w + (int64_t)nb * p.nkb * 1024 + lane * 16;
  i32x4 wf[DEPTH];
  auto weights = [&](int kb) {
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
      if (kb + d * W < kb1) wf[d] = __builtin_nontemporal_load((const i32x4*)(wp + (int64_t)(kb + d * W) * 1024));
  };
  weights(kb0 + wave);
  const int pitch = p.nkb * 64 + 16;   // (16 rows at one multiple of 64 bytes would share their banks)
  if constexpr (FLOAT) quantize_block<W, T>(f, p.M, p.K, s_q, pitch, s_scale, s_amax, threadIdx.x);
  const int8_t* xp[TM];
  int xq[TM];   // FLOAT: in LDS
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const unsigned m = min(m0 + i * 16 + fr, p.M - 1);
    xp[i] = FLOAT ? nullptr : p.q + ph_row_off(p.qr, m);
    xq[i] = (int)m * pitch;
  }
  typedef i32x4 any __attribute__((aligned(1)));
  const int last = p.loose ? p.K - 16 : p.K;   // where the last 16 bytes start: nothing is read behind a loose row's end
  i32x4 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; i++) acc[i] = i32x4{0, 0, 0, 0};
  for (int kb = kb0 + wave; kb < kb1; kb += W * DEPTH) {
    i32x4 xf[DEPTH][TM], w[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      if (kb + d * W >= kb1) break;
      int k = (kb + d * W) * 64 + fq * 16;
      k = k < p.K ? k : 0;   // units behind the row's end meet zero weights
#pragma unroll
      for (int i = 0; i < TM; i++) {
        if constexpr (FLOAT) xf[d][i] = *(const i32x4*)(s_q + xq[i] + k);
        else xf[d][i] = *(const any*)(xp[i] + min(k, last));
      }
      w[d] = wf[d];
    }
    if (!FLOAT && p.loose) {
#pragma unroll
      for (int d = 0; d < DEPTH; d++) {
        if (kb + d * W >= kb1 || (kb + d * W + 1) * 64 <= p.K) continue;   // (only the last fragment of a row has an end inside)
        const int k = (kb + d * W) * 64 + fq * 16;
        if (k > last && k < p.K)
#pragma unroll
          for (int i = 0; i < TM; i++) xf[d][i] = tail_16(xf[d][i], p.K);
      }
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
    const unsigned m = m0 + wave * 16 + fr;
    const int n = nb * 16 + fq * 4;
    if (m >= p.M || n >= p.N) return;
    if (SPLIT) *(i32x4*)(p.parts + ((int64_t)blockIdx.y * p.M + m) * (p.nnb * 16) + n) = a;
    else w8_finish4<O>(p, a, m, n, FLOAT ? s_scale[m] : p.qs[m]);
  }
}

// sums of the parts of K -> out; integers, so that their order does not matter.  J lanes, 64 / J apart, share four channels' parts.
template <int J, typename O>
__global__ __launch_bounds__(256) void w8_join_kernel(const PhW8Params p, int parts) {
  const int q4 = (p.N + 3) / 4, lane = threadIdx.x & 63, j = lane / (64 / J);
  const int64_t pieces = (int64_t)p.M * q4;
  const int64_t t = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / J) + lane % (64 / J);
  const int64_t at_t = min(t, pieces - 1);   // (lanes beyond the end: the last one's again)
  const unsigned m = (unsigned)(at_t / q4);
  const int n = (int)(at_t - (int64_t)m * q4) * 4;
  const int64_t pitch = (int64_t)p.M * (p.nnb * 16);
  const int* at = p.parts + (int64_t)m * (p.nnb * 16) + n;
  i32x4 a = i32x4{0, 0, 0, 0};
  for (int s0 = j; s0 < parts; s0 += 8 * J) {   // eight at a time on their way
    i32x4 b[8];
#pragma unroll
    for (int s = 0; s < 8; s++) b[s] = s0 + s * J < parts ? *(const i32x4*)(at + (s0 + s * J) * pitch) : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 8; s++) a += b[s];
  }
#pragma unroll
  for (int d = 64 / J; d < 64; d *= 2)
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] += __shfl_xor(a[e], d);
  if (j == 0 && t < pieces) w8_finish4<O>(p, a, m, n, p.qs[m]);
}

template <int TM, bool SPLIT, typename O>
static int launch_few(const PhW8Params& p, int parts, hipStream_t st) {
  const unsigned tokens = (p.M - 1) / (16 * TM) + 1, y = SPLIT ? parts : (p.M - 1) / FEW_Z + 1, z = SPLIT ? tokens : (tokens - 1) / y + 1;
  if (ph_w8_launchable((int64_t)p.nnb * y * z, 512)) return -1;
  hipLaunchKernelGGL((w8_few_kernel<TM, 8, SPLIT, int8_t, O>), dim3(p.nnb, y, z), dim3(512), 0, st, p, FloatRows{});
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

// the parts' sums to memory, back, and the launch that joins them
static float join_us(int64_t M, int64_t n16, int parts) { return parts > 1 ? 3.3f + (float)M * n16 * 4e-6f * parts / 2.f : 0.f; }   // (2 TB/s)

// Splitting K pays where there are far fewer blocks than CUs: the parts' sums (4 bytes each) are written, read and
// joined by a second launch.
PhW8Choice ph_w8_choose(int64_t M, int N, int nkb) {
  const int steps = nkb / 2;
  const int64_t n16 = (N + 15) / 16 * 16;
  const float wire = (float)n16 * nkb * 64 / 5.5e6f;   // the weights, once, from memory
  PhW8Choice best = {K_64, 1, 1e30f};
  const int64_t small = (M + 63) / 64 * ((N + 63) / 64);   // blocks of the smallest tile: two rounds of them need no parts
  for (int parts = 1; parts <= 32 && parts <= steps; parts *= 2) {
    if (parts > 1 && (small >= 1024 || (float)M * n16 * parts > (float)(1 << 24))) break;
    const int s = (steps + parts - 1) / parts;
    for (int k = 0; k < N_KERNELS; k++) {
      const Kernel& c = kernels[k];
      const int64_t blocks = (M + c.bm - 1) / c.bm * ((N + c.bn - 1) / c.bn) * parts;
      const int64_t each = (blocks + 255) / 256, rounds = (each + c.fit - 1) / c.fit;
      const float run = (float)s * (each * c.full > rounds * c.alone ? each * c.full : rounds * c.alone);
      const float t = (run > wire ? run : wire) + rounds * c.fixed + join_us(M, n16, parts);
      if (t < best.us) best = {k, parts, t};
    }
    if (M <= 64) {   // a wave's step is one fragment of 64 k; blocks' loads share the memory's rate
      const int tm = (int)(M + 15) / 16;
      const int64_t blocks = n16 / 16 * parts, rounds = (blocks + 511) / 512;
      const float run = (s * 2 + 31) / 32 * rounds * (0.35f + 0.45f * tm), w = wire * (0.8f + 0.2f * tm);
      const float t = 1.f + 0.5f * tm + (run > w ? run : w) + join_us(M, n16, parts);
      if (t < best.us) best = {K_FEW, parts, t};
    }
  }
  return best;
}

// Rows of any alignment: the few-token kernel takes them as they are, 64 tokens to a block, as long as that costs less than a
// launch that lays them out anew (3.4 us and 16-byte pieces at 2 TB/s) and a product of those.  A load of 16 rows' 64 bytes that
// start anywhere takes a CU 0.07 us (a fragment of aligned rows hardly anything), so long rows go the other way.
// us, direct | laid out anew:
//   1613 x 55 -> 22 3.6 | 7.3, 500 x 301 -> 300 4.7 | 7.5, 5000 x 31 -> 100 5.3 | 7.3, 70 x 1001 -> 40 6.1 | 8.1
//   37 x 2047 -> 1001 11.2 | 8.7, 70 x 2001 -> 40 in one part 10.8, in four 6.6 | 9.4, 64 x 4001 -> 2000 23 | 12.5
PhW8Choice ph_w8_choose_loose(int64_t M, int K, int N) {
  const int nkb = (K + 63) / 64;
  const PhW8Choice c = ph_w8_choose(M, N, (K + 127) / 128 * 2);
  PhW8Choice best = {-1, 1, c.us + 3.4f + (float)M * K * 1e-6f};
  if (K < 16) return best;
  const int64_t n16 = (N + 15) / 16 * 16;
  const int tm = M > 48 ? 4 : (int)(M + 15) / 16;
  for (int parts = 1; parts <= 8 && parts <= (nkb + 1) / 2; parts *= 2) {
    if (parts > 1 && (float)M * n16 * parts > (float)(1 << 22)) break;
    const int64_t blocks = (M + 63) / 64 * (n16 / 16) * parts, rounds = (blocks + 255) / 256;
    if (!ph_w8_fits_launch(blocks, 512)) break;   // (the tiles' blocks, of 64 channels and 256 threads, are far fewer)
    const float t = 2.5f + (float)rounds * (0.7f + 0.07f * tm * ((nkb + parts - 1) / parts)) + join_us(M, n16, parts);
    if (t < best.us) best = {K_FEW, parts, t};
  }
  return best;
}

int64_t ph_w8_parts_bytes(const PhW8Choice& c, int64_t M, int N) {
  return c.parts > 1 ? (int64_t)c.parts * M * ((N + 15) / 16 * 16) * 4 : 0;
}

template <bool SPLIT, typename O>
static int launch_kernel(const PhW8Params& p, const PhW8Choice& c, hipStream_t st) {
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

// ph_w8_parts_bytes() of workspace at p.parts
template <typename O>
static int launch_product_t(const PhW8Params& p, const PhW8Choice& c, hipStream_t st) {
  if (c.parts == 1) return launch_kernel<false, O>(p, c, st);
  if (launch_kernel<true, O>(p, c, st)) return -1;
  const int64_t pieces = (int64_t)p.M * ((p.N + 3) / 4);
  if (ph_w8_launchable(pieces, 1)) return -1;
  // few sums of many parts: a lane that adds them all up waits for memory several times over (61 x 32500 -> 187 in 32
  // parts 11.3 -> 9.5 us)
  if (c.parts >= 8 && pieces < 65536) hipLaunchKernelGGL((w8_join_kernel<8, O>), dim3((unsigned)((pieces + 31) / 32)), dim3(256), 0, st, p, c.parts);
  else hipLaunchKernelGGL((w8_join_kernel<1, O>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, st, p, c.parts);
  PH_CHECK(hipGetLastError());
  return 0;
}

// Up to 64 tokens of up to 32 K values in all: the product's blocks quantise the rows themselves.  us on the GPU, against two
// launches: 1 x 4096 -> 4096 6.0 (7.2), 12 x 1001 -> 512 5.2 (5.8), 8 x 4096 -> 4096 9.0 (8.2); a call from Python takes 8.3
// in the last case, with two launches 12.  16 x 4096: 12.7 (8.9).
bool ph_w8_few_float(int64_t M, int K) { return M <= 64 && M * K <= 32768; }

template <int TM, typename T, typename O>
static int launch_few_float_t(const PhW8Params& p, const FloatRows& f, hipStream_t st) {
  const int lds = (int)p.M * (p.nkb * 64 + 16);   // at most 41 KB
  static int granted[PH_MAX_DEVICES];
  if (lds > 16 * 1024 && ph_ensure_lds((const void*)w8_few_kernel<TM, 8, false, T, O>, lds, granted)) return -1;
  hipLaunchKernelGGL((w8_few_kernel<TM, 8, false, T, O>), dim3(p.nnb), dim3(512), lds, st, p, f);
  PH_CHECK(hipGetLastError());
  return 0;
}
template <typename O>
static int launch_few_float(const PhW8Params& p, int x_type, const FloatRows& f, hipStream_t st) {
  switch (x_type) {
    case PH_F32: return p.M <= 16 ? launch_few_float_t<1, float, O>(p, f, st) : launch_few_float_t<4, float, O>(p, f, st);
    case PH_F16: return p.M <= 16 ? launch_few_float_t<1, _Float16, O>(p, f, st) : launch_few_float_t<4, _Float16, O>(p, f, st);
    default: return p.M <= 16 ? launch_few_float_t<1, bf16, O>(p, f, st) : launch_few_float_t<4, bf16, O>(p, f, st);
  }
}
int ph_launch_w8_few_float(const PhW8Params& p, const FloatRows& f, int x_type, int out_type, hipStream_t st) {
  switch (out_type) {
    case PH_F32: return launch_few_float<float>(p, x_type, f, st);
    case PH_F16: return launch_few_float<_Float16>(p, x_type, f, st);
    default: return launch_few_float<bf16>(p, x_type, f, st);
  }
}

int ph_launch_w8_product(const PhW8Params& p, const PhW8Choice& c, int out_type, hipStream_t st) {
  switch (out_type) {
    case PH_F32: return launch_product_t<float>(p, c, st);
    case PH_F16: return launch_product_t<_Float16>(p, c, st);
    default: return launch_product_t<bf16>(p, c, st);
  }
}
