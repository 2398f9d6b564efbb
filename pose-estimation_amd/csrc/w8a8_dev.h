// Device code that the 8-bit kernels share: rounding of rows to 8 bits, and what follows an integer sum.
#pragma once
#include "w8a8.h"

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void glb_void;

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
  float s, inv, half;   // scale, 1 / scale to 2^-23 of it, scale / 2
  bool finite;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.finite = amax < __builtin_inff();
  // amax / 127, rounded as a division rounds it (compared for every f32)
  const float y = amax * (1.f / 127.f);
  r.s = r.finite ? fmaxf(__builtin_fmaf(__builtin_fmaf(-127.f, y, amax), 1.f / 127.f, y), 0x1p-126f) : 1.f;
  r.inv = __builtin_amdgcn_rcpf(r.s);
  r.half = 0.5f * r.s;
  return r;
}
__device__ __forceinline__ float scale_out(const RowScale& r) { return r.finite ? r.s : __builtin_nanf(""); }

// round_half_even(x / s), N values to N bytes; ZERO: zeros for a row that is not finite (else anything).  Adding 1.5 * 2^23
// rounds to a whole number, which then stands in the low bits of the sum.  x * (1/s) is within 127 * 2^-22 of the quotient, so
// that number is the wanted one or its neighbour; the remainder x - q s is exact in one fused operation and tells which.
// Where no remainder reaches half a step, as almost always, all stand.  (One rounding that leaves the fraction in the sum's
// low bits takes an operation less, but shifts and integer minima run at half the rate of fma and add: 28 -> 30 us.)
template <bool ZERO, int N>
__device__ __forceinline__ void quantize_n(const float (&x)[N], const RowScale& r, unsigned (&out)[N / 4]) {
  constexpr float MAGIC = 12582912.f;
  float t[N], worst = 0.f;
#pragma unroll
  for (int i = 0; i < N; i++) {
    t[i] = __builtin_fmaf(x[i], r.inv, MAGIC);
    worst = fmaxf(worst, fabsf(__builtin_fmaf(-(t[i] - MAGIC), r.s, x[i])));
  }
  if (worst >= r.half) {
    const float up = r.s < 1.f ? 0x1p64f : 1.f, s = r.s * up, half = 0.5f * s;   // (half the smallest scales is no float)
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float rem = __builtin_fmaf(-(t[i] - MAGIC), s, x[i] * up), a = fabsf(rem);
      const bool odd = __float_as_uint(t[i]) & 1;
      const float far = odd ? a : __uint_as_float(__float_as_uint(a) - (a > 0.f));   // a tie moves an odd number only
      t[i] += far >= half ? __builtin_copysignf(1.f, rem) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < N / 4; i++) {
    const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 1]), __float_as_uint(t[4 * i]), 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 3]), __float_as_uint(t[4 * i + 2]), 0x04000c0cu);
    out[i] = ZERO && !r.finite ? 0 : lo | hi;
  }
}

template <bool ZERO = false>
__device__ __forceinline__ uint64_t quantize_8(const float (&x)[8], const RowScale& r) {
  unsigned o[2];
  quantize_n<ZERO>(x, r, o);
  return (uint64_t)o[1] << 32 | o[0];
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
  __device__ __forceinline__ void to_floats(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)v[i];
  }
  template <bool ZERO = false>
  __device__ __forceinline__ uint64_t quantize(const RowScale& r) const {
    float x[8];
    to_floats(x);
    return quantize_8<ZERO>(x, r);
  }
};

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

__device__ __forceinline__ f32x4 w8_values_of(const i32x4 acc, const Channels& c, float s, int act) {
  if (act == PH_ACT_RELU) return w8_values<PH_ACT_RELU>(acc, c, s);
  if (act == PH_ACT_PRELU) return w8_values<PH_ACT_PRELU>(acc, c, s);
  return w8_values<PH_ACT_NONE>(acc, c, s);
}
// one sum of four channels -> out
template <typename O>
__device__ __forceinline__ void w8_finish4(const PhW8Params& p, const i32x4 a, unsigned m, int n, float s) {
  w8_store4<O>((O*)p.out + ph_row_off(p.outr, m) + n, w8_values_of(a, w8_channels(p, n), s, p.act), p.N - n);
}

// A wave's TM x TN fragments -> out, tokens m0 + .. (s: the scales of a lane's tokens), channels n0 + ...  In a fragment the
// 16 lanes side by side hold 16 tokens (rows of out) and 4 channels each: stored like that, every 8-byte piece is a request of
// its own (13 us for a 256 x 256 tile of bf16).  So two fragments' tokens at a time go through the wave's own LDS piece and
// leave as whole rows of its channels, 16 bytes a lane.
template <int TM, int TN, typename O>
struct WaveOut {
  static constexpr int ROW = TN * 16 * (int)sizeof(O);
  static constexpr int PITCH = ROW + 16;
  static constexpr int STEP = TM < 2 ? 1 : 2;
  static constexpr int BYTES = STEP * 16 * PITCH;
  typedef O oe __attribute__((ext_vector_type(16 / sizeof(O)), aligned(sizeof(O))));
  typedef O o4 __attribute__((ext_vector_type(4)));

  // channels(j): those of this lane in fragment column j
  template <int ACT, bool STREAM, typename F>
  static __device__ __forceinline__ void put(const PhW8Params& p, const i32x4 (&acc)[TN][TM], const float (&s)[TM], unsigned m0, int n0,
                                             char* buf, int lane, const F& channels) {
    const int fr = lane & 15, fq = lane >> 4;
    constexpr int PER = 16 / (int)sizeof(O);          // values of a 16-byte unit
    constexpr int UNITS = STEP * 16 * (ROW / 16);     // units of a pass
#pragma unroll
    for (int i0 = 0; i0 < TM; i0 += STEP) {
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const Channels c = channels(j);
#pragma unroll
        for (int i = 0; i < STEP; i++) {
          const f32x4 v = w8_values<ACT>(acc[j][i0 + i], c, s[i0 + i]);
          o4 w;
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = (O)v[e];
          *(o4*)(buf + (i * 16 + fr) * PITCH + (j * 16 + fq * 4) * (int)sizeof(O)) = w;
        }
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
  template <typename F>
  static __device__ __forceinline__ void store(const PhW8Params& p, const i32x4 (&acc)[TN][TM], const float (&s)[TM], unsigned m0,
                                               int n0, char* buf, int lane, const F& channels) {
    if (p.stream) store_act<true>(p, acc, s, m0, n0, buf, lane, channels);
    else store_act<false>(p, acc, s, m0, n0, buf, lane, channels);
  }
  template <bool STREAM, typename F>
  static __device__ __forceinline__ void store_act(const PhW8Params& p, const i32x4 (&acc)[TN][TM], const float (&s)[TM],
                                                   unsigned m0, int n0, char* buf, int lane, const F& channels) {
    if (p.act == PH_ACT_RELU) put<PH_ACT_RELU, STREAM>(p, acc, s, m0, n0, buf, lane, channels);
    else if (p.act == PH_ACT_PRELU) put<PH_ACT_PRELU, STREAM>(p, acc, s, m0, n0, buf, lane, channels);
    else put<PH_ACT_NONE, STREAM>(p, acc, s, m0, n0, buf, lane, channels);
  }
};
