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

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }

// |v| as an integer that orders like it; NaN and infinities are >= 0x7f800000
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct RowScale {
  float s, inv, half;   // scale, 1 / scale, scale / 2
};
__device__ __forceinline__ RowScale row_scale(unsigned amax_bits, bool& finite) {
  finite = amax_bits < 0x7f800000u;
  RowScale r;
  r.s = finite ? fmaxf(__uint_as_float(amax_bits) / 127.f, 0x1p-126f) : 1.f;
  r.inv = 1.f / r.s;
  r.half = 0.5f * r.s;
  return r;
}
// round_half_even(x / s): x * (1/s) is within 127 * 2^-23 of the quotient, so its rounding is the wanted number or its
// neighbour; the remainder x - q s is exact in one fused operation and tells which.
__device__ __forceinline__ int quant_one(float x, const RowScale& r) {
  const float q = rintf(x * r.inv);
  const float rem = __builtin_fmaf(-q, r.s, x);
  const float a = fabsf(rem);
  const int qi = (int)q;
  const bool move = a > r.half || (a == r.half && (qi & 1));
  return qi + (move ? (rem > 0.f ? 1 : -1) : 0);
}

template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
  f32x4 a, b;
  __device__ __forceinline__ float get(int i) const { return i < 4 ? a[i] : b[i - 4]; }
};
template <>
struct Vec8<_Float16> {
  _Float16 v __attribute__((ext_vector_type(8)));
  __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
};
template <>
struct Vec8<bf16> {
  bf16x8 v;
  __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
};

// A group of 64 * NW threads owns a row; a thread holds its values of up to CH chunks of 8 (in registers between the
// two passes; rows longer than that are read again).  VEC: rows are 16-byte aligned, chunks are loaded whole.
template <typename T, bool VEC, int NW, int CH>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void quantize_rows_kernel(const T* __restrict__ x, PhRowMap xr, unsigned M,
                                                                               int K, int8_t* __restrict__ q,
                                                                               int64_t q_pitch, float* __restrict__ scale) {
  constexpr int TPR = 64 * NW;
  const int lane = threadIdx.x & (TPR - 1);
  const unsigned m = NW == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (NW == 1 && m >= M) return;
  const T* row = x + ph_row_off(xr, m);
  const int step = TPR * 8;
  float v[CH][8];
  unsigned am = 0;
  auto load = [&](int k, float* o) {
    if (VEC && k + 8 <= K) {
      const Vec8<T> c = *(const Vec8<T>*)(row + k);
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = c.get(i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = k + i < K ? to_f32(row[k + i]) : 0.f;
    }
  };
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int k = c * step + lane * 8;
    if (k < K) {
      load(k, v[c]);
#pragma unroll
      for (int i = 0; i < 8; i++) am = max(am, abs_bits(v[c][i]));
    }
  }
  for (int k = CH * step + lane * 8; k < K; k += step) {
    float t[8];
    load(k, t);
#pragma unroll
    for (int i = 0; i < 8; i++) am = max(am, abs_bits(t[i]));
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) am = max(am, (unsigned)__shfl_xor((int)am, d));
  if (NW > 1) {
    __shared__ unsigned s_am[NW];
    if ((lane & 63) == 0) s_am[lane >> 6] = am;
    __syncthreads();
    am = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) am = max(am, s_am[w]);
  }
  bool finite;
  const RowScale r = row_scale(am, finite);
  if (lane == 0) scale[m] = finite ? r.s : __uint_as_float(0x7fc00000u);
  int8_t* qrow = q + (int64_t)m * q_pitch;
  auto store = [&](int k, const float* o) {   // (pitch and base are multiples of 16: whole chunks, also the last)
    union { int8_t b[8]; uint64_t u; } p;
#pragma unroll
    for (int i = 0; i < 8; i++) p.b[i] = finite ? (int8_t)quant_one(o[i], r) : (int8_t)0;
    *(uint64_t*)(qrow + k) = p.u;
  };
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int k = c * step + lane * 8;
    if (k < K) store(k, v[c]);
  }
  for (int k = CH * step + lane * 8; k < K; k += step) {
    float t[8];
    load(k, t);
    store(k, t);
  }
}

template <typename T>
static int launch_quantize_t(const T* x, const PhRowMap& xr, unsigned M, int K, int8_t* q, int64_t pitch, float* scale,
                             hipStream_t st) {
  const int64_t strides = xr.flat ? xr.s2 : (xr.s0 | xr.s1 | xr.s2);
  const bool vec = ((uintptr_t)x & 15) == 0 && (strides * (int64_t)sizeof(T)) % 16 == 0;
  const bool wave = K <= 2048;   // a wave holds 4 chunks of 512 values
#define PH_Q(V, NW, CH)                                                                                         \
  hipLaunchKernelGGL((quantize_rows_kernel<T, V, NW, CH>), dim3(NW == 1 ? (M + 3) / 4 : M), dim3(NW == 1 ? 256 : 64 * NW), 0, \
                     st, x, xr, M, K, q, pitch, scale)
  if (wave) {
    if (vec) { if (K <= 512) PH_Q(true, 1, 1); else PH_Q(true, 1, 4); }
    else { if (K <= 512) PH_Q(false, 1, 1); else PH_Q(false, 1, 4); }
  } else {
    if (vec) PH_Q(true, 8, 2); else PH_Q(false, 8, 2);
  }
#undef PH_Q
  PH_CHECK(hipGetLastError());
  return 0;
}

// ---- weights ---------------------------------------------------------------------------------------------------------

// int8 [N][K] -> fragments of the 16 x 64 operand of the matrix instruction, [N16/16][Kp/64][lane][16]: lane l of a
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

__device__ __forceinline__ float w8_act(float v, int act, float slope) {
  if (act == PH_ACT_RELU) return v < 0.f ? 0.f : v;
  if (act == PH_ACT_PRELU) return v < 0.f ? v * slope : v;
  return v;
}
__device__ __forceinline__ float w8_value(int acc, float ws, float s, float bias, int act, float slope) {
  return w8_act(((float)acc * ws) * s + bias, act, slope);
}

// ---- product: fragments straight from memory ----------------------------------------------------------------------------

template <typename O>
__global__ __launch_bounds__(256) void w8_product_kernel(const PhW8Params p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int nb = blockIdx.y * 4 + wave;
  if (nb >= p.nnb) return;
  const unsigned m0 = blockIdx.x * 64;
  const int8_t* xp[4];
#pragma unroll
  for (int i = 0; i < 4; i++) xp[i] = p.q + ph_row_off(p.qr, min(m0 + i * 16 + fr, p.M - 1));
  const int8_t* wp = p.w + (int64_t)nb * p.nkb * 1024 + lane * 16;
  i32x4 acc[4] = {};
  for (int kb = 0; kb < p.nkb; kb++) {
    const i32x4 wf = *(const i32x4*)(wp + (int64_t)kb * 1024);
    int k = kb * 64 + fq * 16;
    k = k < p.K ? k : 0;   // pieces behind the row's end meet zero weights: any readable ones will do
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const i32x4 xf = *(const i32x4*)(xp[i] + k);
      acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf, acc[i], 0, 0, 0);
    }
  }
  const int n = nb * 16 + fq * 4;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const unsigned m = m0 + i * 16 + fr;
    if (m >= p.M) continue;
    const float s = p.qs[m];
    O* o = (O*)p.out + ph_row_off(p.outr, m) + n;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (n + e < p.N)
        o[e] = (O)w8_value(acc[i][e], p.ws[n + e], s, p.bias ? p.bias[n + e] : 0.f, p.act, p.slope ? p.slope[n + e] : 0.f);
  }
}

static int launch_product(const PhW8Params& p, int out_type, hipStream_t st) {
  const dim3 grid((p.M + 63) / 64, (p.nnb + 3) / 4), block(256);
  switch (out_type) {
    case PH_F32: hipLaunchKernelGGL((w8_product_kernel<float>), grid, block, 0, st, p); break;
    case PH_F16: hipLaunchKernelGGL((w8_product_kernel<_Float16>), grid, block, 0, st, p); break;
    default: hipLaunchKernelGGL((w8_product_kernel<bf16>), grid, block, 0, st, p); break;
  }
  PH_CHECK(hipGetLastError());
  return 0;
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

bool aligned16(const void* p, const PhRowMap& r, int64_t elem) {
  return ((uintptr_t)p & 15) == 0 && ((r.s0 | r.s1 | r.s2) * elem) % 16 == 0;
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
                          const PhRowMap& outr) {
  PhW8Params p;
  p.q = q, p.qr = qr, p.qs = qs, p.w = l.packed, p.ws = l.scale, p.bias = l.bias, p.slope = l.slope, p.act = l.act;
  p.M = M, p.N = l.n, p.K = l.k, p.nkb = (l.k + 63) / 64, p.nnb = (l.n + 15) / 16, p.out = out, p.outr = outr;
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

}  // namespace

extern "C" {

int64_t ph_w8_packed_bytes(int n, int k) {
  if (n < 1 || n > W8_MAX_N || k < 1 || k > W8_MAX_K) {
    ph_set_error("ph_w8_packed_bytes: 1 <= n <= %d and 1 <= k <= %d, got %d and %d", W8_MAX_N, W8_MAX_K, n, k);
    return -1;
  }
  return up(n, 16) * up(k, 64);
}

int ph_w8_pack(int device, void* stream, const int8_t* w, int64_t row_stride, int n, int k, int8_t* packed) {
  if (ph_w8_packed_bytes(n, k) < 0 || !some("ph_w8_pack", w, packed)) return -1;
  if ((uintptr_t)packed & 15) {
    ph_set_error("ph_w8_pack: packed weights need 16-byte alignment");
    return -1;
  }
  W8_DEVICE(device);
  const int nkb = (k + 63) / 64, nnb = (n + 15) / 16;
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
  if (m < 0 || m > 0x7fffffff || k < 1 || h < 0 || n < 1) {
    ph_set_error("ph_w8_workspace: bad sizes");
    return -1;
  }
  Pieces w = {nullptr};
  switch (op) {
    case PH_W8_MATMUL:   // rows that are not 16-byte aligned are laid out anew
      w.take<int8_t>(m * q_pitch_of(k));
      break;
    case PH_W8_LINEAR:
      w.take<int8_t>(m * q_pitch_of(k));
      w.take<float>(m);
      break;
    case PH_W8_FEED_FORWARD:
      w.take<int8_t>(m * q_pitch_of(k));
      w.take<float>(m);
      w.take<float>(m * up(h, 4));
      w.take<int8_t>(m * q_pitch_of(h));
      w.take<float>(m);
      break;
    default:
      ph_set_error("ph_w8_workspace: unknown operator %d", op);
      return -1;
  }
  return w.used;
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
  const bool direct = aligned16(q, qr, 1);
  if (!direct && !ws_ok(who, ws, ws_bytes, ph_w8_workspace(PH_W8_MATMUL, M, layer->k, 0, layer->n))) return -3;
  W8_DEVICE(device);
  if (!direct) {
    const int64_t pitch = q_pitch_of(layer->k), pieces = M * (pitch / 16);
    hipLaunchKernelGGL(repitch_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream, q, qr,
                       (unsigned)M, layer->k, (int8_t*)ws, pitch);
    PH_CHECK(hipGetLastError());
    q = (const int8_t*)ws;
    qr = even_rows(pitch);
  }
  return launch_product(product_params(q, qr, scale, (unsigned)M, *layer, out, row_map(orow)), out_type, (hipStream_t)stream);
}

int ph_w8_linear(int device, void* stream, const void* x, int x_type, const ph_rows* rows, const ph_w8_layer* layer, void* out,
                 int out_type, const int64_t* out_stride, void* ws, int64_t ws_bytes) {
  const char* who = "ph_w8_linear";
  int64_t M;
  if (!rows_ok(who, rows, M) || !layer_ok(who, layer) || !type_ok(who, x_type) || !type_ok(who, out_type)) return -1;
  if (M == 0) return 0;
  if (!some(who, x, out) || !some(who, out, out_stride)) return -1;
  if (!ws_ok(who, ws, ws_bytes, ph_w8_workspace(PH_W8_LINEAR, M, layer->k, 0, layer->n))) return -3;
  ph_rows orow = *rows;
  for (int d = 0; d < 3; d++) orow.stride[d] = out_stride[d];
  W8_DEVICE(device);
  const int64_t pitch = q_pitch_of(layer->k);
  Pieces w = {(char*)ws};
  int8_t* q = w.take<int8_t>(M * pitch);
  float* s = w.take<float>(M);
  if (quantize(x, x_type, row_map(*rows), (unsigned)M, layer->k, q, pitch, s, (hipStream_t)stream)) return -1;
  return launch_product(product_params(q, even_rows(pitch), s, (unsigned)M, *layer, out, row_map(orow)), out_type,
                        (hipStream_t)stream);
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
  if (!ws_ok(who, ws, ws_bytes, ph_w8_workspace(PH_W8_FEED_FORWARD, M, layer1->k, layer1->n, layer2->n))) return -3;
  ph_rows orow = *rows;
  for (int d = 0; d < 3; d++) orow.stride[d] = out_stride[d];
  W8_DEVICE(device);
  hipStream_t st = (hipStream_t)stream;
  const int K = layer1->k, H = layer1->n;
  const int64_t pitch = q_pitch_of(K), hpitch = up(H, 4), pitch2 = q_pitch_of(H);
  Pieces w = {(char*)ws};
  int8_t* q = w.take<int8_t>(M * pitch);
  float* s = w.take<float>(M);
  float* h = w.take<float>(M * hpitch);
  int8_t* q2 = w.take<int8_t>(M * pitch2);
  float* s2 = w.take<float>(M);
  if (quantize(x, x_type, row_map(*rows), (unsigned)M, K, q, pitch, s, st)) return -1;
  if (launch_product(product_params(q, even_rows(pitch), s, (unsigned)M, *layer1, h, even_rows(hpitch)), PH_F32, st)) return -1;
  if (quantize(h, PH_F32, even_rows(hpitch), (unsigned)M, H, q2, pitch2, s2, st)) return -1;
  return launch_product(product_params(q2, even_rows(pitch2), s2, (unsigned)M, *layer2, out, row_map(orow)), out_type, st);
}

}  // extern "C"
