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
#include "w8a8_dev.h"

// ---- quantisation of rows ------------------------------------------------------------------------------------------

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
    if (k < K) *(uint64_t*)(qrow + k) = v[c].template quantize<true>(r) >> Eight<T>::shift(k, K);
  }
  for (int k = CH * STEP + lane * 8; k < K; k += STEP) {
    Eight<T> t;
    t.load(row, k, K);
    *(uint64_t*)(qrow + k) = t.template quantize<true>(r) >> Eight<T>::shift(k, K);
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
  if (ph_w8_launchable(M, groups[g])) return -1;
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

// rows of any alignment -> rows of `pitch` bytes, 16-byte aligned; a thread moves 4 pieces of 16 bytes of a row
__global__ void repitch_kernel(const int8_t* __restrict__ q, PhRowMap qr, unsigned M, int K, int8_t* __restrict__ out,
                               int64_t pitch) {
  typedef u32x4 u16b __attribute__((aligned(1)));
  const int per = (int)((pitch + 63) >> 6);   // threads of a row
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const unsigned m = (unsigned)(t / per);
  if (m >= M) return;
  const int p0 = (int)(t - (int64_t)m * per);
  const int8_t* row = q + ph_row_off(qr, m);
  int8_t* const to = out + (int64_t)m * pitch;
  u32x4 v[4];
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int k = (p0 + u * per) * 16;
    if (k + 16 <= K) v[u] = *(const u16b*)(row + k);
  }
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const int k = (p0 + u * per) * 16;
    if (k + 16 <= K) *(u32x4*)(to + k) = v[u];
    else
      for (int i = k; i < K; i++) to[i] = row[i];
  }
}

// ---- entry points --------------------------------------------------------------------------------------------------------

#define W8_MAX_K 131071      // 128 * 128 * K < 2^31
#define W8_MAX_N (1 << 20)
#define W8_MAX_ROW (1 << 30)   // of quantised rows: indexes past a row's end by one step stay ints

namespace {

// the call's device is current inside, the caller's again afterwards
struct DeviceScope {
  int prev = -1;
  bool ok = false;
  explicit DeviceScope(int device) {
    if (hipGetDevice(&prev) != hipSuccess) {
      prev = -1;
      (void)hipGetLastError();
      return;
    }
    if (prev == device) prev = -1, ok = true;
    else ok = hipSetDevice(device) == hipSuccess;
    if (!ok) (void)hipGetLastError();   // (else the next call's check of its launch would find it)
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
  const uintptr_t at = l ? (uintptr_t)l->packed | (uintptr_t)l->scale | (uintptr_t)l->bias | (uintptr_t)l->slope : 0;
  if (!l || !l->packed || !l->scale || (at & 15) || l->n < 1 || l->n > W8_MAX_N || l->k < 1 || l->k > W8_MAX_K ||
      l->act < PH_ACT_NONE || l->act > PH_ACT_PRELU || (l->act == PH_ACT_PRELU && !l->slope)) {
    ph_set_error("%s: bad layer (1 <= n <= %d, 1 <= k <= %d, PReLU needs slopes, arrays 16-byte aligned)", who, W8_MAX_N, W8_MAX_K);
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
                          const PhRowMap& outr, int* parts, int out_type) {
  PhW8Params p;
  p.q = q, p.qr = qr, p.qs = qs, p.w = l.packed, p.ws = l.scale, p.bias = l.bias, p.slope = l.slope, p.act = l.act;
  p.parts = parts;
  p.loose = 0;
  // Long rows of a large output go past the caches: 120704 x 512 bf16 of K = 384 69 -> 55 us, 16384 x 4096 of K = 4096
  // 263 -> 247 us.  Rows that end inside a line lose by it (N = 52: 17.5 -> 18.7 us).
  const int64_t row = (int64_t)l.n * (out_type == PH_F32 ? 4 : 2);
  p.stream = row >= 512 && row * M >= (4 << 20);
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
  int* parts;
  int8_t* q = nullptr;
  float* s = nullptr;
  RowsSpace(void* ws, const PhW8Choice& choice, int64_t M, int K, int N, bool rows, bool scales) : w{(char*)ws} {
    parts = (int*)w.take<char>(ph_w8_parts_bytes(choice, M, N));
    if (rows) q = w.take<int8_t>(M * q_pitch_of(K));
    if (scales) s = w.take<float>(M);
  }
  int64_t used() const { return w.used; }
};
// rows of a layer that quantises them itself need no space
bool itself(int64_t M, int K, int N) { return ph_w8_few_float(M, K) || ph_w8_rows_fit(M, K, N); }
int64_t linear_space(int64_t M, int K, int N) {
  return itself(M, K, N) ? 0 : RowsSpace(nullptr, ph_w8_choose(M, N, nkb_of(K)), M, K, N, true, true).used();
}

// How a product of given 8-bit rows is done, and whether they are laid out anew first.
struct MatmulWay {
  PhW8Choice choice;
  bool anew, loose;
  MatmulWay(int64_t M, int K, int N, bool even) {
    anew = loose = false;
    if (!even) {
      choice = ph_w8_choose_loose(M, K, N);
      loose = choice.kernel >= 0;
      anew = !loose;
    }
    if (!loose) choice = ph_w8_choose(M, N, nkb_of(K));
  }
};

int linear(const void* x, int x_type, const PhRowMap& xr, unsigned M, const ph_w8_layer& l, void* out, int out_type,
           const PhRowMap& outr, void* ws, hipStream_t st) {
  if (itself(M, l.k, l.n)) {
    const FloatRows f = {x, xr};
    const PhW8Params p = product_params(nullptr, xr, nullptr, M, l, out, outr, nullptr, out_type);
    return ph_w8_few_float(M, l.k) ? ph_launch_w8_few_float(p, f, x_type, out_type, st) : ph_launch_w8_rows(p, f, x_type, out_type, st);
  }
  const PhW8Choice choice = ph_w8_choose(M, l.n, nkb_of(l.k));
  const RowsSpace w(ws, choice, M, l.k, l.n, true, true);
  const int64_t pitch = q_pitch_of(l.k);
  if (quantize(x, x_type, xr, M, l.k, w.q, pitch, w.s, st)) return -1;
  return ph_launch_w8_product(product_params(w.q, even_rows(pitch), w.s, M, l, out, outr, w.parts, out_type), choice, out_type, st);
}

int64_t matmul_space(int64_t M, int K, int N, bool even) {
  const MatmulWay way(M, K, N, even);
  return RowsSpace(nullptr, way.choice, M, K, N, way.anew, false).used();
}

// Of two layers: the inner rows in f32, and the larger of the two layers' spaces, one after the other in one place.
int64_t inner_bytes(int64_t M, int H) { return up(M * up(H, 4) * 4, 256); }
int64_t pair_space(int64_t M, int K, int H, int N) {
  const int64_t a = linear_space(M, K, H), b = linear_space(M, H, N);
  return inner_bytes(M, H) + (a > b ? a : b);
}

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
  if (ph_w8_launchable(pieces, 1)) return -1;
  hipLaunchKernelGGL(pack_weight_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream, w,
                     row_stride, n, k, nkb, nnb, packed);
  PH_CHECK(hipGetLastError());
  return 0;
}

int ph_w8_quantize_rows(int device, void* stream, const void* x, int x_type, const ph_rows* rows, int k, int8_t* q,
                        int64_t q_pitch, float* scale) {
  int64_t M;
  if (!rows_ok("ph_w8_quantize_rows", rows, M) || !type_ok("ph_w8_quantize_rows", x_type)) return -1;
  if (k < 1 || k > W8_MAX_ROW || q_pitch < q_pitch_of(k) || q_pitch % 16 || ((uintptr_t)q & 15)) {
    ph_set_error("ph_w8_quantize_rows: k %d, q_pitch %lld: 1 <= k <= 2^30, rows of 8-bit values are 16-byte aligned and hold k "
                 "rounded up to 16", k, (long long)q_pitch);
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
    case PH_W8_MATMUL: return matmul_space(m, k, n, true);
    case PH_W8_MATMUL_ANY: {   // rows that turn out to be aligned are done the other way
      const int64_t a = matmul_space(m, k, n, true), b = matmul_space(m, k, n, false);
      return a > b ? a : b;
    }
    case PH_W8_LINEAR: return linear_space(m, k, n);
    case PH_W8_FEED_FORWARD:
      if (h < 1) {
        ph_set_error("ph_w8_workspace: a feed-forward's inner width is 1 or more");
        return -1;
      }
      return ph_w8_pair_fits(k, h, n) ? 0 : pair_space(m, k, h, n);
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
  const bool even = aligned16(q, qr);
  const MatmulWay way(M, layer->k, layer->n, even);
  const RowsSpace w(ws, way.choice, M, layer->k, layer->n, way.anew, false);
  if (!ws_ok(who, ws, ws_bytes, w.used())) return -3;
  W8_DEVICE(device);
  if (way.anew) {
    const int64_t pitch = q_pitch_of(layer->k), threads = M * ((pitch + 63) / 64);
    if (ph_w8_launchable(threads, 1)) return -1;
    hipLaunchKernelGGL(repitch_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, (hipStream_t)stream, q, qr,
                       (unsigned)M, layer->k, w.q, pitch);
    PH_CHECK(hipGetLastError());
    q = w.q;
    qr = even_rows(pitch);
  }
  PhW8Params p = product_params(q, qr, scale, (unsigned)M, *layer, out, row_map(orow), w.parts, out_type);
  p.loose = way.loose;
  return ph_launch_w8_product(p, way.choice, out_type, (hipStream_t)stream);
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
  if (!ws_ok(who, ws, ws_bytes, linear_space(M, layer->k, layer->n))) return -3;
  W8_DEVICE(device);
  return linear(x, x_type, row_map(*rows), (unsigned)M, *layer, out, out_type, row_map(orow), ws, (hipStream_t)stream);
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
  if (ph_w8_pair_fits(K, H, layer2->n)) {
    W8_DEVICE(device);
    const ph_w8_layer &a = *layer1, &b = *layer2;
    PhW8Pair p = {x, row_map(*rows), (unsigned)M, K, H, b.n, nkb_of(K), (H + 15) / 16, nkb_of(H), (b.n + 15) / 16, a.act, b.act,
                  a.packed, b.packed, a.scale, a.bias, a.slope, b.scale, b.bias, b.slope, 1, {}};
    p.out[0] = {out, row_map(orow), 1, out_type};
    return ph_launch_w8_pair(p, x_type, st);
  }
  if (!ws_ok(who, ws, ws_bytes, pair_space(M, K, H, layer2->n))) return -3;
  W8_DEVICE(device);
  float* const h = (float*)ws;
  void* const more = (char*)ws + inner_bytes(M, H);
  const PhRowMap inner = even_rows(up(H, 4));
  if (linear(x, x_type, row_map(*rows), (unsigned)M, *layer1, h, PH_F32, inner, more, st)) return -1;
  return linear(h, PH_F32, inner, (unsigned)M, *layer2, out, out_type, row_map(orow), more, st);
}

}  // extern "C"
