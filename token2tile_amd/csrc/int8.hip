// 8-bit linear layers: symmetric codes -127 .. 127 with one fp32 scale a row (a
// token of the activations, a channel of the weights); quantisation, the values
// back, and the linear layer on the 8-bit MFMA.
//
// An 8-bit matrix [M, K]: codes in rows, row m at m * stride bytes (a multiple of
// 16), columns K .. Kp - 1 zero, Kp = K rounded up to 128; scales [M].
#include "t2t_linear.h"
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

#define I8_MAX_K 131071  // 2^7 2^7 K stays below 2^31
static inline int i8_kp(int K) { return (K + 127) / 128 * 128; }

extern "C" size_t t2t_int8_row_bytes(int K) { return K < 1 || K > I8_MAX_K ? 0 : (size_t)i8_kp(K); }

static int i8_check_sizes(const char* what, int M, int K) {
  T2T_REQUIRE(M >= 0 && M <= (1 << 30) && K >= 1 && K <= I8_MAX_K, "%s: M=%d K=%d (M <= 2^30, 1 <= K < 2^17)",
              what, M, K);
  return T2T_OK;
}
static int i8_check_matrix(const char* what, const void* codes, long long stride, const void* scales, int M,
                           int K) {
  T2T_REQUIRE(codes && scales, "%s: null pointer", what);
  T2T_REQUIRE((uintptr_t)codes % 16 == 0 && stride % 16 == 0 && stride >= i8_kp(K) && (uintptr_t)scales % 4 == 0,
              "%s: rows of codes must be 16-byte aligned and hold K rounded up to 128, stride %lld", what, stride);
  return T2T_OK;
}
// a 16-bit matrix
static int i8_check_rows(const char* what, const void* x, int dtype, long long row_stride, int M, int K) {
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "%s: dtype %d", what, dtype);
  T2T_REQUIRE(x, "%s: null pointer", what);
  T2T_REQUIRE(M == 1 || row_stride >= K, "%s: row stride %lld < %d", what, row_stride, K);
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// One row's scale and codes: s = max|x| / 127, not below 2^-120 (whose reciprocal
// and products stay in range), codes x / s to nearest, ties to even.  A row with
// an inf or NaN has scale NaN and codes 0.
//
// The quotient is exact: n = x (1 / s) to nearest is off by one at most, and only
// next to a border; r = x - n s is a multiple of both numbers' last places and no
// larger than s, so the fused product gives it without rounding, and |r| against
// s / 2 says on which side of the border x lies.
// ---------------------------------------------------------------------------
struct I8Scale {
  float s, inv, half;
};
__device__ inline I8Scale i8_scale(float top) {
  const float s = __builtin_fmaxf(top / 127.f, 0x1p-120f);
  return {s, 1.f / s, 0.5f * s};
}
template <typename T> struct I8Inf;
template <> struct I8Inf<BF16T> { static constexpr uint32_t bits = 0x7f80u; };
template <> struct I8Inf<F16T> { static constexpr uint32_t bits = 0x7c00u; };

// eight values -> eight codes
template <typename T>
__device__ inline u32x2 i8_codes(const u32x4& x, const I8Scale& k) {
  constexpr float MAGIC = 0x1.8p23f;  // a sum with it is rounded to a whole number, in its low bits
  float m[8], top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = T::to_f((uint16_t)(x[i >> 1] >> (16 * (i & 1))));
    m[i] = __builtin_fmaf(f, k.inv, MAGIC);
    top = __builtin_fmaxf(top, __builtin_fabsf(__builtin_fmaf(-(m[i] - MAGIC), k.s, f)));
  }
  if (top >= k.half) {  // (rare: a value next to a border, or on it)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = T::to_f((uint16_t)(x[i >> 1] >> (16 * (i & 1))));
      const float n = m[i] - MAGIC, r = __builtin_fmaf(-n, k.s, f);
      const bool odd = (int)n & 1;
      if (r > k.half || (r == k.half && odd)) m[i] += 1.f;
      if (r < -k.half || (r == -k.half && odd)) m[i] -= 1.f;
    }
  }
  u32x2 c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __builtin_bit_cast(uint32_t, m[4 * i + e]);
    // byte 0 of each
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    c[i] = lo | hi;
  }
  return c;
}

// eight values of a row at any alignment, the first n of which are inside
__device__ inline u32x4 i8_load(const uint16_t* p, int n) {
  u32x4 v{0u, 0u, 0u, 0u};
  if (n >= 8)
    __builtin_memcpy(&v, p, 16);
  else
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
  return v;
}
__device__ inline uint32_t i8_top(uint32_t top, const u32x4& v) {  // both halves' largest magnitudes
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu)));
  return top;
}

// TPR threads a row, which stays in registers between its maximum and its codes:
// one read of x, one write of the codes.
template <typename T, int TPR, int I>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void i8_quantize_kernel(
    const uint16_t* __restrict__ x, long long row_stride, char* __restrict__ codes, long long stride,
    float* __restrict__ scales, int M, int K, int Kp) {
  constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
  __shared__ uint32_t tops[16];
  const int t = threadIdx.x % TPR;
  for (long long row = (long long)blockIdx.x * ROWS + threadIdx.x / TPR; row < M; row += (long long)gridDim.x * ROWS) {
    const uint16_t* src = x + row * row_stride;
    u32x4 v[I];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < I; ++i) v[i] = i8_load(src + 8 * (t + i * TPR), K - 8 * (t + i * TPR));
#pragma unroll
    for (int i = 0; i < I; ++i) top = i8_top(top, v[i]);
    top = max(top & 0xffffu, top >> 16);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    if constexpr (TPR > 64) {
      __syncthreads();  // the last row's are read
      if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) top = max(top, tops[w]);
    }
    const bool bad = top >= I8Inf<T>::bits;
    const I8Scale k = i8_scale(T::to_f((uint16_t)top));
    char* dst = codes + row * stride;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int c = 8 * (t + i * TPR);
      if (c < Kp) *(u32x2*)(dst + c) = bad ? u32x2{0u, 0u} : i8_codes<T>(v[i], k);
    }
    if (t == 0) scales[row] = bad ? __builtin_nanf("") : k.s;
  }
}

template <typename T>
static void i8_quantize_launch(const uint16_t* x, long long row_stride, char* codes, long long stride,
                               float* scales, int M, int K, hipStream_t st) {
  const int Kp = i8_kp(K);
  auto go = [&](auto tpr, auto its) {
    constexpr int TPR = decltype(tpr)::value, I = decltype(its)::value, ROWS = TPR < 256 ? 256 / TPR : 1;
    const int wgs = cdiv(M, ROWS);
    hipLaunchKernelGGL((i8_quantize_kernel<T, TPR, I>), dim3(wgs < (1 << 20) ? wgs : 1 << 20),
                       dim3(TPR < 256 ? 256 : TPR), 0, st, x, row_stride, codes, stride, scales, M, K, Kp);
  };
#define I8_GO(TPR, I) go(std::integral_constant<int, TPR>{}, std::integral_constant<int, I>{})
  if (Kp <= 512) I8_GO(64, 1);
  else if (Kp <= 1024) I8_GO(64, 2);
  else if (Kp <= 2048) I8_GO(64, 4);
  else if (Kp <= 4096) I8_GO(256, 2);
  else if (Kp <= 6144) I8_GO(256, 3);
  else if (Kp <= 8192) I8_GO(256, 4);
  else if (Kp <= 16384) I8_GO(256, 8);
  else if (Kp <= 32768) I8_GO(1024, 4);
  else I8_GO(1024, 16);
#undef I8_GO
}

extern "C" int t2t_int8_quantize(const void* x, int dtype, long long row_stride, void* codes,
                                 long long code_stride, float* scales, int M, int K, void* stream) {
  int rc = i8_check_sizes("int8_quantize", M, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_rows("int8_quantize", x, dtype, row_stride, M, K);
  if (rc == T2T_OK) rc = i8_check_matrix("int8_quantize", codes, code_stride, scales, M, K);
  if (rc != T2T_OK) return rc;
  (dtype == T2T_BF16 ? i8_quantize_launch<BF16T> : i8_quantize_launch<F16T>)(
      (const uint16_t*)x, row_stride, (char*)codes, code_stride, scales, M, K, (hipStream_t)stream);
  T2T_LAUNCH_CHECK("int8_quantize");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// the values back: eight a thread.  Bound: writing them.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void i8_dequantize_kernel(const char* __restrict__ codes, long long stride,
                                                            const float* __restrict__ scales,
                                                            uint16_t* __restrict__ out, long long row_stride,
                                                            long long units, int per_row, int K) {
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
    const long long row = u / per_row;
    const int c = 8 * (int)(u - row * per_row);
    const u32x2 v = *(const u32x2*)(codes + row * stride + c);
    const float s = scales[row];
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(v[e >> 2] >> (8 * (e & 3))) * s;
    lin_put(out + row * row_stride + c,
            u32x4{Pk<T>::pack(f[0], f[1]), Pk<T>::pack(f[2], f[3]), Pk<T>::pack(f[4], f[5]), Pk<T>::pack(f[6], f[7])},
            K - c);
  }
}

extern "C" int t2t_int8_dequantize(const void* codes, long long code_stride, const float* scales, void* out,
                                   int dtype, long long row_stride, int M, int K, void* stream) {
  int rc = i8_check_sizes("int8_dequantize", M, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_rows("int8_dequantize", out, dtype, row_stride, M, K);
  if (rc == T2T_OK) rc = i8_check_matrix("int8_dequantize", codes, code_stride, scales, M, K);
  if (rc != T2T_OK) return rc;
  const int per_row = (K + 7) / 8;
  const long long units = (long long)M * per_row, wgs = (units + 255) / 256;
  const dim3 grid((unsigned)(wgs < (1 << 20) ? wgs : 1 << 20));
  auto kernel = dtype == T2T_BF16 ? i8_dequantize_kernel<BF16T> : i8_dequantize_kernel<F16T>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, (const char*)codes, code_stride, scales,
                     (uint16_t*)out, row_stride, units, per_row, K);
  T2T_LAUNCH_CHECK("int8_dequantize");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// the linear layer: y[m, n] = act((sum_k a[m, k] w[n, k]) sw[n] sa[m] + bias[n]).  The sum is exact
// in 32 bits; the channel's scale comes first, so that a row of extreme scale leaves the product in
// range for ordinary weights.
// ---------------------------------------------------------------------------
struct I8Mat {
  const char* codes;
  long long stride;
  const float* scales;
  int rows, blocks;  // rows, row blocks of 32
};

template <typename T, bool GELU>
__device__ inline float i8_out(int acc, float sw, float sa, float bias) {
  const float y = __builtin_fmaf((float)acc * sw, sa, bias);
  return GELU ? lin_gelu(y) : y;
}

// ---- small launches: the columns split over the waves ------------------------
// 32 features x 32 tokens a work-group; its eight waves take units of 128 columns
// in turn, loaded straight into registers, DEPTH units ahead.  The waves' sums
// meet in LDS.
template <typename T, int DEPTH, bool GELU>
__global__ __launch_bounds__(512) void i8_split_kernel(I8Mat a, I8Mat w, const uint16_t* __restrict__ bias,
                                                       uint16_t* __restrict__ out, long long ldo, int units,
                                                       int mt, int nt, int per_xcd) {
  constexpr int WAVES = 8;
  __shared__ i32x4 part[WAVES][4][64];
  const int id = lin_first(per_xcd);
  if (id >= lin_end(mt, nt, per_xcd)) return;
  int mb, nb;
  lin_place(id, mt, nt, 1, 1, mb, nb);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = mb * 32 + (lane & 31), feat = nb * 32 + (lane & 31);
  // (any order of the columns will do that is the same for both: a lane takes 64 bytes of a unit)
  const char* pw = w.codes + min(feat, w.rows - 1) * w.stride + 64 * (lane >> 5);
  const char* pa = a.codes + min(row, a.rows - 1) * a.stride + 64 * (lane >> 5);
  struct Unit {
    i32x4 w[4], a[4];
  };
  auto load = [&](int s, Unit& t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.w[i] = *(const i32x4*)(pw + (size_t)s * 128 + 16 * i);
      t.a[i] = *(const i32x4*)(pa + (size_t)s * 128 + 16 * i);
    }
  };
  i32x16 acc = {};
  Unit ring[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (wave + d * WAVES < units) load(wave + d * WAVES, ring[d]);
  for (int s = wave; s < units; s += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      Unit& t = ring[d];
      if (s + d * WAVES < units)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(t.w[i], t.a[i], acc, 0, 0, 0);
      if (s + (d + DEPTH) * WAVES < units) load(s + (d + DEPTH) * WAVES, t);
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    part[wave][q][lane] = i32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  if (wave >= 4) return;
  // quarter q: four features of each token
  const int q = wave, f = nb * 32 + 8 * q + 4 * (lane >> 5);
  i32x4 v = part[0][q][lane];
#pragma unroll
  for (int x = 1; x < WAVES; ++x) v += part[x][q][lane];
  if (row < a.rows && f < w.rows) {
    const float sa = a.scales[row];
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = min(f + e, w.rows - 1);
      y[e] = i8_out<T, GELU>(v[e], w.scales[n], sa, bias ? T::to_f(bias[n]) : 0.f);
    }
    lin_put(out + row * ldo + f, u32x2{Pk<T>::pack(y[0], y[1]), Pk<T>::pack(y[2], y[3])}, w.rows - f);
  }
}

template <typename T, int DEPTH>
static int i8_split_launch(const I8Mat& a, const I8Mat& w, const uint16_t* bias, int act, uint16_t* out,
                           long long ldo, int units, hipStream_t st) {
  const long long tiles = (long long)a.blocks * w.blocks;
  if ((tiles + 7) / 8 > (1 << 19)) {  // 2^31 threads
    t2t_set_error("int8_product: M=%d N=%d", a.rows, w.rows);
    return T2T_ERR_UNSUPPORTED;
  }
  const int per = cdiv(tiles, 8);
  auto kernel = act == T2T_ACT_GELU_TANH ? i8_split_kernel<T, DEPTH, true> : i8_split_kernel<T, DEPTH, false>;
  hipLaunchKernelGGL(kernel, dim3(8 * per), dim3(512), 0, st, a, w, bias, out, ldo, units, a.blocks, w.blocks, per);
  T2T_LAUNCH_CHECK("int8_product");
  return T2T_OK;
}

template <typename T>
static int i8_product(const I8Mat& a, const I8Mat& w, const uint16_t* bias, int act, uint16_t* out, long long ldo,
                      int units, hipStream_t st) {
  return i8_split_launch<T, 2>(a, w, bias, act, out, ldo, units, st);
}

static int i8_check_product(const char* what, const void* w_codes, long long w_stride, const float* w_scales,
                            int act, const void* out, int dtype, long long out_row_stride, int M, int N, int K) {
  int rc = i8_check_sizes(what, M, K);
  if (rc != T2T_OK) return rc;
  T2T_REQUIRE(act == T2T_ACT_NONE || act == T2T_ACT_GELU_TANH, "%s: activation %d", what, act);
  T2T_REQUIRE(N >= 1 && N <= (1 << 30), "%s: N=%d (1 <= N <= 2^30)", what, N);
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "%s: dtype %d", what, dtype);
  if (M == 0) return T2T_OK;
  rc = i8_check_rows(what, out, dtype, out_row_stride, M, N);
  return rc != T2T_OK ? rc : i8_check_matrix(what, w_codes, w_stride, w_scales, N, K);
}

extern "C" int t2t_int8_product(const void* a_codes, long long a_stride, const float* a_scales,
                                const void* w_codes, long long w_stride, const float* w_scales, const void* bias,
                                int act, void* out, int dtype, long long out_row_stride, int M, int N, int K,
                                void* stream) {
  int rc = i8_check_product("int8_product", w_codes, w_stride, w_scales, act, out, dtype, out_row_stride, M, N, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_matrix("int8_product", a_codes, a_stride, a_scales, M, K);
  if (rc != T2T_OK) return rc;
  const I8Mat a{(const char*)a_codes, a_stride, a_scales, M, cdiv(M, 32)};
  const I8Mat w{(const char*)w_codes, w_stride, w_scales, N, cdiv(N, 32)};
  return (dtype == T2T_BF16 ? i8_product<BF16T> : i8_product<F16T>)(a, w, (const uint16_t*)bias, act, (uint16_t*)out,
                                                                   out_row_stride, i8_kp(K) / 128,
                                                                   (hipStream_t)stream);
}

// codes, then scales
extern "C" size_t t2t_int8_linear_ws_bytes(int M, int N, int K) {
  (void)N;
  return M < 1 || M > (1 << 30) || K < 1 || K > I8_MAX_K ? 0 : (size_t)M * i8_kp(K) + t2t_align256((size_t)M * 4);
}

extern "C" int t2t_int8_linear(const void* x, int dtype, long long x_row_stride, const void* w_codes,
                               long long w_stride, const float* w_scales, const void* bias, int act, void* out,
                               long long out_row_stride, int M, int N, int K, void* ws, size_t ws_bytes,
                               void* stream) {
  // everything before the first launch
  int rc = i8_check_product("int8_linear", w_codes, w_stride, w_scales, act, out, dtype, out_row_stride, M, N, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_rows("int8_linear", x, dtype, x_row_stride, M, K);
  if (rc != T2T_OK) return rc;
  const size_t need = t2t_int8_linear_ws_bytes(M, N, K);
  if (!ws || ws_bytes < need) {
    t2t_set_error("int8_linear: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
    return T2T_ERR_WORKSPACE;
  }
  T2T_REQUIRE((uintptr_t)ws % 16 == 0, "int8_linear: workspace must be 16-byte aligned");
  float* scales = (float*)((char*)ws + (size_t)M * i8_kp(K));
  rc = t2t_int8_quantize(x, dtype, x_row_stride, ws, i8_kp(K), scales, M, K, stream);
  if (rc != T2T_OK) return rc;
  return t2t_int8_product(ws, i8_kp(K), scales, w_codes, w_stride, w_scales, bias, act, out, dtype, out_row_stride,
                          M, N, K, stream);
}
