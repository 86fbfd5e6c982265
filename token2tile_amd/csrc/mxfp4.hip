// MXFP4: 4-bit E2M1 codes in blocks of 32 along the columns, one power-of-two
// scale (E8M0 byte) per block; quantisation, the values back, and the linear
// layer on the scaled MFMA.
//
// Layout of an MXFP4 matrix [M, K] (K a multiple of 32).  It is that of the
// operands of v_mfma_scale_f32_32x32x64_f8f6f4, whose lane l supplies the 32
// values (16 bytes) of row l % 32 and columns 32 (l / 32) .. + 31 and their
// scale, so fragments are read whole, 1 KB contiguous per wave:
//   codes   [ceil(M / 32)][Kp / 64][64 lanes][16 bytes], Kp = K rounded up to 256:
//           lane l of chunk c: row l % 32 of the row block, columns
//           64 c + 32 (l / 32) + j, value j in nibble j % 2 of byte j / 2
//   scales  [ceil(M / 32)][Kp / 256][64 lanes][4 bytes]: byte j of lane l in
//           group g: the block of row l % 32, columns 256 g + 64 j + 32 (l / 32)
// Rows past M and columns past K hold zero codes and zero scale bytes (a zero
// code under a scale of 255, which stands for NaN, would be NaN).
#include "t2t_common.h"

typedef int i32x8 __attribute__((ext_vector_type(8)));

static inline long long mx_row_blocks(int M) { return ((long long)M + 31) / 32; }
static inline int mx_kp(int K) { return (K + 255) / 256 * 256; }

extern "C" size_t t2t_mxfp4_code_bytes(int M, int K) {
  return M <= 0 || K <= 0 ? 0 : (size_t)mx_row_blocks(M) * mx_kp(K) * 16;
}
extern "C" size_t t2t_mxfp4_scale_bytes(int M, int K) {
  return M <= 0 || K <= 0 ? 0 : (size_t)mx_row_blocks(M) * mx_kp(K);
}

// a 16-bit matrix beside its codes and scales
static int mx_check_rows(const char* what, const void* x, int dtype, long long row_stride,
                         const void* codes, const void* scales, int M, int K) {
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "%s: dtype %d", what, dtype);
  T2T_REQUIRE(M >= 0 && K >= 32 && K % 32 == 0 && K <= INT_MAX - 255, "%s: M=%d K=%d (K a multiple of 32)",
              what, M, K);
  if (M == 0) return T2T_OK;
  T2T_REQUIRE(x && codes && scales, "%s: null pointer", what);
  T2T_REQUIRE(((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) % 16 == 0 && row_stride % 8 == 0 &&
                  (M == 1 || row_stride >= K),
              "%s: rows must be 16-byte aligned, row stride %lld >= K", what, row_stride);
  T2T_REQUIRE(mx_row_blocks(M) * (mx_kp(K) / 256) <= INT_MAX, "%s: M=%d K=%d", what, M, K);
  return T2T_OK;
}

template <typename T> struct MxCvt;
template <> struct MxCvt<BF16T> {
  template <int S> __device__ static inline uint32_t enc(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, pair), scale, S);
  }
  template <int S> __device__ static inline uint32_t dec(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, S));
  }
  static constexpr uint32_t nan_pair = 0x7fc07fc0u;
  static constexpr uint32_t inf = 0x7f80u;
};
template <> struct MxCvt<F16T> {
  template <int S> __device__ static inline uint32_t enc(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, pair), scale, S);
  }
  template <int S> __device__ static inline uint32_t dec(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, S));
  }
  static constexpr uint32_t nan_pair = 0x7e007e00u;
  static constexpr uint32_t inf = 0x7c00u;
};

// One block: 32 values (16 pairs) -> codes and scale byte.  The largest
// magnitude is found on the bit patterns, which order like the magnitudes
// (an inf or NaN pattern is >= inf: byte 255, zero codes).  The scale is
// 2^(floor(log2 max) - 2), not below 2^-126, which brings the maximum to
// [4, 8); the conversion rounds to nearest even and saturates at 6.
template <typename T>
__device__ inline void mx_block(const u32x4 (&x)[4], u32x4& codes, uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int v = 0; v < 4; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = x[v][i] & 0x7fffu, hi = (x[v][i] >> 16) & 0x7fffu;
      top = max(top, max(lo, hi));
    }
  if (top >= MxCvt<T>::inf) {
    byte = 255;
    codes = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  const int e = (int)(__builtin_bit_cast(uint32_t, T::to_f((uint16_t)top)) >> 23);  // 0: below 2^-126
  byte = (uint32_t)max(e - 2, 1);
  const float scale = __builtin_bit_cast(float, byte << 23);
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    uint32_t c = 0;
    c = MxCvt<T>::template enc<0>(c, x[v][0], scale);
    c = MxCvt<T>::template enc<1>(c, x[v][1], scale);
    c = MxCvt<T>::template enc<2>(c, x[v][2], scale);
    c = MxCvt<T>::template enc<3>(c, x[v][3], scale);
    codes[v] = c;
  }
}

// ---------------------------------------------------------------------------
// quantise: a work-group per 32 rows x 256 columns, a thread per block
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const uint16_t* __restrict__ x,
                                                          long long row_stride,
                                                          uint32_t* __restrict__ codes,
                                                          uint32_t* __restrict__ scales, int M, int K,
                                                          int groups) {
  const long long rb = blockIdx.x / groups;
  const int g = (int)(blockIdx.x - rb * groups);
  const int r = threadIdx.x >> 3, blk = threadIdx.x & 7;
  const long long row = rb * 32 + r;
  const int col = 256 * g + 32 * blk;
  u32x4 c{0u, 0u, 0u, 0u};
  uint32_t byte = 0;
  if (row < M && col < K) {
    const u32x4* src = (const u32x4*)(x + row * row_stride + col);
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = src[i];
    mx_block<T>(v, c, byte);
  }
  const int half = blk & 1, j = blk >> 1;
  char* cp = (char*)codes + (rb * groups + g) * 4096 + j * 1024 + (r + 32 * half) * 16;
  *(u32x4*)cp = c;
  // the four bytes of a lane's dword sit in blocks half, half + 2, ...
  uint32_t word = byte << (8 * j);
  word |= __shfl_xor(word, 2, 64);
  word |= __shfl_xor(word, 4, 64);
  if (j == 0) scales[(rb * groups + g) * 64 + r + 32 * half] = word;
}

extern "C" int t2t_mxfp4_quantize(const void* x, int dtype, long long row_stride, void* codes,
                                  void* scales, int M, int K, void* stream) {
  const int rc = mx_check_rows("mxfp4_quantize", x, dtype, row_stride, codes, scales, M, K);
  if (rc != T2T_OK || M == 0) return rc;
  const int groups = mx_kp(K) / 256;
  const long long wgs = mx_row_blocks(M) * groups;
  if (dtype == T2T_BF16)
    hipLaunchKernelGGL(mx_quantize_kernel<BF16T>, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,
                       (const uint16_t*)x, row_stride, (uint32_t*)codes, (uint32_t*)scales, M, K, groups);
  else
    hipLaunchKernelGGL(mx_quantize_kernel<F16T>, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream,
                       (const uint16_t*)x, row_stride, (uint32_t*)codes, (uint32_t*)scales, M, K, groups);
  T2T_LAUNCH_CHECK("mxfp4_quantize");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// the values back: the same thread per block
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                            const uint32_t* __restrict__ scales,
                                                            uint16_t* __restrict__ out,
                                                            long long row_stride, int M, int K,
                                                            int groups) {
  const long long rb = blockIdx.x / groups;
  const int g = (int)(blockIdx.x - rb * groups);
  const int r = threadIdx.x >> 3, blk = threadIdx.x & 7;
  const long long row = rb * 32 + r;
  const int col = 256 * g + 32 * blk;
  if (row >= M || col >= K) return;
  const int half = blk & 1, j = blk >> 1;
  const u32x4 c = *(const u32x4*)((const char*)codes + (rb * groups + g) * 4096 + j * 1024 +
                                  (r + 32 * half) * 16);
  const uint32_t byte = (scales[(rb * groups + g) * 64 + r + 32 * half] >> (8 * j)) & 255u;
  const float scale = __builtin_bit_cast(float, byte << 23);
  u32x4* dst = (u32x4*)(out + row * row_stride + col);
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    u32x4 o;
    o[0] = MxCvt<T>::template dec<0>(c[v], scale);
    o[1] = MxCvt<T>::template dec<1>(c[v], scale);
    o[2] = MxCvt<T>::template dec<2>(c[v], scale);
    o[3] = MxCvt<T>::template dec<3>(c[v], scale);
    if (byte == 255) o = u32x4{MxCvt<T>::nan_pair, MxCvt<T>::nan_pair, MxCvt<T>::nan_pair, MxCvt<T>::nan_pair};
    dst[v] = o;
  }
}

extern "C" int t2t_mxfp4_dequantize(const void* codes, const void* scales, void* out, int dtype,
                                    long long row_stride, int M, int K, void* stream) {
  const int rc = mx_check_rows("mxfp4_dequantize", out, dtype, row_stride, codes, scales, M, K);
  if (rc != T2T_OK || M == 0) return rc;
  const int groups = mx_kp(K) / 256;
  const long long wgs = mx_row_blocks(M) * groups;
  if (dtype == T2T_BF16)
    hipLaunchKernelGGL(mx_dequantize_kernel<BF16T>, dim3((unsigned)wgs), dim3(256), 0,
                       (hipStream_t)stream, (const uint32_t*)codes, (const uint32_t*)scales,
                       (uint16_t*)out, row_stride, M, K, groups);
  else
    hipLaunchKernelGGL(mx_dequantize_kernel<F16T>, dim3((unsigned)wgs), dim3(256), 0,
                       (hipStream_t)stream, (const uint32_t*)codes, (const uint32_t*)scales,
                       (uint16_t*)out, row_stride, M, K, groups);
  T2T_LAUNCH_CHECK("mxfp4_dequantize");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// the linear layer: y[m, n] = act(sum_k a[m, k] w[n, k] + bias[n])
// ---------------------------------------------------------------------------
// fp4 x fp4 32x32x64, scale byte S of each operand's dword
template <int S>
__device__ inline f32x16 mx_mfma(const u32x4& a, const u32x4& b, const f32x16& c, uint32_t sa,
                                 uint32_t sb) {
  const i32x8 A{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 B{(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, c, 4, 4, S, (int)sa, S, (int)sb);
}

// gelu(x) = x / 2 (1 + tanh u) = x / (1 + e^(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
__device__ inline float mx_gelu(float x) {
  const float u2 = 1.5957691216057308f * x * (1.f + 0.044715f * x * x);
  return x / (1.f + __expf(-u2));
}

struct MxMat {
  const char* codes;
  const uint32_t* scales;
  int rows, blocks;  // rows, row blocks of 32
};

// One wave per 32 x 32 outputs, fragments straight from memory.  The weights
// are the A operand, so a lane holds one token's features 8 (i / 4) +
// 4 (l / 32) + i % 4.
template <typename T>
__global__ __launch_bounds__(256) void mx_linear_kernel(MxMat a, MxMat w,
                                                        const uint16_t* __restrict__ bias, int act,
                                                        uint16_t* __restrict__ out, long long ldo,
                                                        int groups, long long tiles) {
  const int lane = threadIdx.x & 63;
  const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const long long mb = tile / w.blocks;
  const int nb = (int)(tile - mb * w.blocks);
  const char* ap = a.codes + mb * groups * 4096 + lane * 16;
  const char* wp = w.codes + (long long)nb * groups * 4096 + lane * 16;
  const uint32_t* as = a.scales + mb * groups * 64 + lane;
  const uint32_t* wsc = w.scales + (long long)nb * groups * 64 + lane;
  f32x16 acc = zero16();
  for (int g = 0; g < groups; ++g) {
    const uint32_t sa = as[g * 64], sw = wsc[g * 64];
    const u32x4* pa = (const u32x4*)(ap + (size_t)g * 4096);
    const u32x4* pw = (const u32x4*)(wp + (size_t)g * 4096);
    acc = mx_mfma<0>(pw[0], pa[0], acc, sw, sa);
    acc = mx_mfma<1>(pw[64], pa[64], acc, sw, sa);
    acc = mx_mfma<2>(pw[128], pa[128], acc, sw, sa);
    acc = mx_mfma<3>(pw[192], pa[192], acc, sw, sa);
  }
  const long long m = mb * 32 + (lane & 31);
  if (m >= a.rows) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = nb * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
    if (n < w.rows) {
      float v = acc[i];
      if (bias) v += T::to_f(bias[n]);
      if (act) v = mx_gelu(v);
      out[m * ldo + n] = T::from_f(v);
    }
  }
}

static int mx_check_product(const char* what, const void* a_codes, const void* a_scales,
                            const void* w_codes, const void* w_scales, int act, const void* out, int dtype,
                            long long out_row_stride, int M, int N, int K) {
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "%s: dtype %d", what, dtype);
  T2T_REQUIRE(act == T2T_ACT_NONE || act == T2T_ACT_GELU_TANH, "%s: activation %d", what, act);
  T2T_REQUIRE(M >= 0 && N >= 1 && K >= 32 && K % 32 == 0, "%s: M=%d N=%d K=%d (K a multiple of 32)", what, M,
              N, K);
  if (M == 0) return T2T_OK;
  T2T_REQUIRE(a_codes && a_scales && w_codes && w_scales && out, "%s: null pointer", what);
  T2T_REQUIRE(((uintptr_t)a_codes | (uintptr_t)a_scales | (uintptr_t)w_codes | (uintptr_t)w_scales) % 16 == 0,
              "%s: codes and scales must be 16-byte aligned", what);
  T2T_REQUIRE(M == 1 || out_row_stride >= N, "%s: row stride %lld < N=%d", what, out_row_stride, N);
  return T2T_OK;
}

extern "C" int t2t_mxfp4_product(const void* a_codes, const void* a_scales, const void* w_codes,
                                 const void* w_scales, const void* bias, int act, void* out, int dtype,
                                 long long out_row_stride, int M, int N, int K, void* stream) {
  const int rc = mx_check_product("mxfp4_product", a_codes, a_scales, w_codes, w_scales, act, out, dtype,
                                  out_row_stride, M, N, K);
  if (rc != T2T_OK || M == 0) return rc;
  const MxMat a{(const char*)a_codes, (const uint32_t*)a_scales, M, (int)mx_row_blocks(M)};
  const MxMat w{(const char*)w_codes, (const uint32_t*)w_scales, N, (int)mx_row_blocks(N)};
  const long long tiles = (long long)a.blocks * w.blocks;
  const long long wgs = (tiles + 3) / 4;
  T2T_REQUIRE(wgs <= INT_MAX, "mxfp4_product: M=%d N=%d", M, N);
  if (dtype == T2T_BF16)
    hipLaunchKernelGGL(mx_linear_kernel<BF16T>, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, a,
                       w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, mx_kp(K) / 256, tiles);
  else
    hipLaunchKernelGGL(mx_linear_kernel<F16T>, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, a,
                       w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, mx_kp(K) / 256, tiles);
  T2T_LAUNCH_CHECK("mxfp4_product");
  return T2T_OK;
}

// codes, then scales
extern "C" size_t t2t_mxfp4_linear_ws_bytes(int M, int N, int K) {
  (void)N;
  return t2t_align256(t2t_mxfp4_code_bytes(M, K)) + t2t_mxfp4_scale_bytes(M, K);
}

extern "C" int t2t_mxfp4_linear(const void* x, int dtype, long long x_row_stride, const void* w_codes,
                                const void* w_scales, const void* bias, int act, void* out,
                                long long out_row_stride, int M, int N, int K, void* ws, size_t ws_bytes,
                                void* stream) {
  // everything before the first launch
  int rc = mx_check_product("mxfp4_linear", x, x, w_codes, w_scales, act, out, dtype, out_row_stride, M, N, K);
  if (rc == T2T_OK) rc = mx_check_rows("mxfp4_linear", x, dtype, x_row_stride, w_codes, w_scales, M, K);
  if (rc != T2T_OK || M == 0) return rc;
  if (!ws || ws_bytes < t2t_mxfp4_linear_ws_bytes(M, N, K)) {
    t2t_set_error("mxfp4_linear: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0,
                  t2t_mxfp4_linear_ws_bytes(M, N, K));
    return T2T_ERR_WORKSPACE;
  }
  char* scales = (char*)ws + t2t_align256(t2t_mxfp4_code_bytes(M, K));
  T2T_REQUIRE((uintptr_t)ws % 16 == 0, "mxfp4_linear: workspace must be 16-byte aligned");
  rc = t2t_mxfp4_quantize(x, dtype, x_row_stride, ws, scales, M, K, stream);
  if (rc != T2T_OK) return rc;
  return t2t_mxfp4_product(ws, scales, w_codes, w_scales, bias, act, out, dtype, out_row_stride, M, N, K,
                           stream);
}
