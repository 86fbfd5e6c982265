// 8-bit linear layers: symmetric codes -127 .. 127 with one fp32 scale a row (a
// token of the activations, a channel of the weights); quantisation, the values
// back, and the linear layer on the 8-bit MFMA.
//
// Layout of the codes of a matrix [M, K]: blocks of 16 rows x 64 columns, 1 KB each,
//   [ceil(M / 16)][Kp / 64][16 rows][4 chunks of 16 bytes], Kp = K rounded up to 128,
// chunk c of row r at place c ^ ((r >> 2) & 3).  It is the order in which the tiles
// lie in LDS (the places let the operand reads of sixteen rows meet all banks), so a
// tile is fetched in whole kilobytes: from plain rows, 64 bytes of each at a time,
// every fetch took half lines, and 75,600 x 13,824 x 5,120 5.09 ms.  Columns K .. Kp -
// 1 are zero, rows from M on anything.
#include "t2t_linear.h"
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

#define I8_MAX_K 131071  // 2^7 2^7 K stays below 2^31
static inline int i8_kp(int K) { return (K + 127) / 128 * 128; }
// where column c of row r lies, blk bytes to 16 rows (Kp * 16)
__host__ __device__ static inline int i8_swz(int row) { return (row >> 2) & 3; }
__device__ inline long long i8_at(long long r, int c, long long blk) {
  return (r >> 4) * blk + ((c >> 6) << 10) + ((int)(r & 15) << 6) + ((((c >> 4) & 3) ^ i8_swz((int)r)) << 4) + (c & 15);
}

extern "C" size_t t2t_int8_code_bytes(int M, int K) {
  return M < 1 || M > (1 << 30) || K < 1 || K > I8_MAX_K ? 0 : ((size_t)M + 15) / 16 * 16 * i8_kp(K);
}

static int i8_check_sizes(const char* what, int M, int K) {
  T2T_REQUIRE(M >= 0 && M <= (1 << 30) && K >= 1 && K <= I8_MAX_K, "%s: M=%d K=%d (M <= 2^30, 1 <= K < 2^17)",
              what, M, K);
  return T2T_OK;
}
static int i8_check_matrix(const char* what, const void* codes, const void* scales) {
  T2T_REQUIRE(codes && scales, "%s: null pointer", what);
  T2T_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 4 == 0, "%s: codes must be 16-byte aligned", what);
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
// one read of x, one write of the codes, which bound it (75,600 x 5,120: 4.6 to 5.5 TB/s; 4,099 x
// 1,531 is one round of waves, each a chain of loads, maximum and codes: 8.5 us, 7.6 at 1,536 columns).  A
// work-group has several rows where it can:
// a row writes half lines (64 bytes of every block), its neighbour the other halves
// (75,600 x 5,120: 217 us with two rows, 260 with one).
template <typename T, int TPR, int I, int ROWS>
__global__ __launch_bounds__(TPR * ROWS) void i8_quantize_kernel(
    const uint16_t* __restrict__ x, long long row_stride, char* __restrict__ codes, float* __restrict__ scales, int M,
    int K, int Kp) {
  __shared__ uint32_t tops[16];
  const int t = threadIdx.x % TPR;
  for (long long row0 = (long long)blockIdx.x * ROWS; row0 < M; row0 += (long long)gridDim.x * ROWS) {
    const long long row = row0 + threadIdx.x / TPR;
    if (TPR == 64 && row >= M) return;
    const uint16_t* src = x + row * row_stride;
    u32x4 v[I];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < I; ++i) v[i] = i8_load(src + 8 * (t + i * TPR), row < M ? K - 8 * (t + i * TPR) : 0);
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
      for (int w = 0; w < TPR / 64; ++w) top = max(top, tops[threadIdx.x / TPR * (TPR / 64) + w]);
    }
    const bool bad = top >= I8Inf<T>::bits;
    const I8Scale k = i8_scale(T::to_f((uint16_t)top));
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int c = 8 * (t + i * TPR);
      if (c < Kp && row < M) *(u32x2*)(codes + i8_at(row, c, 16LL * Kp)) = bad ? u32x2{0u, 0u} : i8_codes<T>(v[i], k);
    }
    if (t == 0 && row < M) scales[row] = bad ? __builtin_nanf("") : k.s;
  }
}

template <typename T>
static void i8_quantize_launch(const uint16_t* x, long long row_stride, char* codes, float* scales, int M, int K,
                               hipStream_t st) {
  const int Kp = i8_kp(K);
  auto go = [&](auto tpr, auto its, auto rows) {
    constexpr int TPR = decltype(tpr)::value, I = decltype(its)::value, ROWS = decltype(rows)::value;
    const int wgs = cdiv(M, ROWS);
    hipLaunchKernelGGL((i8_quantize_kernel<T, TPR, I, ROWS>), dim3(wgs < (1 << 20) ? wgs : 1 << 20), dim3(TPR * ROWS),
                       0, st, x, row_stride, codes, scales, M, K, Kp);
  };
#define I8_GO(TPR, I, ROWS) \
  go(std::integral_constant<int, TPR>{}, std::integral_constant<int, I>{}, std::integral_constant<int, ROWS>{})
  // enough threads a row that its loads come at once (us, 10 x 16 bytes a thread of 64 against 3 of 256,
  // K = 5,120: 64 rows 7.3 and 4.0, 2,048 rows 11.9 and 9.3, 75,600 rows 225 and 217); more shorten
  // small launches alone (K = 1,536, 3 of 64 against 1 of 256: 256 rows 3.7 and 3.1, 4,680 rows 7.0 and 10.1)
  const bool many = M >= 1024;
  if (Kp <= 512) I8_GO(64, 1, 4);
  else if (Kp <= 1024) I8_GO(64, 2, 4);
  else if (Kp <= 2048 && !many) I8_GO(256, 1, 2);
  else if (Kp <= 1536) I8_GO(64, 3, 4);
  else if (Kp <= 2048) I8_GO(128, 2, 4);
  else if (Kp <= 4096) I8_GO(256, 2, 2);
  else if (Kp <= 6144) I8_GO(256, 3, 2);
  else if (Kp <= 8192) I8_GO(256, 4, 2);
  else if (Kp <= 16384) I8_GO(512, 4, 2);
  else if (Kp <= 32768) I8_GO(1024, 4, 1);
  else I8_GO(1024, 16, 1);
#undef I8_GO
}

extern "C" int t2t_int8_quantize(const void* x, int dtype, long long row_stride, void* codes, float* scales, int M,
                                 int K, void* stream) {
  int rc = i8_check_sizes("int8_quantize", M, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_rows("int8_quantize", x, dtype, row_stride, M, K);
  if (rc == T2T_OK) rc = i8_check_matrix("int8_quantize", codes, scales);
  if (rc != T2T_OK) return rc;
  (dtype == T2T_BF16 ? i8_quantize_launch<BF16T> : i8_quantize_launch<F16T>)(
      (const uint16_t*)x, row_stride, (char*)codes, scales, M, K, (hipStream_t)stream);
  T2T_LAUNCH_CHECK("int8_quantize");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// the values back: eight a thread, the codes read in order, so that a row of a
// block is stored whole (128 bytes).  Bound: writing them (75,600 x 5,120: 205 us, 5.7 TB/s).
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void i8_dequantize_kernel(const char* __restrict__ codes, long long blk,
                                                            const float* __restrict__ scales,
                                                            uint16_t* __restrict__ out, long long row_stride,
                                                            long long units, int M, int K) {
  const int per = (int)(blk >> 3);  // units of 16 rows
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
    const long long rb = u / per;
    const int in = (int)(u - rb * per), r = in >> 3 & 15;
    const int c = 64 * (in >> 7) + 16 * ((in >> 1 & 3) ^ i8_swz(r)) + 8 * (in & 1);
    const long long row = 16 * rb + r;
    if (row >= M || c >= K) continue;
    const u32x2 v = *(const u32x2*)(codes + 8 * u);
    const float s = scales[row];
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(v[e >> 2] >> (8 * (e & 3))) * s;
    lin_put(out + row * row_stride + c,
            u32x4{Pk<T>::pack(f[0], f[1]), Pk<T>::pack(f[2], f[3]), Pk<T>::pack(f[4], f[5]), Pk<T>::pack(f[6], f[7])},
            K - c);
  }
}

extern "C" int t2t_int8_dequantize(const void* codes, const float* scales, void* out, int dtype, long long row_stride,
                                   int M, int K, void* stream) {
  int rc = i8_check_sizes("int8_dequantize", M, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_rows("int8_dequantize", out, dtype, row_stride, M, K);
  if (rc == T2T_OK) rc = i8_check_matrix("int8_dequantize", codes, scales);
  if (rc != T2T_OK) return rc;
  const long long units = (long long)(t2t_int8_code_bytes(M, K) / 8), wgs = (units + 255) / 256;
  const dim3 grid((unsigned)(wgs < (1 << 20) ? wgs : 1 << 20));
  auto kernel = dtype == T2T_BF16 ? i8_dequantize_kernel<BF16T> : i8_dequantize_kernel<F16T>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, (const char*)codes, 16LL * i8_kp(K), scales,
                     (uint16_t*)out, row_stride, units, M, K);
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
  long long blk;  // bytes of 16 rows
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
// meet in LDS.  With X16 the tokens come in 16 bits, and every work-group quantises
// them into LDS first, under the loads of its first weights, in the place of a launch
// before this one.  Bound: the weights' loads, of which 160 of 256 CUs have one round
// each (1 x 5,120 x 5,120: 10.5 us with weights from memory, 2.5 TB/s; 7.4 on one weight again and again).
#define I8_X16_BYTES 32768  // codes that the LDS holds
struct I8Src {
  I8Mat m;            // in 8 bits (its row count in either case), or
  const uint16_t* x;  // in 16 bits
  long long stride;
  int K;
};

template <typename T, int DEPTH, bool GELU, bool X16>
__global__ __launch_bounds__(512) void i8_split_kernel(I8Src a, I8Mat w, const uint16_t* __restrict__ bias,
                                                       uint16_t* __restrict__ out, long long ldo, int units,
                                                       int mt, int nt, int per_xcd) {
  constexpr int WAVES = 8;
  __shared__ i32x4 part[WAVES][4][64];
  __shared__ __attribute__((aligned(16))) char codes[X16 ? I8_X16_BYTES + 32 * 16 : 16];
  __shared__ uint32_t tops[X16 ? 32 : 1][WAVES];
  __shared__ float scales[X16 ? 32 : 1];
  const int id = lin_first(per_xcd);
  if (id >= lin_end(mt, nt, per_xcd)) return;
  int mb, nb;
  lin_place(id, mt, nt, 1, 1, mb, nb);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = mb * 32 + (lane & 31), feat = nb * 32 + (lane & 31);
  // (rows past the last are read from its block of sixteen, and not stored)
  const char* pw = w.codes + (min(feat, w.rows - 1) >> 4) * w.blk + (feat & 15) * 64;
  const char* pa = X16 ? nullptr : a.m.codes + (min(row, a.m.rows - 1) >> 4) * a.m.blk + (row & 15) * 64;
  int at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = (i >> 1) * 1024 + (((2 * (i & 1) + (lane >> 5)) ^ i8_swz(lane)) << 4);
  struct Unit {
    i32x4 w[4], a[4];
  };
  auto load = [&](int s, Unit& t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.w[i] = *(const i32x4*)(pw + (size_t)s * 2048 + at[i]);
      if constexpr (!X16) t.a[i] = *(const i32x4*)(pa + (size_t)s * 2048 + at[i]);
    }
  };
  const int pitch = 128 * units + 16;  // of the codes' rows in LDS
  auto fetch = [&](int s, Unit& t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.a[i] = i32x4{};
      if (row < a.m.rows) t.a[i] = *(const i32x4*)(codes + row * pitch + 128 * s + 64 * (i >> 1) + 32 * (i & 1) + 16 * (lane >> 5));
    }
  };
  i32x16 acc = {};
  Unit ring[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (wave + d * WAVES < units) load(wave + d * WAVES, ring[d]);
  if constexpr (X16) {
    for (int r = 0; r < a.m.rows; ++r) {
      uint32_t top = 0;
      for (int c = 8 * threadIdx.x; c < a.K; c += 8 * 64 * WAVES) top = i8_top(top, i8_load(a.x + r * a.stride + c, a.K - c));
      top = max(top & 0xffffu, top >> 16);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
      if (lane == 0) tops[r][wave] = top;
    }
    __syncthreads();
    for (int r = 0; r < a.m.rows; ++r) {
      uint32_t top = 0;
#pragma unroll
      for (int x = 0; x < WAVES; ++x) top = max(top, tops[r][x]);
      const bool bad = top >= I8Inf<T>::bits;
      const I8Scale k = i8_scale(T::to_f((uint16_t)top));
      for (int c = 8 * threadIdx.x; c < 128 * units; c += 8 * 64 * WAVES)
        *(u32x2*)(codes + r * pitch + c) = bad ? u32x2{0u, 0u} : i8_codes<T>(i8_load(a.x + r * a.stride + c, a.K - c), k);
      if (threadIdx.x == 0) scales[r] = bad ? __builtin_nanf("") : k.s;
    }
    __syncthreads();
  }
  for (int s = wave; s < units; s += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      Unit& t = ring[d];
      if (s + d * WAVES < units) {
        if constexpr (X16) fetch(s + d * WAVES, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(t.w[i], t.a[i], acc, 0, 0, 0);
      }
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
  if (row < a.m.rows && f < w.rows) {
    const float sa = X16 ? scales[row] : a.m.scales[row];
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = min(f + e, w.rows - 1);
      y[e] = i8_out<T, GELU>(v[e], w.scales[n], sa, bias ? T::to_f(bias[n]) : 0.f);
    }
    lin_put(out + row * ldo + f, u32x2{Pk<T>::pack(y[0], y[1]), Pk<T>::pack(y[2], y[3])}, w.rows - f);
  }
}

template <typename T, int DEPTH, bool X16>
static int i8_split_launch(const I8Src& a, const I8Mat& w, const uint16_t* bias, int act, uint16_t* out,
                           long long ldo, int units, hipStream_t st) {
  const long long tiles = (long long)a.m.blocks * w.blocks;
  if ((tiles + 7) / 8 > (1 << 19)) {  // 2^31 threads
    t2t_set_error("int8_product: M=%d N=%d", a.m.rows, w.rows);
    return T2T_ERR_UNSUPPORTED;
  }
  const int per = cdiv(tiles, 8);
  auto kernel =
      act == T2T_ACT_GELU_TANH ? i8_split_kernel<T, DEPTH, true, X16> : i8_split_kernel<T, DEPTH, false, X16>;
  hipLaunchKernelGGL(kernel, dim3(8 * per), dim3(512), 0, st, a, w, bias, out, ldo, units, a.m.blocks, w.blocks, per);
  T2T_LAUNCH_CHECK("int8_product");
  return T2T_OK;
}

// ---- tiles staged through LDS ------------------------------------------------
// Tiles of 64 TW features x 64 TA tokens, four waves of 32 TW x 32 TA each (2 x 2).
// The weights are the A operand, so a lane holds one token's features 8 (i / 4) +
// 4 (l / 32) + i % 4 of a block.  A stage is 64 columns, the blocks of the weights
// before those of the tokens, fetched as they are by DMA (1 KB an instruction); step
// s of a stage reads row l % 32, chunk 2 s + l / 32 in lane l.  Four stages are kept.
template <int TW, int TA> struct I8Tile {
  static constexpr int STAGE = 64 * (TW + TA) * 64;
};

// A wave's 32 TA tokens from m on, 32 TW features from n on: 32 tokens x 64 features at a time are
// scaled, packed, turned through 4 KB of LDS of the wave's own (16-byte chunk c of token t at c ^ (t &
// 7)) and stored as rows, a step behind, so that the reads have the next step's packing to land.  (DS
// operations of a wave run in order: the next writes follow the last reads.)  VEC: widths and strides
// are multiples of eight and out is 16-byte aligned, so a chunk is inside or outside as a whole.
// `par`: the wave's 32 TW channel scales and as many biases, in LDS.
template <typename T, int TW, int TA, bool GELU, bool VEC>
__device__ inline void i8_store(const i32x16 (&acc)[TW][TA], char* so, const float* par, const I8Mat& a,
                                uint16_t* __restrict__ out, long long ldo, int m, int n, int N) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (or its addresses are kept in registers through the products)
  const int hh = lane >> 5, c = lane & 7, t0 = lane >> 3, M = a.rows;
  const long long lane_at = t0 * ldo + 8 * c;
  float sa[TA];
#pragma unroll
  for (int j = 0; j < TA; ++j) sa[j] = a.scales[min(m + 32 * j + (lane & 31), M - 1)];
  u32x4 v[4];
  auto put = [&](int j, int i) {
    const int left = N - (n + 32 * i + 8 * c), rows = left > 0 ? M - (m + 32 * j) : 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      uint16_t* o = out + ((long long)(m + 32 * j + 8 * r) * ldo + n + 32 * i);
      if (8 * r + t0 < rows) {
        if constexpr (VEC)
          *(u32x4*)(o + lane_at) = v[r];
        else
          lin_put(o + lane_at, v[r], left);
      }
    }
  };
#pragma unroll
  for (int ii = 0; ii < TW; ii += 2) {
    f32x4 sw[2][4], sb[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sw[i][q] = *(const f32x4*)(par + 32 * (ii + i) + 8 * q + 4 * hh);
        sb[i][q] = *(const f32x4*)(par + 32 * (TW + ii + i) + 8 * q + 4 * hh);
      }
#pragma unroll
    for (int j = 0; j < TA; ++j) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = i8_out<T, GELU>(acc[ii + i][j][4 * q + e], sw[i][q][e], sa[j], sb[i][q][e]);
          *(u32x2*)(so + (lane & 31) * 128 + (((4 * i + q) ^ (lane & 7)) * 16) + 8 * hh) =
              u32x2{Pk<T>::pack(f[0], f[1]), Pk<T>::pack(f[2], f[3])};
        }
      __builtin_amdgcn_sched_barrier(0);
      if (ii || j) put(j ? j - 1 : TA - 1, j ? ii : ii - 2);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 8 * r + t0;
        v[r] = *(const u32x4*)(so + t * 128 + ((c ^ (t & 7)) * 16));
      }
    }
  }
  put(TA - 1, TW - 2);
}
// the wave's scales and biases to LDS of its own
template <typename T, int TW>
__device__ inline void i8_params(float* par, const I8Mat& w, const uint16_t* __restrict__ bias, int n) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = lane; i < 32 * TW; i += 64) {
    const int f = min(n + i, w.rows - 1);
    par[i] = w.scales[f];
    par[32 * TW + i] = bias ? T::to_f(bias[f]) : 0.f;
  }
}

// ---- the 256 x 256 tile: its inner loop is written out ----------------------
// With 256 accumulators a SIMD holds one wave, so no other wave covers a wait.  A
// step is one asm block of sixteen products (32 columns): the next step's eight
// fragment reads and half a stage's DMA go between them, and the one wait at its
// end finds the reads old.  A block waits for its own reads, so none of its
// outputs is in flight outside it.
#define I8_P(i, j) "v_mfma_i32_32x32x32_i8 %[c" #i #j "], %[w" #i "], %[a" #j "], %[c" #i #j "]\n\t"
#define I8_R(d, base, o) "ds_read_b128 %[" d "], %[" base "] offset:%c[" o "]\n\t"
// 1 KB (16 bytes a lane) to LDS at m0, which moves on
#define I8_D(i) "global_load_lds_dwordx4 %[v" #i "], %[g]\n\ts_add_u32 m0, m0, 0x400\n\t"
#define I8_ACC                                                                                          \
  [c00] "+a"(acc[0][0]), [c01] "+a"(acc[0][1]), [c02] "+a"(acc[0][2]), [c03] "+a"(acc[0][3]),           \
      [c10] "+a"(acc[1][0]), [c11] "+a"(acc[1][1]), [c12] "+a"(acc[1][2]), [c13] "+a"(acc[1][3]),       \
      [c20] "+a"(acc[2][0]), [c21] "+a"(acc[2][1]), [c22] "+a"(acc[2][2]), [c23] "+a"(acc[2][3]),       \
      [c30] "+a"(acc[3][0]), [c31] "+a"(acc[3][1]), [c32] "+a"(acc[3][2]), [c33] "+a"(acc[3][3])
#define I8_NEXT(f)                                                                                      \
  [x0] "=&v"(f.w[0]), [x1] "=&v"(f.w[1]), [x2] "=&v"(f.w[2]), [x3] "=&v"(f.w[3]), [y0] "=&v"(f.a[0]),   \
      [y1] "=&v"(f.a[1]), [y2] "=&v"(f.a[2]), [y3] "=&v"(f.a[3])
#define I8_CUR(f)                                                                                       \
  [w0] "v"(f.w[0]), [w1] "v"(f.w[1]), [w2] "v"(f.w[2]), [w3] "v"(f.w[3]), [a0] "v"(f.a[0]),             \
      [a1] "v"(f.a[1]), [a2] "v"(f.a[2]), [a3] "v"(f.a[3])
#define I8_READS(OFF)                                                                                   \
  [bw] "v"(bw), [ba] "v"(ba), [o0] "n"(OFF), [o1] "n"((OFF) + 2048), [o2] "n"((OFF) + 4096),            \
      [o3] "n"((OFF) + 6144)
#define I8_DMA_IN [v0] "v"(v[0]), [v1] "v"(v[1]), [v2] "v"(v[2]), [v3] "v"(v[3]), [g] "s"(g), [m] "s"(m)
#define I8_STEP                                                                                         \
  I8_P(0, 0) I8_R("x0", "bw", "o0") I8_P(0, 1) I8_R("y0", "ba", "o0") I8_P(0, 2) I8_R("x1", "bw", "o1") \
      I8_P(0, 3) I8_D(0) I8_P(1, 3) I8_R("y1", "ba", "o1") I8_P(1, 2) I8_R("x2", "bw", "o2")            \
          I8_P(1, 1) I8_R("y2", "ba", "o2") I8_P(1, 0) I8_D(1) I8_P(2, 0) I8_R("x3", "bw", "o3")        \
              I8_P(2, 1) I8_R("y3", "ba", "o3") I8_P(2, 2) I8_P(2, 3) I8_D(2) I8_P(3, 3)                \
                  I8_P(3, 2) I8_D(3) I8_P(3, 1) I8_P(3, 0) "s_waitcnt lgkmcnt(0)"

struct I8Frags {
  i32x4 w[4], a[4];
};
// First step of a stage: reads the stage's second fragments at OFF; fetches the second half of the
// stage three further on.
template <int OFF>
__device__ inline void i8_step0(i32x16 (&acc)[4][4], const I8Frags& f, I8Frags& nx, uint32_t bw, uint32_t ba,
                                const uint32_t* v, const char* g, uint32_t m) {
  asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 1\n\t" I8_STEP
               : I8_ACC, I8_NEXT(nx)
               : I8_CUR(f), I8_READS(OFF), I8_DMA_IN
               : "memory", "scc");
}
// Second step: once the next stage has landed for every wave (the two after it may be under way) and
// this one's reads are done, reads the next stage's first fragments at OFF and fetches the first half
// of the stage four further on into this one's place.
template <int OFF>
__device__ inline void i8_step1(i32x16 (&acc)[4][4], const I8Frags& f, I8Frags& nx, uint32_t bw, uint32_t ba,
                                const uint32_t* v, const char* g, uint32_t m) {
  asm volatile("s_mov_b32 m0, %[m]\n\ts_waitcnt vmcnt(16)\n\ts_barrier\n\t" I8_STEP
               : I8_ACC, I8_NEXT(nx)
               : I8_CUR(f), I8_READS(OFF), I8_DMA_IN
               : "memory", "scc");
}

// 256 x 256 for four waves of 128 x 128: a step's sixteen products take 512 cycles, the
// eight fragments that they need 256 of LDS reads a CU (waves of 64 x 64: as many as the
// products).  Bound: the matrix units are busy for 69% of the cycles, and the clock falls
// under their load (75,600 x 13,824 x 5,120 with GELU: 4.2 ms, 2.5 POP/s; a large library
// product in 8 bits 2.1).
// Work-groups stay for many tiles.  The DMA runs four stages ahead of the products
// as one stream over all of them, so a tile's first stages are loaded under the last
// products and the epilogue of the one before; the epilogue has LDS of its own.
template <typename T, bool GELU, bool VEC>
__global__ __launch_bounds__(256, 1) void i8_big_kernel(I8Mat a, I8Mat w, const uint16_t* __restrict__ bias,
                                                        uint16_t* __restrict__ out, long long ldo, int n,
                                                        int mt, int nt, int per_xcd) {
  constexpr int ST = I8Tile<4, 4>::STAGE, PAIR = 2 * ST, OWN = 4096 + 1024;
  static_assert(ST + 8192 < 65536, "LDS offsets of 16 bits");
  __shared__ __attribute__((aligned(1024))) char lds[4 * ST + 4 * OWN];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 1, wm = wave >> 1;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lin_lds_t*)lds;
  const int step = gridDim.x >> 3;
  int id = lin_first(per_xcd);
  const int end = lin_end(mt, nt, per_xcd);
  if (id >= end) return;

  // the stream of stages (n a tile, an even number): tile ld, its stage ls; this wave fetches 128 rows
  // of the weights (waves 0 and 1) or the tokens, KB i the block i of them
  const char* g;
  uint32_t v[8];
  int ld = id, ls = 0;
  auto aim = [&]() {
    int m0, n0;
    lin_place(ld, mt, nt, 8, 8, m0, n0);
    const I8Mat& x = wave < 2 ? w : a;
    const int first = 2 * (wave < 2 ? n0 : m0), last = (x.rows - 1) / 16 - first;
    g = x.codes + first * x.blk;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (uint32_t)(min(8 * (wave & 1) + i, last) * x.blk) + 16 * lane;
  };
  auto next_pair = [&]() {
    if (ld >= end) return;
    ls += 2;
    if (ls < n) return;
    ld += step;
    if (ld < end) {
      ls = 0;
      aim();
    } else {  // after the last tile every lane reads one place, so that the counts of loads stay
      ls = n - 2;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0;
    }
  };
  auto at = [&](int odd) { return g + (size_t)(ls + odd) * 1024; };
  const uint32_t dst = lds0 + wave * 8192;
  auto issue = [&](uint32_t off, int i) {  // KB i of a pair
    asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %[v], %[g]" ::[m] "s"(
                     dst + off + (i >> 3) * ST + (i & 7) * 1024),
                 [v] "v"(v[i & 7]), [g] "s"(at(i >> 3))
                 : "memory");
  };
  // two pairs but for the last half stage, which the first step fetches
  aim();
#pragma unroll
  for (int i = 0; i < 16; ++i) issue(0, i);
  next_pair();
#pragma unroll
  for (int i = 0; i < 12; ++i) issue(PAIR, i);
  // fragment addresses in the pair in use: of a stage's first and second steps
  const uint32_t row = (lane & 31) * 64, hh = lane >> 5, z = i8_swz(lane & 31);
  const uint32_t f0at = row + 16 * (hh ^ z), f1at = row + 16 * ((2 + hh) ^ z);
  uint32_t bw = lds0 + wn * 8192, ba = lds0 + 16384 + wm * 8192, off = 0;
  I8Frags f0, f1;
  {
    const uint32_t w0 = bw + f0at, a0 = ba + f0at;
    asm volatile("s_waitcnt vmcnt(20)\n\ts_barrier\n\t" I8_R("x0", "bw", "o0") I8_R("y0", "ba", "o0")
                 I8_R("x1", "bw", "o1") I8_R("y1", "ba", "o1") I8_R("x2", "bw", "o2") I8_R("y2", "ba", "o2")
                 I8_R("x3", "bw", "o3") I8_R("y3", "ba", "o3") "s_waitcnt lgkmcnt(0)"
                 : I8_NEXT(f0)
                 : [bw] "v"(w0), [ba] "v"(a0), [o0] "n"(0), [o1] "n"(2048), [o2] "n"(4096), [o3] "n"(6144)
                 : "memory");
  }
  char* own = lds + 4 * ST + wave * OWN;
  i32x16 acc[4][4];
  for (;;) {
    int m0, n0;
    lin_place(id, mt, nt, 8, 8, m0, n0);
    i8_params<T, 4>((float*)(own + 4096), w, bias, (n0 + wn * 4) * 32);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = i32x16{};
        asm volatile("" : "+a"(acc[i][j]));  // a register set each, now
      }
    for (int s = n; s > 0; s -= 2) {
      const uint32_t other = PAIR - 2 * off;  // from this pair to the other one (off: 0 or PAIR)
      i8_step0<0>(acc, f0, f1, bw + f1at, ba + f1at, v + 4, at(1), dst + PAIR - off + ST + 4096);
      next_pair();
      i8_step1<ST>(acc, f1, f0, bw + f0at, ba + f0at, v, at(0), dst + off);
      i8_step0<ST>(acc, f0, f1, bw + f1at, ba + f1at, v + 4, at(0), dst + off + 4096);
      bw += other, ba += other;
      i8_step1<0>(acc, f1, f0, bw + f0at, ba + f0at, v, at(1), dst + off + ST);
      off = PAIR - off;
    }
    // the last products' registers are readable after 18 cycles of issue
    asm volatile("s_nop 15\n\ts_nop 15" : I8_ACC);
    i8_store<T, 4, 4, GELU, VEC>(acc, own, (const float*)(own + 4096), a, out, ldo, (m0 + wm * 4) * 32,
                                 (n0 + wn * 4) * 32, w.rows);
    id += step;
    if (id >= end) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- the 128 x 128 tile ------------------------------------------------------
// The same with a whole stage a step: eight products, the next stage's eight
// fragment reads and the DMA of the stage four further on.  Two work-groups fit a
// CU, and one's products pass under the other's start and epilogue.  Bound: 0.43 us a
// stage with two on every CU (2.7 POP/s), and about 6 us beside the stages, of which the
// outputs' bytes are a half (4,680 x 1,536 x 1,536: 15.4 us).
#define I8_Q(c, i, j) "v_mfma_i32_32x32x32_i8 %[c" #i #j "], %[w" #c #i "], %[a" #c #j "], %[c" #i #j "]\n\t"
#define I8_MID_STEP                                                                                     \
  "s_mov_b32 m0, %[m]\n\ts_waitcnt vmcnt(8)\n\ts_barrier\n\t" I8_Q(0, 0, 0) I8_R("x00", "bw0", "o0")    \
      I8_R("y00", "ba0", "o0") I8_Q(0, 0, 1) I8_R("x01", "bw0", "o1") I8_R("y01", "ba0", "o1")          \
          I8_Q(0, 1, 1) I8_D(0) I8_R("x10", "bw1", "o0") I8_Q(0, 1, 0) I8_R("y10", "ba1", "o0") I8_D(1) \
              I8_Q(1, 0, 0) I8_R("x11", "bw1", "o1") I8_R("y11", "ba1", "o1") I8_Q(1, 0, 1) I8_D(2)     \
                  I8_Q(1, 1, 1) I8_D(3) I8_Q(1, 1, 0) "s_waitcnt lgkmcnt(0)"
struct I8MidFrags {
  i32x4 w[2][2], a[2][2];  // [fragment of the stage][block]
};
#define I8_MID_NEXT(nx)                                                                                 \
  [x00] "=&v"(nx.w[0][0]), [x01] "=&v"(nx.w[0][1]), [x10] "=&v"(nx.w[1][0]), [x11] "=&v"(nx.w[1][1]),   \
      [y00] "=&v"(nx.a[0][0]), [y01] "=&v"(nx.a[0][1]), [y10] "=&v"(nx.a[1][0]), [y11] "=&v"(nx.a[1][1])
// OFF: where the next stage lies
template <int OFF>
__device__ inline void i8_mid_step(i32x16 (&acc)[2][2], const I8MidFrags& f, I8MidFrags& nx, uint32_t bw0,
                                   uint32_t bw1, uint32_t ba0, uint32_t ba1, const uint32_t (&v)[4], const char* g,
                                   uint32_t m) {
  asm volatile(I8_MID_STEP
               : [c00] "+v"(acc[0][0]), [c01] "+v"(acc[0][1]), [c10] "+v"(acc[1][0]), [c11] "+v"(acc[1][1]),
                 I8_MID_NEXT(nx)
               : [w00] "v"(f.w[0][0]), [w01] "v"(f.w[0][1]), [w10] "v"(f.w[1][0]), [w11] "v"(f.w[1][1]),
                 [a00] "v"(f.a[0][0]), [a01] "v"(f.a[0][1]), [a10] "v"(f.a[1][0]), [a11] "v"(f.a[1][1]),
                 [bw0] "v"(bw0), [bw1] "v"(bw1), [ba0] "v"(ba0), [ba1] "v"(ba1), [o0] "n"(OFF), [o1] "n"(OFF + 2048),
                 I8_DMA_IN
               : "memory", "scc");
}

template <typename T, bool GELU, bool VEC>
__global__ __launch_bounds__(256, 2) void i8_mid_kernel(I8Mat a, I8Mat w, const uint16_t* __restrict__ bias,
                                                        uint16_t* __restrict__ out, long long ldo, int n, int mt,
                                                        int nt, int per_xcd) {
  constexpr int ST = I8Tile<2, 2>::STAGE, PAIR = 2 * ST;
  __shared__ __attribute__((aligned(1024))) char lds[4 * ST];
  __shared__ __attribute__((aligned(16))) float par[4][128];
  const int id = lin_first(per_xcd);
  if (id >= lin_end(mt, nt, per_xcd)) return;
  int m0, n0;
  lin_place(id, mt, nt, 4, 4, m0, n0);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 1, wm = wave >> 1;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lin_lds_t*)lds;
  const I8Mat& x = wave < 2 ? w : a;
  const int first = 2 * (wave < 2 ? n0 : m0), last = (x.rows - 1) / 16 - first;
  const char* g = x.codes + first * x.blk;
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (uint32_t)(min(4 * (wave & 1) + i, last) * x.blk) + 16 * lane;
  const uint32_t dst = lds0 + wave * 4096;
  // (past the last stage it is fetched again, so that the counts of loads in flight stay)
  auto at = [&](int s) { return g + (size_t)min(s, n - 1) * 1024; };
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %[v], %[g]" ::[m] "s"(
                       dst + s * ST + i * 1024),
                   [v] "v"(v[i]), [g] "s"(at(s))
                   : "memory");
  i8_params<T, 2>(par[wave], w, bias, (n0 + wn * 2) * 32);
  i32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = i32x16{};
  const uint32_t row = (lane & 31) * 64, hh = lane >> 5, z = i8_swz(lane & 31);
  const uint32_t at0 = row + 16 * (hh ^ z), at1 = row + 16 * ((2 + hh) ^ z);
  uint32_t bw0 = lds0 + wn * 4096 + at0, bw1 = lds0 + wn * 4096 + at1;
  uint32_t ba0 = lds0 + 8192 + wm * 4096 + at0, ba1 = lds0 + 8192 + wm * 4096 + at1, off = 0;
  I8MidFrags f0, f1;
  asm volatile("s_waitcnt vmcnt(12)\n\ts_barrier\n\t" I8_R("x00", "bw0", "o0") I8_R("x01", "bw0", "o1")
               I8_R("x10", "bw1", "o0") I8_R("x11", "bw1", "o1") I8_R("y00", "ba0", "o0") I8_R("y01", "ba0", "o1")
               I8_R("y10", "ba1", "o0") I8_R("y11", "ba1", "o1") "s_waitcnt lgkmcnt(0)"
               : I8_MID_NEXT(f0)
               : [bw0] "v"(bw0), [bw1] "v"(bw1), [ba0] "v"(ba0), [ba1] "v"(ba1), [o0] "n"(0), [o1] "n"(2048)
               : "memory");
  for (int s = 0; s < n; s += 2) {
    const uint32_t other = PAIR - 2 * off;  // from this pair of stages to the other one
    i8_mid_step<ST>(acc, f0, f1, bw0, bw1, ba0, ba1, v, at(s + 4), dst + off);
    bw0 += other, bw1 += other, ba0 += other, ba1 += other;
    i8_mid_step<0>(acc, f1, f0, bw0, bw1, ba0, ba1, v, at(s + 5), dst + off + ST);
    off = PAIR - off;
  }
  // every load has landed and every wave's reads are done: LDS is free; the products' registers are
  // readable
  asm volatile("s_nop 15\n\ts_nop 15\n\ts_waitcnt vmcnt(0)\n\ts_barrier"
               : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1])
               :
               : "memory");
  i8_store<T, 2, 2, GELU, VEC>(acc, lds + wave * 4096, par[wave], a, out, ldo, (m0 + wm * 2) * 32, (n0 + wn * 2) * 32,
                               w.rows);
}

// tiles of 64 TW x 64 TA
template <typename T, int TW, int TA>
static int i8_tile_launch(const I8Mat& a, const I8Mat& w, const uint16_t* bias, int act, uint16_t* out,
                          long long ldo, int units, hipStream_t st) {
  const int mt = cdiv(a.blocks, 2 * TA), nt = cdiv(w.blocks, 2 * TW);
  const long long tiles = (long long)mt * nt;
  if (tiles > (1 << 23)) {  // 2^31 threads of 128 x 128 tiles; as many large ones are a TB of outputs
    t2t_set_error("int8_product: M=%d N=%d", a.rows, w.rows);
    return T2T_ERR_UNSUPPORTED;
  }
  const int per = cdiv(tiles, 8);
  auto launch = [&](auto kernel, int slots) {
    hipLaunchKernelGGL(kernel, dim3(8 * slots), dim3(256), 0, st, a, w, bias, out, ldo, 2 * units, mt, nt, per);
  };
  auto form = [&](auto G, auto V) {
    constexpr bool GELU = decltype(G)::value, VEC = decltype(V)::value;
    if constexpr (TW == 4)  // fills a CU: 32 work-groups an XCD, which go through the tiles
      launch(i8_big_kernel<T, GELU, VEC>, per < 32 ? per : 32);
    else
      launch(i8_mid_kernel<T, GELU, VEC>, per);
  };
  const bool gelu = act == T2T_ACT_GELU_TANH;
  const bool vec = w.rows % 8 == 0 && ldo % 8 == 0 && (uintptr_t)out % 16 == 0;
  if (gelu)
    vec ? form(std::true_type{}, std::true_type{}) : form(std::true_type{}, std::false_type{});
  else
    vec ? form(std::false_type{}, std::true_type{}) : form(std::false_type{}, std::false_type{});
  T2T_LAUNCH_CHECK("int8_product");
  return T2T_OK;
}

// Which tile, measured in graphs of twenty launches, us (K = 5,120 / 1,536):
//                       32 x 32 blocks     split       128 x 128       256 x 256
//   96 x 5,120                       480  13.2 /  6.2   15.2 /  7.2    46.6 / 19.3
//   128 x 5,120                      640  18.6 /  8.6   15.4 /  7.3    46.6 / 19.8
//   2,048 x 5,120 (160 of 256 x 256)                    55.5 / 20.9    53.2 / 24.4
//   3,000 x 5,120 (240)                                 75.9 / 28.1    66.1 / 27.5
//   4,096 x 4,096 (256)                                 78.6 / 29.7    70.1 / 28.7
//   9,000 x 2,048 (288)                                 90.9 / 34.1     110 / 44.1
//   2,700 x 13,824 (594)                                 185 / 70.3     172 / 67.1
// The small tiles' time goes with their number (two fit a CU, of which one goes on while the other
// starts or ends); the large ones go by rounds of 256, of which a full one takes that of 890 small tiles
// and an empty one more than half of it.
template <typename T>
static int i8_product(const I8Mat& a, const I8Mat& w, const uint16_t* bias, int act, uint16_t* out, long long ldo,
                      int units, hipStream_t st) {
  if ((long long)a.blocks * w.blocks <= 512)
    return i8_split_launch<T, 4, false>(I8Src{a, nullptr, 0, 0}, w, bias, act, out, ldo, units, st);
  const long long big = (long long)cdiv(a.blocks, 8) * cdiv(w.blocks, 8), rest = big % 256;
  const long long mid = (long long)cdiv(a.blocks, 4) * cdiv(w.blocks, 4);
  if (big / 256 * 890 + (rest ? 470 + 420 * rest / 256 : 0) < mid + 25)
    return i8_tile_launch<T, 4, 4>(a, w, bias, act, out, ldo, units, st);
  return i8_tile_launch<T, 2, 2>(a, w, bias, act, out, ldo, units, st);
}

static int i8_check_product(const char* what, const void* w_codes, const float* w_scales, int act, const void* out,
                            int dtype, long long out_row_stride, int M, int N, int K) {
  int rc = i8_check_sizes(what, M, K);
  if (rc != T2T_OK) return rc;
  T2T_REQUIRE(act == T2T_ACT_NONE || act == T2T_ACT_GELU_TANH, "%s: activation %d", what, act);
  T2T_REQUIRE(N >= 1 && N <= (1 << 30), "%s: N=%d (1 <= N <= 2^30)", what, N);
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "%s: dtype %d", what, dtype);
  if (M == 0) return T2T_OK;
  rc = i8_check_rows(what, out, dtype, out_row_stride, M, N);
  return rc != T2T_OK ? rc : i8_check_matrix(what, w_codes, w_scales);
}

extern "C" int t2t_int8_product(const void* a_codes, const float* a_scales, const void* w_codes,
                                const float* w_scales, const void* bias, int act, void* out, int dtype,
                                long long out_row_stride, int M, int N, int K, void* stream) {
  int rc = i8_check_product("int8_product", w_codes, w_scales, act, out, dtype, out_row_stride, M, N, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_matrix("int8_product", a_codes, a_scales);
  if (rc != T2T_OK) return rc;
  const long long blk = 16LL * i8_kp(K);
  const I8Mat a{(const char*)a_codes, blk, a_scales, M, cdiv(M, 32)};
  const I8Mat w{(const char*)w_codes, blk, w_scales, N, cdiv(N, 32)};
  return (dtype == T2T_BF16 ? i8_product<BF16T> : i8_product<F16T>)(a, w, (const uint16_t*)bias, act, (uint16_t*)out,
                                                                   out_row_stride, i8_kp(K) / 128,
                                                                   (hipStream_t)stream);
}

// Few rows are quantised by the product itself: every work-group does it again (5120 x 5120, weights
// from memory: one row 10.5 us, two 11.8, three 14.5, four 14.8; with a launch before it 14.4, 14.1, 14.2, 14.8).
static bool i8_few(int M, int K) { return M <= 2 && M * i8_kp(K) <= I8_X16_BYTES; }

// codes, then scales
extern "C" size_t t2t_int8_linear_ws_bytes(int M, int N, int K) {
  (void)N;
  const size_t codes = t2t_int8_code_bytes(M, K);
  return codes && !i8_few(M, K) ? codes + t2t_align256((size_t)M * 4) : 0;
}

extern "C" int t2t_int8_linear(const void* x, int dtype, long long x_row_stride, const void* w_codes,
                               const float* w_scales, const void* bias, int act, void* out,
                               long long out_row_stride, int M, int N, int K, void* ws, size_t ws_bytes,
                               void* stream) {
  // everything before the first launch
  int rc = i8_check_product("int8_linear", w_codes, w_scales, act, out, dtype, out_row_stride, M, N, K);
  if (rc != T2T_OK || M == 0) return rc;
  rc = i8_check_rows("int8_linear", x, dtype, x_row_stride, M, K);
  if (rc != T2T_OK) return rc;
  if (i8_few(M, K)) {
    const I8Src a{I8Mat{nullptr, 0, nullptr, M, 1}, (const uint16_t*)x, x_row_stride, K};
    const I8Mat w{(const char*)w_codes, 16LL * i8_kp(K), w_scales, N, cdiv(N, 32)};
    return (dtype == T2T_BF16 ? i8_split_launch<BF16T, 5, true> : i8_split_launch<F16T, 5, true>)(
        a, w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, i8_kp(K) / 128, (hipStream_t)stream);
  }
  const size_t need = t2t_int8_linear_ws_bytes(M, N, K);
  if (!ws || ws_bytes < need) {
    t2t_set_error("int8_linear: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0, need);
    return T2T_ERR_WORKSPACE;
  }
  T2T_REQUIRE((uintptr_t)ws % 16 == 0, "int8_linear: workspace must be 16-byte aligned");
  float* scales = (float*)((char*)ws + t2t_int8_code_bytes(M, K));
  rc = t2t_int8_quantize(x, dtype, x_row_stride, ws, scales, M, K, stream);
  if (rc != T2T_OK) return rc;
  return t2t_int8_product(ws, scales, w_codes, w_scales, bias, act, out, dtype, out_row_stride, M, N, K, stream);
}
