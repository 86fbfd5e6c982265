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
#include <type_traits>

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

static inline long long mx_row_blocks(int M) { return ((long long)M + 31) / 32; }
static inline int mx_kp(int K) { return (K + 255) / 256 * 256; }

extern "C" size_t t2t_mxfp4_scale_bytes(int M, int K) {
  return M <= 0 || K <= 0 ? 0 : (size_t)mx_row_blocks(M) * (((size_t)K + 255) / 256 * 256);
}
extern "C" size_t t2t_mxfp4_code_bytes(int M, int K) { return 16 * t2t_mxfp4_scale_bytes(M, K); }

// a 16-bit matrix beside its codes and scales
static int mx_check_rows(const char* what, const void* x, int dtype, long long row_stride,
                         const void* codes, const void* scales, int M, int K) {
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "%s: dtype %d", what, dtype);
  T2T_REQUIRE(M >= 0 && M <= (1 << 30) && K >= 32 && K % 32 == 0 && K <= (1 << 27),
              "%s: M=%d K=%d (M <= 2^30, K a multiple of 32, K <= 2^27)", what, M, K);
  if (M == 0) return T2T_OK;
  T2T_REQUIRE(x && codes && scales, "%s: null pointer", what);
  T2T_REQUIRE(((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) % 16 == 0 && row_stride % 8 == 0 &&
                  (M == 1 || row_stride >= K),
              "%s: rows must be 16-byte aligned, row stride %lld >= K", what, row_stride);
  return T2T_OK;
}

// work-groups of the two conversions, which go through the tiles of 32 rows x 256 columns (a grid
// may not hold 2^32 threads)
static inline dim3 mx_grid(long long wgs) { return dim3((unsigned)(wgs < 65536 ? wgs : 65536)); }

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
  u16x2 both{0, 0};
#pragma unroll
  for (int v = 0; v < 4; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      both = __builtin_elementwise_max(both, __builtin_bit_cast(u16x2, x[v][i] & 0x7fff7fffu));
  const uint32_t top = max((uint32_t)both[0], (uint32_t)both[1]);
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
// quantise: a work-group per 32 rows x 256 columns, a thread per block (64 bytes
// of a row; the four loads' lines meet in L1).  Bound: reading x, 75,600 x 5,120
// in 185 us, 5.3 TB/s with the codes written.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const uint16_t* __restrict__ x,
                                                          long long row_stride,
                                                          uint32_t* __restrict__ codes,
                                                          uint32_t* __restrict__ scales, int M, int K,
                                                          int groups, long long wgs) {
  const int r = threadIdx.x >> 3, blk = threadIdx.x & 7, half = blk & 1, j = blk >> 1;
  for (long long wg = blockIdx.x; wg < wgs; wg += gridDim.x) {
    const long long row = wg / groups * 32 + r;
    const int col = 256 * (int)(wg % groups) + 32 * blk;
    u32x4 c{0u, 0u, 0u, 0u};
    uint32_t byte = 0;
    if (row < M && col < K) {
      const u32x4* src = (const u32x4*)(x + row * row_stride + col);
      u32x4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = src[i];
      mx_block<T>(v, c, byte);
    }
    *(u32x4*)((char*)codes + wg * 4096 + j * 1024 + (r + 32 * half) * 16) = c;
    // the four bytes of a lane's dword sit in blocks half, half + 2, ...
    uint32_t word = byte << (8 * j);
    word |= __shfl_xor(word, 2, 64);
    word |= __shfl_xor(word, 4, 64);
    if (j == 0) scales[wg * 64 + r + 32 * half] = word;
  }
}

extern "C" int t2t_mxfp4_quantize(const void* x, int dtype, long long row_stride, void* codes,
                                  void* scales, int M, int K, void* stream) {
  const int rc = mx_check_rows("mxfp4_quantize", x, dtype, row_stride, codes, scales, M, K);
  if (rc != T2T_OK || M == 0) return rc;
  const int groups = mx_kp(K) / 256;
  const long long wgs = mx_row_blocks(M) * groups;
  if (dtype == T2T_BF16)
    hipLaunchKernelGGL(mx_quantize_kernel<BF16T>, mx_grid(wgs), dim3(256), 0, (hipStream_t)stream,
                       (const uint16_t*)x, row_stride, (uint32_t*)codes, (uint32_t*)scales, M, K, groups,
                       wgs);
  else
    hipLaunchKernelGGL(mx_quantize_kernel<F16T>, mx_grid(wgs), dim3(256), 0, (hipStream_t)stream,
                       (const uint16_t*)x, row_stride, (uint32_t*)codes, (uint32_t*)scales, M, K, groups,
                       wgs);
  T2T_LAUNCH_CHECK("mxfp4_quantize");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// the values back: 32 lanes take a row of the 256 columns, eight values each, so
// that the stores are whole rows (a thread per block, with its four stores 64
// bytes apart from its neighbour's, took 260 us at 75,600 x 5,120; this takes
// 194, 5.0 TB/s).  Bound: writing the values.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales,
                                                            uint16_t* __restrict__ out,
                                                            long long row_stride, int M, int K,
                                                            int groups, long long wgs) {
  const int part = threadIdx.x & 31, blk = part >> 2, half = blk & 1, j = blk >> 1;
  for (long long wg = blockIdx.x; wg < wgs; wg += gridDim.x) {
    const int col = 256 * (int)(wg % groups) + 8 * part;
    if (col >= K) continue;
    const uint32_t* cp = codes + wg * 1024 + j * 256 + half * 128 + (part & 3);
    const uint8_t* sp = scales + wg * 256 + half * 128 + j;
    uint32_t c[4], byte[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (threadIdx.x >> 5);
      c[i] = cp[4 * r];
      byte[i] = sp[4 * r];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = wg / groups * 32 + 8 * i + (threadIdx.x >> 5);
      const float scale = __builtin_bit_cast(float, byte[i] << 23);
      u32x4 o;
      o[0] = MxCvt<T>::template dec<0>(c[i], scale);
      o[1] = MxCvt<T>::template dec<1>(c[i], scale);
      o[2] = MxCvt<T>::template dec<2>(c[i], scale);
      o[3] = MxCvt<T>::template dec<3>(c[i], scale);
      if (byte[i] == 255)
        o = u32x4{MxCvt<T>::nan_pair, MxCvt<T>::nan_pair, MxCvt<T>::nan_pair, MxCvt<T>::nan_pair};
      if (row < M) *(u32x4*)(out + row * row_stride + col) = o;
    }
  }
}

extern "C" int t2t_mxfp4_dequantize(const void* codes, const void* scales, void* out, int dtype,
                                    long long row_stride, int M, int K, void* stream) {
  const int rc = mx_check_rows("mxfp4_dequantize", out, dtype, row_stride, codes, scales, M, K);
  if (rc != T2T_OK || M == 0) return rc;
  const int groups = mx_kp(K) / 256;
  const long long wgs = mx_row_blocks(M) * groups;
  if (dtype == T2T_BF16)
    hipLaunchKernelGGL(mx_dequantize_kernel<BF16T>, mx_grid(wgs), dim3(256), 0,
                       (hipStream_t)stream, (const uint32_t*)codes, (const uint8_t*)scales,
                       (uint16_t*)out, row_stride, M, K, groups,
                       wgs);
  else
    hipLaunchKernelGGL(mx_dequantize_kernel<F16T>, mx_grid(wgs), dim3(256), 0,
                       (hipStream_t)stream, (const uint32_t*)codes, (const uint8_t*)scales,
                       (uint16_t*)out, row_stride, M, K, groups,
                       wgs);
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

// gelu(x) = x / 2 (1 + tanh u) = x / (1 + e^(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3), with the
// constants of e^(-2 u) = 2^(x (c0 + c1 x^2)).  v_exp_f32 and v_rcp_f32 are within 1 ulp.
__device__ inline float mx_gelu(float x) {
  const float z = x * __builtin_fmaf(-0.10294324f, x * x, -2.3022082f);
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z));
}

struct MxMat {
  const char* codes;
  const uint32_t* scales;
  int rows, blocks;  // rows, row blocks of 32
};

// Tiles of 64 TW features x 64 TA tokens, four waves of 32 TW x 32 TA each (2 x
// 2).  The weights are the A operand, so a lane holds one token's features 8
// (i / 4) + 4 (l / 32) + i % 4 of a block.  Operands are staged through LDS by
// DMA, in the order they are held in memory, which is the order of the
// fragments: both the DMA and the fragment reads are linear (no conflicts, no
// address arithmetic).  A stage is 128 columns (two fragments a row block) and
// four stages are kept, so a stage's loads have the time of three to land.
typedef __attribute__((address_space(3))) void mx_lds_t;
typedef __attribute__((address_space(1))) void mx_glb_t;

template <int TW, int TA> struct MxTile {
  static constexpr int RB = 2 * (TW + TA);          // row blocks: 2 TW of weights, 2 TA of tokens
  static constexpr int CODES = RB * 2048;           // a stage's codes
  static constexpr int STAGE = CODES + RB * 256;    // with its scales (of every second stage)
};

// Consecutive work-groups go to the eight XCDs in turn: each takes a run of
// tiles, eight token tiles by all feature tiles, so that the 32 tiles an XCD
// has under way share their panels in its L2.
__device__ inline int mx_first(int per_xcd) { return (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3); }
__device__ inline int mx_end(int mt, int nt, int per_xcd) {
  return min(mt * nt, ((int)(blockIdx.x & 7) + 1) * per_xcd);
}
// a tile's first row blocks
__device__ inline void mx_place(int id, int mt, int nt, int mb, int nb, int& m0, int& n0) {
  const int grp = id / (8 * nt), in = id - grp * 8 * nt;
  const int gm = min(8, mt - grp * 8);
  m0 = (grp * 8 + in % gm) * mb;
  n0 = (in / gm) * nb;
}

// The sums start at the bias, which comes through LDS of the wave's own (128 TW bytes): a lane needs
// 16 TW of the wave's 32 TW features.
template <typename T, int TW, int TA>
__device__ inline void mx_start(f32x16 (&acc)[TW][TA], const uint16_t* __restrict__ bias, float* own, int f0,
                                int rows) {
  const int lane = threadIdx.x & 63, hh = lane >> 5;
  if (bias)
#pragma unroll
    for (int i = lane; i < 32 * TW; i += 64) own[i] = T::to_f(bias[min(f0 + i, rows - 1)]);
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    f32x16 b0 = zero16();
    if (bias)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 v = *(const f32x4*)(own + 32 * i + 8 * q + 4 * hh);
#pragma unroll
        for (int e = 0; e < 4; ++e) b0[4 * q + e] = v[e];
      }
#pragma unroll
    for (int j = 0; j < TA; ++j) {
      acc[i][j] = b0;
      if constexpr (TW == 4) asm volatile("" : "+a"(acc[i][j]));  // a register set each, now
    }
  }
}

// The values of one row, the first n of which are inside, to an o of any alignment (rows of odd
// widths: the store takes 16 bytes at any address, two at a time it cost 16 us at 4099 x 2041)
template <typename VT>
__device__ inline void mx_put(uint16_t* o, const VT& v, int n) {
  if (n >= (int)sizeof(VT) / 2)
    __builtin_memcpy(o, &v, sizeof(VT));
  else
#pragma unroll
    for (int e = 0; e < (int)sizeof(VT) / 2; ++e)
      if (e < n) o[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
}

// A wave's 32 TA tokens from m on, 32 TW features from n on: 32 tokens x 64 features at a time are
// packed, turned through 4 KB of LDS of the wave's own (16-byte chunk c of token t at c ^ (t & 7)) and
// stored as rows, a step behind, so that the reads have the next step's packing to land.  (DS
// operations of a wave run in order: the next writes follow the last reads.)  VEC: widths and strides
// are multiples of eight and out is 16-byte aligned, so a chunk is inside or outside as a whole, and a
// store takes one scalar address, one offset a lane for all of them and one comparison.
template <typename T, int TW, int TA, bool GELU, bool VEC>
__device__ inline void mx_store(const f32x16 (&acc)[TW][TA], char* so, uint16_t* __restrict__ out,
                                long long ldo, int m, int M, int n, int N) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (or its addresses are kept in registers through the products)
  const int hh = lane >> 5, c = lane & 7, t0 = lane >> 3;
  const long long lane_at = t0 * ldo + 8 * c;
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
          mx_put(o + lane_at, v[r], left);
      }
    }
  };
#pragma unroll
  for (int k = 0; k < TA * (TW / 2); ++k) {
    const int j = k / (TW / 2), ii = k % (TW / 2) * 2;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f[e] = GELU ? mx_gelu(acc[ii + i][j][4 * q + e]) : acc[ii + i][j][4 * q + e];
        *(u32x2*)(so + (lane & 31) * 128 + (((4 * i + q) ^ (lane & 7)) * 16) + 8 * hh) =
            u32x2{Pk<T>::pack(f[0], f[1]), Pk<T>::pack(f[2], f[3])};
      }
    __builtin_amdgcn_sched_barrier(0);
    if (k) put((k - 1) / (TW / 2), (k - 1) % (TW / 2) * 2);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 8 * r + t0;
      v[r] = *(const u32x4*)(so + t * 128 + ((c ^ (t & 7)) * 16));
    }
  }
  put(TA - 1, TW - 2);
}

// ---- the 256 x 256 tile: its inner loop is written out ----------------------
// With 256 accumulators a SIMD holds one wave, so no other wave covers a wait,
// and left to itself the compiler issues a fragment read right before the
// product that needs it (2.93 ms at 75,600 x 13,824 x 5,120; 2.52 written out).
// A step is one asm block of sixteen products (64 columns): the next step's eight
// fragment reads and half a stage's DMA go between them, and the one wait at its
// end finds the reads old.  A block waits for its own reads, so none of its
// outputs is in flight outside it.
// Why this tile: per stage a CU moves 36 KB to LDS (64 bytes a cycle at most) and
// reads 64 KB from it for 1024 cycles of products; with 128 x 128 it is LDS that
// bounds.  Measured: 1203 cycles a stage, 1024 of them products, and 12,000 a tile
// beside them (its start and its epilogue, which only DMA overlaps: a fifth of the
// time at K = 5120); 4.4 PFLOP/s at K = 5120, 4.9 at 13,824.  Bounds: those idle
// cycles, and power: the card holds 1.5 to 1.75 GHz of 2.4 on random codes, and
// with zero codes the time is 1.3 times shorter.  With loads that always hit L2, or
// reads and DMA placed otherwise, it is the same.  How much of the idle fifth the
// clock would take back is not measured.
#define MX_P(i, j)                                                                                      \
  "v_mfma_scale_f32_32x32x64_f8f6f4 %[c" #i #j "], %[w" #i "], %[a" #j "], %[c" #i #j "], %[p" #i     \
  "], %[q" #j "] " MX_SEL " cbsz:4 blgp:4\n\t"
#define MX_R(d, base, o) "ds_read_b128 %[" d "], %[" base "] offset:%c[" o "]\n\t"
#define MX_RS(d, base, o) "ds_read_b32 %[" d "], %[" base "] offset:%c[" o "]\n\t"
// 1 KB (16 bytes a lane) to LDS at m0, which moves on
#define MX_D(i) "global_load_lds_dwordx4 %[v], %[g" #i "]\n\ts_add_u32 m0, m0, 0x400\n\t"
#define MX_ACC                                                                                          \
  [c00] "+a"(acc[0][0]), [c01] "+a"(acc[0][1]), [c02] "+a"(acc[0][2]), [c03] "+a"(acc[0][3]),           \
      [c10] "+a"(acc[1][0]), [c11] "+a"(acc[1][1]), [c12] "+a"(acc[1][2]), [c13] "+a"(acc[1][3]),       \
      [c20] "+a"(acc[2][0]), [c21] "+a"(acc[2][1]), [c22] "+a"(acc[2][2]), [c23] "+a"(acc[2][3]),       \
      [c30] "+a"(acc[3][0]), [c31] "+a"(acc[3][1]), [c32] "+a"(acc[3][2]), [c33] "+a"(acc[3][3])
#define MX_NEXT(f)                                                                                      \
  [x0] "=&v"(f.w[0]), [x1] "=&v"(f.w[1]), [x2] "=&v"(f.w[2]), [x3] "=&v"(f.w[3]), [y0] "=&v"(f.a[0]),   \
      [y1] "=&v"(f.a[1]), [y2] "=&v"(f.a[2]), [y3] "=&v"(f.a[3])
#define MX_CUR(f, sc)                                                                                   \
  [w0] "v"(f.w[0]), [w1] "v"(f.w[1]), [w2] "v"(f.w[2]), [w3] "v"(f.w[3]), [a0] "v"(f.a[0]),             \
      [a1] "v"(f.a[1]), [a2] "v"(f.a[2]), [a3] "v"(f.a[3]), [p0] "v"(sc.w[0]), [p1] "v"(sc.w[1]),       \
      [p2] "v"(sc.w[2]), [p3] "v"(sc.w[3]), [q0] "v"(sc.a[0]), [q1] "v"(sc.a[1]), [q2] "v"(sc.a[2]),    \
      [q3] "v"(sc.a[3])
#define MX_READS(OFF)                                                                                   \
  [bw] "v"(bw), [ba] "v"(ba), [o0] "n"(OFF), [o1] "n"((OFF) + 2048), [o2] "n"((OFF) + 4096),            \
      [o3] "n"((OFF) + 6144)
// where the reads and the DMA of a step go; X0 .. X3: what else it has to issue (products in an order
// that changes one operand at a time)
#define MX_STEP(X0, X1, X2, X3)                                                                         \
  MX_P(0, 0) MX_R("x0", "bw", "o0") MX_P(0, 1) MX_R("y0", "ba", "o0") MX_P(0, 2) MX_R("x1", "bw", "o1") \
      MX_P(0, 3) MX_D(0) X0 MX_P(1, 3) MX_R("y1", "ba", "o1") MX_P(1, 2) MX_R("x2", "bw", "o2")         \
          MX_P(1, 1) MX_R("y2", "ba", "o2") MX_P(1, 0) MX_D(1) X1 MX_P(2, 0) MX_R("x3", "bw", "o3")     \
              MX_P(2, 1) MX_R("y3", "ba", "o3") MX_P(2, 2) X2 MX_P(2, 3) MX_D(2) MX_P(3, 3) X3          \
                  MX_P(3, 2) MX_D(3) MX_P(3, 1) MX_P(3, 0) "s_waitcnt lgkmcnt(0)"

struct MxFrags {
  u32x4 w[4], a[4];
};
struct MxScales {
  uint32_t w[4], a[4];
};
struct MxDma {
  const char* g[8];    // this wave's eight KB of a stage, at stage 0
  const char* scales;  // its KB of scales, per lane
};

// half a stage's DMA: four KB from g[0 .. 3] + v to LDS at m
#define MX_DMA_IN                                                                                       \
  [v] "v"(v), [m] "s"(m), [g0] "s"(g[0]), [g1] "s"(g[1]), [g2] "s"(g[2]), [g3] "s"(g[3])

// First step of a stage: reads the stage's second fragments at OFF; fetches the second half of the
// stage three further on (after an odd stage, that is of an even one, its scales too).
template <int ODD, int OFF>
__device__ inline void mx_step0(f32x16 (&acc)[4][4], const MxFrags& f, MxFrags& nx, const MxScales& sc,
                                uint32_t bw, uint32_t ba, const char* const* g, uint32_t m, uint32_t v,
                                uint32_t ms, const char* vs) {
  if constexpr (!ODD) {
#define MX_SEL "op_sel:[0,0,0] op_sel_hi:[0,0,0]"
    asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 1\n\t" MX_STEP("", "", "", "")
                 : MX_ACC, MX_NEXT(nx)
                 : MX_CUR(f, sc), MX_READS(OFF), MX_DMA_IN
                 : "memory", "scc");
#undef MX_SEL
  } else {
#define MX_SEL "op_sel:[0,0,0] op_sel_hi:[1,1,0]"
    asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 1\n\t" MX_STEP("", "", "", "")
                 "\n\ts_mov_b32 m0, %[ms]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[vs], off"
                 : MX_ACC, MX_NEXT(nx)
                 : MX_CUR(f, sc), MX_READS(OFF), MX_DMA_IN, [ms] "s"(ms), [vs] "v"(vs)
                 : "memory", "scc");
#undef MX_SEL
  }
}

// Second step of a stage: once the next stage has landed for every wave (the two after it may be
// under way) and this one's reads are done, reads the next stage's first fragments at OFF (after an
// odd stage also the next group's scales at SOFF) and fetches the first half of the stage four
// further on into this one's place.
template <int ODD, int OFF, int SOFF>
__device__ inline void mx_step1(f32x16 (&acc)[4][4], const MxFrags& f, MxFrags& nx, const MxScales& sc,
                                MxScales& nsc, uint32_t bw, uint32_t ba, uint32_t sbw, uint32_t sba,
                                const char* const* g, uint32_t m, uint32_t v) {
  if constexpr (!ODD) {
#define MX_SEL "op_sel:[1,1,0] op_sel_hi:[0,0,0]"
    asm volatile("s_mov_b32 m0, %[m]\n\ts_waitcnt vmcnt(17)\n\ts_barrier\n\t" MX_STEP("", "", "", "")
                 : MX_ACC, MX_NEXT(nx)
                 : MX_CUR(f, sc), MX_READS(OFF), MX_DMA_IN
                 : "memory", "scc");
#undef MX_SEL
  } else {
#define MX_SEL "op_sel:[1,1,0] op_sel_hi:[1,1,0]"
    asm volatile("s_mov_b32 m0, %[m]\n\ts_waitcnt vmcnt(17)\n\ts_barrier\n\t" MX_STEP(
                     MX_RS("n0", "sbw", "t0") MX_RS("n1", "sbw", "t1"),
                     MX_RS("n2", "sbw", "t2") MX_RS("n3", "sbw", "t3"),
                     MX_RS("r0", "sba", "t0") MX_RS("r1", "sba", "t1"),
                     MX_RS("r2", "sba", "t2") MX_RS("r3", "sba", "t3"))
                 : MX_ACC, MX_NEXT(nx), [n0] "=&v"(nsc.w[0]), [n1] "=&v"(nsc.w[1]), [n2] "=&v"(nsc.w[2]),
                   [n3] "=&v"(nsc.w[3]), [r0] "=&v"(nsc.a[0]), [r1] "=&v"(nsc.a[1]), [r2] "=&v"(nsc.a[2]),
                   [r3] "=&v"(nsc.a[3])
                 : MX_CUR(f, sc), MX_READS(OFF), MX_DMA_IN, [sbw] "v"(sbw), [sba] "v"(sba), [t0] "n"(SOFF),
                   [t1] "n"(SOFF + 256), [t2] "n"(SOFF + 512), [t3] "n"(SOFF + 768)
                 : "memory", "scc");
#undef MX_SEL
  }
}
#undef MX_DMA_IN

// Work-groups stay for many tiles.  The DMA runs four stages ahead of the
// products as one stream over all of them, so a tile's first stages are loaded
// under the last products and the epilogue of the one before; the epilogue has
// LDS of its own (4 KB a wave).
template <typename T, bool GELU, bool VEC>
__global__ __launch_bounds__(256, 1) void mx_big_kernel(MxMat a, MxMat w, const uint16_t* __restrict__ bias,
                                                        uint16_t* __restrict__ out, long long ldo,
                                                        int groups, int mt, int nt, int per_xcd) {
  using C = MxTile<4, 4>;
  constexpr int ST = C::STAGE, PAIR = 2 * ST;
  static_assert(ST + 8192 < 65536 && C::CODES + 1024 < 65536, "LDS offsets of 16 bits");
  __shared__ __attribute__((aligned(1024))) char lds[4 * ST + 4 * 4096];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 1, wm = wave >> 1;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(mx_lds_t*)lds, l16 = lane * 16;
  const int n = 2 * groups, step = gridDim.x >> 3;
  int id = mx_first(per_xcd);
  const int end = mx_end(mt, nt, per_xcd);
  if (id >= end) return;

  // the stream of stages: tile ld, its stage ls
  MxDma d;
  int ld = id, ls = 0;
  auto aim = [&]() {
    int m0, n0;
    mx_place(ld, mt, nt, 8, 8, m0, n0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rb = wave * 4 + (i >> 1);
      const long long row = rb < 8 ? min(n0 + rb, w.blocks - 1) : min(m0 + rb - 8, a.blocks - 1);
      d.g[i] = (rb < 8 ? w.codes : a.codes) + row * groups * 4096 + (i & 1) * 1024;
    }
    const int rb = 4 * wave + (lane >> 4);
    const long long row = rb < 8 ? min(n0 + rb, w.blocks - 1) : min(m0 + rb - 8, a.blocks - 1);
    d.scales = (const char*)(rb < 8 ? w.scales : a.scales) + row * groups * 256 + (lane & 15) * 16;
  };
  // column offset of stage ls (+ 1); after the last tile every lane reads one line of its last
  // stage, so that the counts of loads in flight stay what they are
  auto col = [&](int odd) { return (uint32_t)(ls + odd) * 2048 + (ld < end ? l16 : 0); };
  auto next_pair = [&]() {
    if (ld >= end) return;
    ls += 2;
    if (ls < n) return;
    ld += step;
    if (ld < end) {
      ls = 0;
      aim();
    } else {
      ls = n - 2;
    }
  };
  const uint32_t dst = lds0 + wave * 8192, sdst = lds0 + C::CODES + wave * 1024;
  auto issue = [&](uint32_t off, int i) {  // KB i of a pair
    asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %[v], %[g]" ::[m] "s"(
                     dst + off + (i >> 3) * ST + (i & 7) * 1024),
                 [v] "v"(col(i >> 3)), [g] "s"(d.g[i & 7])
                 : "memory");
    if (i == 7)  // in the order of the steps: the scales after the even stage
      asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[v], off" ::[m] "s"(sdst + off),
                   [v] "v"(d.scales + (size_t)ls * 128)
                   : "memory");
  };
  // two pairs but for the last half stage, which the first step fetches
  aim();
#pragma unroll
  for (int i = 0; i < 16; ++i) issue(0, i);
  next_pair();
#pragma unroll
  for (int i = 0; i < 12; ++i) issue(PAIR, i);
  // fragment and scale addresses of the pair in use and of the other one
  uint32_t bw = lds0 + wn * 8192 + l16, ba = lds0 + 16384 + wm * 8192 + l16;
  uint32_t sw = lds0 + wn * 1024 + lane * 4, sa = lds0 + 2048 + wm * 1024 + lane * 4;
  uint32_t off = 0;
  MxFrags f0, f1;
  MxScales sc, nsc;
  asm volatile("s_waitcnt vmcnt(13)\n\ts_barrier\n\t" MX_R("x0", "bw", "o0") MX_R("y0", "ba", "o0")
               MX_R("x1", "bw", "o1") MX_R("y1", "ba", "o1") MX_R("x2", "bw", "o2") MX_R("y2", "ba", "o2")
               MX_R("x3", "bw", "o3") MX_R("y3", "ba", "o3") MX_RS("n0", "sbw", "t0") MX_RS("n1", "sbw", "t1")
               MX_RS("n2", "sbw", "t2") MX_RS("n3", "sbw", "t3") MX_RS("r0", "sba", "t0")
               MX_RS("r1", "sba", "t1") MX_RS("r2", "sba", "t2") MX_RS("r3", "sba", "t3")
               "s_waitcnt lgkmcnt(0)"
               : MX_NEXT(f0), [n0] "=&v"(sc.w[0]), [n1] "=&v"(sc.w[1]), [n2] "=&v"(sc.w[2]),
                 [n3] "=&v"(sc.w[3]), [r0] "=&v"(sc.a[0]), [r1] "=&v"(sc.a[1]), [r2] "=&v"(sc.a[2]),
                 [r3] "=&v"(sc.a[3])
               : MX_READS(0), [sbw] "v"(sw), [sba] "v"(sa), [t0] "n"(C::CODES), [t1] "n"(C::CODES + 256),
                 [t2] "n"(C::CODES + 512), [t3] "n"(C::CODES + 768)
               : "memory");
  char* own = lds + 4 * ST + wave * 4096;
  f32x16 acc[4][4];
  for (;;) {
    int m0, n0;
    mx_place(id, mt, nt, 8, 8, m0, n0);
    mx_start<T>(acc, bias, (float*)own, (n0 + wn * 4) * 32, w.rows);
    for (int g = groups; g > 0; --g) {
      const uint32_t other = PAIR - 2 * off;  // from this pair to the other one (off: 0 or PAIR)
      mx_step0<0, 1024>(acc, f0, f1, sc, bw, ba, d.g + 4, dst + PAIR - off + ST + 4096, col(1), 0, nullptr);
      next_pair();
      mx_step1<0, ST, 0>(acc, f1, f0, sc, nsc, bw, ba, sw, sa, d.g, dst + off, col(0));
      mx_step0<1, ST + 1024>(acc, f0, f1, sc, bw, ba, d.g + 4, dst + off + 4096, col(0), sdst + off,
                             d.scales + (size_t)ls * 128);
      const uint32_t o_bw = bw + other, o_ba = ba + other, o_sw = sw + other, o_sa = sa + other;
      mx_step1<1, 0, C::CODES>(acc, f1, f0, sc, nsc, o_bw, o_ba, o_sw, o_sa, d.g, dst + off + ST, col(1));
      sc = nsc;
      bw = o_bw, ba = o_ba, sw = o_sw, sa = o_sa, off = PAIR - off;
    }
    // the last products' registers are readable after 18 cycles of issue
    asm volatile("s_nop 15\n\ts_nop 15" : MX_ACC);
    mx_store<T, 4, 4, GELU, VEC>(acc, own, out, ldo, (m0 + wm * 4) * 32, a.rows, (n0 + wn * 4) * 32, w.rows);
    id += step;
    if (id >= end) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- the 128 x 128 tile ------------------------------------------------------
// The same with a whole stage a step: eight products, the next stage's eight
// fragment reads and the DMA of the stage four further on.  Bound by LDS: at 128
// bytes a cycle a stage's reads (32 KB) and the DMA's writes (18 KB) take 400
// cycles, its products 256.  Two work-groups fit a CU; eight stages instead
// (one work-group a CU) gained nothing at 512 x 5120 x 5120 (11.5 and 12.3 us;
// 17.0 with the compiler's schedule).
#define MX_Q(c, i, j, SEL)                                                                              \
  "v_mfma_scale_f32_32x32x64_f8f6f4 %[c" #i #j "], %[w" #c #i "], %[a" #c #j "], %[c" #i #j           \
  "], %[p" #i "], %[q" #j "] " SEL " cbsz:4 blgp:4\n\t"
#define MX_MID_STEP(S0, S1, X)                                                                          \
  "s_mov_b32 m0, %[m]\n\ts_waitcnt vmcnt(9)\n\ts_barrier\n\t" MX_Q(0, 0, 0, S0) MX_R("x00", "bw", "o0") \
      MX_R("y00", "ba", "o0") MX_Q(0, 0, 1, S0) MX_R("x01", "bw", "o1") MX_R("y01", "ba", "o1")         \
          MX_Q(0, 1, 1, S0) MX_D(0) MX_R("x10", "bw", "o2") MX_Q(0, 1, 0, S0) MX_R("y10", "ba", "o2")   \
              MX_D(1) MX_Q(1, 0, 0, S1) MX_R("x11", "bw", "o3") MX_R("y11", "ba", "o3") X               \
                  MX_Q(1, 0, 1, S1) MX_D(2) MX_Q(1, 1, 1, S1) MX_D(3) MX_Q(1, 1, 0, S1)
struct MxMidFrags {
  u32x4 w[2][2], a[2][2];  // [fragment of the stage][block]
};
struct MxMidScales {
  uint32_t w[2], a[2];
};
// OFF: where the next stage lies; after an odd stage its scales are read too (SOFF), with an even
// one the DMA fetches scales
template <int ODD, int OFF, int SOFF>
__device__ inline void mx_mid_step(f32x16 (&acc)[2][2], const MxMidFrags& f, MxMidFrags& nx,
                                   const MxMidScales& sc, MxMidScales& nsc, uint32_t bw, uint32_t ba,
                                   uint32_t sbw, uint32_t sba, const char* const (&g)[4], uint32_t m, uint32_t v,
                                   uint32_t ms, const char* vs) {
#define MX_MID_OUT                                                                                      \
  [c00] "+v"(acc[0][0]), [c01] "+v"(acc[0][1]), [c10] "+v"(acc[1][0]), [c11] "+v"(acc[1][1]),           \
      [x00] "=&v"(nx.w[0][0]), [x01] "=&v"(nx.w[0][1]), [x10] "=&v"(nx.w[1][0]), [x11] "=&v"(nx.w[1][1]), \
      [y00] "=&v"(nx.a[0][0]), [y01] "=&v"(nx.a[0][1]), [y10] "=&v"(nx.a[1][0]), [y11] "=&v"(nx.a[1][1])
#define MX_MID_IN                                                                                       \
  [w00] "v"(f.w[0][0]), [w01] "v"(f.w[0][1]), [w10] "v"(f.w[1][0]), [w11] "v"(f.w[1][1]),               \
      [a00] "v"(f.a[0][0]), [a01] "v"(f.a[0][1]), [a10] "v"(f.a[1][0]), [a11] "v"(f.a[1][1]),           \
      [p0] "v"(sc.w[0]), [p1] "v"(sc.w[1]), [q0] "v"(sc.a[0]), [q1] "v"(sc.a[1]), [bw] "v"(bw),         \
      [ba] "v"(ba), [o0] "n"(OFF), [o1] "n"(OFF + 2048), [o2] "n"(OFF + 1024), [o3] "n"(OFF + 3 * 1024),    \
      [m] "s"(m), [v] "v"(v), [g0] "s"(g[0]), [g1] "s"(g[1]), [g2] "s"(g[2]), [g3] "s"(g[3])
  if constexpr (!ODD)
    asm volatile(MX_MID_STEP("op_sel:[0,0,0] op_sel_hi:[0,0,0]", "op_sel:[1,1,0] op_sel_hi:[0,0,0]", "")
                 "s_mov_b32 m0, %[ms]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[vs], off\n\ts_waitcnt lgkmcnt(0)"
                 : MX_MID_OUT
                 : MX_MID_IN, [ms] "s"(ms), [vs] "v"(vs)
                 : "memory", "scc");
  else
    asm volatile(MX_MID_STEP("op_sel:[0,0,0] op_sel_hi:[1,1,0]", "op_sel:[1,1,0] op_sel_hi:[1,1,0]",
                             MX_RS("n0", "sbw", "t0") MX_RS("n1", "sbw", "t1") MX_RS("r0", "sba", "t0")
                                 MX_RS("r1", "sba", "t1")) "s_waitcnt lgkmcnt(0)"
                 : MX_MID_OUT, [n0] "=&v"(nsc.w[0]), [n1] "=&v"(nsc.w[1]), [r0] "=&v"(nsc.a[0]),
                   [r1] "=&v"(nsc.a[1])
                 : MX_MID_IN, [sbw] "v"(sbw), [sba] "v"(sba), [t0] "n"(SOFF), [t1] "n"(SOFF + 256)
                 : "memory", "scc");
#undef MX_MID_OUT
#undef MX_MID_IN
}

template <typename T, bool GELU, bool VEC>
__global__ __launch_bounds__(256, 2) void mx_mid_kernel(MxMat a, MxMat w, const uint16_t* __restrict__ bias,
                                                        uint16_t* __restrict__ out, long long ldo, int groups,
                                                        int mt, int nt, int per_xcd) {
  using C = MxTile<2, 2>;
  constexpr int ST = C::STAGE, PAIR = 2 * ST;
  __shared__ __attribute__((aligned(1024))) char lds[4 * ST];
  __shared__ __attribute__((aligned(16))) float sbias[4][64];
  const int id = mx_first(per_xcd);
  if (id >= mx_end(mt, nt, per_xcd)) return;
  int m0, n0;
  mx_place(id, mt, nt, 4, 4, m0, n0);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 1, wm = wave >> 1, n = 2 * groups;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(mx_lds_t*)lds, l16 = lane * 16;
  const char* g[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rb = wave * 2 + (i >> 1);
    const long long row = rb < 4 ? min(n0 + rb, w.blocks - 1) : min(m0 + rb - 4, a.blocks - 1);
    g[i] = (rb < 4 ? w.codes : a.codes) + row * groups * 4096 + (i & 1) * 1024;
  }
  // 1 KB of scales, four row blocks; waves 0 and 2, 1 and 3 fetch the same
  const int srb = 4 * wn + (lane >> 4);
  const long long srow = srb < 4 ? min(n0 + srb, w.blocks - 1) : min(m0 + srb - 4, a.blocks - 1);
  const char* gs = (const char*)(srb < 4 ? w.scales : a.scales) + srow * groups * 256 + (lane & 15) * 16;
  const uint32_t dst = lds0 + wave * 4096, sdst = lds0 + C::CODES + wn * 1024;
  // past the last stage every lane reads one line of it, so that the counts of loads in flight stay
  auto col = [&](int s) { return (uint32_t)min(s, n - 2 + (s & 1)) * 2048 + (s < n ? l16 : 0); };
  auto scol = [&](int s) { return gs + (size_t)(min(s, n - 2) >> 1) * 256; };
#pragma unroll
  for (int s = 0; s < 4; ++s) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %[v], %[g]" ::[m] "s"(
                       dst + s * ST + i * 1024),
                   [v] "v"(col(s)), [g] "s"(g[i])
                   : "memory");
    if (!(s & 1))
      asm volatile("s_mov_b32 m0, %[m]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[v], off" ::[m] "s"(sdst + s * ST),
                   [v] "v"(scol(s))
                   : "memory");
  }
  f32x16 acc[2][2];
  mx_start<T>(acc, bias, sbias[wave], (n0 + wn * 2) * 32, w.rows);
  uint32_t bw = lds0 + wn * 4096 + l16, ba = lds0 + 8192 + wm * 4096 + l16;
  uint32_t sw = lds0 + wn * 512 + lane * 4, sa = lds0 + 1024 + wm * 512 + lane * 4;
  uint32_t off = 0;
  MxMidFrags f0, f1;
  MxMidScales sc, nsc;
  asm volatile("s_waitcnt vmcnt(13)\n\ts_barrier\n\t" MX_R("x00", "bw", "o0") MX_R("x01", "bw", "o1")
               MX_R("x10", "bw", "o2") MX_R("x11", "bw", "o3") MX_R("y00", "ba", "o0") MX_R("y01", "ba", "o1")
               MX_R("y10", "ba", "o2") MX_R("y11", "ba", "o3") MX_RS("n0", "sbw", "t0") MX_RS("n1", "sbw", "t1")
               MX_RS("r0", "sba", "t0") MX_RS("r1", "sba", "t1") "s_waitcnt lgkmcnt(0)"
               : [x00] "=&v"(f0.w[0][0]), [x01] "=&v"(f0.w[0][1]), [x10] "=&v"(f0.w[1][0]),
                 [x11] "=&v"(f0.w[1][1]), [y00] "=&v"(f0.a[0][0]), [y01] "=&v"(f0.a[0][1]),
                 [y10] "=&v"(f0.a[1][0]), [y11] "=&v"(f0.a[1][1]), [n0] "=&v"(sc.w[0]), [n1] "=&v"(sc.w[1]),
                 [r0] "=&v"(sc.a[0]), [r1] "=&v"(sc.a[1])
               : [bw] "v"(bw), [ba] "v"(ba), [o0] "n"(0), [o1] "n"(2048), [o2] "n"(1024), [o3] "n"(3 * 1024),
                 [sbw] "v"(sw), [sba] "v"(sa), [t0] "n"(C::CODES), [t1] "n"(C::CODES + 256)
               : "memory");
  for (int s = 0; s < n; s += 2) {
    const uint32_t other = PAIR - 2 * off;  // from this pair of stages to the other one
    mx_mid_step<0, ST, 0>(acc, f0, f1, sc, nsc, bw, ba, sw, sa, g, dst + off, col(s + 4), sdst + off,
                          scol(s + 4));
    const uint32_t o_bw = bw + other, o_ba = ba + other, o_sw = sw + other, o_sa = sa + other;
    mx_mid_step<1, 0, C::CODES>(acc, f1, f0, sc, nsc, o_bw, o_ba, o_sw, o_sa, g, dst + off + ST, col(s + 5), 0,
                                nullptr);
    sc = nsc;
    bw = o_bw, ba = o_ba, sw = o_sw, sa = o_sa, off = PAIR - off;
  }
  // every load has landed and every wave's reads are done: LDS is free; the products' registers are
  // readable
  asm volatile("s_nop 15\n\ts_nop 15\n\ts_waitcnt vmcnt(0)\n\ts_barrier"
               : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1])
               :
               : "memory");
  char* own = lds + wave * 4096;
  mx_store<T, 2, 2, GELU, VEC>(acc, own, out, ldo, (m0 + wm * 2) * 32, a.rows, (n0 + wn * 2) * 32, w.rows);
}

// ---- small launches: the columns split over the waves ------------------------
// 32 features x 32 tokens a work-group; its eight waves take units of 128 columns
// in turn, so every fragment is loaded once, straight into registers (no staging,
// no barrier in the loop), DEPTH units ahead.  The waves' sums meet in LDS, in
// the order of the waves.  With X16 the tokens come in 16 bits and every
// work-group quantises them into LDS first (MX_X16_BLOCKS blocks at most), under
// the loads of its first weights, in the place of a launch before this one.
// Bound: one round of loads and the exchange (1 x 5120 x 5120, 160 work-groups for
// 256 CUs: 5.3 us, with X16 5.4, against 2.7 more for a launch that quantises); with
// more tokens the bytes from L2, which every 32 x 32 block reads for itself.
#define MX_X16_BLOCKS 2048
struct MxSrc {
  MxMat m;            // in MXFP4 (its row count in either case), or
  const uint16_t* x;  // in 16 bits
  long long stride;
  int K;
};

template <typename T, int DEPTH, bool GELU, bool X16>
__global__ __launch_bounds__(512) void mx_split_kernel(MxSrc a, MxMat w, const uint16_t* __restrict__ bias,
                                                       uint16_t* __restrict__ out, long long ldo, int groups,
                                                       int mt, int nt, int per_xcd) {
  constexpr int WAVES = 8;
  __shared__ f32x4 part[WAVES][4][64];
  __shared__ u32x4 xc[X16 ? MX_X16_BLOCKS : 1];
  __shared__ uint8_t xs[X16 ? MX_X16_BLOCKS : 1];
  const int id = mx_first(per_xcd);
  if (id >= mx_end(mt, nt, per_xcd)) return;
  int mb, nb;
  mx_place(id, mt, nt, 1, 1, mb, nb);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = 2 * groups;
  const char* pw = w.codes + (long long)nb * groups * 4096;
  const uint32_t* qw = w.scales + (long long)nb * groups * 64;
  const char* pa = X16 ? nullptr : a.m.codes + (long long)mb * groups * 4096;
  const uint32_t* qa = X16 ? nullptr : a.m.scales + (long long)mb * groups * 64;
  const int row = mb * 32 + (lane & 31);
  struct Unit {
    u32x4 w[2], a[2];
    uint32_t sw, sa;
  };
  auto load = [&](int s, Unit& t) {
    const size_t o = (size_t)s * 2048 + lane * 16, os = (size_t)(s >> 1) * 64 + lane;
    const int sh = 16 * (s & 1);  // an odd unit's scales are the upper half
    t.w[0] = *(const u32x4*)(pw + o);
    t.w[1] = *(const u32x4*)(pw + o + 1024);
    t.sw = qw[os] >> sh;
    if constexpr (!X16) {
      t.a[0] = *(const u32x4*)(pa + o);
      t.a[1] = *(const u32x4*)(pa + o + 1024);
      t.sa = qa[os] >> sh;
    }
  };
  // X16: block b of row r at r 8 groups + b
  auto fetch = [&](int s, Unit& t) {
    const int b = row * 8 * groups + 4 * s + (lane >> 5);
    t.a[0] = t.a[1] = u32x4{0u, 0u, 0u, 0u};
    t.sa = 0;
    if (row < a.m.rows) {
      t.a[0] = xc[b], t.a[1] = xc[b + 2];
      t.sa = xs[b] | (xs[b + 2] << 8);
    }
  };
  f32x16 acc = zero16();
  Unit ring[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (wave + d * WAVES < n) load(wave + d * WAVES, ring[d]);
  if constexpr (X16) {
    for (int b = threadIdx.x; b < a.m.rows * 8 * groups; b += 64 * WAVES) {
      const int r = b / (8 * groups), c = 32 * (b - r * 8 * groups);
      u32x4 v[4], codes{0u, 0u, 0u, 0u};
      uint32_t byte = 0;
      if (c < a.K) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *(const u32x4*)(a.x + r * a.stride + c + 8 * i);
        mx_block<T>(v, codes, byte);
      }
      xc[b] = codes;
      xs[b] = (uint8_t)byte;
    }
    __syncthreads();
  }
  for (int s = wave; s < n; s += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      Unit& t = ring[d];
      if (s + d * WAVES < n) {
        if constexpr (X16) fetch(s + d * WAVES, t);
        acc = mx_mfma<0>(t.w[0], t.a[0], acc, t.sw, t.sa);
        acc = mx_mfma<1>(t.w[1], t.a[1], acc, t.sw, t.sa);
      }
      if (s + (d + DEPTH) * WAVES < n) load(s + (d + DEPTH) * WAVES, t);
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    part[wave][q][lane] = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  if (wave >= 4) return;
  // quarter q: four features of each token
  const int q = wave, f = nb * 32 + 8 * q + 4 * (lane >> 5);
  f32x4 v = part[0][q][lane];
#pragma unroll
  for (int x = 1; x < WAVES; ++x) {
    const f32x4 y = part[x][q][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += y[e];
  }
  if (row < a.m.rows && f < w.rows) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (bias) v[e] += T::to_f(bias[min(f + e, w.rows - 1)]);
      if (GELU) v[e] = mx_gelu(v[e]);
    }
    mx_put(out + row * ldo + f, u32x2{Pk<T>::pack(v[0], v[1]), Pk<T>::pack(v[2], v[3])}, w.rows - f);
  }
}

template <typename T, int DEPTH, bool X16>
static int mx_split_launch(const MxSrc& a, const MxMat& w, const uint16_t* bias, int act, uint16_t* out,
                           long long ldo, int groups, hipStream_t st) {
  const long long tiles = (long long)a.m.blocks * w.blocks;
  const int per = cdiv(tiles, 8);
  if (per > (1 << 19)) {  // 2^31 threads
    t2t_set_error("mxfp4_product: M=%d N=%d", a.m.rows, w.rows);
    return T2T_ERR_UNSUPPORTED;
  }
  auto kernel =
      act == T2T_ACT_GELU_TANH ? mx_split_kernel<T, DEPTH, true, X16> : mx_split_kernel<T, DEPTH, false, X16>;
  hipLaunchKernelGGL(kernel, dim3(8 * per), dim3(512), 0, st, a, w, bias, out, ldo, groups, a.m.blocks,
                     w.blocks, per);
  T2T_LAUNCH_CHECK("mxfp4_product");
  return T2T_OK;
}

// tiles of 64 TW x 64 TA
template <typename T, int TW, int TA>
static int mx_tile_launch(const MxMat& a, const MxMat& w, const uint16_t* bias, int act, uint16_t* out,
                          long long ldo, int groups, hipStream_t st) {
  const int mt = cdiv(a.blocks, 2 * TA), nt = cdiv(w.blocks, 2 * TW);
  const long long tiles = (long long)mt * nt;
  if (tiles > (1 << 23)) {  // 2^31 threads of 128 x 128 tiles; as many large ones are a TB of outputs
    t2t_set_error("mxfp4_product: M=%d N=%d", a.rows, w.rows);
    return T2T_ERR_UNSUPPORTED;
  }
  const int per = cdiv(tiles, 8);
  auto launch = [&](auto kernel, int slots) {
    hipLaunchKernelGGL(kernel, dim3(8 * slots), dim3(256), 0, st, a, w, bias, out, ldo, groups, mt, nt, per);
  };
  auto form = [&](auto G, auto V) {
    constexpr bool GELU = decltype(G)::value, VEC = decltype(V)::value;
    if constexpr (TW == 4)  // fills a CU: 32 work-groups an XCD, which go through the tiles
      launch(mx_big_kernel<T, GELU, VEC>, per < 32 ? per : 32);
    else
      launch(mx_mid_kernel<T, GELU, VEC>, per);
  };
  const bool gelu = act == T2T_ACT_GELU_TANH;
  const bool vec = w.rows % 8 == 0 && ldo % 8 == 0 && (uintptr_t)out % 16 == 0;
  if (gelu)
    vec ? form(std::true_type{}, std::true_type{}) : form(std::true_type{}, std::false_type{});
  else
    vec ? form(std::false_type{}, std::true_type{}) : form(std::false_type{}, std::false_type{});
  T2T_LAUNCH_CHECK("mxfp4_product");
  return T2T_OK;
}

// Which product: by the number of outputs.  Below 512 blocks of 32 x 32 too few tiles would go through
// all of K one stage after another (64 x 5120 x 5120: split 7.6 us, 128 x 128 tiles 10.6; 128 x 5120 x
// 5120: 10.7 and 10.8; 256 x: 15.8 and 11.0).  From 256 large tiles on they fill the chip (4096^3: 37.4
// us, 128 x 128 tiles 38.4; 1500 x 5120 x 5120, 120 large tiles: 33.3 and 25.9), unless K is short and
// they are few (9000 x 2048 x 512: 20.4 and 15.8; 75,600 x 5120 x 128: 172 and 208) or they would be
// padded by more than a quarter over the small ones (75,600 x 96 x 1536: 34.1 and 17.7).  Rounds of 256
// work-groups are not counted, which loses where the second holds few tiles (K = 4096, 289 of them: 52.7
// and 42.5; 324: 51.9 and 50.3; 400: 55.6 and 58.5; 504: 62.2 and 69.8; 576: 83.2 and 78.8).
template <typename T>
static int mx_product(const MxMat& a, const MxMat& w, const uint16_t* bias, int act, uint16_t* out,
                      long long ldo, int groups, hipStream_t st) {
  const long long big = (long long)cdiv(a.blocks, 8) * cdiv(w.blocks, 8);
  const long long mid = (long long)cdiv(a.blocks, 4) * cdiv(w.blocks, 4);
  if ((long long)a.blocks * w.blocks <= 512)
    return mx_split_launch<T, 4, false>(MxSrc{a, nullptr, 0, 0}, w, bias, act, out, ldo, groups, st);
  if (big >= 256 && (groups >= 4 || big >= 1024) && 4 * big <= mid + mid / 4)
    return mx_tile_launch<T, 4, 4>(a, w, bias, act, out, ldo, groups, st);
  return mx_tile_launch<T, 2, 2>(a, w, bias, act, out, ldo, groups, st);
}

static int mx_check_product(const char* what, const void* a_codes, const void* a_scales,
                            const void* w_codes, const void* w_scales, int act, const void* out, int dtype,
                            long long out_row_stride, int M, int N, int K) {
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "%s: dtype %d", what, dtype);
  T2T_REQUIRE(act == T2T_ACT_NONE || act == T2T_ACT_GELU_TANH, "%s: activation %d", what, act);
  T2T_REQUIRE(M >= 0 && M <= (1 << 30) && N >= 1 && N <= (1 << 30) && K >= 32 && K % 32 == 0 && K <= (1 << 27),
              "%s: M=%d N=%d K=%d (M, N <= 2^30, K a multiple of 32, K <= 2^27)", what, M, N, K);
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
  const int groups = mx_kp(K) / 256;
  if (dtype == T2T_BF16)
    return mx_product<BF16T>(a, w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, groups,
                             (hipStream_t)stream);
  return mx_product<F16T>(a, w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, groups,
                          (hipStream_t)stream);
}

// Few rows are quantised by the product itself, as far as its LDS holds them: every work-group does it
// again, which costs what the saved launch gains at 12 x 5120 (8.2 us either way; 1 x: 5.4 and 8.0).
static bool mx_few(int M, int K) { return M <= 32 && (long long)M * (mx_kp(K) / 32) <= MX_X16_BLOCKS; }

// codes, then scales
extern "C" size_t t2t_mxfp4_linear_ws_bytes(int M, int N, int K) {
  (void)N;
  return mx_few(M, K) ? 0 : t2t_align256(t2t_mxfp4_code_bytes(M, K)) + t2t_mxfp4_scale_bytes(M, K);
}

extern "C" int t2t_mxfp4_linear(const void* x, int dtype, long long x_row_stride, const void* w_codes,
                                const void* w_scales, const void* bias, int act, void* out,
                                long long out_row_stride, int M, int N, int K, void* ws, size_t ws_bytes,
                                void* stream) {
  // everything before the first launch
  int rc = mx_check_product("mxfp4_linear", x, x, w_codes, w_scales, act, out, dtype, out_row_stride, M, N, K);
  if (rc == T2T_OK) rc = mx_check_rows("mxfp4_linear", x, dtype, x_row_stride, w_codes, w_scales, M, K);
  if (rc != T2T_OK || M == 0) return rc;
  if (mx_few(M, K)) {
    const MxSrc a{MxMat{nullptr, nullptr, M, (int)mx_row_blocks(M)}, (const uint16_t*)x, x_row_stride, K};
    const MxMat w{(const char*)w_codes, (const uint32_t*)w_scales, N, (int)mx_row_blocks(N)};
    auto run = dtype == T2T_BF16 ? mx_split_launch<BF16T, 2, true> : mx_split_launch<F16T, 2, true>;
    return run(a, w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, mx_kp(K) / 256,
               (hipStream_t)stream);
  }
  if (!ws || ws_bytes < t2t_mxfp4_linear_ws_bytes(M, N, K)) {
    t2t_set_error("mxfp4_linear: workspace %zu < %zu bytes", ws ? ws_bytes : (size_t)0,
                  t2t_mxfp4_linear_ws_bytes(M, N, K));
    return T2T_ERR_WORKSPACE;
  }
  T2T_REQUIRE((uintptr_t)ws % 16 == 0, "mxfp4_linear: workspace must be 16-byte aligned");
  char* scales = (char*)ws + t2t_align256(t2t_mxfp4_code_bytes(M, K));
  rc = t2t_mxfp4_quantize(x, dtype, x_row_stride, ws, scales, M, K, stream);
  if (rc != T2T_OK) return rc;
  return t2t_mxfp4_product(ws, scales, w_codes, w_scales, bias, act, out, dtype, out_row_stride, M, N, K,
                           stream);
}
