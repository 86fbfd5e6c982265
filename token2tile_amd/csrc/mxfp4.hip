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
  static constexpr int PITCH = 64 * TW + 16;        // a token's staged outputs (bytes)
  static constexpr int SCALES = RB * 256;
  static constexpr int STAGE = CODES + SCALES > 4 * 32 * PITCH ? CODES + SCALES : 4 * 32 * PITCH;
};

template <typename T, int TW, int TA, bool GELU>
__global__ __launch_bounds__(256, TW * TA >= 16 ? 1 : 2) void mx_tile_kernel(
    MxMat a, MxMat w, const uint16_t* __restrict__ bias, uint16_t* __restrict__ out, long long ldo, int vec,
    int groups, int mt, int nt, int per_xcd) {
  using C = MxTile<TW, TA>;
  __shared__ __attribute__((aligned(1024))) char st0[C::STAGE];
  __shared__ __attribute__((aligned(1024))) char st1[C::STAGE];
  __shared__ __attribute__((aligned(1024))) char st2[C::STAGE];
  __shared__ __attribute__((aligned(1024))) char st3[C::STAGE];
  // consecutive work-groups go to the eight XCDs in turn: each takes a run of
  // tiles, eight token tiles by all feature tiles, so that the 32 tiles an XCD
  // has under way share their panels in its L2
  const int id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (id >= mt * nt) return;
  const int grp = id / (8 * nt), in = id - grp * 8 * nt;
  const int gm = min(8, mt - grp * 8);
  const int m0 = (grp * 8 + in % gm) * 2 * TA, n0 = (in / gm) * 2 * TW;  // row blocks

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 1, wm = wave >> 1, hh = lane >> 5;
  // this wave's share of the stage's DMA: TW + TA KB of codes, and 1 KB of scales (four row
  // blocks; with fewer than sixteen some waves fetch the same)
  const char* src[TW + TA];
#pragma unroll
  for (int i = 0; i < TW + TA; ++i) {
    const int q = wave * (TW + TA) + i, rb = q >> 1;
    const long long row = rb < 2 * TW ? min(n0 + rb, w.blocks - 1) : min(m0 + rb - 2 * TW, a.blocks - 1);
    src[i] = (rb < 2 * TW ? w.codes : a.codes) + row * groups * 4096 + (q & 1) * 1024;
  }
  constexpr int SI = (C::RB + 3) / 4;
  const int srb = min(4 * (wave % SI) + (lane >> 4), C::RB - 1);
  const long long srow = srb < 2 * TW ? min(n0 + srb, w.blocks - 1) : min(m0 + srb - 2 * TW, a.blocks - 1);
  const char* ssrc = (const char*)(srb < 2 * TW ? w.scales : a.scales) + srow * groups * 256 + (lane & 15) * 16;
  const int n = 2 * groups;  // stages
  // Stages past the last keep the counts of loads in flight what they are, at the price of one
  // line each: every lane reads the same 16 bytes of the last stage.
  auto issue = [&](int s, char* st, auto ODD) {
    constexpr int O = decltype(ODD)::value;
    const int t = min(s, n - 2 + O);
    const uint32_t voff = s < n ? lane * 16 : 0;
#pragma unroll
    for (int i = 0; i < TW + TA; ++i)
      __builtin_amdgcn_global_load_lds((const mx_glb_t*)(src[i] + (size_t)t * 2048 + voff),
                                       (mx_lds_t*)(st + (wave * (TW + TA) + i) * 1024), 16, 0, 0);
    if constexpr (!O)
      __builtin_amdgcn_global_load_lds((const mx_glb_t*)(ssrc + (size_t)(t >> 1) * 256),
                                       (mx_lds_t*)(st + C::CODES + (wave % SI) * 1024), 16, 0, 0);
  };
  f32x16 acc[TW][TA];
#pragma unroll
  for (int i = 0; i < TW; ++i) {
    f32x16 b0 = zero16();
    if (bias)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        b0[e] = T::to_f(bias[min((n0 + wn * TW + i) * 32 + 8 * (e >> 2) + 4 * hh + (e & 3), w.rows - 1)]);
#pragma unroll
    for (int j = 0; j < TA; ++j) acc[i][j] = b0;
  }
  u32x4 fw[2][TW], fa[2][TA];
  uint32_t sw[TW], sa[TA];
  auto frags = [&](const char* st, int c) {
#pragma unroll
    for (int i = 0; i < TW; ++i)
      fw[c][i] = *(const u32x4*)(st + ((wn * TW + i) * 2 + c) * 1024 + lane * 16);
#pragma unroll
    for (int j = 0; j < TA; ++j)
      fa[c][j] = *(const u32x4*)(st + ((2 * TW + wm * TA + j) * 2 + c) * 1024 + lane * 16);
  };
  auto mul = [&](auto S, int c) {
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
      for (int j = 0; j < TA; ++j)
        acc[i][j] = mx_mfma<decltype(S)::value>(fw[c][i], fa[c][j], acc[i][j], sw[i], sa[j]);
  };
  // one stage: its first fragments are in registers; the second ones are read under the first
  // products, the next stage's first ones under the second products
  auto stage = [&](int s, char* cur, const char* nxt, auto ODD) {
    constexpr int O = decltype(ODD)::value;
    if constexpr (!O) {
#pragma unroll
      for (int i = 0; i < TW; ++i) sw[i] = *(const uint32_t*)(cur + C::CODES + (wn * TW + i) * 256 + lane * 4);
#pragma unroll
      for (int j = 0; j < TA; ++j)
        sa[j] = *(const uint32_t*)(cur + C::CODES + (2 * TW + wm * TA + j) * 256 + lane * 4);
    }
    frags(cur, 1);
    mul(std::integral_constant<int, 2 * O>{}, 0);
    // stage s + 1 of every wave has landed and this stage's reads are done; the two stages
    // after it may still be under way
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * (TW + TA) + 1) : "memory");
    issue(s + 4, cur, ODD);
    frags(nxt, 0);
    mul(std::integral_constant<int, 2 * O + 1>{}, 1);
  };
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 1>;
  issue(0, st0, Even{});
  issue(1, st1, Odd{});
  issue(2, st2, Even{});
  issue(3, st3, Odd{});
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(3 * (TW + TA) + 1) : "memory");
  frags(st0, 0);
  for (int s = 0;; s += 4) {
    stage(s, st0, st1, Even{});
    stage(s + 1, st1, st2, Odd{});
    if (s + 2 >= n) break;
    stage(s + 2, st2, st3, Even{});
    stage(s + 3, st3, st0, Odd{});
    if (s + 4 >= n) break;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  // epilogue: 32 tokens at a time through a staging area of the wave's own, then whole rows
  char* so = st0 + wave * 32 * C::PITCH;
  constexpr int LR = 4 * TW;  // lanes per row, 8 features each
  const int f0 = (n0 + wn * TW) * 32 + (lane % LR) * 8;
  const bool whole = vec && f0 + 8 <= w.rows;
#pragma unroll
  for (int j = 0; j < TA; ++j) {
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = GELU ? mx_gelu(acc[i][j][4 * q + e]) : acc[i][j][4 * q + e];
        *(u32x2*)(so + (lane & 31) * C::PITCH + (32 * i + 8 * q + 4 * hh) * 2) =
            u32x2{Pk<T>::pack(v[0], v[1]), Pk<T>::pack(v[2], v[3])};
      }
    const int mb = (m0 + wm * TA + j) * 32;
#pragma unroll 1
    for (int t = lane / LR; t < 32 && mb + t < a.rows; t += 64 / LR) {
      const u32x4 v = *(const u32x4*)(so + t * C::PITCH + (lane % LR) * 16);
      uint16_t* o = out + (long long)(mb + t) * ldo + f0;
      if (whole)
        *(u32x4*)o = v;
      else
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (f0 + e < w.rows) o[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <typename T, int TW, int TA>
static int mx_tile_launch(const MxMat& a, const MxMat& w, const uint16_t* bias, int act, uint16_t* out,
                          long long ldo, int groups, hipStream_t st) {
  const int mt = cdiv(a.blocks, 2 * TA), nt = cdiv(w.blocks, 2 * TW);
  const long long tiles = (long long)mt * nt;
  T2T_REQUIRE(tiles <= INT_MAX / 2, "mxfp4_product: M=%d N=%d", a.rows, w.rows);
  const int per = cdiv(tiles, 8);
  const int vec = ldo % 8 == 0 && (uintptr_t)out % 16 == 0;
  if (act == T2T_ACT_GELU_TANH)
    hipLaunchKernelGGL((mx_tile_kernel<T, TW, TA, true>), dim3(8 * per), dim3(256), 0, st, a, w, bias, out,
                       ldo, vec, groups, mt, nt, per);
  else
    hipLaunchKernelGGL((mx_tile_kernel<T, TW, TA, false>), dim3(8 * per), dim3(256), 0, st, a, w, bias, out,
                       ldo, vec, groups, mt, nt, per);
  T2T_LAUNCH_CHECK("mxfp4_product");
  return T2T_OK;
}

template <typename T>
static int mx_product(const MxMat& a, const MxMat& w, const uint16_t* bias, int act, uint16_t* out,
                      long long ldo, int groups, hipStream_t st) {
  if ((long long)a.blocks * w.blocks >= 64 * 256)
    return mx_tile_launch<T, 4, 4>(a, w, bias, act, out, ldo, groups, st);
  if ((long long)a.blocks * w.blocks >= 16 * 256)
    return mx_tile_launch<T, 2, 2>(a, w, bias, act, out, ldo, groups, st);
  return mx_tile_launch<T, 1, 1>(a, w, bias, act, out, ldo, groups, st);
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
  const int groups = mx_kp(K) / 256;
  if (dtype == T2T_BF16)
    return mx_product<BF16T>(a, w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, groups,
                             (hipStream_t)stream);
  return mx_product<F16T>(a, w, (const uint16_t*)bias, act, (uint16_t*)out, out_row_stride, groups,
                          (hipStream_t)stream);
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
