// Rotary positions: the cos / sin tables of a set of positions, and the
// rotation of q and k with the RMS norm that stands before it.
#include "t2t_common.h"
#include <type_traits>

// ---------------------------------------------------------------------------
// cos[t, i] = m cos(p[t, a] f[i]), sin likewise; pair i belongs to the axis a
// with start[a] <= i < start[a + 1].  The angle is one fp64 product (a far
// position leaves no fraction in fp32) and its sine and cosine are taken in
// fp64, so the fp32 entries are off by one rounding.  A thread keeps one pair
// and goes through the positions.  75,600 x 64 entries take 15 us into the same
// buffers again, 17 into others (2.6 and 2.3 TB/s of writes).  Counted: 77 vector
// instructions an entry, 9.5 us of issue, of which the 23 in fp64 are 3; the
// others are addresses and a thread's setup for its four positions.  With the
// device library's sincos, which takes any angle, 24 us.
// ---------------------------------------------------------------------------
struct TableAxes {
  int n;
  int start[5];
};

// m sin x and m cos x by the Taylor series on [-pi/4, pi/4], to below 1e-15 (r^15, r^14), after taking
// the nearest multiple of pi/2 off in two parts; |x| < 2^51.  The coefficients are kept in scalar
// registers (left to itself the compiler moves each into vector registers at every use).
struct TableCoef {
  double s[7], c[6];
  __device__ TableCoef()
      : s{-1.0 / 1307674368000.0, 1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0, -1.0 / 5040.0,
          1.0 / 120.0, -1.0 / 6.0},
        c{-1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0, 1.0 / 40320.0, -1.0 / 720.0, 1.0 / 24.0} {
#pragma unroll
    for (int i = 0; i < 7; ++i) asm("" : "+s"(s[i]));
#pragma unroll
    for (int i = 0; i < 6; ++i) asm("" : "+s"(c[i]));
  }
};
__device__ inline void table_sincos(const TableCoef& k_, double x, double m, float& s, float& c) {
  const double k = __builtin_rint(x * 0.6366197723675814);
  double r = __builtin_fma(-k, 1.5707963267948966, x);
  r = __builtin_fma(-k, 6.123233995736766e-17, r);
  const double t = r * r;
  double u = k_.s[0], v = k_.c[0];
#pragma unroll
  for (int i = 1; i < 7; ++i) u = __builtin_fma(u, t, k_.s[i]);
#pragma unroll
  for (int i = 1; i < 6; ++i) v = __builtin_fma(v, t, k_.c[i]);
  u = __builtin_fma(u * t, r, r);
  v = __builtin_fma(__builtin_fma(v, t, -0.5), t, 1.0);
  // which is which, and the signs, after the rounding to fp32; k modulo 2^32 stands in the low bits of
  // k + 1.5 2^52 (a conversion to an integer ends at 2^31)
  const uint32_t q = (uint32_t)__builtin_bit_cast(uint64_t, k + 0x1.8p52);
  const uint32_t fu = __builtin_bit_cast(uint32_t, (float)(m * u)), fv = __builtin_bit_cast(uint32_t, (float)(m * v));
  s = __builtin_bit_cast(float, (q & 1 ? fv : fu) ^ ((q & 2) << 30));
  c = __builtin_bit_cast(float, (q & 1 ? fu : fv) ^ (((q + 1) & 2) << 30));
}

template <typename P>
__global__ __launch_bounds__(256) void rotary_table_kernel(const P* __restrict__ pos,
                                                           const double* __restrict__ freqs,
                                                           TableAxes ax, double m,
                                                           float* __restrict__ cosv,
                                                           float* __restrict__ sinv, int pairs,
                                                           long long T) {
  const int rows = pairs < 256 ? 256 / pairs : 1;  // positions a work-group takes at once
  const int r = pairs < 256 ? threadIdx.x / pairs : 0;
  if (r >= rows) return;
  const TableCoef coef;
  for (int p = pairs < 256 ? threadIdx.x - r * pairs : threadIdx.x; p < pairs; p += pairs < 256 ? pairs : 256) {
    int a = 0;
    for (int k = 1; k < ax.n; ++k) a += p >= ax.start[k];
    const double f = freqs[p];
    const long long step = (long long)gridDim.x * rows;
    for (long long t0 = (long long)blockIdx.x * rows + r; t0 < T; t0 += 4 * step) {
      P at[4];  // four positions' loads under way at once
#pragma unroll
      for (int i = 0; i < 4; ++i) at[i] = pos[min(t0 + i * step, T - 1) * ax.n + a];
      // neighbouring fp64 angles are half a radian apart from 2^51 on: these entries are NaN (a choice
      // at every entry instead of the rare second store takes 15.4 for 14.9 us)
      bool far = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long t = t0 + i * step;
        const double x = (double)at[i] * f;
        far |= !(__builtin_fabs(x) < 0x1p51);
        float s, c;
        table_sincos(coef, x, m, s, c);
        if (t < T) cosv[t * pairs + p] = c, sinv[t * pairs + p] = s;
      }
      if (far) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long t = t0 + i * step;
          if (t < T && !(__builtin_fabs((double)at[i] * f) < 0x1p51))
            cosv[t * pairs + p] = sinv[t * pairs + p] = __builtin_nanf("");
        }
      }
    }
  }
}

extern "C" int t2t_rotary_table(const void* positions, int pos_bits, long long T, int axes,
                                const int* axis_pairs, const double* freqs, double factor, float* cosv,
                                float* sinv, void* stream) {
  T2T_REQUIRE(axis_pairs, "rotary_table: null pointer");
  T2T_REQUIRE(pos_bits == 32 || pos_bits == 64, "rotary_table: positions of %d bits", pos_bits);
  T2T_REQUIRE(T >= 0 && axes >= 1 && axes <= 4, "rotary_table: T=%lld axes=%d", T, axes);
  TableAxes ax{axes, {0, 0, 0, 0, 0}};
  for (int a = 0; a < axes; ++a) {
    T2T_REQUIRE(axis_pairs[a] >= 1 && axis_pairs[a] <= 4096, "rotary_table: %d pairs on axis %d",
                axis_pairs[a], a);
    ax.start[a + 1] = ax.start[a] + axis_pairs[a];
  }
  const int pairs = ax.start[axes];
  T2T_REQUIRE(T <= LLONG_MAX / 4 / pairs, "rotary_table: T=%lld", T);
  if (T == 0) return T2T_OK;
  T2T_REQUIRE(positions && freqs && cosv && sinv, "rotary_table: null pointer");
  const long long rows = pairs < 256 ? 256 / pairs : 1, g = (T + rows - 1) / rows;
  // four positions a thread, where that leaves enough work-groups
  const long long wgs = g < 2048 ? g : (g + 3) / 4;
  const dim3 grid((unsigned)(wgs < (1 << 20) ? wgs : 1 << 20));
  if (pos_bits == 32)
    hipLaunchKernelGGL(rotary_table_kernel<int32_t>, grid, dim3(256), 0, (hipStream_t)stream,
                       (const int32_t*)positions, freqs, ax, factor, cosv, sinv, pairs, T);
  else
    hipLaunchKernelGGL(rotary_table_kernel<long long>, grid, dim3(256), 0, (hipStream_t)stream,
                       (const long long*)positions, freqs, ax, factor, cosv, sinv, pairs, T);
  T2T_LAUNCH_CHECK("rotary_table");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// y = rotate(x rsqrt(mean(x^2) + eps) w), fp32 inside, one rounding at the
// end.  Bound: one read and one write of every element (q and k of 75,600 tokens
// x 40 heads x 128: 575 us, 5.4 TB/s; one element off their alignment, pair by
// pair in the general form below, 2.5 ms; 4 tokens: 4.8 us).
//
// A head is cut into units of 2 V channels that turn together (V: 8, or 4 where
// widths, strides or addresses ask for it): with paired halves channels V u .. +
// V - 1 and R / 2 + V u .. + V - 1, else 2 V u .. + 2 V - 1; unit u reads entries
// V u .. + V - 1 of the tables in both layouts.  The lanes of a wave are units of
// heads of tokens: L lanes a head (units rounded up to a power of two), then as
// many heads as there are or fit, then tokens, where few heads leave lanes over.
// A lane's table entries are read once a token, the norm's sums run over
// neighbouring lanes, and a token's heads stay in registers (ITS of them a lane)
// between the sum and the turn, as do the token norm's weights from token to
// token: a work-group goes through many.  (One head of 64 in 75,600 tokens: 15 us,
// 73 with a token a wave; 32 + 8 heads of 96 in 20,000: 77 us.)
// ---------------------------------------------------------------------------
struct RotaryArgs {
  const float* cosv;
  const float* sinv;
  long long table_batch;  // table rows from one sequence to the next
  long long tokens;
  int N, D, R, half;
  float sign, eps;
  int units, shift;          // units of a head, log2(L)
  int hshift[2], chunks[2];  // q and k: log2 of a wave's heads, rounds of ITS that a token takes
};

// What every form below computes alike, so that a result hardly depends on the form that its call's
// shape and strides take: the turn (one product rounded, one fused), and the norm's sum, fp32 over
// each four channels of a head in their order and fp64 over these (the order differs between the forms,
// which shows only where two sums a few fp64 steps apart round to different fp32 values).
__device__ inline void rope_turn(float a, float e, float c, float s, float& y0, float& y1) {
  y0 = __builtin_fmaf(a, c, -(e * s));
  y1 = __builtin_fmaf(a, s, e * c);
}
__device__ inline double rope_sum(double v, int lanes) {  // over groups of `lanes` neighbours
  for (int d = 1; d < lanes; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ inline double rope_squares(float a, float b, float c, float d) {
  return (double)__builtin_fmaf(d, d, __builtin_fmaf(c, c, __builtin_fmaf(b, b, a * a)));
}
__device__ inline float rope_inv(double sum, double one_over_n, float eps) {
  return rsqrtf((float)(sum * one_over_n) + eps);
}

template <int V> struct RopeVec;
template <> struct RopeVec<8> {
  typedef u32x4 type;
};
template <> struct RopeVec<4> {
  typedef u32x2 type;
};
template <typename T, int V>
__device__ inline void rope_unpack(const typename RopeVec<V>::type& v, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    f[2 * i] = T::to_f((uint16_t)(v[i] & 0xffff));
    f[2 * i + 1] = T::to_f((uint16_t)(v[i] >> 16));
  }
}
template <typename T, int V>
__device__ inline typename RopeVec<V>::type rope_pack(const float (&f)[V]) {
  typename RopeVec<V>::type v;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) v[i] = Pk<T>::pack(f[2 * i], f[2 * i + 1]);
  return v;
}

// ---- into a paged cache ------------------------------------------------------
// The forms with SLOTS are those of an append: the first tensor's rows go to their slots (its out
// strides are the cache's), the second, if any, is an ordinary one, and the grid's last row of
// work-groups stores v.  Bound: one read and one write of every element (4,680 tokens of 40 heads:
// 72 us, 4.0 TB/s; 10,007 of 32 and 8, head norm, 96 of 128: 52 us, 4.8 TB/s; 68 and 43.5 on inputs just
// seen; four tokens: 4.9 us).
struct RopeSlots {
  const void* slots;
  int wide;               // 64-bit slots
  int page;
  unsigned long long all;  // slots there are
  t2t_rotary_tensor v;
  // the place of a token's row; false where it has none
  __device__ bool place(long long tok, long long out_batch, long long out_row, long long& at) const {
    const unsigned long long s = wide ? (unsigned long long)((const long long*)slots)[tok]
                                      : (unsigned long long)(long long)((const int32_t*)slots)[tok];
    if (s >= all) return false;
    // (fewer than 2^32 in nearly every cache: a division of 32 bits)
    const long long p = all >> 32 ? (long long)(s / page) : (long long)((uint32_t)s / (uint32_t)page);
    at = p * out_batch + ((long long)s - p * page) * out_row;
    return true;
  }
};
// v [T, H, D] into its slots, V channels a thread
template <int V>
__device__ inline void rope_store_v(const RopeSlots& S, long long tokens, int D) {
  const t2t_rotary_tensor& g = S.v;
  const int per_head = D / V, per = per_head * g.heads;
  const long long units = tokens * per, step = (long long)gridDim.x * 256;
  for (long long u0 = (long long)blockIdx.x * 256 + threadIdx.x; u0 < units; u0 += 4 * step) {
    typedef uint16_t vec __attribute__((ext_vector_type(V)));
    vec x[4];
    long long at[4];
    bool on[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long u = u0 + i * step;
      on[i] = u < units;
      const long long tok = on[i] ? u / per : 0;
      const int in = on[i] ? (int)(u - tok * per) : 0, h = in / per_head, c = (in - h * per_head) * V;
      on[i] = on[i] && S.place(tok, g.out_batch, g.out_row, at[i]);
      if (!on[i]) continue;
      at[i] += h * g.out_head + c;
      x[i] = *(const vec*)((const uint16_t*)g.x + tok * g.x_row + h * g.x_head + c);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (on[i]) *(vec*)((uint16_t*)g.out + at[i]) = x[i];
  }
}

// NORM as T2T_NORM_*.  WPT waves to a token: 1, or 4 under the token norm where the tokens are few
// or a wave's registers do not hold their heads.
template <typename T, int NORM, int WPT, int ITS, int V, typename SLOTS>
__global__ __launch_bounds__(256) void rotary_kernel(t2t_rotary_tensor q, t2t_rotary_tensor k, RotaryArgs A,
                                                     SLOTS slots) {
  typedef typename RopeVec<V>::type vec;
  constexpr bool APPEND = std::is_same<SLOTS, RopeSlots>::value;
  if constexpr (APPEND)
    if (blockIdx.y + 1 == gridDim.y) return rope_store_v<V>(slots, A.tokens, A.D);
  const t2t_rotary_tensor& g = blockIdx.y ? k : q;
  __shared__ double part[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hshift = A.hshift[blockIdx.y], chunks = A.chunks[blockIdx.y];
  const int L = 1 << A.shift, per = 1 << hshift, span = A.shift + hshift;  // 2^span lanes a token
  const int u = lane & (L - 1), hl = (lane >> A.shift) & (per - 1), slot = lane >> span;
  const int hstep = WPT * per;
  // the unit's two halves: where they lie, whether they are there and turn
  const int tu = A.half ? A.R / (2 * V) : (A.R + 2 * V - 1) / (2 * V);  // units that turn
  const bool pair = A.half && u < tu;
  const int rest = A.R + 2 * V * (u - tu);
  const int c0 = pair ? V * u : A.half ? rest : 2 * V * u;
  const int c1 = pair ? A.R / 2 + V * u : c0 + V;
  const bool on0 = u < A.units, on1 = on0 && c1 < A.D;
  const bool turn0 = on0 && (A.half ? u < tu : c0 < A.R), turn1 = on1 && (A.half ? u < tu : c1 < A.R);
  const int H = g.heads;
  const double one_over_n = 1.0 / (NORM == T2T_NORM_TOKEN ? (double)H * A.D : (double)A.D);
  const uint16_t* w = (const uint16_t*)g.weight;
  const vec none = {};
  vec wr[ITS][2];  // the token norm's weights, the same for every token
  if constexpr (NORM == T2T_NORM_TOKEN) {
#pragma unroll
    for (int i = 0; i < ITS; ++i) {
      const int h = (WPT == 1 ? 0 : wave * per) + hl + i * hstep;
      wr[i][0] = wr[i][1] = none;
      if (on0 && h < H) wr[i][0] = *(const vec*)(w + (long long)h * A.D + c0);
      if (on1 && h < H) wr[i][1] = *(const vec*)(w + (long long)h * A.D + c1);
    }
  } else if constexpr (NORM == T2T_NORM_HEAD) {
    wr[0][0] = wr[0][1] = none;
    if (on0) wr[0][0] = *(const vec*)(w + c0);
    if (on1) wr[0][1] = *(const vec*)(w + c1);
  }
  const long long items = ((A.tokens + (64 >> span) - 1) >> (6 - span)) * chunks;
  constexpr int IPB = 4 / WPT;  // items under way in a work-group
  for (long long item = (long long)blockIdx.x * IPB + (WPT == 1 ? wave : 0); item < items;
       item += (long long)gridDim.x * IPB) {
    // (chunks is 1 but where the heads of a token go in several items)
    const long long group = chunks == 1 ? item : item / chunks;
    const int first = WPT == 1 ? (int)(item - group * chunks) * ITS * per : wave * per;  // the wave's heads
    const long long tok = (group << (6 - span)) + slot;
    bool live = tok < A.tokens;
    const uint32_t t32 = (uint32_t)(live ? tok : A.tokens - 1), b = t32 / (uint32_t)A.N, n = t32 - b * A.N;
    const uint16_t* x = (const uint16_t*)g.x + b * g.x_batch + n * g.x_row;
    uint16_t* o = (uint16_t*)g.out + b * g.out_batch + n * g.out_row;
    if constexpr (APPEND)
      if (blockIdx.y == 0) {
        long long at = 0;
        live = slots.place(t32, g.out_batch, g.out_row, at) && live;
        o = (uint16_t*)g.out + at;
      }
    float cs[V], sn[V];
    {
      const long long row = (b * A.table_batch + n) * (A.R / 2) + V * u;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        // (the unit's first and second half of entries)
#pragma unroll
        for (int i = 0; i < V / 2; ++i) cs[V / 2 * v + i] = 1.f, sn[V / 2 * v + i] = 0.f;
        if (v ? turn1 : turn0) {
          typedef float fvec __attribute__((ext_vector_type(V / 2)));
          const fvec cv = *(const fvec*)(A.cosv + row + V / 2 * v), sv = *(const fvec*)(A.sinv + row + V / 2 * v);
#pragma unroll
          for (int i = 0; i < V / 2; ++i) cs[V / 2 * v + i] = cv[i], sn[V / 2 * v + i] = A.sign * sv[i];
        }
      }
    }
    vec r[ITS][2];
#pragma unroll
    for (int i = 0; i < ITS; ++i) {
      const int h = first + hl + i * hstep;
      r[i][0] = r[i][1] = none;
      if (on0 && h < H) r[i][0] = *(const vec*)(x + h * g.x_head + c0);
      if (on1 && h < H) r[i][1] = *(const vec*)(x + h * g.x_head + c1);
    }
    float inv[ITS];
    if constexpr (NORM != T2T_NORM_NONE) {
      double sum[ITS], all = 0.0;
#pragma unroll
      for (int i = 0; i < ITS; ++i) {
        sum[i] = 0.0;
        if (first + i * hstep < H) {  // (the same for the wave)
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            float f[V];
            rope_unpack<T, V>(r[i][v], f);
#pragma unroll
            for (int e = 0; e < V; e += 4) sum[i] += rope_squares(f[e], f[e + 1], f[e + 2], f[e + 3]);
          }
        }
        all += sum[i];
      }
      if constexpr (NORM == T2T_NORM_TOKEN) {
        all = rope_sum(all, 1 << span);
        if constexpr (WPT > 1) {
          __syncthreads();  // the last token's sums are read
          if (lane == 0) part[wave] = all;
          __syncthreads();
          all = part[0] + part[1] + part[2] + part[3];
        }
        const float v = rope_inv(all, one_over_n, A.eps);
#pragma unroll
        for (int i = 0; i < ITS; ++i) inv[i] = v;
      } else {
#pragma unroll
        for (int i = 0; i < ITS; ++i) inv[i] = rope_inv(rope_sum(sum[i], L), one_over_n, A.eps);
      }
    }
#pragma unroll
    for (int i = 0; i < ITS; ++i) {
      if (first + i * hstep >= H) break;
      const int h = first + hl + i * hstep;
      // the packed values are kept, not their fp32 forms from the sum or the last token
      asm volatile("" : "+v"(r[i][0]), "+v"(r[i][1]));
      if constexpr (NORM != T2T_NORM_NONE) {
        constexpr int last = NORM == T2T_NORM_TOKEN ? ITS - 1 : 0;
        asm volatile("" : "+v"(wr[i < last ? i : last][0]), "+v"(wr[i < last ? i : last][1]));
      }
      float f0[V], f1[V], y0[V], y1[V];
      rope_unpack<T, V>(r[i][0], f0);
      rope_unpack<T, V>(r[i][1], f1);
      if constexpr (NORM != T2T_NORM_NONE) {
        float w0[V], w1[V];
        const int wi = NORM == T2T_NORM_TOKEN ? i : 0;
        rope_unpack<T, V>(wr[wi][0], w0);
        rope_unpack<T, V>(wr[wi][1], w1);
#pragma unroll
        for (int e = 0; e < V; ++e) f0[e] *= inv[i] * w0[e], f1[e] *= inv[i] * w1[e];
      }
      if (pair) {
#pragma unroll
        for (int e = 0; e < V; ++e) rope_turn(f0[e], f1[e], cs[e], sn[e], y0[e], y1[e]);
      } else {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          y0[2 * e] = f0[2 * e], y0[2 * e + 1] = f0[2 * e + 1];
          y1[2 * e] = f1[2 * e], y1[2 * e + 1] = f1[2 * e + 1];
          if (turn0) rope_turn(f0[2 * e], f0[2 * e + 1], cs[e], sn[e], y0[2 * e], y0[2 * e + 1]);
          if (turn1)
            rope_turn(f1[2 * e], f1[2 * e + 1], cs[V / 2 + e], sn[V / 2 + e], y1[2 * e], y1[2 * e + 1]);
        }
      }
      if (on0 && h < H && live) *(vec*)(o + h * g.out_head + c0) = rope_pack<T, V>(y0);
      if (on1 && h < H && live) *(vec*)(o + h * g.out_head + c1) = rope_pack<T, V>(y1);
    }
  }
}

// The sum of a head's squares, by a wave.
template <typename T>
__device__ inline double rope_head_squares(const uint16_t* x, int D, int lane) {
  double sum = 0.0;
  for (int c = 4 * lane; c < D; c += 256) {
    float f[4];
    for (int e = 0; e < 4; ++e) f[e] = c + e < D ? T::to_f(x[c + e]) : 0.f;
    sum += rope_squares(f[0], f[1], f[2], f[3]);
  }
  return sum;
}

// Any strides, widths and alignment: one work-group per token and tensor, pair by pair, a wave to
// a head; the token norm's sum comes first.
template <typename T, typename SLOTS>
__global__ __launch_bounds__(256) void rotary_any_kernel(t2t_rotary_tensor q, t2t_rotary_tensor k,
                                                         RotaryArgs A, int norm, SLOTS slots) {
  constexpr bool APPEND = std::is_same<SLOTS, RopeSlots>::value;
  if constexpr (APPEND)
    if (blockIdx.y + 1 == gridDim.y) return rope_store_v<1>(slots, A.tokens, A.D);
  const t2t_rotary_tensor& g = blockIdx.y ? k : q;
  __shared__ double part[4];
  const int D = A.D, R = A.R;
  for (long long tok = blockIdx.x; tok < A.tokens; tok += gridDim.x) {
    const int b = (int)(tok / A.N), n = (int)(tok - (long long)b * A.N);
    const uint16_t* x = (const uint16_t*)g.x + b * g.x_batch + n * g.x_row;
    uint16_t* o = (uint16_t*)g.out + b * g.out_batch + n * g.out_row;
    if constexpr (APPEND)
      if (blockIdx.y == 0) {
        long long at = 0;
        if (!slots.place(tok, g.out_batch, g.out_row, at)) continue;  // (the same for the work-group)
        o = (uint16_t*)g.out + at;
      }
    const uint16_t* w = (const uint16_t*)g.weight;
    const float* c = A.cosv + (b * A.table_batch + n) * (R / 2);
    const float* s = A.sinv + (b * A.table_batch + n) * (R / 2);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float inv = 1.f;
    if (norm == T2T_NORM_TOKEN) {
      double sum = 0.0;
      for (int h = wave; h < g.heads; h += 4) sum += rope_head_squares<T>(x + h * g.x_head, D, lane);
      sum = rope_sum(sum, 64);
      __syncthreads();  // the last token's sums are read
      if (lane == 0) part[wave] = sum;
      __syncthreads();
      inv = rope_inv(part[0] + part[1] + part[2] + part[3], 1.0 / ((double)g.heads * D), A.eps);
    }
    const int units = R / 2 + (D - R);  // pairs, then channels that are not turned
    for (int h = wave; h < g.heads; h += 4) {
      const uint16_t* xh = x + h * g.x_head;
      uint16_t* oh = o + h * g.out_head;
      const uint16_t* wh = norm == T2T_NORM_TOKEN ? w + (long long)h * D : w;
      if (norm == T2T_NORM_HEAD) {
        inv = rope_inv(rope_sum(rope_head_squares<T>(xh, D, lane), 64), 1.0 / D, A.eps);
      }
      for (int u = lane; u < units; u += 64) {
        if (u < R / 2) {
          const int i0 = A.half ? u : 2 * u, i1 = A.half ? u + R / 2 : 2 * u + 1;
          float a = T::to_f(xh[i0]), e = T::to_f(xh[i1]);
          if (norm) {
            a *= inv * T::to_f(wh[i0]);
            e *= inv * T::to_f(wh[i1]);
          }
          float y0, y1;
          rope_turn(a, e, c[u], A.sign * s[u], y0, y1);
          oh[i0] = T::from_f(y0);
          oh[i1] = T::from_f(y1);
        } else {
          const int d = R + (u - R / 2);
          float a = T::to_f(xh[d]);
          if (norm) a *= inv * T::to_f(wh[d]);
          oh[d] = T::from_f(a);
        }
      }
    }
  }
}

// vectors of V channels: widths, strides and pointers allow them
static bool rope_vectors(const t2t_rotary_tensor& t, bool weight, int V) {
  return ((t.x_batch | t.x_row | t.x_head | t.out_batch | t.out_row | t.out_head) & (V - 1)) == 0 &&
         (((uintptr_t)t.x | (uintptr_t)t.out | (weight ? (uintptr_t)t.weight : 0)) & (2 * V - 1)) == 0;
}

struct RopeInPlace {};  // an ordinary call: no slots
template <typename SLOTS> static constexpr int rope_rows(int tensors) {
  return tensors + std::is_same<SLOTS, RopeSlots>::value;
}

template <typename T, int NORM, int WPT, int ITS, int V, typename SLOTS>
static void rope_launch(const t2t_rotary_tensor& q, const t2t_rotary_tensor& k, const RotaryArgs& A, int tensors,
                        hipStream_t st, const SLOTS& slots) {
  long long items = 0;
  for (int i = 0; i < tensors; ++i) {
    const int span = A.shift + A.hshift[i];
    const long long n = ((A.tokens + (64 >> span) - 1) >> (6 - span)) * A.chunks[i];
    items = n > items ? n : items;
  }
  const long long wgs = (items + 4 / WPT - 1) / (4 / WPT);
  // evenly several items a work-group from 16,384 of them on, so that the weights are read once for
  // several tokens (75,600 tokens of 40 + 40 heads: two each 578 us, one 599, up to five 590)
  const long long turns = (wgs + 16383) / 16384, grid = (wgs + turns - 1) / turns;
  hipLaunchKernelGGL((rotary_kernel<T, NORM, WPT, ITS, V, SLOTS>), dim3((unsigned)grid, rope_rows<SLOTS>(tensors)),
                     dim3(256), 0, st, q, k, A, slots);
}

// the vector kernel, if it takes the call
template <typename T, int V, typename SLOTS>
static bool rope_vector_run(const t2t_rotary_tensor& q, const t2t_rotary_tensor& k, RotaryArgs A, int norm,
                            int tensors, hipStream_t st, const SLOTS& slots) {
  if constexpr (std::is_same<SLOTS, RopeSlots>::value)
    if (!rope_vectors(slots.v, false, V)) return false;
  if (A.D % V || A.R % (A.half ? 2 * V : V) || !rope_vectors(q, norm, V) ||
      (tensors == 2 && !rope_vectors(k, norm, V)) || (((uintptr_t)A.cosv | (uintptr_t)A.sinv) & (2 * V - 1)))
    return false;
  A.units = A.half ? A.R / (2 * V) + (A.D - A.R + 2 * V - 1) / (2 * V) : (A.D + 2 * V - 1) / (2 * V);
  for (A.shift = 0; (1 << A.shift) < A.units;) ++A.shift;
  if (A.shift > 6) return false;
  int its = 1;  // rounds of a token's heads
  const int heads[2] = {q.heads, k.heads};
  for (int i = 0; i < tensors; ++i) {
    for (A.hshift[i] = 0; A.hshift[i] < 6 - A.shift && (1 << A.hshift[i]) < heads[i];) ++A.hshift[i];
    its = max(its, cdiv(heads[i], 1 << A.hshift[i]));
    A.chunks[i] = 1;
  }
  if (norm == T2T_NORM_TOKEN) {
    // a whole work-group takes a token where the tokens are few (latency) or its heads too many for
    // a wave's registers (3000 tokens of 32 + 8 heads x 256: eight rounds in a wave 43 us, two in four
    // waves 28)
    if (A.tokens >= 1024 && its <= 5) {
      switch (its) {
        case 1: rope_launch<T, T2T_NORM_TOKEN, 1, 1, V>(q, k, A, tensors, st, slots); return true;
        case 2: rope_launch<T, T2T_NORM_TOKEN, 1, 2, V>(q, k, A, tensors, st, slots); return true;
        case 3: rope_launch<T, T2T_NORM_TOKEN, 1, 3, V>(q, k, A, tensors, st, slots); return true;
        case 4: rope_launch<T, T2T_NORM_TOKEN, 1, 4, V>(q, k, A, tensors, st, slots); return true;
        default: rope_launch<T, T2T_NORM_TOKEN, 1, 5, V>(q, k, A, tensors, st, slots); return true;
      }
    }
    A.hshift[0] = A.hshift[1] = 6 - A.shift;
    its = cdiv(max(heads[0], tensors == 2 ? heads[1] : 0), 4 << (6 - A.shift));
    if (its <= 1) rope_launch<T, T2T_NORM_TOKEN, 4, 1, V>(q, k, A, tensors, st, slots);
    else if (its <= 2) rope_launch<T, T2T_NORM_TOKEN, 4, 2, V>(q, k, A, tensors, st, slots);
    else if (its <= 4) rope_launch<T, T2T_NORM_TOKEN, 4, 4, V>(q, k, A, tensors, st, slots);
    else if (its <= 8) rope_launch<T, T2T_NORM_TOKEN, 4, 8, V>(q, k, A, tensors, st, slots);
    return its <= 8;
  }
  // heads on their own: up to four rounds an item (table entries serve them all), one where the items
  // would be few
  const int r = its >= 4 ? 4 : its >= 2 ? 2 : 1, rounds = A.tokens * cdiv(its, r) < 8192 ? 1 : r;
  for (int i = 0; i < tensors; ++i) A.chunks[i] = cdiv(heads[i], rounds << A.hshift[i]);
  if (norm == T2T_NORM_HEAD) {
    if (rounds == 4) rope_launch<T, T2T_NORM_HEAD, 1, 4, V>(q, k, A, tensors, st, slots);
    else if (rounds == 2) rope_launch<T, T2T_NORM_HEAD, 1, 2, V>(q, k, A, tensors, st, slots);
    else rope_launch<T, T2T_NORM_HEAD, 1, 1, V>(q, k, A, tensors, st, slots);
  } else {
    if (rounds == 4) rope_launch<T, T2T_NORM_NONE, 1, 4, V>(q, k, A, tensors, st, slots);
    else if (rounds == 2) rope_launch<T, T2T_NORM_NONE, 1, 2, V>(q, k, A, tensors, st, slots);
    else rope_launch<T, T2T_NORM_NONE, 1, 1, V>(q, k, A, tensors, st, slots);
  }
  return true;
}

template <typename T, typename SLOTS>
static void rope_run(const t2t_rotary_tensor& q, const t2t_rotary_tensor& k, const RotaryArgs& A, int norm,
                     int tensors, hipStream_t st, const SLOTS& slots) {
  if (rope_vector_run<T, 8>(q, k, A, norm, tensors, st, slots) ||
      rope_vector_run<T, 4>(q, k, A, norm, tensors, st, slots))
    return;
  hipLaunchKernelGGL((rotary_any_kernel<T, SLOTS>),
                     dim3((unsigned)(A.tokens < 65536 ? A.tokens : 65536), rope_rows<SLOTS>(tensors)), dim3(256), 0,
                     st, q, k, A, norm, slots);
}

extern "C" int t2t_rotary(const t2t_rotary_tensor* q, const t2t_rotary_tensor* k, int dtype,
                          const float* cosv, const float* sinv, int table_batched, int B, int N, int D,
                          int R, int layout, int inverse, int norm, float eps, void* stream) {
  T2T_REQUIRE(q, "rotary: null pointer");
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "rotary: dtype %d", dtype);
  T2T_REQUIRE(B >= 0 && N >= 0 && (long long)B * N <= INT_MAX, "rotary: B=%d N=%d", B, N);
  T2T_REQUIRE(D >= 1 && D <= 256 && R >= 2 && R <= D && R % 2 == 0,
              "rotary: D=%d R=%d (1 <= D <= 256, R even, 2 <= R <= D)", D, R);
  T2T_REQUIRE(layout == T2T_ROPE_INTERLEAVED || layout == T2T_ROPE_HALF, "rotary: layout %d", layout);
  T2T_REQUIRE(norm >= T2T_NORM_NONE && norm <= T2T_NORM_HEAD, "rotary: norm %d", norm);
  T2T_REQUIRE(!(inverse && norm), "rotary: the inverse rotation takes no norm");
  const t2t_rotary_tensor* ts[2] = {q, k ? k : q};
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    T2T_REQUIRE(ts[i]->heads >= 1 && ts[i]->heads <= 65536, "rotary: heads=%d", ts[i]->heads);
    T2T_REQUIRE(!norm || ts[i]->weight, "rotary: the norm needs a weight");
  }
  const long long tokens = (long long)B * N;
  if (tokens == 0) return T2T_OK;
  T2T_REQUIRE(cosv && sinv && ts[0]->x && ts[0]->out && ts[1]->x && ts[1]->out, "rotary: null pointer");
  RotaryArgs A{};
  A.cosv = cosv, A.sinv = sinv;
  A.table_batch = table_batched ? N : 0;
  A.tokens = tokens, A.N = N, A.D = D, A.R = R;
  A.half = layout == T2T_ROPE_HALF;
  A.sign = inverse ? -1.f : 1.f, A.eps = eps;
  if (dtype == T2T_BF16)
    rope_run<BF16T>(*ts[0], *ts[1], A, norm, k ? 2 : 1, (hipStream_t)stream, RopeInPlace{});
  else
    rope_run<F16T>(*ts[0], *ts[1], A, norm, k ? 2 : 1, (hipStream_t)stream, RopeInPlace{});
  T2T_LAUNCH_CHECK("rotary");
  return T2T_OK;
}

extern "C" int t2t_cache_append(const t2t_rotary_tensor* q, const t2t_rotary_tensor* k, const t2t_rotary_tensor* v,
                                int dtype, const float* cosv, const float* sinv, const void* slots, int slot_bits,
                                int pages, int page_size, long long T, int D, int R, int layout, int norm, float eps,
                                void* stream) {
  T2T_REQUIRE(k && v, "cache_append: null pointer");
  T2T_REQUIRE(dtype == T2T_F16 || dtype == T2T_BF16, "cache_append: dtype %d", dtype);
  T2T_REQUIRE(slot_bits == 32 || slot_bits == 64, "cache_append: slots of %d bits", slot_bits);
  T2T_REQUIRE(pages >= 1 && page_size >= 1, "cache_append: %d pages of %d", pages, page_size);
  T2T_REQUIRE(T >= 0 && T <= INT_MAX, "cache_append: T=%lld", T);
  T2T_REQUIRE(D >= 1 && D <= 256 && R >= 2 && R <= D && R % 2 == 0,
              "cache_append: D=%d R=%d (1 <= D <= 256, R even, 2 <= R <= D)", D, R);
  T2T_REQUIRE(layout == T2T_ROPE_INTERLEAVED || layout == T2T_ROPE_HALF, "cache_append: layout %d", layout);
  T2T_REQUIRE(norm >= T2T_NORM_NONE && norm <= T2T_NORM_HEAD, "cache_append: norm %d", norm);
  const t2t_rotary_tensor* ts[3] = {k, v, q ? q : k};
  for (int i = 0; i < 3; ++i) {
    T2T_REQUIRE(ts[i]->heads >= 1 && ts[i]->heads <= 65536, "cache_append: heads=%d", ts[i]->heads);
    T2T_REQUIRE(!norm || i == 1 || ts[i]->weight, "cache_append: the norm needs a weight");
  }
  T2T_REQUIRE(k->heads == v->heads, "cache_append: %d heads of keys, %d of values", k->heads, v->heads);
  if (T == 0) return T2T_OK;
  T2T_REQUIRE(cosv && sinv && slots, "cache_append: null pointer");
  for (int i = 0; i < 3; ++i) T2T_REQUIRE(ts[i]->x && ts[i]->out, "cache_append: null pointer");
  t2t_rotary_tensor kt = *k, qt = q ? *q : *k;
  kt.x_batch = 0, qt.x_batch = 0;  // one sequence
  if (q) qt.out_batch = 0;
  RotaryArgs A{};
  A.cosv = cosv, A.sinv = sinv;
  A.tokens = T, A.N = (int)T, A.D = D, A.R = R;
  A.half = layout == T2T_ROPE_HALF;
  A.sign = 1.f, A.eps = eps;
  RopeSlots S{slots, slot_bits == 64, page_size, (unsigned long long)pages * page_size, *v};
  S.v.x_batch = 0;
  if (dtype == T2T_BF16)
    rope_run<BF16T>(kt, qt, A, norm, q ? 2 : 1, (hipStream_t)stream, S);
  else
    rope_run<F16T>(kt, qt, A, norm, q ? 2 : 1, (hipStream_t)stream, S);
  T2T_LAUNCH_CHECK("cache_append");
  return T2T_OK;
}
