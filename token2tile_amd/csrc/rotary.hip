// Rotary positions: the cos / sin tables of a set of positions, and the
// rotation of q and k with the RMS norm that stands before it.
#include "t2t_common.h"

// ---------------------------------------------------------------------------
// cos[t, i] = m cos(p[t, a] f[i]), sin likewise; pair i belongs to the axis a
// with start[a] <= i < start[a + 1].  The angle is one fp64 product (a far
// position leaves no fraction in fp32) and its sine and cosine are taken in
// fp64, so the fp32 entries are off by one rounding.  Bound: writing the
// tables.
// ---------------------------------------------------------------------------
struct TableAxes {
  int n;
  int start[5];
};

template <typename P>
__global__ __launch_bounds__(256) void rotary_table_kernel(const P* __restrict__ pos,
                                                           const double* __restrict__ freqs,
                                                           TableAxes ax, double m,
                                                           float* __restrict__ cosv,
                                                           float* __restrict__ sinv, int pairs,
                                                           long long total) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (long long)gridDim.x * 256) {
    const long long t = i / pairs;
    const int p = (int)(i - t * pairs);
    int a = 0;
    for (int k = 1; k < ax.n; ++k) a += p >= ax.start[k];
    double s, c;
    sincos((double)pos[t * ax.n + a] * freqs[p], &s, &c);
    cosv[i] = (float)(m * c);
    sinv[i] = (float)(m * s);
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
  const long long total = T * pairs;
  const long long g = (total + 255) / 256;
  const dim3 grid((unsigned)(g < 16384 ? g : 16384));
  if (pos_bits == 32)
    hipLaunchKernelGGL(rotary_table_kernel<int32_t>, grid, dim3(256), 0, (hipStream_t)stream,
                       (const int32_t*)positions, freqs, ax, factor, cosv, sinv, pairs, total);
  else
    hipLaunchKernelGGL(rotary_table_kernel<long long>, grid, dim3(256), 0, (hipStream_t)stream,
                       (const long long*)positions, freqs, ax, factor, cosv, sinv, pairs, total);
  T2T_LAUNCH_CHECK("rotary_table");
  return T2T_OK;
}

// ---------------------------------------------------------------------------
// y = rotate(x rsqrt(mean(x^2) + eps) w), fp32 inside, one rounding at the
// end.  One work-group of 256 threads per token and tensor (blockIdx.y: q or
// k); the norm's sums are taken first (over the token's H D values, or one
// wave per head), then every thread turns pairs.  Any strides, widths and
// alignment.
// ---------------------------------------------------------------------------
static __device__ inline float rope_sum64(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(t2t_rotary_tensor q, t2t_rotary_tensor k,
                                                         const float* __restrict__ cosv,
                                                         const float* __restrict__ sinv,
                                                         long long table_batch, int N, int D, int R,
                                                         int half, float sign, int norm, float eps) {
  const t2t_rotary_tensor& g = blockIdx.y ? k : q;
  __shared__ float part[4];
  const long long tok = blockIdx.x;
  const int b = (int)(tok / N), n = (int)(tok - (long long)b * N);
  const uint16_t* x = (const uint16_t*)g.x + b * g.x_batch + n * g.x_row;
  uint16_t* o = (uint16_t*)g.out + b * g.out_batch + n * g.out_row;
  const uint16_t* w = (const uint16_t*)g.weight;
  const float* c = cosv + (b * table_batch + n) * (R / 2);
  const float* s = sinv + (b * table_batch + n) * (R / 2);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float inv = 1.f;
  if (norm == T2T_NORM_TOKEN) {
    float sum = 0.f;
    for (int h = wave; h < g.heads; h += 4)
      for (int d = lane; d < D; d += 64) {
        const float v = T::to_f(x[h * g.x_head + d]);
        sum += v * v;
      }
    sum = rope_sum64(sum);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    inv = rsqrtf((part[0] + part[1] + part[2] + part[3]) / ((float)g.heads * D) + eps);
  }
  const int units = R / 2 + (D - R);  // pairs, then channels that are not turned
  for (int h = wave; h < g.heads; h += 4) {
    const uint16_t* xh = x + h * g.x_head;
    uint16_t* oh = o + h * g.out_head;
    const uint16_t* wh = norm == T2T_NORM_TOKEN ? w + (long long)h * D : w;
    if (norm == T2T_NORM_HEAD) {
      float sum = 0.f;
      for (int d = lane; d < D; d += 64) {
        const float v = T::to_f(xh[d]);
        sum += v * v;
      }
      inv = rsqrtf(rope_sum64(sum) / D + eps);
    }
    for (int u = lane; u < units; u += 64) {
      if (u < R / 2) {
        const int i0 = half ? u : 2 * u, i1 = half ? u + R / 2 : 2 * u + 1;
        float a = T::to_f(xh[i0]), e = T::to_f(xh[i1]);
        if (norm) {
          a = a * inv * T::to_f(wh[i0]);
          e = e * inv * T::to_f(wh[i1]);
        }
        const float cc = c[u], ss = sign * s[u];
        oh[i0] = T::from_f(a * cc - e * ss);
        oh[i1] = T::from_f(a * ss + e * cc);
      } else {
        const int d = R + (u - R / 2);
        float a = T::to_f(xh[d]);
        if (norm) a = a * inv * T::to_f(wh[d]);
        oh[d] = T::from_f(a);
      }
    }
  }
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
  const dim3 grid((unsigned)tokens, k ? 2 : 1);
  const long long tb = table_batched ? N : 0;
  if (dtype == T2T_BF16)
    hipLaunchKernelGGL(rotary_any_kernel<BF16T>, grid, dim3(256), 0, (hipStream_t)stream, *ts[0], *ts[1],
                       cosv, sinv, tb, N, D, R, layout == T2T_ROPE_HALF, inverse ? -1.f : 1.f, norm, eps);
  else
    hipLaunchKernelGGL(rotary_any_kernel<F16T>, grid, dim3(256), 0, (hipStream_t)stream, *ts[0], *ts[1],
                       cosv, sinv, tb, N, D, R, layout == T2T_ROPE_HALF, inverse ? -1.f : 1.f, norm, eps);
  T2T_LAUNCH_CHECK("rotary");
  return T2T_OK;
}
