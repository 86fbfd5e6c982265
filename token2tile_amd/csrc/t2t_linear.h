// What the linear layers (mxfp4.hip, int8.hip) have in common: the activation,
// the order of their tiles and the stores of odd rows.
#pragma once
#include "t2t_common.h"

// gelu(x) = x / 2 (1 + tanh u) = x / (1 + e^(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3), with the
// constants of e^(-2 u) = 2^(x (c0 + c1 x^2)).  v_exp_f32 and v_rcp_f32 are within 1 ulp.
__device__ inline float lin_gelu(float x) {
  const float z = x * __builtin_fmaf(-0.10294324f, x * x, -2.3022082f);
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z));
}

typedef __attribute__((address_space(3))) void lin_lds_t;

// Consecutive work-groups go to the eight XCDs in turn: each takes a run of
// tiles, eight token tiles by all feature tiles, so that the 32 tiles an XCD
// has under way share their panels in its L2.
__device__ inline int lin_first(int per_xcd) { return (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3); }
__device__ inline int lin_end(int mt, int nt, int per_xcd) {
  return min(mt * nt, ((int)(blockIdx.x & 7) + 1) * per_xcd);
}
// a tile's first row blocks
__device__ inline void lin_place(int id, int mt, int nt, int mb, int nb, int& m0, int& n0) {
  const int grp = id / (8 * nt), in = id - grp * 8 * nt;
  const int gm = min(8, mt - grp * 8);
  m0 = (grp * 8 + in % gm) * mb;
  n0 = (in / gm) * nb;
}

// The values of one row, the first n of which are inside, to an o of any alignment (rows of odd
// widths: the store takes 16 bytes at any address, two at a time it cost 16 us at 4099 x 2041)
template <typename VT>
__device__ inline void lin_put(uint16_t* o, const VT& v, int n) {
  if (n >= (int)sizeof(VT) / 2)
    __builtin_memcpy(o, &v, sizeof(VT));
  else
#pragma unroll
    for (int e = 0; e < (int)sizeof(VT) / 2; ++e)
      if (e < n) o[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
}

