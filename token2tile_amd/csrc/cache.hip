// Attention of new tokens over a paged cache of keys and values.
//
// Row (token, head) of a sequence whose cache holds L keys, the last n of them
// those of its n new tokens:  o = sum_j p_j v_j,  p = softmax over the seen j of
// scale q . k_j.  Seen are the L - n older keys, and of the new ones all, those up
// to the row's own token, or those that the mask names.  A row that sees nothing is
// zero (log-sum -inf).  Keys that are not seen have no part in the result whatever
// they hold.
#include "t2t_common.h"
#include <type_traits>

typedef __attribute__((address_space(3))) void ca_lds_t;
typedef const __attribute__((address_space(1))) void ca_glb_t;

#define CA_NONE (-1.0e30f)  // the running maximum before any key: finite, so that rows of hidden keys add 0

struct CacheArgs {
  const char *q, *k, *v;
  char* out;
  float* lse;
  const int32_t *table, *lengths, *offsets;
  const uint8_t* mask;
  long long q_batch, q_row, q_head, o_batch, o_row, o_head, kv_page, kv_row, kv_head;  // bytes
  long long table_row, mask_batch, mask_row;
  int B, N, T, HQ, HK, G, pages, page, shift, width, mask_cols, causal;
  float c;  // scale log2(e)
  int S;    // most parts of a sequence's keys
  float* opart;
  float* mlpart;
};

// parts that a sequence of L keys goes in
#define CA_PART 512
__device__ inline int ca_parts(int L, int S) { return min(S, max(1, (L + CA_PART - 1) / CA_PART)); }

// A work-group's rows: row block `tile` of ROWS packed rows (token, head of the group) of a
// sequence.  Sequence b owns blocks from offsets[b] G / ROWS + b on, at least as many as it needs.
struct CacheRows {
  int b, n, L, first;   // sequence, its new tokens, keys, older keys
  int r0, rows;         // packed rows from r0 on, how many there are in the sequence
  long long row0;       // its first row among all
};
template <int ROWS>
__device__ inline bool ca_rows(const CacheArgs& A, int tile, CacheRows& w) {
  int first_tile;
  if (A.offsets) {
    const int lane = __lane_id();
    int count = 0;
    for (int b0 = 0; b0 < A.B; b0 += 64) {
      const int b = b0 + lane;
      const long long off = b < A.B ? min(max(A.offsets[b], 0), A.T) : 0;
      count += __popcll(__ballot(b < A.B && off * A.G / ROWS + b <= tile));
    }
    w.b = max(count - 1, 0);
    const int lo = min(max(A.offsets[w.b], 0), A.T), hi = min(max(A.offsets[w.b + 1], 0), A.T);
    w.row0 = lo, w.n = max(hi - lo, 0);
    first_tile = (int)((long long)lo * A.G / ROWS) + w.b;
  } else {
    const int per = (int)(((long long)A.N * A.G + ROWS - 1) / ROWS);
    w.b = tile / per;
    w.row0 = (long long)w.b * A.N, w.n = A.N;
    first_tile = w.b * per;
  }
  w.rows = w.n * A.G;
  w.r0 = (tile - first_tile) * ROWS;
  if (w.b >= A.B || w.r0 < 0 || w.r0 >= w.rows) return false;
  w.L = min((long long)max(A.lengths[w.b], 0), (long long)A.width * A.page);
  w.first = w.L - w.n;
  return true;
}
__device__ inline const char* ca_token(const char* p, const CacheArgs& A, const CacheRows& w, long long batch,
                                       long long row, int i) {
  return p + (A.offsets ? (w.row0 + i) * row : w.b * batch + i * row);
}

// Where the bytes of a tile lie in LDS: rows of D halves, 16-byte chunk c of row r at c ^ swizzle(r),
// so that the 16-byte reads of sixteen keys (K) and the transposing reads of four (V) meet all banks.
template <int D> __device__ inline int ca_kswz(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D> __device__ inline int ca_vswz(int row) { return D == 128 ? (row & 3) << 2 : (row & 2) << 1; }

// Rows of a tile are fetched by position: the cache row of position pos of a sequence, in units of
// 16 bytes from the head's base (which spans less than 64 GiB).  A table entry outside the cache
// leaves its keys out: `ok` is false and row 0 is fetched in their place.
__device__ inline uint32_t ca_entry(const CacheArgs& A, const int32_t* table, int pos) {
  return (uint32_t)table[A.shift >= 0 ? pos >> A.shift : pos / A.page];
}
__device__ inline uint32_t ca_offset(const CacheArgs& A, uint32_t entry, int pos, bool& ok) {
  ok = entry < (uint32_t)A.pages;
  const int in = A.shift >= 0 ? pos & (A.page - 1) : pos % A.page;
  return ok ? (uint32_t)((entry * A.kv_page + in * A.kv_row) >> 4) : 0u;
}

template <typename T> struct CaType;
template <> struct CaType<BF16T> {
  static constexpr float top = 0.f, limit = 0x1p64f;  // log2 of the largest weight, most of a tile's sum
  static constexpr uint32_t inf = 0x7f80u;
};
template <> struct CaType<F16T> {
  static constexpr float top = 8.f, limit = 0x1p14f;  // (weights down to 2^-22 of the largest keep their bits)
  static constexpr uint32_t inf = 0x7c00u;
};

// ---- one tile of NK x 32 keys for 32 rows ------------------------------------
// S^T = K Q^T and O^T = V^T P^T: lane l holds row l % 32 throughout, keys 8 (a / 4)
// + 4 (l / 32) + a % 4 of a 32-key block in element a, dims likewise.
template <typename T, int D>
struct CacheState {
  u32x4 q[D / 16];  // dims 16 s + 8 (l / 32) .. + 7
  f32x16 o[D / 32];
  float m, l;
};

// the four operand parts of 32 keys and dim block nb, from the transposing reads: lane l gets dim l %
// 32 of keys 16 i / 2 + 8 (i % 2) + 4 (l / 32) + 0 .. 3
template <int D, int BASE>
__device__ inline void ca_vread(u32x2 (&f)[4], uint32_t a) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%c5\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%c6\n\t"
      "ds_read_b64_tr_b16 %2, %4 offset:%c7\n\t"
      "ds_read_b64_tr_b16 %3, %4 offset:%c8"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
      : "v"(a), "n"(BASE), "n"(BASE + 16 * D), "n"(BASE + 32 * D), "n"(BASE + 48 * D));
}
#define CA_WAIT4(f, n) \
  asm volatile("s_waitcnt lgkmcnt(" #n ")" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]))

// The lane's row in the mask: hidden are positions past the length, new ones past `last` (causal)
// and, with a mask, those it does not name.
struct CacheSight {
  const uint8_t* mask;  // the row's bytes for new token 0, or NULL
  int first, last, cols;
  __device__ bool sees(int pos) const {
    if (pos > last) return false;
    if (!mask || pos < first) return true;
    return pos - first < cols && mask[pos - first] != 0;
  }
};

// s -> weights against the running maximum (exp2 scales exactly, so it only has to keep the weights in
// the range of T: it moves where they leave it, and the sums so far with it)
template <typename T, int D, int NK>
__device__ inline void ca_weights(CacheState<T, D>& w, const f32x16 (&s)[NK], u32x4 (&p)[2 * NK], float c) {
  auto expo = [&](float nm) __attribute__((always_inline)) {
    float acc = 0.f;
#pragma unroll
    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
      for (int a = 0; a < 16; a += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][a], c, nm));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][a + 1], c, nm));
        const uint32_t pk = Pk<T>::pack(p0, p1);
        acc = Pk<T>::sum2(pk, acc);
        p[2 * kb + a / 8][(a % 8) / 2] = pk;
      }
    return acc;
  };
  float lt = expo(-w.m);
  if (__builtin_amdgcn_readfirstlane((int)(__ballot(!(lt <= CaType<T>::limit)) != 0ull))) {
    float mr = -__builtin_inff();
#pragma unroll
    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
      for (int a = 0; a < 16; ++a) mr = __builtin_elementwise_maximum(mr, s[kb][a]);
    const float mx = half_max(mr) * c - CaType<T>::top;
    const float mnew = mx > w.m || mx != mx ? mx : w.m;
    const float alpha = __builtin_amdgcn_exp2f(w.m - mnew);
    w.m = mnew;
    w.l *= alpha;
#pragma unroll
    for (int nb = 0; nb < D / 32; ++nb)
#pragma unroll
      for (int a = 0; a < 16; ++a) w.o[nb][a] *= alpha;
    lt = expo(-w.m);
  }
  w.l += lt;
}

// Whether a tile's operand parts hold an inf or NaN, and those parts without them
template <typename T>
__device__ inline bool ca_clean(u32x2 (&f)[4]) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t lo = (f[i][e] & CaType<T>::inf) == CaType<T>::inf ? 0u : f[i][e] & 0xffffu;
      const uint32_t hi = (f[i][e] >> 16 & CaType<T>::inf) == CaType<T>::inf ? 0u : f[i][e] & 0xffff0000u;
      any |= (lo | hi) != f[i][e];
      f[i][e] = lo | hi;
    }
  return any;
}

// ---- few rows: a work-group's waves take the keys in turn --------------------
// 32 packed rows a work-group, 32 keys a tile; a wave fetches its own tiles (DMA to
// its own LDS, one ahead) and keeps sums of its own, which meet at the end.  Where
// the row blocks are few, a sequence's keys go in parts to several work-groups,
// whose sums ca_combine_kernel joins.
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void ca_few_kernel(CacheArgs A) {
  constexpr int WAVES = 4, TILE = 32 * D, LPR = D / 8, RPI = 64 / LPR;  // lanes a row, rows an instruction
  __shared__ __attribute__((aligned(1024))) uint16_t sK0[WAVES * TILE], sK1[WAVES * TILE];
  __shared__ __attribute__((aligned(1024))) uint16_t sV0[WAVES * TILE], sV1[WAVES * TILE];
  __shared__ float sM[WAVES][32], sL[WAVES][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int jl = lane & 31, hh = lane >> 5;
  const int part = blockIdx.x % A.S, kh = blockIdx.x / A.S % A.HK, tile = blockIdx.x / A.S / A.HK;
  CacheRows w;
  if (!ca_rows<32>(A, tile, w)) return;
  const int parts = ca_parts(w.L, A.S);
  if (part >= parts) return;
  const int r = min(w.r0 + jl, w.rows - 1), tok = r / A.G, head = kh * A.G + r - tok * A.G;
  CacheSight sight{A.mask ? A.mask + (A.offsets ? (w.row0 + tok) * A.mask_row : w.b * A.mask_batch + tok * A.mask_row)
                          : nullptr,
                   w.first, A.causal ? w.first + tok : w.L - 1, A.mask_cols};
  const bool masked = A.mask || A.causal;
  CacheState<T, D> st;
  st.m = CA_NONE, st.l = 0.f;
  {
    const char* qr = ca_token(A.q, A, w, A.q_batch, A.q_row, tok) + head * A.q_head + 16 * hh;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) st.q[s] = *(const u32x4*)(qr + 32 * s);
  }
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb) st.o[nb] = zero16();
  const char* kbase = A.k + kh * A.kv_head;
  const char* vbase = A.v + kh * A.kv_head;
  const int32_t* table = A.table + w.b * A.table_row;

  const int tiles = (w.L + 31) / 32;
  const int t0 = (int)((long long)part * tiles / parts) + wave, t1 = (int)((long long)(part + 1) * tiles / parts);
  auto pos_of = [&](int t) { return min(32 * t + jl, w.L - 1); };
  auto issue = [&](uint32_t off, auto BUF) __attribute__((always_inline)) {
    uint16_t* dk = (decltype(BUF)::value ? sK1 : sK0) + wave * TILE;
    uint16_t* dv = (decltype(BUF)::value ? sV1 : sV0) + wave * TILE;
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) {
      const int row = RPI * i + lane / LPR;
      const size_t at = (size_t)(uint32_t)__shfl((int)off, row, 64) * 16;
      __builtin_amdgcn_global_load_lds((ca_glb_t*)(kbase + at + 16 * ((lane & (LPR - 1)) ^ ca_kswz<D>(row))),
                                       (ca_lds_t*)(dk + i * 512), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((ca_glb_t*)(vbase + at + 16 * ((lane & (LPR - 1)) ^ ca_vswz<D>(row))),
                                       (ca_lds_t*)(dv + i * 512), 16, 0, 0);
    }
  };
  const int trkey = 4 * hh + ((lane & 15) >> 2), trdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  // BAD: lanes whose key's table entry lies outside the cache
  auto step = [&](int t, uint64_t bad, auto BUF) __attribute__((always_inline)) {
    const uint16_t* sk = (decltype(BUF)::value ? sK1 : sK0) + wave * TILE;
    const uint16_t* sv = (decltype(BUF)::value ? sV1 : sV0) + wave * TILE;
    const uint32_t va = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint16_t*)sv;
    f32x16 s[1] = {zero16()};
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      s[0] = Mfma<T>::run(*(const u32x4*)(sk + jl * D + 8 * ((2 * i + hh) ^ ca_kswz<D>(jl))), st.q[i], s[0]);
    const bool hide = 32 * t + 32 > (masked ? w.first : w.L) || bad;  // (of the wave)
    uint32_t seen = 0;  // by the lane's row, of all 32 keys
    if (hide) {
#pragma unroll
      for (int a = 0; a < 16; ++a) {
        const int j = 8 * (a / 4) + 4 * hh + a % 4;
        const bool see = sight.sees(32 * t + j) && !(bad >> j & 1);
        seen |= (uint32_t)see << j;
        if (!see) s[0][a] = -__builtin_inff();
      }
      seen |= half_partner(seen);
    }
    u32x4 p[2];
    ca_weights<T, D, 1>(st, s, p, A.c);
    bool odd = false;
#pragma unroll
    for (int nb = 0; nb < D / 32; ++nb) {
      u32x2 f[4];
      ca_vread<D, 0>(f, va + 2 * (trkey * D + 8 * ((4 * nb + (trdim >> 3)) ^ ca_vswz<D>(trkey)) + (trdim & 7)));
      CA_WAIT4(f, 0);
      if (hide) odd |= ca_clean<T>(f);
#pragma unroll
      for (int mm = 0; mm < 2; ++mm)
        st.o[nb] = Mfma<T>::run(u32x4{f[2 * mm][0], f[2 * mm][1], f[2 * mm + 1][0], f[2 * mm + 1][1]}, p[mm], st.o[nb]);
    }
    // an inf or NaN among the values (left out above, or a weight of 0 would make it NaN) goes to
    // the rows that see it
    if (hide && __ballot(odd)) {
      for (int j = 0; j < 32; ++j)
#pragma unroll
        for (int nb = 0; nb < D / 32; ++nb)
#pragma unroll
          for (int a = 0; a < 16; ++a) {
            const int d = 32 * nb + 8 * (a / 4) + 4 * hh + a % 4;
            const uint16_t u = sv[j * D + 8 * ((d >> 3) ^ ca_vswz<D>(j)) + (d & 7)];
            if ((u & CaType<T>::inf) == CaType<T>::inf && (seen >> j & 1)) st.o[nb][a] += T::to_f(u);
          }
    }
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  uint32_t entry = 0;
  bool ok;
  uint64_t bad0 = 0, bad1 = 0;
  if (t0 < t1) {
    const uint32_t off = ca_offset(A, ca_entry(A, table, pos_of(t0)), pos_of(t0), ok);
    bad0 = __ballot(!ok);
    issue(off, B0{});
    if (t0 + WAVES < t1) entry = ca_entry(A, table, pos_of(t0 + WAVES));
  }
  // tile t has been issued and the entry of the one after it is under way
  auto turn = [&](int t, uint64_t bad, uint64_t& next_bad, auto BUF) __attribute__((always_inline)) {
    constexpr int buf = decltype(BUF)::value;
    uint32_t off = 0;
    if (t + WAVES < t1) {
      off = ca_offset(A, entry, pos_of(t + WAVES), ok);
      next_bad = __ballot(!ok);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (t + WAVES < t1) issue(off, std::integral_constant<int, 1 - buf>{});
    if (t + 2 * WAVES < t1) entry = ca_entry(A, table, pos_of(t + 2 * WAVES));
    step(t, bad, BUF);
  };
  for (int t = t0; t < t1; t += 2 * WAVES) {
    turn(t, bad0, bad1, B0{});
    if (t + WAVES < t1) turn(t + WAVES, bad1, bad0, B1{});
  }
  // the waves' sums
  const float l = half_sum(st.l);
  if (hh == 0) sM[wave][jl] = st.m, sL[wave][jl] = l;
  __syncthreads();
  float M = sM[0][jl], total = 0.f;
#pragma unroll
  for (int x = 1; x < WAVES; ++x) M = __builtin_elementwise_maximum(M, sM[x][jl]);
#pragma unroll
  for (int x = 0; x < WAVES; ++x) total += sL[x][jl] * __builtin_amdgcn_exp2f(sM[x][jl] - M);
  const float mine = __builtin_amdgcn_exp2f(st.m - M);
  auto sums = [&](int x) { return (float*)(x < 2 ? sK0 : sK1) + (x & 1) * 32 * D; };
  float* to = sums(wave);
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int ch = (8 * nb + 2 * g + hh) ^ (jl & 15);
      *(f32x4*)(to + jl * D + 4 * ch) = f32x4{st.o[nb][4 * g] * mine, st.o[nb][4 * g + 1] * mine,
                                              st.o[nb][4 * g + 2] * mine, st.o[nb][4 * g + 3] * mine};
    }
  if (wave == 0 && hh == 0) sM[0][jl] = M;
  __syncthreads();
  if (wave == 0 && hh == 0) sL[0][jl] = total;
  __syncthreads();
  // a row by eight threads, D / 8 dims each
  const int rr = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * (D / 8);
  if (w.r0 + rr >= w.rows) return;
  const int tok2 = (w.r0 + rr) / A.G, head2 = kh * A.G + w.r0 + rr - tok2 * A.G;
  const float lt = sL[0][rr];
  const long long at = (w.row0 + tok2) * A.HQ + head2;
  float o[D / 8];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < WAVES; ++y) x += *(const f32x4*)(sums(y) + rr * D + 4 * ((d0 / 4 + i) ^ (rr & 15)));
#pragma unroll
    for (int e = 0; e < 4; ++e) o[4 * i + e] = x[e];
  }
  if (parts > 1) {
    const long long pr = (long long)part * A.T * A.HQ + at;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      *(f32x4*)(A.opart + pr * D + d0 + 4 * i) = f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
    if (d0 == 0) A.mlpart[2 * pr] = sM[0][rr], A.mlpart[2 * pr + 1] = lt;
    return;
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  char* dst = (char*)ca_token(A.out, A, w, A.o_batch, A.o_row, tok2) + head2 * A.o_head + 2 * d0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    *(u32x4*)(dst + 16 * i) = u32x4{Pk<T>::pack(o[8 * i] * inv, o[8 * i + 1] * inv), Pk<T>::pack(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                    Pk<T>::pack(o[8 * i + 4] * inv, o[8 * i + 5] * inv), Pk<T>::pack(o[8 * i + 6] * inv, o[8 * i + 7] * inv)};
  if (A.lse && d0 == 0) A.lse[at] = lt == 0.f ? -__builtin_inff() : 0.6931471805599453f * (sM[0][rr] + __log2f(lt));
}

// joins the parts of a row block's rows, eight threads a row
template <typename T, int D>
__global__ __launch_bounds__(256) void ca_combine_kernel(CacheArgs A) {
  const int kh = blockIdx.x % A.HK, tile = blockIdx.x / A.HK;
  CacheRows w;
  if (!ca_rows<32>(A, tile, w)) return;
  const int parts = ca_parts(w.L, A.S), rr = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * (D / 8);
  if (parts < 2 || w.r0 + rr >= w.rows) return;  // (its work-group has written the rows)
  const int tok = (w.r0 + rr) / A.G, head = kh * A.G + w.r0 + rr - tok * A.G;
  const long long at = (w.row0 + tok) * A.HQ + head, step = (long long)A.T * A.HQ;
  float M = CA_NONE, total = 0.f, o[D / 8];
  for (int i = 0; i < parts; ++i) M = __builtin_elementwise_maximum(M, A.mlpart[2 * (at + i * step)]);
#pragma unroll
  for (int e = 0; e < D / 8; ++e) o[e] = 0.f;
  for (int i = 0; i < parts; ++i) {
    const float a = __builtin_amdgcn_exp2f(A.mlpart[2 * (at + i * step)] - M);
    total = __builtin_fmaf(a, A.mlpart[2 * (at + i * step) + 1], total);
#pragma unroll
    for (int e = 0; e < D / 8; e += 4) {
      const f32x4 x = *(const f32x4*)(A.opart + (at + i * step) * D + d0 + e);
#pragma unroll
      for (int f = 0; f < 4; ++f) o[e + f] = __builtin_fmaf(a, x[f], o[e + f]);
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  char* dst = (char*)ca_token(A.out, A, w, A.o_batch, A.o_row, tok) + head * A.o_head + 2 * d0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    *(u32x4*)(dst + 16 * i) = u32x4{Pk<T>::pack(o[8 * i] * inv, o[8 * i + 1] * inv), Pk<T>::pack(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                    Pk<T>::pack(o[8 * i + 4] * inv, o[8 * i + 5] * inv), Pk<T>::pack(o[8 * i + 6] * inv, o[8 * i + 7] * inv)};
  if (A.lse && d0 == 0) A.lse[at] = total == 0.f ? -__builtin_inff() : 0.6931471805599453f * (M + __log2f(total));
}

// Most parts of a sequence's keys: as many as bring the launch to two rounds of work-groups, of
// CA_PART keys at least.
static int ca_split(long long tiles, int HK, long long keys) {
  const long long wgs = tiles * HK, most = (keys + CA_PART - 1) / CA_PART;
  if (wgs >= 512 || most < 2) return 1;
  const long long s = (512 + wgs - 1) / wgs;
  return (int)(s < most ? (s < 64 ? s : 64) : (most < 64 ? most : 64));
}
// row blocks of 32 packed rows
static long long ca_tiles(int ragged, int B, long long T, int G) {
  return ragged ? T * G / 32 + B : B * ((T / B * G + 31) / 32);
}
static size_t ca_ws(int S, long long rows, int D) { return S < 2 ? 0 : (size_t)S * rows * (D + 2) * 4; }

extern "C" size_t t2t_cache_attention_ws_bytes(int ragged, int B, long long T, int HQ, int HK, int D, long long keys) {
  if (B < 1 || T < 1 || HK < 1 || HQ < HK || keys < 1) return 0;
  return ca_ws(ca_split(ca_tiles(ragged, B, T, HQ / HK), HK, keys), T * HQ, D);
}

extern "C" int t2t_cache_attention(const t2t_cache_attention_args* a, void* ws, size_t ws_bytes, void* stream) {
  T2T_REQUIRE(a && a->struct_bytes == sizeof(*a), "cache_attention: struct of %zu bytes, not %zu",
              a ? a->struct_bytes : (size_t)0, sizeof(*a));
  T2T_REQUIRE(a->dtype == T2T_F16 || a->dtype == T2T_BF16, "cache_attention: dtype %d", a->dtype);
  T2T_REQUIRE(a->D == 64 || a->D == 128, "cache_attention: D=%d (64 or 128)", a->D);
  T2T_REQUIRE(a->HK >= 1 && a->HQ >= 1 && a->HQ <= 65536 && a->HQ % a->HK == 0, "cache_attention: %d heads over %d",
              a->HQ, a->HK);
  T2T_REQUIRE(a->B >= 0 && a->B <= (1 << 20) && a->N >= 0 && (a->offsets || (long long)a->B * a->N <= INT_MAX),
              "cache_attention: B=%d N=%d", a->B, a->N);
  const long long T = a->offsets ? a->N : (long long)a->B * a->N;
  if (T == 0 || a->B == 0) return T2T_OK;
  T2T_REQUIRE(T * a->HQ <= INT_MAX, "cache_attention: %lld rows of %d heads", T, a->HQ);
  T2T_REQUIRE(a->pages >= 1 && a->page_size >= 1 && a->width >= 0 && (long long)a->width * a->page_size <= INT_MAX - 64,
              "cache_attention: %d pages of %d, %d a sequence", a->pages, a->page_size, a->width);
  T2T_REQUIRE(a->scale > 0.f && a->scale < __builtin_inff(), "cache_attention: scale %g", a->scale);
  T2T_REQUIRE(!(a->mask && a->causal), "cache_attention: a mask and causal");
  T2T_REQUIRE(!a->mask || a->mask_cols >= 0, "cache_attention: mask of %d columns", a->mask_cols);
  T2T_REQUIRE(a->q && a->k && a->v && a->out && a->lengths && (a->table || a->width == 0),
              "cache_attention: null pointer");
  const long long strides = a->q_batch | a->q_row | a->q_head | a->out_batch | a->out_row | a->out_head | a->kv_page |
                            a->kv_row | a->kv_head;
  T2T_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) % 16 == 0 && strides % 8 == 0,
              "cache_attention: rows must be 16-byte aligned");
  T2T_REQUIRE(a->kv_page >= 0 && a->kv_row >= 0 && a->kv_head >= 0 && a->kv_page <= (1LL << 40) && a->kv_row <= (1LL << 40) &&
                  (a->pages - 1) * (__int128)a->kv_page + (a->page_size - 1) * (__int128)a->kv_row < (1LL << 35),
              "cache_attention: one head's keys must span less than 64 GiB");
  CacheArgs A{};
  A.q = (const char*)a->q, A.k = (const char*)a->k, A.v = (const char*)a->v, A.out = (char*)a->out, A.lse = a->lse;
  A.table = a->table, A.lengths = a->lengths, A.offsets = a->offsets, A.mask = a->mask;
  A.q_batch = 2 * a->q_batch, A.q_row = 2 * a->q_row, A.q_head = 2 * a->q_head;
  A.o_batch = 2 * a->out_batch, A.o_row = 2 * a->out_row, A.o_head = 2 * a->out_head;
  A.kv_page = 2 * a->kv_page, A.kv_row = 2 * a->kv_row, A.kv_head = 2 * a->kv_head;
  A.table_row = a->table_row, A.mask_batch = a->mask_batch, A.mask_row = a->mask_row;
  A.B = a->B, A.N = a->N, A.T = (int)T, A.HQ = a->HQ, A.HK = a->HK, A.G = a->HQ / a->HK;
  A.pages = a->pages, A.page = a->page_size, A.width = a->width, A.mask_cols = a->mask_cols, A.causal = a->causal;
  A.shift = (a->page_size & (a->page_size - 1)) ? -1 : __builtin_ctz(a->page_size);
  A.c = a->scale * 1.4426950408889634f;
  const long long tiles = ca_tiles(a->offsets != nullptr, a->B, T, A.G);
  const long long keys = (long long)a->width * a->page_size;
  A.S = ca_split(tiles, a->HK, keys < 1 ? 1 : keys);
  // (as many parts as the workspace holds)
  while (A.S > 1 && (!ws || ws_bytes < ca_ws(A.S, T * a->HQ, a->D))) --A.S;
  if (A.S > 1) {
    T2T_REQUIRE((uintptr_t)ws % 16 == 0, "cache_attention: workspace must be 16-byte aligned");
    A.opart = (float*)ws;
    A.mlpart = A.opart + (size_t)A.S * T * a->HQ * a->D;
  }
  if (tiles * a->HK * A.S > (1 << 23)) {  // 2^31 threads
    t2t_set_error("cache_attention: %lld row blocks of %d heads", tiles, a->HK);
    return T2T_ERR_UNSUPPORTED;
  }
  auto run = [&](auto t, auto d) {
    using TT = decltype(t);
    constexpr int D = decltype(d)::value;
    hipLaunchKernelGGL((ca_few_kernel<TT, D>), dim3((unsigned)(tiles * a->HK * A.S)), dim3(256), 0, (hipStream_t)stream, A);
    if (A.S > 1)
      hipLaunchKernelGGL((ca_combine_kernel<TT, D>), dim3((unsigned)(tiles * a->HK)), dim3(256), 0, (hipStream_t)stream, A);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (a->dtype == T2T_BF16)
    a->D == 64 ? run(BF16T{}, D64{}) : run(BF16T{}, D128{});
  else
    a->D == 64 ? run(F16T{}, D64{}) : run(F16T{}, D128{});
  T2T_LAUNCH_CHECK("cache_attention");
  return T2T_OK;
}
