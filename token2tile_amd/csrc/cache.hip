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

// 1 KB to LDS, 16 bytes a lane in the order of the lanes; ONCE: of what no other work-group reads
// (sixteen tokens over 32,760 keys: 302 us, 326 without).  (In assembly: of the builtin the compiler
// knows no more than that it writes LDS, and has the transposing reads wait for every one in flight.
// The waits and barriers that order them are written out.)
template <bool ONCE = false> __device__ inline void ca_dma(const char* from, uint16_t* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(ca_lds_t*)to);
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(at), "v"(from) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
}

// the same from a scalar base and an offset a lane
__device__ inline void ca_dma_at(const char* base, uint32_t off, uint16_t* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                   __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(ca_lds_t*)to)),
               "v"(off), "s"(base)
               : "memory");
}

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
  int S, target;  // most parts of a sequence's keys; work-groups of a key head that are aimed at
  float* opart;
  float* mlpart;
  int* size;  // keys of a part, as the launch has found it
};

// A sequence's keys go in parts of one size, so that all work-groups have about the same to do. The
// launch finds the size from the lengths themselves (ca_part): a table is as wide as its longest
// sequence may become, above all in a captured graph, and lengths differ (single tokens of 40 heads over
// 8, parts by the lengths and by the table's width: one of 4,000 keys in a table for 65,536 14.1 and 26.6
// us, one of 32,000 keys and fifteen of 1,000 50 and 207; with equal lengths it costs 0.5). CA_PART keys
// at least, a tile of each of two waves.
#define CA_PART 64
#define CA_SPAN 256  // columns of a mask from which on the many-row form searches it
__device__ inline int ca_parts(int size, int L) { return L < 1 ? 1 : (L - 1) / size + 1; }

// A work-group's rows: a row block of ROWS packed rows (token, head of the group) of a sequence.
struct CacheRows {
  int b, n, L, first;   // sequence, its new tokens, keys, older keys
  int r0, rows;         // packed rows from r0 on, how many there are in the sequence
  long long row0;       // its first row among all
};
// sequence b: offsets and lengths are held to what there is
__device__ inline void ca_sequence(const CacheArgs& A, int b, CacheRows& w) {
  w.b = b;
  if (A.offsets) {
    const int lo = min(max(A.offsets[b], 0), A.T), hi = min(max(A.offsets[b + 1], 0), A.T);
    w.row0 = lo, w.n = max(hi - lo, 0);
  } else {
    w.row0 = (long long)b * A.N, w.n = A.N;
  }
  w.rows = w.n * A.G;
  w.L = (int)min((long long)max(A.lengths[b], 0), (long long)A.width * A.page);
  w.first = w.L - w.n;
}
// Row block `tile` of a launch that does not go by the parts: sequence b owns blocks from offsets[b] G
// / ROWS + b on, at least as many as it needs.
template <int ROWS>
__device__ inline bool ca_rows(const CacheArgs& A, int tile, CacheRows& w) {
  const int per = A.offsets ? 0 : (int)(((long long)A.N * A.G + ROWS - 1) / ROWS);
  int b, first;
  if (A.offsets) {
    int count = 0;
    for (int b0 = 0; b0 < A.B; b0 += 64) {
      const int x = b0 + (int)__lane_id();
      const long long off = x < A.B ? min(max(A.offsets[x], 0), A.T) : 0;
      count += __popcll(__ballot(x < A.B && off * A.G / ROWS + x <= tile));
    }
    b = max(count - 1, 0);
    first = (int)((long long)min(max(A.offsets[b], 0), A.T) * A.G / ROWS) + b;
  } else {
    b = tile / per, first = b * per;
  }
  if (b >= A.B) return false;
  ca_sequence(A, b, w);
  w.r0 = (tile - first) * ROWS;
  return w.r0 >= 0 && w.r0 < w.rows;
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
  // log2 of the largest weight as the maximum moves, and the most that a lane's weights of a half tile (16
  // keys) may add up to before it moves again.  Weights are then 1 on average at most, so the sums stay
  // below keys x max |v| (with 2^64 for the limit, values of 2^100 overflowed where scores rose by 45)
  static constexpr float top = -10.f, limit = 16.f;
  static constexpr uint32_t inf = 0x7f80u;
};
template <> struct CaType<F16T> {
  static constexpr float top = 8.f, limit = 0x1p14f;  // (weights down to 2^-22 of the largest keep their bits)
  static constexpr uint32_t inf = 0x7c00u;
};

// ---- 32 keys for 32 rows -----------------------------------------------------
// S^T = K Q^T and O^T = V^T P^T: lane l holds row l % 32 throughout, keys 8 (a / 4)
// + 4 (l / 32) + a % 4 of a 32-key block in element a, dims likewise.
template <typename T, int D>
struct CacheState {
  u32x4 q[D / 16];  // dims 16 s + 8 (l / 32) .. + 7
  f32x16 o[D / 32];
  float m, l;
};

// the four operand parts of 32 keys and a block of dims, from the transposing reads: in a 16-lane group
// lane i gets, in slot k, element i % 4 of the 8 bytes that lane 4 k + i / 4 addresses.  Lane l
// addresses key 8 r + 4 (l / 32) + (l % 16) / 4 at dims 16 ((l / 16) % 2) + 4 (l % 4) .. + 3 and so gets
// dim l % 32 of keys 8 r + 4 (l / 32) + 0 .. 3, the order the weights are packed in.
__device__ inline int ca_trkey(int lane) { return 4 * (lane >> 5) + ((lane & 15) >> 2); }
template <int D> __device__ inline int ca_trat(int lane, int nb) {  // halves; + 8 r D for r
  const int key = ca_trkey(lane), dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  return key * D + 8 * ((4 * nb + (dim >> 3)) ^ ca_vswz<D>(key)) + (dim & 7);
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ inline u32x2 ca_trread(const uint16_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)p));
}

// What the lane's row sees: positions up to `last` (the length's, or under causal its own), and of the
// new ones, with a mask, those it names.
struct CacheSight {
  const uint8_t* mask;  // the row's bytes for new token 0, or NULL
  int first, last, cols;
  // four positions' bytes of the mask, not 0 where they are seen
  __device__ uint32_t peek(int pos) const {
    const int i = pos - first;
    uint32_t x = 0x01010101u;
    if (i >= 0 && i + 3 < cols) {
      __builtin_memcpy(&x, mask + i, 4);
    } else if (i > -4) {
      x = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < 0 || (i + e < cols && mask[i + e])) x |= 1u << (8 * e);
    }
    return x;
  }
  // a bit for each of the 32 positions from base on; raw: peek() of base + 8 g + 4 (lane / 32)
  __device__ uint32_t bits(int base, const uint32_t (&raw)[4]) const {
    uint32_t seen = 0;
    if (mask) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t x = (((raw[g] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | raw[g]) >> 7 & 0x01010101u;
        seen |= (x * 0x01020408u >> 24 & 0xfu) << (8 * g + 4 * (__lane_id() >> 5));
      }
      seen |= half_partner(seen);
    } else {
      seen = 0xffffffffu;
    }
    const int n = last - base + 1;
    return n >= 32 ? seen : n <= 0 ? 0u : seen & ((1u << n) - 1u);
  }
};

// Row blocks and keys of the sequences, a lane each, 64 at a time; up to 64 are loaded once.
template <int ROWS> struct CacheBatch {
  const CacheArgs& A;
  int n, L;
  __device__ CacheBatch(const CacheArgs& a) : A(a), n(0), L(0) {
    if (A.B <= 64) load(0);
  }
  __device__ void load(int b0) {
    const int b = b0 + (int)__lane_id();
    n = L = 0;
    if (b >= A.B) return;
    CacheRows w;
    ca_sequence(A, b, w);
    n = (w.rows + ROWS - 1) / ROWS, L = w.L;
  }
  __device__ void at(int b0) {
    if (A.B > 64) load(b0);
  }
};
// Keys of a part: the smallest size (in CA_PART keys, to a sixteenth) at which the row blocks' parts are
// no more than the launch aims at, and a sequence's no more than the workspace has room for.
template <int ROWS> __device__ inline int ca_part(CacheBatch<ROWS>& s) {
  const CacheArgs& A = s.A;
  if (A.S == 1) return INT_MAX;
  auto units = [&]() { return max(s.L - 1, 0) / CA_PART + 1; };
  // over the lanes; past 2^23 a lane's is enough to be too many (a launch has fewer work-groups)
  auto all = [&](int x) { return wave_sum((int)min((long long)s.n * x, 1ll << 23)); };
  int total = 0, hi = 1;
  for (int b0 = 0; b0 < A.B; b0 += 64) {
    s.at(b0);
    total = min(total + all(units()), 1 << 30);
    hi = max(hi, __builtin_amdgcn_readlane(wave_incl_max(s.n ? units() : 0), 63));
  }
  auto fits = [&](int p) {
    int parts = 0;
    for (int b0 = 0; b0 < A.B; b0 += 64) s.at(b0), parts = min(parts + all((units() + p - 1) / p), 1 << 30);
    return parts <= A.target;
  };
  int lo = max(min((total - 1) / A.target + 1, hi), max((hi - 1) / A.S + 1, 1));
  if (lo < hi && !fits(lo)) {
    ++lo;
    while (hi - lo > lo / 16) {
      const int mid = lo + (hi - lo) / 2;
      if (fits(mid)) hi = mid;
      else lo = mid + 1;
    }
    lo = hi;
  }
  return lo * CA_PART;
}

// Which key head, sequence, part and row block a work-group takes.  Those that there are (row blocks
// times parts of every sequence, which the lanes count) come without gaps, so that the launch's spare
// work-groups are its last: dealt among the others, they left CUs without work while others had two.
// Consecutive work-groups go to the eight XCDs in turn: each takes a run of items, the row blocks of
// one part and key head next to each other, which then share their keys in its L2.  Under causal the
// last row blocks, which see the most, go first: of a uniform batch without parts, and where there are
// fewer key heads and sequences than XCDs, items are dealt one by one, all heads' and sequences' longest
// before their next (8,184 tokens of 24 heads over one: 400 us, 580 in runs, of which an XCD had long ones
// alone; 4 x 2,000 tokens of 16 heads 96 and 118; with as many heads as XCDs a head stays on its XCD).
template <int ROWS>
__device__ inline bool ca_item(const CacheArgs& A, int& part, int& parts, int& kh, CacheRows& w) {
  const int lane = __lane_id();
  auto blocks = [&](const CacheRows& x) { return (x.rows + ROWS - 1) / ROWS; };
  if (A.offsets && A.S == 1 && A.B > 64) {
    // (to count many sequences would take longer than a work-group's own part: 4,096 of one token over 200
    // keys 3.3 ms.  Sequence b owns row blocks from offsets[b] G / ROWS + b on, which is at least as many as
    // it needs, and the lanes look for the last one that starts no later)
    const long long tiles = (long long)A.T * A.G / ROWS + A.B;
    const int all = (int)(tiles * A.HK), per = (all + 7) / 8, in = (int)(blockIdx.x >> 3);
    const int id = (int)(blockIdx.x & 7) * per + in;
    if (in >= per || id >= all) return false;
    kh = id / (int)tiles;
    const int local = id - kh * (int)tiles;
    auto start = [&](int b) { return (long long)min(max(A.offsets[b], 0), A.T) * A.G / ROWS + b; };
    int lo = 0, n = A.B;
    while (n > 1) {
      const int step = (n + 63) / 64, at = lane * step;
      const bool on = at < n && start(lo + min(at, n - 1)) <= local;
      const int started = __popcll(__ballot(on)), skip = max(started - 1, 0) * step;
      lo += skip, n = min(step, n - skip);
    }
    ca_sequence(A, lo, w);
    const long long tile = local - start(lo);
    const int n_blocks = blocks(w);
    part = 0, parts = 1;
    w.r0 = (int)(A.causal ? n_blocks - 1 - tile : tile) * ROWS;
    return tile >= 0 && tile < n_blocks;
  }
  const bool alike = !A.offsets && A.S == 1;
  long long each = 0;  // items of a key head
  CacheBatch<ROWS> s(A);
  int size = INT_MAX;
  if (alike) {
    each = (long long)A.B * (((long long)A.N * A.G + ROWS - 1) / ROWS);
  } else {
    size = ca_part(s);
    for (int b0 = 0; b0 < A.B; b0 += 64) s.at(b0), each += wave_sum(s.n * ca_parts(size, s.L));
    if (A.S > 1 && blockIdx.x == 0 && threadIdx.x == 0) *A.size = size;
  }
  if (each * A.HK > gridDim.x) return false;  // (offsets that go back, whose sequences overlap)
  const int all = (int)(each * A.HK), per = (all + 7) / 8, in = (int)(blockIdx.x >> 3);
  const bool deal = A.causal && (alike || A.HK * A.B < 8);
  const int id = deal ? (int)blockIdx.x : (int)(blockIdx.x & 7) * per + in;
  if (in >= per || id >= all) return false;
  kh = deal ? id % A.HK : id / (int)each;
  int local = deal ? id / A.HK : id - kh * (int)each, b = 0;
  if (alike) {
    const int n = (int)each / A.B;
    if (deal) {
      const int x = local / A.B;
      b = local - x * A.B, local = x;
    } else {
      b = local / n, local -= b * n;
    }
  } else {
    for (int b0 = 0; b0 < A.B; b0 += 64) {
      s.at(b0);
      const int n = s.n * ca_parts(size, s.L), end = wave_incl_scan(n), sum = __builtin_amdgcn_readlane(end, 63);
      if (local < sum) {  // (the same for the wave)
        const int at = __ffsll((unsigned long long)__ballot(end > local)) - 1;
        b = b0 + at;
        local -= __builtin_amdgcn_readlane(end, at) - __builtin_amdgcn_readlane(n, at);
        break;
      }
      local -= sum;
    }
  }
  ca_sequence(A, __builtin_amdgcn_readfirstlane(b), w);
  local = __builtin_amdgcn_readfirstlane(local), kh = __builtin_amdgcn_readfirstlane(kh);
  const int n = blocks(w), tile = local % n;
  part = local / n, parts = ca_parts(size, w.L);
  w.r0 = (A.causal ? n - 1 - tile : tile) * ROWS;
  return true;
}

// s -> weights against the running maximum (exp2 scales exactly, so it only has to keep the weights in
// the range of T: it moves where they leave it, and the sums so far with it).  The many-row kernel's
// weigh() and settle() are the same steps between its products: they change together.
template <typename T, int D>
__device__ inline void ca_weights(CacheState<T, D>& w, const f32x16& s, u32x4 (&p)[2], float c) {
  auto expo = [&](float nm) __attribute__((always_inline)) {
    float acc = 0.f;
#pragma unroll
    for (int a = 0; a < 16; a += 2) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[a], c, nm));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[a + 1], c, nm));
      acc += p0 + p1;
      p[a / 8][(a % 8) / 2] = Pk<T>::pack(p0, p1);
    }
    return acc;
  };
  float lt = expo(-w.m);
  if (__builtin_amdgcn_readfirstlane((int)(__ballot(!(lt <= CaType<T>::limit)) != 0ull))) {
    float mr = -__builtin_inff();
#pragma unroll
    for (int a = 0; a < 16; ++a) mr = __builtin_elementwise_maximum(mr, s[a]);
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
template <typename T, int N>
__device__ inline bool ca_clean(u32x2 (&f)[N]) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t lo = (f[i][e] & CaType<T>::inf) == CaType<T>::inf ? 0u : f[i][e] & 0xffffu;
      const uint32_t hi = (f[i][e] >> 16 & CaType<T>::inf) == CaType<T>::inf ? 0u : f[i][e] & 0xffff0000u;
      any |= (lo | hi) != f[i][e];
      f[i][e] = lo | hi;
    }
  return any;
}

// D / 8 dims from d0 on of packed row r, of a part of its keys or (part < 0) of all: the sums, or the
// result
template <typename T, int D>
__device__ inline void ca_row(const CacheArgs& A, const CacheRows& w, int kh, int r, int part, float m, float l, int d0,
                              const float (&o)[D / 8]) {
  const int tok = r / A.G, head = kh * A.G + r - tok * A.G;
  const long long at = (w.row0 + tok) * A.HQ + head;
  if (part >= 0) {
    const long long pr = (long long)part * A.T * A.HQ + at;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      *(f32x4*)(A.opart + pr * D + d0 + 4 * i) = f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
    if (d0 == 0) A.mlpart[2 * pr] = m, A.mlpart[2 * pr + 1] = l;
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* dst = (char*)ca_token(A.out, A, w, A.o_batch, A.o_row, tok) + head * A.o_head + 2 * d0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    *(u32x4*)(dst + 16 * i) =
        u32x4{Pk<T>::pack(o[8 * i] * inv, o[8 * i + 1] * inv), Pk<T>::pack(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
              Pk<T>::pack(o[8 * i + 4] * inv, o[8 * i + 5] * inv), Pk<T>::pack(o[8 * i + 6] * inv, o[8 * i + 7] * inv)};
  if (A.lse && d0 == 0) A.lse[at] = l == 0.f ? -__builtin_inff() : 0.6931471805599453f * (m + __log2f(l));
}

// ---- few rows: a work-group's waves take the keys in turn --------------------
// 32 packed rows a work-group, 32 keys a tile; a wave fetches its own tiles (DMA to
// its own LDS, one ahead) and keeps sums of its own, which meet at the end.  Where
// the row blocks are few, a sequence's keys go in parts to several work-groups,
// whose sums ca_combine_kernel joins.  Two waves a work-group, two work-groups a CU:
// one's start and end pass under the other's loads.  Bound: reading the cache (sixteen
// tokens of 40 heads over up to 32,760 keys of 8: 286 us, 5.7 TB/s).
template <typename T, int D>
__global__ __launch_bounds__(128, 1) void ca_few_kernel(CacheArgs A) {
  constexpr int WAVES = 2, TILE = 32 * D, LPR = D / 8, RPI = 64 / LPR;  // lanes a row, rows an instruction
  __shared__ __attribute__((aligned(1024))) uint16_t sK0[WAVES * TILE], sK1[WAVES * TILE];
  __shared__ __attribute__((aligned(1024))) uint16_t sV0[WAVES * TILE], sV1[WAVES * TILE];
  __shared__ float sM[WAVES][32], sL[WAVES][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int jl = lane & 31, hh = lane >> 5;
  int part, parts, kh;
  CacheRows w;
  if (!ca_item<32>(A, part, parts, kh, w)) return;
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
      ca_dma<true>(kbase + at + 16 * ((lane & (LPR - 1)) ^ ca_kswz<D>(row)), dk + i * 512);
      ca_dma<true>(vbase + at + 16 * ((lane & (LPR - 1)) ^ ca_vswz<D>(row)), dv + i * 512);
    }
  };
  // BAD: lanes whose key's table entry lies outside the cache
  auto step = [&](int t, uint64_t bad, auto BUF) __attribute__((always_inline)) {
    const uint16_t* sk = (decltype(BUF)::value ? sK1 : sK0) + wave * TILE;
    const uint16_t* sv = (decltype(BUF)::value ? sV1 : sV0) + wave * TILE;
    f32x16 s = zero16();
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      s = Mfma<T>::run(*(const u32x4*)(sk + jl * D + 8 * ((2 * i + hh) ^ ca_kswz<D>(jl))), st.q[i], s);
    const bool hide = 32 * t + 32 > (masked ? w.first : w.L) || bad;  // (of the wave)
    uint32_t seen = 0;  // by the lane's row
    if (hide) {
      uint32_t raw[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) raw[g] = A.mask ? sight.peek(32 * t + 8 * g + 4 * hh) : 0u;
      seen = sight.bits(32 * t, raw) & ~(uint32_t)bad;
#pragma unroll
      for (int a = 0; a < 16; ++a)
        if (!(seen >> (8 * (a / 4) + 4 * hh + a % 4) & 1)) s[a] = -__builtin_inff();
    }
    u32x4 p[2];
    ca_weights<T, D>(st, s, p, A.c);
    bool odd = false;
#pragma unroll
    for (int nb = 0; nb < D / 32; ++nb) {
      u32x2 f[4];
      const uint16_t* at = sv + ca_trat<D>(lane, nb);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = ca_trread(at + 8 * i * D);
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
  auto sums = [&](int x) { return (float*)(x ? sK1 : sK0); };
  float* to = sums(wave);
#pragma unroll
  for (int nb = 0; nb < D / 32; ++nb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int ch = (8 * nb + 2 * g + hh) ^ (jl & 15);
      *(f32x4*)(to + jl * D + 4 * ch) = f32x4{st.o[nb][4 * g] * mine, st.o[nb][4 * g + 1] * mine,
                                              st.o[nb][4 * g + 2] * mine, st.o[nb][4 * g + 3] * mine};
    }
  __syncthreads();
  if (wave == 0 && hh == 0) sM[0][jl] = M, sL[0][jl] = total;
  __syncthreads();
  // a row by eight threads, D / 8 dims each
  for (int rr = threadIdx.x >> 3; rr < 32; rr += 8 * WAVES) {
    if (w.r0 + rr >= w.rows) return;
    const int d0 = (threadIdx.x & 7) * (D / 8);
    float o[D / 8];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int ch = 4 * ((d0 / 4 + i) ^ (rr & 15));
      const f32x4 x = *(const f32x4*)(sums(0) + rr * D + ch) + *(const f32x4*)(sums(1) + rr * D + ch);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[4 * i + e] = x[e];
    }
    ca_row<T, D>(A, w, kh, w.r0 + rr, parts > 1 ? part : -1, sM[0][rr], sL[0][rr], d0, o);
  }
}

// The products of the pipeline below, with the sums and the queries in accumulation registers (the
// compiler's choice moved them back and forth).  Two wait states come before each:
// the compiler may have moved an operand just before, and does not know what this is.  Who reads a
// result waits, or comes two products later.
#define CA_MFMA(dst, c, dst_, q_)                                                                       \
  if constexpr (T::code == T2T_BF16)                                                                    \
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, " c : dst_(dst) : "v"(a), q_(b));               \
  else                                                                                                  \
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, " c : dst_(dst) : "v"(a), q_(b))
template <typename T> __device__ inline void ca_mfma_sum(f32x16& c, const u32x4& a, const u32x4& b) {
  CA_MFMA(c, "%0", "+a", "v");
}
template <typename T, bool FIRST>
__device__ inline void ca_mfma_score(f32x16& c, const u32x4& a, const u32x4& b) {
  if constexpr (FIRST) { CA_MFMA(c, "0", "=&v", "a"); }
  else { CA_MFMA(c, "%0", "+v", "a"); }
}
#undef CA_MFMA

// The new tokens that all of a work-group's tokens tok0 .. tok1 see, up to the first that one does not,
// and one behind the last that any sees: columns of the mask's rows at `rows`, of cols >= 16.  A wave
// takes every W-th row, sixteen at once, and a KB of each from either end until it has met its column.
template <int W>
__device__ inline void ca_span(const uint8_t* rows, long long stride, int count, int cols, int (&sFirst)[W],
                               int (&sLast)[W], int& first, int& last) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto flags = [](uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u; };  // of bytes that are not 0
  constexpr int AT_ONCE = 16;
  auto gather = [&](int col, uint32_t (&every)[4], uint32_t (&any)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) every[e] = ~0u, any[e] = 0u;
    for (int r = wave; r < count; r += AT_ONCE * W) {
      u32x4 x[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) __builtin_memcpy(&x[i], rows + min(r + i * W, count - 1) * stride + col, 16);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t y = flags(x[i][e]);
          every[e] &= y, any[e] |= y;
        }
    }
  };
  int lo = cols, hi = 0;
  uint32_t every[4], any[4];
  auto behind = [&](int col) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (any[e]) hi = col + 4 * e + 4 - (__builtin_clz(any[e]) >> 3);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) hi = max(hi, __shfl_xor(hi, d, 64));
  };
  for (int b = 0; b < cols && lo == cols; b += 1024) {
    const int col = min(b + 16 * lane, cols - 16);
    gather(col, every, any);
#pragma unroll
    for (int e = 3; e >= 0; --e) {
      const uint32_t none = ~every[e] & 0x80808080u;
      if (none) lo = col + 4 * e + (__builtin_ctz(none) >> 3);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) lo = min(lo, __shfl_xor(lo, d, 64));
    if (cols <= 1024) behind(col);  // (all columns at once)
  }
  for (int b = cols; cols > 1024 && b > 0 && hi == 0; b -= 1024) {
    const int col = max(b - 1024 + 16 * lane, 0);
    gather(col, every, any);
    behind(col);
  }
  if (lane == 0) sFirst[wave] = lo, sLast[wave] = hi;
  __syncthreads();
  first = cols, last = 0;
#pragma unroll
  for (int x = 0; x < W; ++x) first = min(first, sFirst[x]), last = max(last, sLast[x]);
  first = __builtin_amdgcn_readfirstlane(first), last = __builtin_amdgcn_readfirstlane(last);
}

// ---- many rows: a work-group's waves share the keys --------------------------
// 32 W packed rows a work-group of W waves; tiles of 64 keys, fetched by all waves for
// all (DMA, one barrier a tile).  Tiles of which every row sees every key go through a
// pipeline of half tiles: a turn computes the scores of the next half, the weights of
// this one and the sums of the last, product by product with the weights' vector
// operations between them, so that the matrix unit has work while the exponentials
// are taken.  The other tiles follow, one after the other.  Under a mask the pipeline
// goes on through the new tokens that all of the work-group's rows see, and the tiles
// behind the last that one of them sees are not fetched (4,096 tokens in eight frames
// over 8,192 keys, 16 heads: 246 us, 479 with every tile of new tokens looked through).
// Eight waves of 32 rows, two to a SIMD (four of 64 rows take the same time, one of 32 to
// a SIMD 9% more): the queries and sums are in accumulation registers.  Bound: a turn's
// sixteen products are 512 cycles of the matrix unit, its exponentials 140 of the vector
// unit's beside them; the matrix units are busy for 62% of the cycles, and the clock falls
// to 1.75 GHz under the load (4,680 tokens over 32,760 keys, 40 heads: 2.7 to 2.85 ms, 1.1
// to 1.17 PFLOP/s; a large library product in bf16 1.35 to 1.6).
template <typename T, int D, int W, bool P16>
__global__ __launch_bounds__(64 * W, 2) void ca_many_kernel(CacheArgs A) {
  constexpr int ROWS = 32 * W, LPR = D / 8, RPI = 64 / LPR, NB = D / 32, NS = D / 16;
  constexpr int KW = 64 / W, IPW = KW / RPI;  // keys of a tile that a wave fetches, in so many instructions
  static_assert(IPW >= 1, "whole instructions");
  constexpr int NBUF = 2;  // tiles that are kept (three gained nothing)
  __shared__ __attribute__((aligned(1024))) uint16_t sK[NBUF * 64 * D], sV[NBUF * 64 * D];
  __shared__ uint32_t sBad[2][W];  // a wave's keys whose table entry lies outside the cache
  __shared__ uint32_t sOdd[2][W];  // whether its values hold an inf or NaN
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int jl = lane & 31, hh = lane >> 5;
  int part, parts, kh;
  CacheRows w;
  if (!ca_item<ROWS>(A, part, parts, kh, w)) return;
  const int wr0 = w.r0 + 32 * wave;  // the wave's first row
  const bool live = wr0 < w.rows;    // (of the wave)
  u32x4 q[NS];
  f32x16 o[NB];
  float m = CA_NONE, l = 0.f;
  // the lane's row (looked up again after the pipeline, which has no registers to spare)
  auto row_of = [&](int& tok, int& head) {
    int x = wr0 + jl;
    asm volatile("" : "+v"(x));
    x = min(x, w.rows - 1);
    tok = x / A.G, head = kh * A.G + x - tok * A.G;
  };
  {
    int tok, head;
    row_of(tok, head);
    const char* qr = ca_token(A.q, A, w, A.q_batch, A.q_row, tok) + head * A.q_head + 16 * hh;
#pragma unroll
    for (int s = 0; s < NS; ++s) q[s] = *(const u32x4*)(qr + 32 * s);
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) o[nb] = zero16();
  // keys that some row of the work-group sees; from `plain` on not every row sees every key
  const int tok0 = w.r0 / A.G, tok1 = (min(w.r0 + ROWS, w.rows) - 1) / A.G;
  const int keys = A.causal ? min(w.L, w.first + tok1 + 1) : w.L;
  int plain = max(0, A.mask ? w.first : A.causal ? w.first + tok0 + 1 : w.L);
  const int all = max(0, (keys + 63) / 64);
  const int t0 = __builtin_amdgcn_readfirstlane((int)((long long)part * all / parts));
  int nt = __builtin_amdgcn_readfirstlane((int)((long long)(part + 1) * all / parts)) - t0;
  const int cols = min(A.mask_cols, w.n);
  if (A.mask && 64 * (t0 + nt) > w.first) {
    __shared__ int sFirst[W], sLast[W];
    int c0 = 0, c1 = cols;
    if (cols >= CA_SPAN)  // (fewer are not worth the search)
      ca_span<W>(A.mask + (A.offsets ? (w.row0 + tok0) * A.mask_row : w.b * A.mask_batch + tok0 * A.mask_row), A.mask_row,
                 tok1 - tok0 + 1, cols, sFirst, sLast, c0, c1);
    plain = max(0, w.first + c0);
    nt = max(0, min(nt, (max(0, w.first + c1) + 63) / 64 - t0));
  }
  const char* kbase = A.k + kh * A.kv_head;
  const char* vbase = A.v + kh * A.kv_head;
  const int32_t* table = A.table + w.b * A.table_row;
  // tiles of the pipeline: none where an entry of the table lies outside the cache
  int nf = min(nt, max(0, plain / 64 - t0));
  {
    bool bad = false;
    const int e0 = nf > 0 ? 64 * t0 / A.page : 0, e1 = nf > 0 ? (64 * (t0 + nf) - 1) / A.page : -1;
    for (int e = e0 + threadIdx.x; e <= e1; e += 64 * W) bad |= (uint32_t)table[e] >= (uint32_t)A.pages;
    if (__syncthreads_or(bad)) nf = 0;
    nf = __builtin_amdgcn_readfirstlane(nf);
  }

  // this wave fetches keys KW wave .. of every tile; lane l looks key l % KW up
  auto pos_of = [&](int t) { return min(64 * (t0 + t) + KW * wave + (lane & (KW - 1)), w.L - 1); };
  // with P16 sixteen keys lie in one page, one stride apart: a scalar base, and offsets that stay
  uint32_t koff[P16 ? IPW : 1], voff[P16 ? IPW : 1];
  if constexpr (P16) {
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
      const int in = RPI * i + lane / LPR, row = KW * wave + in;
      koff[i] = (uint32_t)(in * A.kv_row) + 16 * ((lane & (LPR - 1)) ^ ca_kswz<D>(row));
      voff[i] = (uint32_t)(in * A.kv_row) + 16 * ((lane & (LPR - 1)) ^ ca_vswz<D>(row));
    }
  }
  using Yes = std::true_type;
  using No = std::false_type;
  // 1 KB of a tile's keys (values) to LDS: off is where the wave's keys lie (P16) or the lane's key
  auto one = [&](const char* base, uint16_t* to, auto off, int i, auto KEYS) __attribute__((always_inline)) {
    to += (KW * wave + RPI * i) * D;
    if constexpr (sizeof(off) == 8) {
      ca_dma_at(base + off, decltype(KEYS)::value ? koff[P16 ? i : 0] : voff[P16 ? i : 0], to);
    } else {
      const int in = RPI * i + lane / LPR, row = KW * wave + in;
      const size_t at = (size_t)(uint32_t)__shfl((int)off, in, 64) * 16;
      const int swz = decltype(KEYS)::value ? ca_kswz<D>(row) : ca_vswz<D>(row);
      ca_dma(base + at + 16 * ((lane & (LPR - 1)) ^ swz), to);
    }
  };
  auto whole = [&](const char* base, uint16_t* to, auto off, auto KEYS) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < IPW; ++i) one(base, to, off, i, KEYS);
  };
  // where the lane's operands lie (halves): K of step s, V of dim block nb
  int ka[NS], va[NB];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    ka[s] = jl * D + 8 * ((2 * s + hh) ^ ca_kswz<D>(jl));
    asm volatile("" : "+v"(ka[s]));  // (one register each: not put together again at every read)
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    va[nb] = ca_trat<D>(lane, nb);
    asm volatile("" : "+v"(va[nb]));
  }
  auto kat = [&](int s) { return ka[s]; };
  auto vat = [&](int nb) { return va[nb]; };
  // weight pair i of 8: elements 2 i, + 1
  auto weigh = [&](int i, const f32x16& S, u32x4 (&P)[2], float& lt) __attribute__((always_inline)) {
    const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * i], A.c, -m));
    const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * i + 1], A.c, -m));
    lt += x0 + x1;
    P[i / 4][i % 4] = Pk<T>::pack(x0, x1);
  };
  // the sums are in accumulation registers, written by the assembly below, whose results are
  // readable after 18 cycles of issue
  auto ready = [&]() __attribute__((always_inline)) {
    asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) asm volatile("" : "+a"(o[nb]));
  };
  // a half tile's weights have left the range: the maximum moves, and they are taken again (as in
  // ca_weights)
  auto settle = [&](const f32x16& S, u32x4 (&P)[2], float& lt) __attribute__((always_inline)) {
    if (__ballot(!(lt <= CaType<T>::limit))) {
      ready();
      float mr = -__builtin_inff();
#pragma unroll
      for (int a = 0; a < 16; ++a) mr = __builtin_elementwise_maximum(mr, S[a]);
      const float mx = half_max(mr) * A.c - CaType<T>::top;
      const float mnew = mx > m || mx != mx ? mx : m;
      const float alpha = __builtin_amdgcn_exp2f(m - mnew);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int a = 0; a < 16; ++a) o[nb][a] *= alpha;
      lt = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) weigh(i, S, P, lt);
    }
    l += lt;
  };
  auto scores = [&](f32x16& S, const uint16_t* kt) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < NS; ++s) S = Mfma<T>::run(*(const u32x4*)(kt + kat(s)), q[s], s ? S : zero16());
  };
  // One turn: S of this half tile's scores -> P, the scores SX of the half tile in kt, the sums of the
  // one in vt with its weights PP.  Operands are read AHEAD steps before their products; the first
  // ones by the turn before, which at `mid`, with all its own reads done, meets the other waves where
  // the next turn's tiles have to be there.  extra(i): what else step i issues.
  constexpr int AHEAD = 3, STEPS = NS;
  static_assert(NS == 2 * NB && STEPS % (AHEAD + 1) == 0, "the ring of operands goes on from turn to turn");
  u32x4 kf[AHEAD + 1];
  u32x2 vf[AHEAD + 1][2];
  auto rdk = [&](const uint16_t* kt, int i) __attribute__((always_inline)) {
    kf[i % (AHEAD + 1)] = *(const u32x4*)(kt + kat(i));
  };
  auto rdv = [&](const uint16_t* vt, int i) __attribute__((always_inline)) {
    const uint16_t* at = vt + vat(i / 2) + 16 * (i % 2) * D;
    vf[i % (AHEAD + 1)][0] = ca_trread(at);
    vf[i % (AHEAD + 1)][1] = ca_trread(at + 8 * D);
  };
  auto turn = [&](const f32x16& S, f32x16& SX, u32x4 (&P)[2], const u32x4 (&PP)[2], const uint16_t* kt,
                  const uint16_t* vt, const uint16_t* kn, const uint16_t* vn, auto mid, auto extra)
      __attribute__((always_inline)) {
    float lt = 0.f, x0[2], x1[2];
    // the weights' operations, a slot behind each product: of pair j the products and the first
    // exponential, then the second, with the packing and sum of the pair before (in ordinary
    // additions: a dot product of the packed pair waits for the matrix unit)
    constexpr int EACH = 2 * STEPS / 8;  // slots of a pair: 2 (D = 128), 1
    auto pack = [&](int j) __attribute__((always_inline)) { P[j / 4][j % 4] = Pk<T>::pack(x0[j & 1], x1[j & 1]); };
    auto slot = [&](int n) __attribute__((always_inline)) {
      const int j = n / EACH;
      if (EACH == 1 || n % 2 == 0) {
        x0[j & 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * j], A.c, -m));
        x1[j & 1] = __builtin_fmaf(S[2 * j + 1], A.c, -m);
        if (j) pack(j - 1);
      }
      if (EACH == 1 || n % 2 == 1) {
        x1[j & 1] = __builtin_amdgcn_exp2f(x1[j & 1]);
        if (j) lt += x0[(j - 1) & 1] + x1[(j - 1) & 1];
      }
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i == STEPS - AHEAD) mid();
      rdk(i + AHEAD < STEPS ? kt : kn, (i + AHEAD) % STEPS);
      rdv(i + AHEAD < STEPS ? vt : vn, (i + AHEAD) % STEPS);
      extra(i);
      __builtin_amdgcn_sched_barrier(0);
      if (i == 0) ca_mfma_score<T, true>(SX, kf[0], q[0]);
      else ca_mfma_score<T, false>(SX, kf[i % (AHEAD + 1)], q[i]);
      __builtin_amdgcn_sched_barrier(0);
      slot(2 * i);
      const u32x2 f0 = vf[i % (AHEAD + 1)][0], f1 = vf[i % (AHEAD + 1)][1];
      ca_mfma_sum<T>(o[i / 2], u32x4{f0[0], f0[1], f1[0], f1[1]}, PP[i % 2]);
      __builtin_amdgcn_sched_barrier(0);
      slot(2 * i + 1);
    }
    pack(7);
    lt += x0[1] + x1[1];
    settle(S, P, lt);
  };

  if (nf > 0) {
    f32x16 s0, s1;
    u32x4 p0[2], p1[2];
    // (tiles past the last of the pipeline are fetched like it, and not used)
    auto last = [&](int t) { return min(t, nf - 1); };
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+a"(q[s]));
    // where the wave's keys of a tile lie.  P16: its entry is a lane's of `entries`, those of tiles t0 +
    // 64 i + lane, which are loaded once in 64 tiles
    int first = 0;
    uint32_t entries = 0;
    auto look = [&](int t) {
      first = t;
      entries = ca_entry(A, table, 64 * (t0 + last(t + lane)) + KW * wave);
      asm volatile("" : "+v"(entries));  // (waited for here, not wherever it may be needed)
    };
    auto find = [&](int t) {
      if constexpr (P16) {
        if (t >= first + 64) look(t);
        const uint32_t entry = __builtin_amdgcn_readlane(entries, t - first);
        const int pos = 64 * (t0 + last(t)) + KW * wave;
        return (long long)entry * A.kv_page + (A.shift >= 0 ? pos & (A.page - 1) : pos % A.page) * A.kv_row;
      } else {
        bool ok;
        const int pos = pos_of(last(t));
        return ca_offset(A, ca_entry(A, table, pos), pos, ok);
      }
    };
    if constexpr (P16) look(0);
    // K of tile s + NBUF and V of tile s + NBUF - 1, the ones that round s asks for; offv: where the
    // latter lies
    auto offv = find(0), offk = offv;
    whole(kbase, sK, offk, Yes{});
#pragma unroll
    for (int s = 1 - NBUF; s < 0; ++s) {
      offk = find(s + NBUF);
      whole(kbase, sK + (s + NBUF) * 64 * D, offk, Yes{});
      whole(vbase, sV + (s + NBUF - 1) * 64 * D, offv, No{});
      offv = offk;
    }
    // before the first half tile: values and weights of zero
    for (int i = threadIdx.x; i < 8 * D; i += 64 * W) *(u32x4*)(sV + (NBUF - 1) * 64 * D + 8 * i) = u32x4{0u, 0u, 0u, 0u};
    p1[0] = p1[1] = u32x4{0u, 0u, 0u, 0u};
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NBUF - 1) * 2 * IPW) : "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the zeros
    __builtin_amdgcn_s_barrier();
    if (live) {
      scores(s0, sK);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) rdk(sK + 32 * D, i), rdv(sV + (NBUF - 1) * 64 * D + 32 * D, i);
    }
    // every wave's reads of the tiles before are done, and the loads that have to be there are
    auto meet = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NBUF - 2) * 2 * IPW) : "memory");
    };
    auto nothing = [&](int) __attribute__((always_inline)) {};
    auto none = [&]() __attribute__((always_inline)) {};
    // tile t, in buffer B, whose first half's scores are there
    auto round = [&](int t, auto BUF) __attribute__((always_inline)) {
      constexpr int B = decltype(BUF)::value, BX = (B + 1) % NBUF, BW = (B + NBUF - 1) % NBUF;
      uint16_t *kt = sK + B * 64 * D, *kx = sK + BX * 64 * D, *vt = sV + B * 64 * D, *vw = sV + BW * 64 * D;
      offk = find(t + NBUF);
      if (live) turn(s0, s1, p0, p1, kt + 32 * D, vw + 32 * D, kx, vt, meet, nothing);
      else meet();
      auto ask = [&](int i) __attribute__((always_inline)) {
        if (i < IPW) one(kbase, kt, offk, i, Yes{}), one(vbase, vw, offv, i, No{});
      };
      if (live) {
        turn(s1, s0, p1, p0, kx, vt, kx + 32 * D, vt + 32 * D, none, ask);
      } else {
#pragma unroll
        for (int i = 0; i < IPW; ++i) ask(i);
      }
      offv = offk;
    };
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    for (int t = 0; t < nf; t += 2) {
      round(t, B0{});
      if (t + 1 < nf) round(t + 1, B1{});
    }
    // the last half tile's sums
    if (live) {
      const uint16_t* vt = sV + ((nf - 1) % NBUF * 64 + 32) * D;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mm = 0; mm < 2; ++mm) {
          const uint16_t* at = vt + vat(nb) + 16 * mm * D;
          const u32x2 f0 = ca_trread(at), f1 = ca_trread(at + 8 * D);
          ca_mfma_sum<T>(o[nb], u32x4{f0[0], f0[1], f1[0], f1[1]}, p1[mm]);
        }
      ready();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }

  // ---- tiles with hidden keys: those of a row are not seen, and an inf or NaN among their values
  // (left out of the products, where a weight of 0 would make it NaN) goes to the rows that see it
  int tok, head;
  row_of(tok, head);
  if (nf < nt) {
    const CacheSight sight{
        A.mask ? A.mask + (A.offsets ? (w.row0 + tok) * A.mask_row : w.b * A.mask_batch + tok * A.mask_row) : nullptr,
        w.first, A.causal ? w.first + tok : w.L - 1, A.mask_cols};
    auto at = [&](uint16_t* x, int t) { return x + (t & 1) * 64 * D; };
    uint32_t raw[2][4] = {};
    auto ask = [&](int t) __attribute__((always_inline)) {
      bool ok;
      const uint32_t off = ca_offset(A, ca_entry(A, table, pos_of(t)), pos_of(t), ok);
      const uint64_t bad = __ballot(!ok);
      if (lane == 0) sBad[t & 1][wave] = (uint32_t)bad & ((1u << KW) - 1u);
      whole(kbase, at(sK, t), off, Yes{});
      whole(vbase, at(sV, t), off, No{});
      if (A.mask)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int g = 0; g < 4; ++g) raw[kb][g] = sight.peek(64 * (t0 + t) + 32 * kb + 8 * g + 4 * hh);
    };
    auto hidden = [&](uint32_t seen, bool odd, f32x16& S, const uint16_t* vt) __attribute__((always_inline)) {
      u32x4 P[2];
#pragma unroll
      for (int a = 0; a < 16; ++a)
        if (!(seen >> (8 * (a / 4) + 4 * hh + a % 4) & 1)) S[a] = -__builtin_inff();
      float lt = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) weigh(i, S, P, lt);
      settle(S, P, lt);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mm = 0; mm < 2; ++mm) {
          const uint16_t* x = vt + vat(nb) + 16 * mm * D;
          u32x2 f[2] = {ca_trread(x), ca_trread(x + 8 * D)};
          if (odd) ca_clean<T>(f);
          o[nb] = Mfma<T>::run(u32x4{f[0][0], f[0][1], f[1][0], f[1][1]}, P[mm], o[nb]);
        }
      if (odd) {
        for (int j = 0; j < 32; ++j)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int a = 0; a < 16; ++a) {
              const int d = 32 * nb + 8 * (a / 4) + 4 * hh + a % 4;
              const uint16_t u = vt[j * D + 8 * ((d >> 3) ^ ca_vswz<D>(j)) + (d & 7)];
              if ((u & CaType<T>::inf) == CaType<T>::inf && (seen >> j & 1)) o[nb][a] += T::to_f(u);
            }
      }
    };
    ask(nf);
    for (int t = nf; t < nt; ++t) {
      uint32_t seen[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) seen[kb] = sight.bits(64 * (t0 + t) + 32 * kb, raw[kb]);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      {  // (this wave's own keys have landed)
        u32x2 v[KW * D / 256];
#pragma unroll
        for (int i = 0; i < KW * D / 256; ++i) v[i] = *(const u32x2*)(at(sV, t) + KW * wave * D + 256 * i + 4 * lane);
        const uint64_t any = __ballot(ca_clean<T>(v));
        if (lane == 0) sOdd[t & 1][wave] = any != 0;
      }
      __syncthreads();
      uint32_t bad[2] = {0, 0}, odd = 0;
#pragma unroll
      for (int x = 0; x < W; ++x) bad[x / (W / 2)] |= sBad[t & 1][x] << (KW * (x % (W / 2))), odd |= sOdd[t & 1][x];
      if (t + 1 < nt) ask(t + 1);
      seen[0] &= ~bad[0], seen[1] &= ~bad[1];
      if (!live) continue;
      if constexpr (D == 128) {  // (no registers for both halves' scores)
#pragma clang loop unroll(disable)
        for (int kb = 0; kb < 2; ++kb) {
          const uint32_t see = kb ? seen[1] : seen[0];
          if (!__ballot(see != 0)) continue;
          f32x16 S;
          scores(S, at(sK, t) + 32 * kb * D);
          hidden(see, __builtin_amdgcn_readfirstlane(odd), S, at(sV, t) + 32 * kb * D);
        }
      } else if (__ballot((seen[0] | seen[1]) != 0)) {
        f32x16 S[2];  // (of both halves in turn, as a product waits for the one before of its half)
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
            S[kb] = Mfma<T>::run(*(const u32x4*)(at(sK, t) + 32 * kb * D + kat(s)), q[s], s ? S[kb] : zero16());
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
          if (__ballot(seen[kb] != 0))
            hidden(seen[kb], __builtin_amdgcn_readfirstlane(odd), S[kb], at(sV, t) + 32 * kb * D);
      }
    }
  }
  if (!live) return;
  const float lt = half_sum(l);
  if (wr0 + jl >= w.rows) return;
  const long long at = (w.row0 + tok) * A.HQ + head;
  if (parts > 1) {
    const long long pr = (long long)part * A.T * A.HQ + at;
    float* op = A.opart + pr * D + 4 * hh;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(op + 32 * nb + 8 * g) = f32x4{o[nb][4 * g], o[nb][4 * g + 1], o[nb][4 * g + 2], o[nb][4 * g + 3]};
    if (hh == 0) A.mlpart[2 * pr] = m, A.mlpart[2 * pr + 1] = lt;
    return;
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  char* dst = (char*)ca_token(A.out, A, w, A.o_batch, A.o_row, tok) + head * A.o_head + 8 * hh;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *(u32x2*)(dst + 64 * nb + 16 * g) = u32x2{Pk<T>::pack(o[nb][4 * g] * inv, o[nb][4 * g + 1] * inv),
                                                Pk<T>::pack(o[nb][4 * g + 2] * inv, o[nb][4 * g + 3] * inv)};
  if (A.lse && hh == 0) A.lse[at] = lt == 0.f ? -__builtin_inff() : 0.6931471805599453f * (m + __log2f(lt));
}

// joins the parts of a row block's rows, 32 lanes a row: a lane weighs two parts and sums D / 32 dims
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(256) void ca_combine_kernel(CacheArgs A) {
  const int kh = blockIdx.x % A.HK, tile = blockIdx.x / A.HK, lane = threadIdx.x & 31;
  CacheRows w;
  if (!ca_rows<ROWS>(A, tile, w)) return;
  const int parts = min(ca_parts(max(*A.size, 1), w.L), A.S), r = w.r0 + 8 * blockIdx.y + (threadIdx.x >> 5);
  if (parts < 2 || r >= w.rows) return;  // (its work-group has written the rows)
  const int tok = r / A.G, head = kh * A.G + r - tok * A.G;
  const long long at = (w.row0 + tok) * A.HQ + head, step = (long long)A.T * A.HQ;
  float m[2], l[2], M, total;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool on = lane + 32 * i < parts;
    const u32x2 v = on ? *(const u32x2*)(A.mlpart + 2 * (at + (lane + 32 * i) * step)) : u32x2{0u, 0u};
    m[i] = on ? __builtin_bit_cast(float, (uint32_t)v[0]) : CA_NONE;
    l[i] = __builtin_bit_cast(float, (uint32_t)v[1]);
  }
  M = __builtin_elementwise_maximum(m[0], m[1]);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) M = __builtin_elementwise_maximum(M, __shfl_xor(M, d, 32));
#pragma unroll
  for (int i = 0; i < 2; ++i) m[i] = __builtin_amdgcn_exp2f(m[i] - M);
  total = m[0] * l[0] + m[1] * l[1];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) total += __shfl_xor(total, d, 32);
  typedef float vec __attribute__((ext_vector_type(D / 32)));
  vec o = {};
  const float* src = A.opart + at * D + D / 32 * lane;
  for (int i = 0; i < parts; i += 8) {
    vec x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = *(const vec*)(src + min(i + e, parts - 1) * step * D);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = __shfl(i < 32 ? m[0] : m[1], (i + e) & 31, 32);  // (0 past the last)
#pragma unroll
      for (int f = 0; f < D / 32; ++f) o[f] = i + e < parts ? __builtin_fmaf(a, x[e][f], o[f]) : o[f];
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  char* dst = (char*)ca_token(A.out, A, w, A.o_batch, A.o_row, tok) + head * A.o_head + D / 16 * lane;
#pragma unroll
  for (int f = 0; f < D / 32; f += 2) *(uint32_t*)(dst + 2 * f) = Pk<T>::pack(o[f] * inv, o[f + 1] * inv);
  if (A.lse && lane == 0) A.lse[at] = total == 0.f ? -__builtin_inff() : 0.6931471805599453f * (M + __log2f(total));
}

// Packed rows of a row block and most parts of a sequence's keys, by the least time of an estimate.
// Measured as graphs of ten launches, us, D = 128:
//   rows a sequence, keys, key heads x sequences     blocks of 32      128      256
//   32, 32,000, 40                                            154      170      199
//   48, 32,000, 40                                            249      158      199
//   128, 32,000, 40                                           414      164      206
//   400, 1,000, 320                                           214      102       90
//   4,680, 32,760, 12                                           -      865      823
// so 32 where a sequence has no more rows, else 128 or 256.  Parts: a work-group alone goes through its
// keys at its latency, so there should be about as many as run at once, but a further round costs its
// own, and the parts' sums are written and read again:
//   1 row, 32,760 keys, 40 heads     S = 6: 165   12 (480 work-groups): 118   13 (520): 164   26: 139
//   1,560 rows, 9,360, 12 (256)      S = 1: 195    2: 121    3 (252 work-groups): 103    4: 138
//   400 rows, 1,000, 320 (256)       S = 1:  90    2: 155
//   1 row, 1,000, 8                  S = 2:  19    8: 12
// The estimate: a key of a work-group takes the longer the more run beside it (they share the memory
// and the power); the constants are fitted to such measurements.
// Under causal the first row blocks see few keys: the longest work-group's time, or their mean's over
// all rounds (8,192 rows over as many keys, 8 heads: S = 1: 193 us, 2: 170).  Tiles with hidden keys
// are not pipelined: `extra` us a work-group, more with more rows, so that short sequences under a mask
// go by 128 (blocks of 128 and 256: 653 rows over as many keys, 27 x 40 heads, D = 64, plain 272 and 279,
// causal 235 and 279; 3,306 rows in frames over as many, 3 x 24 heads, 405 and 457; 4,096 in frames over
// 8,192, 16 heads, 255 and 242).
static double ca_time(int block, long long wgs, int S, double keys, double rows, double mean, double extra) {
  const int slots = block == 256 ? 256 : 512;  // work-groups at once
  auto key = [&](long long n) { return block == 32 ? 22e-3 + 45e-6 * n : block == 128 ? 14e-3 + 30e-6 * n : 20e-3 + 20e-6 * n; };
  const long long n = wgs * S, full = n / slots, rest = n % slots;
  const double part = 64.0 * (long long)((keys / S + 63) / 64), start = (block == 256 ? 5.0 : 2.5) + extra;
  double us = (double)full * (part * key(slots) + start);
  if (rest) us += part * key(rest) + start;
  if (mean < 1.0 && full) us = part * key(slots) * (mean * n > slots ? mean * n / slots : 1.0) + start * n / slots;
  return S < 2 ? us : us + 3.0 + 0.1 * S + 0.23e-3 * S * rows;  // (the join: launched, its loads, its bytes)
}
// row blocks of `block` packed rows
static long long ca_tiles(int block, int ragged, int B, long long T, int G) {
  return ragged ? T * G / block + B : B * ((T / B * G + block - 1) / block);
}
// (those of a ragged batch that hold rows: about as many)
static long long ca_full(int block, int ragged, int B, long long T, int G) {
  const long long n = (T * G + block - 1) / block;
  return ragged ? (n > B ? n : B) : ca_tiles(block, ragged, B, T, G);
}
struct CachePlan {
  int block, S, target;
};
// Whether parts may help.  Past 64 sequences every work-group counts them through memory, several times over,
// which costs more than parts gain where the work-groups are enough without and the keys few (one token a
// sequence over tables of so many keys; us with and without parts, equal and random lengths, and four that
// are eight times the others):
//   sequences, key heads, keys      equal     random    four long
//   256, 1, 1,024                   36   34   32   32   17   29
//   400, 1, 2,048                  114   81   81   67   37   55
//   400, 1, 4,096                  182  148  115  118   47  104
//   2,000, 1, 4,096                820  632  664  368  237  159
//   2,000, 1, 16,384              2580 2433 1657 1451  476  618
//   128, 8, 4,096                  344  330  211  222   88  139
//   400, 8, 4,096                 1084 1042  759  557  356  207
static bool ca_divides(int B, long long wgs, long long keys) {
  return B <= 64 || wgs <= 256 || (wgs < 2048 && keys >= 10LL * B);
}
static CachePlan ca_plan(int ragged, int B, long long T, int HQ, int HK, long long keys, int D, int hidden) {
  const int G = HQ / HK;
  // (of a ragged batch: twice the mean, as its sequences are not known to the host)
  long long rows = (T + B - 1) / B * G * (ragged ? 2 : 1);
  if (rows > T * G) rows = T * G;
  const long long parts = (keys + CA_PART - 1) / CA_PART, most = parts < 1 ? 1 : parts < 64 ? parts : 64;
  CachePlan best{rows <= 32 ? 32 : 128, 1, 0};
  // (what a row block sees on average, of the keys)
  const double mean = hidden == 1 ? 1.0 - 0.5 * (double)rows / G / (double)(keys > rows / G ? keys : rows / G) : 1.0;
  double least = 0.0;
  for (int block = best.block; block <= (rows <= 128 ? best.block : 256); block *= 2) {
    const long long wgs = ca_full(block, ragged, B, T, G) * HK, slots = block == 256 ? 256 : 512;
    const double fresh = (double)(rows / G) / 600.0, wide = block == 256 ? 1.0 : 0.0;
    const double extra = block == 32 || !hidden ? 0.0 : (hidden == 1 ? 7.0 + 1.5 * wide : 20.0 + 13.0 * wide) * (fresh < 1.0 ? fresh : 1.0);
    for (int i = 0; i < 11; ++i) {  // 1, 2, 3 and eighths of all that run at once
      const long long S = i < 3 ? i + 1 : (i - 2) * slots / 8 / wgs;
      if (S < 1 || S > most || (S > 1 && !ca_divides(B, wgs, keys))) continue;
      const double us = ca_time(block, wgs, (int)S, (double)keys, (double)T * HQ, mean, extra);
      if (least == 0.0 || us < least) least = us, best = CachePlan{block, (int)S, 0};
    }
  }
  // work-groups of a key head; the parts' number goes by them, and a long sequence among short ones may
  // take more than its share
  const long long full = ca_full(best.block, ragged, B, T, G);
  best.target = (int)(best.S * full);
  if (B > 1 && (best.S > 1 || (best.block == 32 && full * HK < 2048 && keys >= 2048 && ca_divides(B, full * HK, keys)))) {
    // (where there are enough without parts, a round more of them for the long sequences')
    const long long room = (32 << 20) / (T * HQ * (D + 2) * 4);
    if (best.S == 1) best.target += 512 / HK;
    if (room > best.S) best.S = (int)(room < most ? room : most);
  }
  return best;
}
static size_t ca_ws(int S, long long rows, int D) { return S < 2 ? 0 : (size_t)S * rows * (D + 2) * 4 + 16; }

extern "C" size_t t2t_cache_attention_ws_bytes(int ragged, int hidden, int B, long long T, int HQ, int HK, int D,
                                               long long keys) {
  if (B < 1 || T < 1 || HK < 1 || HQ < HK || keys < 1) return 0;
  return ca_ws(ca_plan(ragged, B, T, HQ, HK, keys, D, hidden).S, T * HQ, D);
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
  T2T_REQUIRE(a->scale > 0.f && a->scale * 1.4426950408889634f < __builtin_inff(), "cache_attention: scale %g", a->scale);
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
  const int ragged = a->offsets != nullptr;
  const long long keys = (long long)a->width * a->page_size;
  const CachePlan plan = ca_plan(ragged, a->B, T, a->HQ, a->HK, keys, a->D, a->causal ? 1 : a->mask ? 2 : 0);
  const int block = plan.block;
  const long long tiles = ca_tiles(block, ragged, a->B, T, A.G);
  A.S = plan.S;
  // (as many parts as the workspace holds)
  while (A.S > 1 && (!ws || ws_bytes < ca_ws(A.S, T * a->HQ, a->D))) --A.S;
  if (A.S > 1) {
    T2T_REQUIRE((uintptr_t)ws % 16 == 0, "cache_attention: workspace must be 16-byte aligned");
    A.opart = (float*)ws;
    A.mlpart = A.opart + (size_t)A.S * T * a->HQ * a->D;
    A.size = (int*)(A.mlpart + (size_t)A.S * T * a->HQ * 2);
  }
  A.target = plan.target;
  // (no more work-groups have anything to do: ca_part's, or one part for every row block)
  const long long most = (A.S > 1 && A.target > tiles ? A.target : tiles) * a->HK;
  if (most > (1 << 22)) {  // 2^31 threads
    t2t_set_error("cache_attention: %lld row blocks of %d heads", tiles, a->HK);
    return T2T_ERR_UNSUPPORTED;
  }
  const int items = (int)most;
  // sixteen keys from a multiple of sixteen on lie in one page, at 32-bit offsets
  const bool p16 = a->page_size % 16 == 0 && A.kv_row < (1 << 27);
  auto run = [&](auto t, auto d) {
    using TT = decltype(t);
    constexpr int D = decltype(d)::value;
    auto go = [&](auto kernel, int threads, auto join) {
      hipLaunchKernelGGL(kernel, dim3((items + 7) / 8 * 8), dim3(threads), 0, (hipStream_t)stream, A);
      if (A.S > 1)
        hipLaunchKernelGGL(join, dim3((unsigned)(tiles * a->HK), block / 8), dim3(256), 0, (hipStream_t)stream, A);
    };
    if (block == 32)
      go(ca_few_kernel<TT, D>, 128, ca_combine_kernel<TT, D, 32>);
    else if (block == 128)
      go(p16 ? ca_many_kernel<TT, D, 4, true> : ca_many_kernel<TT, D, 4, false>, 256, ca_combine_kernel<TT, D, 128>);
    else
      go(p16 ? ca_many_kernel<TT, D, 8, true> : ca_many_kernel<TT, D, 8, false>, 512, ca_combine_kernel<TT, D, 256>);
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
