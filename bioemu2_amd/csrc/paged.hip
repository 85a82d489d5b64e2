// Attention of few queries over a paged cache, for gfx950.
//
//   s(i, j) = cap tanh(scale q_i . k_j / cap) + bias[clamp(j - p_i, -R, R)],   o_i = sum_j softmax_j(s) v_j
//   p_i = length - count + i, keys j <= p_i (causal) or j < length; key j is slot j % page_size of page table[j / page_size]
// (none where the table ends)
//
// The queries of a group of heads that share a key head are the rows of one operand, up to 32 of them, so every key and
// value is read once.  A wave takes tiles of 32 keys (bf16) or 16 (fp32), straight from memory into the operands'
// registers; nothing goes through LDS:
//   S^T = K Q^T by 16 x 16 products: lane (m, h) = (lane & 15, lane >> 4) holds values of key m; the accumulator's
//   lane n is a query, its registers keys 4 h + r, which is the order in which the next product takes them;
//   O^T += V^T P^T: lane (m, h) loads DP / 16 neighbouring values of its 8 (fp32: 4) keys, m choosing which, and value t
//   of every key is the operand of a product of its own, whose row m is then channel (DP / 16) m + t.  In bf16 two keys
//   share a register, which takes one byte permutation for each; in fp32 nothing.
// Weights go into the second product as two bf16 parts (16 bits): the matrix cores have time to spare, and the result is
// then rounded once.
//
// Reading the keys and values bounds it; a stream of 2 GB is read at 6.2 TB/s.  Measured, join included, in bf16: 8 tokens
// over 8200 to 32768 keys, 32/8 heads of 128, 116 us (6.2 TB/s); 64 over up to 4000, 32/4 heads of 128, 65 us (4.8).
// Short caches take the latency of a walk, memory read after memory read (lengths, page table, keys): one token over 773
// keys of 16 heads of 64, 10 us; in fp32 4 x 5 tokens over up to 5000, 16/4 heads of 64, 15 us and a join of 5.
#include <algorithm>

#include "attn.h"
#include "paged_parts.h"

namespace bioemu {
namespace {

constexpr float kRescale = 8.f;   // log2 of the largest weight before the maximum moves

struct PagedArgs {
  const char *keys, *values;
  int64_t kpage, kslot, khead, vpage, vslot, vhead;   // bytes
  const int* page_table;
  int64_t table_stride;
  const int *lengths, *counts;
  int pages, page_size, table_width, blocks;   // blocks of rows a key head
  unsigned div_mul, div_shift;                  // key / page_size = key * div_mul >> div_shift, for keys below 2^28
  bool even;                                    // pages are whole blocks of 16 keys
  int groups, least;                            // workgroups at a time, parts of `least` tiles at least; 0: one an item
};

struct Parts {
  float *o, *ml;   // [slots][rows][D], [slots][rows][2]
  int* range;      // [items][2]: the first and last part of an item
};

template <class T>
struct Cache;
template <>
struct Cache<bf16> {
  static constexpr int KEYS = 32;
};
template <>
struct Cache<float> {
  static constexpr int KEYS = 16;
};

__device__ __forceinline__ f32x4 mfma_16x16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_16x16(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// A row's result: a sum of weights is 0 (no key, and values 0), or at least the 1 of the key at its reference.  A
// comparison with 0 would take a NaN for an empty row.
__device__ __forceinline__ float over_sum(float o, float sum) { return o / fmaxf(sum, 0.5f); }

// The largest of the lanes with the same lane % 16: rows of 16 lanes and halves of the wave swapped between two copies.
// Written as instructions: from the builtins the compiler takes both results for one.
__device__ __forceinline__ float max_over_keys(float x) {
  float y = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(x), "+v"(y));   // x: rows 0 0 2 2, y: 1 1 3 3
  x = y = fmaxf(x, y);
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));   // x: halves 0 0, y: 1 1
  return fmaxf(x, y);
}

// Keys of sequence b; the table and the cache bound them.
__device__ __forceinline__ int length_of(const PagedArgs& p, int b) {
  const int most = p.pages > 0 ? p.table_width * p.page_size : 0;
  return min(max(p.lengths[b], 0), most);
}

// Its tiles; none if it has no query.
template <int KEYS>
__device__ __forceinline__ int tiles_of(const PagedArgs& p, int b) {
  const int length = length_of(p, b), count = p.counts ? p.counts[b] : 1;
  return count <= 0 ? 0 : (length + KEYS - 1) / KEYS;
}

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ int scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // from 1, 2, 4, 8 lanes before, in rows of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // the last lane of the row before
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // of the first two rows
  return x;
}

// A workgroup's part of an item (a block of rows of a key head of a sequence): tiles t0 .. t0 + n - 1 of item `item` of
// sequence b; n = 0: none. Every wave by itself, from the sequences' lengths. Every item is cut into equal parts of at most
// part_length's tiles, which may be looked for where a wave has a lane for every sequence. Parts of equal length that begin
// in one item and end in the next cost more (48 sequences of up to 2000 keys, 8 key heads of 128, 61 us; 32 of up to 2048,
// 46; 100 of up to 3000, 4 key heads, 74; 56 of up to 2000, 8 key heads of 80, 61: part_length has the others' times).
struct Part {
  int b, item, t0, n, w;   // w: the part's number
};
// Parts in order over the XCDs (workgroup i runs on XCD i % 8): neighbours, which may read parts of the same cache lines
// or the same keys for other rows, get one L2.  -1: none.
__device__ __forceinline__ int xcd_order(int n) {
  const int per = (n + kAttnXcds - 1) / kAttnXcds, i = blockIdx.x / kAttnXcds, w = blockIdx.x % kAttnXcds * per + i;
  return i < per && w < n ? w : -1;
}
template <int KEYS>
__device__ __forceinline__ Part part_of(const PagedArgs& p, int B, int items) {
  const int lane = threadIdx.x & 63, groups = p.groups;
  int total = 0, live = 0, sums = 0, own = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    own = b0 + lane < B ? tiles_of<KEYS>(p, b0 + lane) : 0;
    sums = scan(own);
    total += __builtin_amdgcn_readlane(sums, 63);
    live += __popcll(__ballot(own > 0));
  }
  total *= items;
  live *= items;
  const auto count = [&](unsigned part) {
    int n = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
      if (B > 64) own = b0 + lane < B ? tiles_of<KEYS>(p, b0 + lane) : 0;
      sums = scan(((unsigned)own + part - 1) / part);
      n += __builtin_amdgcn_readlane(sums, 63);
    }
    return (unsigned)(n * items);
  };
  const unsigned part = part_length(total, live, groups, p.least, B <= 64, count);
  const int n = (int)count(part);   // at most `groups` and one an item
  const int w = xcd_order(n);
  const Part none{0, 0, 0, 0, 0};
  if (w < 0) return none;
  int before = 0, b = 0;
  for (;; b += 64) {
    if (B > 64) own = b + lane < B ? tiles_of<KEYS>(p, b + lane) : 0;
    const int mine = ((unsigned)own + part - 1) / part;
    if (B > 64) sums = scan(mine);
    const uint64_t past = __ballot(before + sums * items > w);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      before += __builtin_amdgcn_readlane(sums - mine, l) * items;
      const unsigned in = w - before, of = __builtin_amdgcn_readlane(mine, l), item = in / of, i = in - item * of;
      const unsigned tiles = __builtin_amdgcn_readlane(own, l), size = tiles / of, rest = tiles - size * of;
      return {b + l, (int)item, (int)(i * size + min(i, rest)), (int)(size + (i < rest)), w};
    }
    before += __builtin_amdgcn_readlane(sums, 63) * items;
    if (b + 64 >= B) return none;   // not with lengths that stay
  }
}

template <class T, int DP, int RB, int CAP, int W, bool EVEN, bool ONCE>
struct Walk {
  static constexpr int KEYS = Cache<T>::KEYS, VC = DP / 16;
  static constexpr int VL = VC * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : VC;   // values a load of V
  static constexpr int KL = sizeof(T) == 2 ? 8 : 4, KS = DP / (4 * KL), KU = KEYS / 16;
  static constexpr int VK = KEYS / 4;   // keys whose values a lane loads
  static constexpr int STEP = 64 * W / (16 * RB);   // threads to a row of the block
  // Four lanes' pieces of a key are 64 bytes, half a cache line, and a second load of the line would wait for the first
  // one's in the cache. So the lanes of two keys read a line of one key, then that line of the other: of the first
  // load an even lane has its key's first half and an odd lane the other key's second half, and of the second load the
  // reverse. The first halves make one product, the second halves another, whose rows (keys) are then swapped in
  // pairs. (One token over 773 keys of 16 heads of 64: 11.4 us, 11.9 by halves; 64 over up to 4000, 72 and 73. In
  // fp32 it gains nothing.)
  static constexpr bool LINES = sizeof(T) == 2 && KS % 2 == 0;
  static constexpr unsigned kAll = KEYS == 32 ? 0xffffffffu : 0xffffu;
  typedef T kvec __attribute__((ext_vector_type(KL)));
  typedef T vvec __attribute__((ext_vector_type(VL)));

  const AttnArgs& a;
  const PagedArgs& p;
  const int lane, m, h;
  const char *kbase, *vbase;
  // byte offsets of the lane's rows among sixteen, and of its pieces of a row (the row's first where it has no more)
  unsigned krow[LINES ? 2 : 1], vrow, kd[LINES ? 2 : 1][LINES ? KS / 2 : KS], vd[VC / VL];
  int64_t kat, kat1, vat, vat1;   // see locate
  kvec kf[KU][KS];
  vvec vf[VK][VC / VL];

  __device__ __forceinline__ Walk(const AttnArgs& a_, const PagedArgs& p_)
      : a(a_), p(p_), lane(threadIdx.x & 63), m(lane & 15), h(lane >> 4) {
    vrow = EVEN ? (unsigned)(4 * h * p.vslot) : 0;
#pragma unroll
    for (int e = 0; e < (LINES ? 2 : 1); ++e) {
      krow[e] = EVEN ? (unsigned)(key_of(e) * p.kslot) : 0;
#pragma unroll
      for (int s = 0; s < (LINES ? KS / 2 : KS); ++s) {
        const int d = KL * (LINES ? 8 * s + 4 * ((m ^ e) & 1) + h : 4 * s + h);
        kd[e][s] = d < a.D ? d * (int)sizeof(T) : 0;
      }
    }
#pragma unroll
    for (int c = 0; c < VC / VL; ++c) vd[c] = 16 * VL * c + VL * m < a.D ? (16 * VL * c + VL * m) * (int)sizeof(T) : 0;
  }

  // key of the lane's load e, among sixteen
  __device__ __forceinline__ int key_of(int e) const { return LINES ? (m & ~1) + e : m; }
  __device__ __forceinline__ int page_index(int j) const { return (int)((uint64_t)(unsigned)j * p.div_mul >> p.div_shift); }
  // Page of the lane's key (key lane % KEYS) of tile t; -1: none.
  __device__ __forceinline__ int page_of(const int* table, int t) const {
    const int at = page_index(t * KEYS + (lane & (KEYS - 1)));
    return at < p.table_width ? table[at] : -1;
  }
  // Which of a tile's keys are there, and where they lie. Sixteen keys of one page: where their rows begin, for all
  // lanes; else each lane's own key, shared as it is loaded. Keys of no page are read as the first page's.
  __device__ __forceinline__ unsigned locate(int t, int page, int length) {
    const int j = t * KEYS + (lane & (KEYS - 1));
    const bool ok = j < length && (unsigned)page < (unsigned)p.pages;
    const unsigned there = (unsigned)__ballot(ok) & kAll;
    const int own = (unsigned)page < (unsigned)p.pages ? page : 0;
    if constexpr (EVEN) {
      place(t * KEYS, __builtin_amdgcn_readlane(own, 0), kat, vat);
      if constexpr (KU == 2) place(t * KEYS + 16, __builtin_amdgcn_readlane(own, 16), kat1, vat1);
    } else {
      place(j, own, kat, vat);
    }
    return there;
  }
  __device__ __forceinline__ void place(int j, int64_t page, int64_t& k, int64_t& v) const {
    const int slot = j - page_index(j) * p.page_size;
    k = page * p.kpage + slot * p.kslot;
    v = page * p.vpage + slot * p.vslot;
  }
  // Keys that no other block of rows reads pass the caches by: eight tokens over 8200 to 32768 keys, 117 us, through the
  // caches 131.  (64 queries of 16/4 heads, 8 blocks, over 4096 keys: 84 and 58.)  Not rows that share lines, with other
  // loads of a tile or other heads: 28 tokens over up to 8000 keys of 16 heads of 80, 155 and 135.
  template <class V>
  __device__ static __forceinline__ V read(const V* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    return *p;
  }
  __device__ __forceinline__ void load_k() {
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int e = 0; e < (LINES ? 2 : 1); ++e) {
        const char* row = EVEN ? kbase + (u == 0 ? kat : kat1) : kbase + __shfl(kat, 16 * u + key_of(e));
#pragma unroll
        for (int s = 0; s < (LINES ? KS / 2 : KS); ++s)
          kf[u][LINES ? 2 * s + e : s] = read((const kvec*)(row + (krow[e] + kd[e][s])));
      }
  }
  // s = K Q^T of rows q, sixteen keys u
  __device__ __forceinline__ f32x4 product(const kvec (&qf)[KS], int u) const {
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      kvec k = kf[u][st];
      if constexpr (LINES) {
        const u32x4 own = __builtin_bit_cast(u32x4, k), other = __builtin_bit_cast(u32x4, kf[u][st ^ 1]);
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = m & 1 ? other[e] : own[e];
        k = __builtin_bit_cast(kvec, w);
      }
      if constexpr (sizeof(T) == 2) {
        s[st & 1] = mfma_16x16(k, qf[st], s[st & 1]);
      } else {
#pragma unroll
        for (int e = 0; e < KL; ++e) s[st & 1] = mfma_16x16(k[e], qf[st][e], s[st & 1]);
      }
    }
    if constexpr (KS > 1) s[0] += LINES ? f32x4{s[1][1], s[1][0], s[1][3], s[1][2]} : s[1];
    return s[0];
  }
  __device__ __forceinline__ void load_v() {
#pragma unroll
    for (int t = 0; t < VK; ++t) {
      const char* row =
          EVEN ? vbase + (t < 4 ? vat : vat1) + (t & 3) * p.vslot : vbase + __shfl(vat, 16 * (t >> 2) + 4 * h + (t & 3));
#pragma unroll
      for (int c = 0; c < VC / VL; ++c) vf[t][c] = read((const vvec*)(row + (vrow + vd[c])));
    }
  }
  // acc += V^T times the tile's weights
  __device__ __forceinline__ void add_values(const float (&x)[RB][KU][4], f32x4 (&acc)[RB][VC]) const {
    if constexpr (sizeof(T) == 2) {
      bf16x8 hi[RB], lo[RB];
#pragma unroll
      for (int q = 0; q < RB; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          hi[q][e] = (bf16)x[q][e >> 2][e & 3];
          lo[q][e] = (bf16)(x[q][e >> 2][e & 3] - (float)hi[q][e]);
        }
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        bf16x8 v;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = vf[k][0][c];
#pragma unroll
        for (int q = 0; q < RB; ++q) acc[q][c] = mfma_16x16(v, hi[q], mfma_16x16(v, lo[q], acc[q][c]));
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
          for (int q = 0; q < RB; ++q) acc[q][c] = mfma_16x16(vf[r][c / VL][c % VL], x[q][0][r], acc[q][c]);
    }
  }
  // Whether v is an infinity or NaN: on its bits, and by size, since the compiler, which is told that there are no NaN,
  // knows the usual test of the exponent for what it is.
  __device__ static __forceinline__ bool not_finite(T v) {
    return __builtin_bit_cast(uint32_t, (float)v) << 1 >= 0xff000000u;
  }
  // Takes the values that are not finite out of the tile; whether there were any.
  __device__ __forceinline__ bool take_not_finite() {
    bool bad = false;
#pragma unroll
    for (int k = 0; k < VK; ++k)
#pragma unroll
      for (int c = 0; c < VC / VL; ++c) {
        vvec v = vf[k][c];
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          const bool is = not_finite(v[e]);
          bad |= is;
          v[e] = is ? (T)0.f : v[e];
        }
        vf[k][c] = v;
      }
    return __ballot(bad) != 0;
  }

  // Tiles [t0, t1) of head hk of sequence b, rows from row0 on; to the output or to part `slot`.
  __device__ __forceinline__ void run(int b, int hk, int row0, int t0, int t1, T* out, Parts parts, int64_t slot,
                                      char* lds) {
    const int wave = wave_id(), length = __builtin_amdgcn_readfirstlane(length_of(p, b));
    const int rows = a.Nq * a.G, n_rows = min(rows - row0, 16 * RB);
    const int count = __builtin_amdgcn_readfirstlane(p.counts ? min(max(p.counts[b], 0), a.Nq) : a.Nq);
    // position of the first query: by the length as given, also where it is past the table (2^30 stands for all beyond it)
    const int first = __builtin_amdgcn_readfirstlane(min(max(p.lengths[b], 0), 1 << 30)) - count;
    const int* table = p.page_table + b * p.table_stride;
    kbase = (const char*)p.keys + hk * p.khead;
    vbase = (const char*)p.values + hk * p.vhead;
    int t = t0 + wave, page = page_of(table, t);

    int pos[RB], lim[RB];
    kvec qf[RB][KS];
#pragma unroll
    for (int q = 0; q < RB; ++q) {
      const int r = row0 + 16 * q + m, i = r < rows ? r / a.G : 0, head = hk * a.G + (r < rows ? r - i * a.G : 0);
      const bool live = r < rows && i < count;
      pos[q] = first + i;
      lim[q] = !live ? 0 : a.causal ? min(pos[q] + 1, length) : length;
      const T* row = static_cast<const T*>(a.q) + b * a.qb + i * a.qn + head * a.qh;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = KL * (4 * s + h);
        qf[q][s] = r < rows && d < a.D ? *reinterpret_cast<const kvec*>(row + d) : kvec{};
      }
    }
    // every row that counts sees the keys below low
    const int low = a.causal ? min(first + 1, length) : length;
    unsigned there = 0;
    // keys, values and the page after next are requested as soon as there is room; behind the last tile it once more (a
    // load that may not be made would have to be waited for at once)
    const auto after = [&](int t) { return t + W < t1 ? t + W : t; };
    // the bias by bucket and row, and the buckets by distance, where the waves' parts go later, requested beside the
    // page and many at once (one by one, 46 x 7 tokens of 32/4 heads and 65 buckets took 18 us, so 16). Past the last
    // one it again, to the same place.
    float* bias = reinterpret_cast<float*>(lds);                         // [buckets][16 RB]
    uint8_t* buckets = reinterpret_cast<uint8_t*>(bias + 256 * 16 * RB);   // [2 radius + 1]
    if (a.table) {
      int self = threadIdx.x;
      asm volatile("" : "+v"(self));
      const int r = self % (16 * RB), head = hk * a.G + (row0 + r) % a.G;
#pragma unroll 1
      for (int n = 0; n * 8 * STEP < a.nb || n * 4 * 64 * W <= 2 * a.radius; ++n) {
        int e[8], d[4];
        uint8_t y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          d[k] = min((4 * n + k) * 64 * W + self, 2 * a.radius);
          y[k] = a.buckets[d[k]];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = min((8 * n + k) * STEP + self / (16 * RB), a.nb - 1);
        const auto fill = [&](auto* table) {
          std::decay_t<decltype(*table)> x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = table[e[k] * a.H + head];
          __builtin_amdgcn_sched_barrier(0);   // all requested before the first is waited for
#pragma unroll
          for (int k = 0; k < 8; ++k) bias[e[k] * 16 * RB + r] = bias_log2((float)x[k]);
        };
        if (a.table_bf16)
          fill(static_cast<const bf16*>(a.table));
        else
          fill(static_cast<const float*>(a.table));
#pragma unroll
        for (int k = 0; k < 4; ++k) buckets[d[k]] = min(y[k], (uint8_t)(a.nb - 1));
      }
    }
    if (t < t1) {
      there = locate(t, page, length);
      load_k();
      page = page_of(table, after(t));
    }
    if (a.table) __syncthreads();

    f32x4 acc[RB][VC];
    float top[RB], ref[RB], l[RB];
#pragma unroll
    for (int q = 0; q < RB; ++q) {
#pragma unroll
      for (int c = 0; c < VC; ++c) acc[q][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      top[q] = -kInf;
      ref[q] = l[q] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) asm volatile("" ::"v"(qf[q][s]));   // waited for here, not in every turn
    }
    const Capped<T, CAP> capped(a);
    const float mult = a.scale * kLog2e;

    bool taken = false;
    for (bool more = t < t1; more;) {
      const int j0 = t * KEYS, next = after(t);
      load_v();
      __builtin_amdgcn_sched_barrier(0);
      const unsigned now = there;
      if (a.D < DP)   // zero times what lies there has to be zero
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int st = 0; st < KS; ++st)
            if (KL * (LINES ? 8 * (st / 2) + 4 * ((m ^ st) & 1) + h : 4 * st + h) >= a.D) kf[u][st] = kvec{};
      f32x4 s[RB][KU];
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int q = 0; q < RB; ++q) s[q][u] = product(qf[q], u);
      __builtin_amdgcn_sched_barrier(0);   // K's registers are free
      there = locate(next, page, length);
      load_k();
      page = page_of(table, after(next));

      float x[RB][KU][4];
      if (a.cap > 0.f) {
        float slope;
#pragma unroll
        for (int q = 0; q < RB; ++q)
#pragma unroll
          for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[q][u][r] = capped.score(s[q][u][r], capped.k3, slope);
      } else {
#pragma unroll
        for (int q = 0; q < RB; ++q)
#pragma unroll
          for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[q][u][r] = s[q][u][r] * mult;
      }
      if (a.table) {
        const int rel0 = j0 - first;   // the first key from the first query
        const auto bucket_of = [&](int rel) { return (int)buckets[min(max(rel, -a.radius), a.radius) + a.radius]; };
        if (rel0 - (a.Nq - 1) >= a.radius || rel0 + KEYS - 1 <= -a.radius) {   // all of one bucket
          const float* one = bias + bucket_of(rel0) * (16 * RB) + m;
#pragma unroll
          for (int q = 0; q < RB; ++q)
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
              for (int r = 0; r < 4; ++r) x[q][u][r] += one[16 * q];
        } else {
          int bucket[RB][KU][4];
#pragma unroll
          for (int q = 0; q < RB; ++q)
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
              for (int r = 0; r < 4; ++r) bucket[q][u][r] = bucket_of(j0 + 16 * u + 4 * h + r - pos[q]);
          __builtin_amdgcn_sched_barrier(0);   // all of them requested before the first is waited for
#pragma unroll
          for (int q = 0; q < RB; ++q)
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
              for (int r = 0; r < 4; ++r) x[q][u][r] += bias[bucket[q][u][r] * (16 * RB) + 16 * q + m];
        }
      }
#pragma unroll
      for (int q = 0; q < RB; ++q) {
        if (now != kAll || j0 + KEYS > low)
#pragma unroll
          for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int k = 16 * u + 4 * h + r;
              x[q][u][r] = j0 + k < lim[q] && (now >> k & 1) ? x[q][u][r] : -kInf;
            }
        float mx = x[q][0][0];
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[q][u][r]);
        mx = max_over_keys(mx);
        if (__ballot(mx > top[q] + kRescale)) {
          const float mn = fmaxf(top[q], mx), to = mn == -kInf ? 0.f : mn;
          const float f = fast_exp2(top[q] - to);
#pragma unroll
          for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[q][c][r] *= f;
          l[q] *= f;
          top[q] = mn;
          ref[q] = to;
        }
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[q][u][r] = fast_exp2(x[q][u][r] - ref[q]);
            l[q] += x[q][u][r];
          }
      }

      if (now != kAll) {
        // what a key that is not there holds has to count nothing, whatever it is
#pragma unroll
        for (int k = 0; k < VK; ++k)
          if (!(now >> (16 * (k >> 2) + 4 * h + (k & 3)) & 1))
#pragma unroll
            for (int c = 0; c < VC / VL; ++c) vf[k][c] = vvec{};
      }
      // where rows differ in what they see, a value that is not finite waits for the end (zero times it is not zero)
      if (a.causal && a.Nq > 1 && j0 + KEYS > first + 1) taken |= take_not_finite();
      add_values(x, acc);
      __builtin_amdgcn_sched_barrier(0);   // and V's
      more = next != t;
      t = next;
    }

    // the waves' parts through LDS.  What follows from the thread's number is worked out here, not kept since the start.
    if (a.table) __syncthreads();
    int self = threadIdx.x;
    asm volatile("" : "+v"(self));
    const int lane = self & 63, m = lane & 15, h = lane >> 4;
    float* sh = reinterpret_cast<float*>(lds);                   // [waves][16 RB][DP]
    float* ml = sh + W * 16 * RB * DP;                           // [waves][16 RB][2]
    int* flags = reinterpret_cast<int*>(ml + W * 16 * RB * 2);   // [waves]
    if (lane == 0) flags[wave] = taken;
#pragma unroll
    for (int q = 0; q < RB; ++q) {
      l[q] += __shfl_xor(l[q], 16);
      l[q] += __shfl_xor(l[q], 32);
      const int at = wave * 16 * RB + 16 * q + m;
      if (h == 0) {
        ml[2 * at] = l[q] == 0.f ? -kInf : ref[q];
        ml[2 * at + 1] = l[q];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < VC; ++c) sh[at * DP + 16 * VL * (c / VL) + VL * (4 * h + r) + c % VL] = acc[q][c][r];
    }
    __syncthreads();
    typedef T quad __attribute__((ext_vector_type(4)));
#pragma unroll 1
    for (int k = self; k < n_rows * (DP / 4); k += 64 * W) {
      const int r = k / (DP / 4), d = (k - r * (DP / 4)) * 4;
      if (d >= a.D) continue;
      f32x2 mls[W];
      float most = -kInf;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        mls[w] = *reinterpret_cast<const f32x2*>(ml + 2 * (w * 16 * RB + r));
        most = fmaxf(most, mls[w][0]);
      }
      const float to = most == -kInf ? 0.f : most;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
      int any = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = fast_exp2(mls[w][0] - to);
        o += f * *reinterpret_cast<const f32x4*>(sh + (w * 16 * RB + r) * DP + d);
        sum += f * mls[w][1];
        any |= flags[w];
      }
      const int i = (row0 + r) / a.G, g = row0 + r - i * a.G;
      if (i >= count) o = f32x4{0.f, 0.f, 0.f, 0.f}, sum = 0.f;   // padding
      if (any) {   // its size does not matter: whatever a seen one weighs, so is the result
        const int seen = i < count ? min(first + i + 1, min(length, t1 * KEYS)) : 0;
#pragma unroll 1
        for (int j = max(max(first + 1, 0) / KEYS, t0) * KEYS; j < seen; ++j) {   // from the first such tile
          const int at = page_index(j), page = table[at];
          if (page < 0 || page >= p.pages) continue;
          const T* v = (const T*)(vbase + page * p.vpage + (j - at * p.page_size) * p.vslot) + d;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (not_finite(v[e])) o[e] += (float)v[e];
        }
      }
      if (slot < 0) {
        quad v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)over_sum(o[e], sum);
        *reinterpret_cast<quad*>(out + (((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D + d) = v;
      } else {
        const int64_t at = slot * min(rows, 16 * RB) + r;
        *reinterpret_cast<f32x4*>(parts.o + at * a.D + d) = o;
        if (d == 0) {
          parts.ml[2 * at] = i >= count || sum == 0.f ? -kInf : to;
          parts.ml[2 * at + 1] = sum;
        }
      }
    }
  }
};

// LDS of a workgroup: the waves' parts, and before them the bias.
template <int DP, int RB, int W>
constexpr int lds_bytes() {
  constexpr int parts = W * (16 * RB * (DP + 2) + 1) * 4, bias = 256 * 16 * RB * 4 + 2 * kMaxRadius + 4;
  return parts > bias ? parts : bias;
}

// Without groups a workgroup takes an item; with them a part of one, for the join, or the whole, which is written at
// once.
template <class T, int DP, int RB, int CAP, int W, bool EVEN, bool ONCE>
__global__ __launch_bounds__(64 * W, 2) void paged_kernel(const AttnArgs a, const PagedArgs p, T* __restrict__ out,
                                                          Parts parts) {
  constexpr int KEYS = Cache<T>::KEYS;
  __shared__ __attribute__((aligned(16))) char lds[lds_bytes<DP, RB, W>()];
  const int items = a.Hk * p.blocks;   // of a sequence
  Part s;
  int64_t slot = -1;
  if (p.groups == 0) {
    const int w = xcd_order(a.B * items);
    if (w < 0) return;
    const int b = w / items, item = w - b * items, tiles = tiles_of<KEYS>(p, b);
    s = {b, item, 0, tiles, w};
    if (tiles == 0) {
      const int hk = item / p.blocks, row0 = item % p.blocks * 16 * RB, n = min(a.Nq * a.G - row0, 16 * RB);
      for (int k = threadIdx.x; k < n * a.D; k += 64 * W) {
        const int r = row0 + k / a.D, i = r / a.G;
        out[(((int64_t)b * a.Nq + i) * a.H + hk * a.G + r - i * a.G) * a.D + k % a.D] = (T)0.f;
      }
      return;
    }
  } else {
    s = part_of<KEYS>(p, a.B, items);
    if (s.n == 0) return;
    const int tiles = tiles_of<KEYS>(p, s.b);
    const int64_t item = (int64_t)s.b * items + s.item;
    if (s.n < tiles) slot = s.w;
    if (threadIdx.x == 0) {
      if (s.t0 == 0) parts.range[2 * item] = s.w;
      if (s.t0 + s.n == tiles) parts.range[2 * item + 1] = s.w;
    }
  }
  Walk<T, DP, RB, CAP, W, EVEN, ONCE>(a, p).run(s.b, s.item / p.blocks, s.item % p.blocks * 16 * RB, s.t0, s.t0 + s.n, out,
                                                parts, slot, lds);
}

// The parts of a row: first .. last of its item; none where the sequence is empty, one where the result is there already.
struct RowParts {
  int64_t row0;   // of the first part
  int n, stride;
};
template <int KEYS>
__device__ __forceinline__ RowParts row_parts(const AttnArgs& a, const PagedArgs& p, const Parts& parts, int64_t row,
                                              int block_rows) {
  const int h = (int)(row % a.H), b = (int)(row / a.H / a.Nq), i = (int)(row / a.H - (int64_t)b * a.Nq);
  const int hk = h / a.G, r = i * a.G + h - hk * a.G, blk = r / block_rows;
  const int64_t item = ((int64_t)b * a.Hk + hk) * p.blocks + blk;
  const int stride = min(a.Nq * a.G, block_rows);
  const int first = parts.range[2 * item], last = parts.range[2 * item + 1];   // not set where the sequence is empty
  if (tiles_of<KEYS>(p, b) == 0) return {0, 0, stride};
  return {(int64_t)first * stride + r - blk * block_rows, last - first + 1, stride};
}

// Parts w, w + step, ... of a row added in order, four at a time and in one pass; N values of each.
template <int N>
struct Sum {
  float top = -kInf, sum = 0.f, o[N] = {};
  __device__ __forceinline__ void merge(float m, float l, const float (&x)[N]) {
    const float to = fmaxf(top, m), ref = to == -kInf ? 0.f : to, f = fast_exp2(top - ref), g = fast_exp2(m - ref);
    top = to;
    sum = sum * f + l * g;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * f + x[i] * g;
  }
  template <class Load>
  __device__ __forceinline__ void add(const Parts& parts, const RowParts& own, int w, int step, const Load& load) {
    for (; w < own.n; w += 4 * step) {
      f32x2 ml[4];
      float x[4][N];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool there = w + k * step < own.n;
        const int64_t at = own.row0 + (int64_t)(there ? w + k * step : w) * own.stride;
        ml[k] = *reinterpret_cast<const f32x2*>(parts.ml + 2 * at);
        load(at, x[k]);
        if (there) continue;
        ml[k] = f32x2{-kInf, 0.f};
#pragma unroll
        for (int i = 0; i < N; ++i) x[k][i] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) merge(ml[k][0], ml[k][1], x[k]);
    }
  }
};

// paged_join: few rows of many parts, a workgroup a row: wave w takes parts w, w + waves, ..., then the waves are added
// in order. Lane d holds values d and 64 + d.
constexpr int kJoinWaves = 8;
template <class T, int KEYS>
__global__ __launch_bounds__(64 * kJoinWaves) void paged_join_kernel(const AttnArgs a, const PagedArgs p,
                                                                     T* __restrict__ out, Parts parts, int block_rows) {
  __shared__ float sh[kJoinWaves][2][64], ml[kJoinWaves][2];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = blockIdx.x;   // (b, i, head)
  const RowParts own = row_parts<KEYS>(a, p, parts, row, block_rows);
  if (own.n == 1) return;
  Sum<2> s;
  const int d0 = min(lane, a.D - 1), d1 = min(lane + 64, a.D - 1);
  s.add(parts, own, wave, kJoinWaves, [&](int64_t at, float (&x)[2]) {
    x[0] = parts.o[at * a.D + d0];
    x[1] = parts.o[at * a.D + d1];
  });
  sh[wave][0][lane] = s.o[0];
  sh[wave][1][lane] = s.o[1];
  if (lane == 0) {
    ml[wave][0] = s.top;
    ml[wave][1] = s.sum;
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) s.merge(ml[w][0], ml[w][1], {sh[w][0][lane], sh[w][1][lane]});
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.D) out[row * a.D + lane + 64 * e] = (T)over_sum(s.o[e], s.sum);
}

// paged_join_rows: many rows of few parts, four values of one a thread, in the parts' order.
template <class T, int KEYS>
__global__ __launch_bounds__(256) void paged_join_rows_kernel(const AttnArgs a, const PagedArgs p, T* __restrict__ out,
                                                              Parts parts, int block_rows, int rows) {
  typedef T quad __attribute__((ext_vector_type(4)));
  const unsigned quads = a.D / 4, k = blockIdx.x * 256 + threadIdx.x, row = k / quads, d = (k - row * quads) * 4;
  if ((int)row >= rows) return;
  const RowParts own = row_parts<KEYS>(a, p, parts, row, block_rows);
  if (own.n == 1) return;
  Sum<4> s;
  s.add(parts, own, 0, 1, [&](int64_t at, float (&x)[4]) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(parts.o + at * a.D + d);
#pragma unroll
    for (int c = 0; c < 4; ++c) x[c] = v[c];
  });
  quad v;
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = (T)over_sum(s.o[c], s.sum);
  *reinterpret_cast<quad*>(out + (int64_t)row * a.D + d) = v;
}

// Whether sixteen keys are always of one page (and their slots' offsets of 32 bits).
bool even_pages(const bioemu_paged_cache& c, bool f32) {
  const int64_t far = (int64_t(1) << 27) / (f32 ? 4 : 2);
  return c.page_size % 16 == 0 && c.keys_stride[1] <= far && c.values_stride[1] <= far;
}

struct Plan {
  int rb, blocks, waves, groups, least;
  bool once;   // keys pass the caches by
  int64_t items, slots;
};

// Rows in blocks of 16 or 32.  Keys shared out over workgroups unless an item's are few (the join costs what the shorter
// walk gains) or the items many.
Plan plan(const AttnArgs& a, const bioemu_paged_cache& c, bool f32) {
  Plan p{};
  p.waves = 4;
  const int rows = a.Nq * a.G;
  p.rb = rows <= 16 ? 1 : 2;
  p.blocks = (rows + 16 * p.rb - 1) / (16 * p.rb);
  p.items = (int64_t)a.B * a.Hk * p.blocks;
  p.once = p.blocks == 1 && a.D * (f32 ? 4 : 2) % 128 == 0;
  const int64_t most = c.pages > 0 ? c.table_width * c.page_size : 0;
  // what a walk of one workgroup takes no longer than parts and the join: up to 1024 keys of 64 values in bf16 (in a
  // graph 8.4 us for 512 and 11.0 for 1024; in parts 9.8 and 10.0, and a second launch)
  // and items enough for 16 a CU, whose lengths the host does not know. Where one is far longer, its walk is what the call
  // takes: 511 sequences of 50 to 400 keys of 8 heads of 128 and one of 400, 100 us; one of 8192, 164; one of 32768, 380.
  if (most * std::max(a.D, 64) * (f32 ? 4 : 2) <= 1024 * 64 * 2 || p.items >= 16 * attn_units()) {
    // With a CU for each, eight waves share a walk (sixteen, where registers allow it, start 1.5 us later: 12.9 us for
    // one token over 773 keys of 16 heads of 64, 11.3 with eight, 17 with four). Two of eight do not fit a CU, two of
    // four do: 273 items of 64 values, 13 keys 6.1 us by four and 10.2 by eight, 1000 keys 18.4 and 23.8.
    if ((p.once || p.rb == 1) && p.items <= attn_units() && (f32 || a.cap <= kFastCap)) p.waves = 8;
    return p;
  }
  // Two a CU: with three or four, where registers allow them, 64 sequences of 4096 keys took 206 us, with these 184.
  // Four where heads are narrow, so that enough is requested at once, and parts are of some length: 64 sequences of
  // 2000 keys of 16 heads of 24 37 us (with two 42), in fp32 75 to 82 (87), but 8 of 8000 keys of 4 heads of 32, eight
  // tiles a part, 15.3 (14.6).
  const bool four = a.D <= 32 && p.rb == 1 && p.items * most >= 4 * attn_units() * 16 * (f32 ? 16 : 32);
  p.groups = (four ? 4 : 2) * attn_units();
  p.least = p.waves;
  p.slots = p.groups + p.items;   // parts at most (see part_of)
  return p;
}

size_t parts_bytes(const AttnArgs& a, const Plan& p) {
  return (size_t)p.slots * std::min(a.Nq * a.G, 16 * p.rb) * (a.D + 2) * sizeof(float) +
         (p.groups ? (size_t)p.items * 2 * sizeof(int) : 0);
}

int paged_args(const bioemu_paged_cache* c, const bioemu_attention_args* in, AttnArgs* a, Plan* pl) {
  if (const int rc = attn_args("paged_attention", in, a)) return rc;
  if (in->Nk || in->k || in->v || in->q_segments || in->k_segments || in->prefix || in->lengths)
    return set_error(BIOEMU_ERR_INVALID_ARG, "paged_attention: keys, lengths and masks come from the cache");
  if (const int rc = paged_cache_args("paged_attention", c, a->B, a->Hk, in->f32 != 0)) return rc;
  *pl = plan(*a, *c, in->f32 != 0);
  const int64_t tiles = (c->table_width * c->page_size + 15) / 16;
  // tiles are counted in 32 bits; a launch of a workgroup an item has fewer than 2^32 threads
  if (pl->items * std::max(tiles, (int64_t)1) >= (int64_t(1) << 31) || round_up(pl->items, kAttnXcds) >= 1 << 24)
    return set_error(BIOEMU_ERR_UNSUPPORTED, "paged_attention: B=%d, Nq=%d, H=%d over %ld keys are too many", a->B,
                     a->Nq, a->H, (long)(c->table_width * c->page_size));
  return BIOEMU_OK;
}

template <class T, int DP>
int launch(const AttnArgs& a, const PagedArgs& p, const Plan& pl, T* out, void* ws, hipStream_t stream) {
  const int block_rows = 16 * pl.rb;
  Parts parts{static_cast<float*>(ws), nullptr, nullptr};
  if (ws) {
    const int64_t part_rows = pl.slots * std::min(a.Nq * a.G, block_rows);
    parts.ml = parts.o + part_rows * a.D;
    parts.range = reinterpret_cast<int*>(parts.ml + 2 * part_rows);
  }
  {
    KernelTimerScope timer("paged_attention", stream);
    const dim3 grid((unsigned)round_up(pl.groups ? pl.slots : pl.items, kAttnXcds));
    const auto go = [&](auto kernel) { kernel<<<grid, 64 * pl.waves, 0, stream>>>(a, p, out, parts); };
    const bool wide = !fast_cap<T>(a);
    // few calls have a wide cap: one form for them (64 tokens over up to 4000 keys, 32/4 heads of 128: 72 us, 64 with a cap
    // of 50)
#define BIOEMU_GO(RB, W, EVEN, ONCE)                                                                 \
  if (pl.rb == RB && !wide && pl.waves == W && p.even == EVEN && pl.once == ONCE)                     \
    go(paged_kernel<T, DP, RB, kCapped, W, EVEN, ONCE>);
#define BIOEMU_GO_RB(RB)                                                            \
  BIOEMU_GO(RB, 4, true, true)                                                      \
  BIOEMU_GO(RB, 4, false, true)                                                     \
  BIOEMU_GO(RB, 8, true, true)                                                      \
  BIOEMU_GO(RB, 8, false, true)                                                     \
  if constexpr (sizeof(T) == 2) {                                                   \
    if (pl.rb == RB && wide) go(paged_kernel<T, DP, RB, kCapWide, 4, false, false>); \
  }
    BIOEMU_GO_RB(1)
    BIOEMU_GO_RB(2)
    BIOEMU_GO(1, 4, true, false)
    BIOEMU_GO(1, 4, false, false)
    BIOEMU_GO(1, 8, true, false)
    BIOEMU_GO(1, 8, false, false)
    BIOEMU_GO(2, 4, true, false)
    BIOEMU_GO(2, 4, false, false)
#undef BIOEMU_GO_RB
#undef BIOEMU_GO
    if (const int rc = check_launch("paged_attention")) return rc;
  }
  if (!pl.groups) return BIOEMU_OK;
  KernelTimerScope timer("paged_join", stream);
  const int64_t rows = (int64_t)a.B * a.Nq * a.H;
  // by parts a row: some 8 (8 tokens over 8192 keys of 8 heads) 50.8 us by quads, 51.2 by a workgroup a row; 16: 30.4 and
  // 29.5; 64: 37.8 and 31.6
  if (pl.groups <= 14 * pl.items)
    paged_join_rows_kernel<T, Cache<T>::KEYS><<<dim3((unsigned)((rows * (a.D / 4) + 255) / 256)), 256, 0, stream>>>(
        a, p, out, parts, block_rows, (int)rows);
  else
    paged_join_kernel<T, Cache<T>::KEYS><<<dim3((unsigned)rows), 64 * kJoinWaves, 0, stream>>>(a, p, out, parts,
                                                                                               block_rows);
  return check_launch("paged_join");
}

}  // namespace
}  // namespace bioemu

using namespace bioemu;

extern "C" size_t bioemu_paged_attention_workspace_bytes(const bioemu_paged_cache* cache,
                                                         const bioemu_attention_args* args) {
  AttnArgs a;
  Plan pl;
  if (paged_args(cache, args, &a, &pl) || a.B == 0 || a.Nq == 0) return 0;
  return parts_bytes(a, pl);
}

extern "C" int bioemu_paged_attention(const bioemu_paged_cache* cache, const bioemu_attention_args* args, void* o,
                                      void* workspace, size_t workspace_bytes, hipStream_t stream) {
  AttnArgs a;
  Plan pl;
  if (const int rc = paged_args(cache, args, &a, &pl)) return rc;
  if (a.B == 0 || a.Nq == 0) return BIOEMU_OK;
  if (!o || !aligned16(o)) return set_error(BIOEMU_ERR_INVALID_ARG, "paged_attention: o must be 16-byte aligned");
  const size_t need = parts_bytes(a, pl);
  if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return set_error(BIOEMU_ERR_WORKSPACE, "paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const int item = args->f32 ? 4 : 2;
  const int64_t *ks = cache->keys_stride, *vs = cache->values_stride;
  // key / page_size: 2^(28 + l) / page_size rounded up, l = log2 of page_size rounded up, is off by less than 2^l /
  // page_size
  unsigned l = 0;
  while ((int64_t(1) << l) < cache->page_size) ++l;
  const unsigned mul = (unsigned)(((int64_t(1) << (28 + l)) + cache->page_size - 1) / cache->page_size);
  const PagedArgs p{static_cast<const char*>(cache->keys), static_cast<const char*>(cache->values), ks[0] * item,
                    ks[1] * item, ks[2] * item, vs[0] * item, vs[1] * item, vs[2] * item, cache->page_table,
                    cache->table_stride, cache->lengths, cache->counts, (int)cache->pages, (int)cache->page_size,
                    (int)cache->table_width, pl.blocks, mul, 28 + l, even_pages(*cache, args->f32 != 0), pl.groups, pl.least};
  const int dp = a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128;
  void* ws = need ? workspace : nullptr;
#define BIOEMU_PAGED(T, P) \
  if (dp == P) return launch<T, P>(a, p, pl, static_cast<T*>(o), ws, stream)
  if (args->f32) {
    BIOEMU_PAGED(float, 32);
    BIOEMU_PAGED(float, 64);
    BIOEMU_PAGED(float, 128);
  } else {
    BIOEMU_PAGED(bf16, 32);
    BIOEMU_PAGED(bf16, 64);
    BIOEMU_PAGED(bf16, 128);
  }
#undef BIOEMU_PAGED
  return BIOEMU_ERR_UNSUPPORTED;
}
