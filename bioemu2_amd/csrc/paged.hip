// Attention of few queries over a paged cache, for gfx950.
//
//   s(i, j) = cap tanh(scale q_i . k_j / cap) + bias[clamp(j - p_i, -R, R)],   o_i = sum_j softmax_j(s) v_j
//   p_i = length - count + i, keys j <= p_i (causal) or j < length; key j is slot j % page_size of page table[j / page_size]
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
#include <algorithm>

#include "attn.h"

namespace bioemu {
namespace {

constexpr int kWaves = 4;
constexpr float kRescale = 8.f;   // log2 of the largest weight before the maximum moves

struct PagedArgs {
  const char *keys, *values;
  int64_t kpage, kslot, khead, vpage, vslot, vhead;   // bytes
  const int* page_table;
  int64_t table_stride;
  const int *lengths, *counts;
  int pages, page_size, table_width, blocks;   // blocks of rows a key head
  int groups, least;                            // workgroups that share the keys, of `least` tiles at least; 0: one an item
};

struct Parts {
  float *o, *ml;   // [slots][rows][D], [slots][rows][2]
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

// Keys of sequence b; the table and the cache bound them.
__device__ __forceinline__ int length_of(const PagedArgs& p, int b) {
  const int most = p.pages > 0 ? p.table_width * p.page_size : 0;
  return min(max(p.lengths[b], 0), most);
}

// Tiles of all items before sequence `upto` (B: of all).  Every wave by itself.
template <int KEYS>
__device__ __forceinline__ int64_t tiles_before(const PagedArgs& p, int upto, int items) {
  const int lane = threadIdx.x & 63;
  int64_t sum = 0;
  for (int b = lane; b < upto; b += 64) sum += (length_of(p, b) + KEYS - 1) / KEYS;
#pragma unroll
  for (int m = 32; m > 0; m /= 2) sum += __shfl_xor(sum, m);
  return sum * items;
}

__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
         (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

template <class T, int DP, int RB, int CAP>
struct Walk {
  static constexpr int KEYS = Cache<T>::KEYS, VC = DP / 16;
  static constexpr int VL = VC * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : VC;   // values a load of V
  static constexpr int KL = sizeof(T) == 2 ? 8 : 4, KS = DP / (4 * KL), KU = KEYS / 16;
  static constexpr int VK = KEYS / 4;   // keys whose values a lane loads
  typedef T kvec __attribute__((ext_vector_type(KL)));
  typedef T vvec __attribute__((ext_vector_type(VL)));

  const AttnArgs& a;
  const PagedArgs& p;
  const int lane, m, h;
  const char *kbase, *vbase;
  int64_t koff[KU], voff[VK];
  kvec kf[KU][KS];
  vvec vf[VK][VC / VL];
  unsigned mask;   // keys of the tile that are there, as loaded

  __device__ __forceinline__ Walk(const AttnArgs& a_, const PagedArgs& p_)
      : a(a_), p(p_), lane(threadIdx.x & 63), m(lane & 15), h(lane >> 4) {}

  // Page of the lane's key (key lane % KEYS) of tile t; -1: none.
  __device__ __forceinline__ int page_of(const int* table, int t) const {
    const int j = t * KEYS + (lane & (KEYS - 1)), at = j / p.page_size;
    return at < p.table_width ? table[at] : -1;
  }
  // Rows of the tile's keys, shared among the lanes.  Keys past the end or of no page read the cache's first row.
  __device__ __forceinline__ void locate(int t, int page, int length, unsigned& there) {
    const int j = t * KEYS + (lane & (KEYS - 1)), slot = j % p.page_size;
    const bool ok = j < length && page >= 0 && page < p.pages;
    there = (unsigned)__ballot(ok) & (KEYS == 32 ? 0xffffffffu : 0xffffu);
    const int64_t k = ok ? page * p.kpage + slot * p.kslot : 0, v = ok ? page * p.vpage + slot * p.vslot : 0;
#pragma unroll
    for (int u = 0; u < KU; ++u) koff[u] = __shfl(k, 16 * u + m);
#pragma unroll
    for (int t = 0; t < VK; ++t) voff[t] = __shfl(v, 16 * (t >> 2) + 4 * h + (t & 3));
  }
  __device__ __forceinline__ void load_k() {
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = KL * (4 * s + h);
        kf[u][s] = *reinterpret_cast<const kvec*>(kbase + koff[u] + (d < a.D ? d : 0) * (int)sizeof(T));
      }
  }
  __device__ __forceinline__ void load_v() {
#pragma unroll
    for (int t = 0; t < VK; ++t)
#pragma unroll
      for (int c = 0; c < VC / VL; ++c) {
        const int d = 16 * VL * c + VL * m;
        vf[t][c] = *reinterpret_cast<const vvec*>(vbase + voff[t] + (d < a.D ? d : 0) * (int)sizeof(T));
      }
  }

  // acc += V^T times the tile's weights; for the lanes that are `mine`, if SOME
  template <bool SOME>
  __device__ __forceinline__ void add_values(const float (&x)[RB][KU][4], f32x4 (&acc)[RB][VC],
                                             const bool (&mine)[RB]) const {
    const auto put = [&](int q, int c, f32x4 sum) {
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[q][c][r] = !SOME || mine[q] ? sum[r] : acc[q][c][r];
    };
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
        for (int q = 0; q < RB; ++q) put(q, c, mfma_16x16(v, hi[q], mfma_16x16(v, lo[q], acc[q][c])));
      }
    } else {
#pragma unroll
      for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int q = 0; q < RB; ++q) {
          f32x4 sum = acc[q][c];
#pragma unroll
          for (int r = 0; r < 4; ++r) sum = mfma_16x16(vf[r][c / VL][c % VL], x[q][0][r], sum);
          put(q, c, sum);
        }
    }
  }
  // Whether the tile's values hold an infinity or NaN: on their bits, and by size, since the compiler, which is told that
  // there are no NaN, knows the usual test of the exponent for what it is.
  __device__ __forceinline__ bool any_not_finite() const {
    bool bad = false;
#pragma unroll
    for (int k = 0; k < VK; ++k)
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        const uint32_t bits = __builtin_bit_cast(uint32_t, (float)vf[k][c / VL][c % VL]);
        bad |= bits << 1 >= 0xff000000u;
      }
    return __ballot(bad) != 0;
  }

  // Tiles [t0, t1) of head hk of sequence b, rows from row0 on; to the output or to part `slot`.
  __device__ __forceinline__ void run(int b, int hk, int row0, int t0, int t1, T* out, Parts parts, int64_t slot,
                                      char* lds) {
    const int wave = wave_id(), length = length_of(p, b);
    const int rows = a.Nq * a.G, n_rows = min(rows - row0, 16 * RB);
    const int count = p.counts ? min(max(p.counts[b], 0), a.Nq) : a.Nq;
    const int* table = p.page_table + b * p.table_stride;
    kbase = p.keys + hk * p.khead;
    vbase = p.values + hk * p.vhead;

    int t = t0 + wave, page = t < t1 ? page_of(table, t) : -1;
    unsigned there = 0;
    if (t < t1) {
      locate(t, page, length, there);
      load_k();
      load_v();
      page = t + kWaves < t1 ? page_of(table, t + kWaves) : -1;
    }

    int pos[RB], lim[RB], head[RB];
    kvec qf[RB][KS];
    float far_lo[RB], far_hi[RB];
#pragma unroll
    for (int q = 0; q < RB; ++q) {
      const int r = row0 + 16 * q + m, i = r < rows ? r / a.G : 0;
      head[q] = hk * a.G + (r < rows ? r - i * a.G : 0);
      const bool live = r < rows && i < count;
      pos[q] = length - count + i;
      lim[q] = !live ? 0 : a.causal ? min(pos[q] + 1, length) : length;
      const T* row = static_cast<const T*>(a.q) + b * a.qb + i * a.qn + head[q] * a.qh;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = KL * (4 * s + h);
        qf[q][s] = live && d < a.D ? *reinterpret_cast<const kvec*>(row + d) : kvec{};
      }
      far_lo[q] = a.table ? table_value(a, 0, head[q]) : 0.f;
      far_hi[q] = a.table ? table_value(a, 2 * a.radius, head[q]) : 0.f;
    }
    const int first = length - count;   // position of the first query

    f32x4 acc[RB][VC];
    float top[RB], ref[RB], l[RB];
#pragma unroll
    for (int q = 0; q < RB; ++q) {
#pragma unroll
      for (int c = 0; c < VC; ++c) acc[q][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      top[q] = -kInf;
      ref[q] = l[q] = 0.f;
    }
    const Capped<T, CAP> capped(a);
    const float mult = a.scale * kLog2e;

    for (; t < t1; t += kWaves) {
      const int j0 = t * KEYS;
      const bool next = t + kWaves < t1;
      const unsigned now = there;
      f32x4 s[RB][KU];
#pragma unroll
      for (int q = 0; q < RB; ++q)
#pragma unroll
        for (int u = 0; u < KU; ++u) s[q][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int st = 0; st < KS; ++st) {
          kvec k = kf[u][st];
          if (KL * (4 * st + h) >= a.D) k = kvec{};   // zero times what lies there has to be zero
#pragma unroll
          for (int q = 0; q < RB; ++q) {
            if constexpr (sizeof(T) == 2) {
              s[q][u] = mfma_16x16(k, qf[q][st], s[q][u]);
            } else {
#pragma unroll
              for (int e = 0; e < KL; ++e) s[q][u] = mfma_16x16(k[e], qf[q][st][e], s[q][u]);
            }
          }
        }
      int64_t vnext[VK];
      if (next) {
        int64_t vnow[VK];
#pragma unroll
        for (int k = 0; k < VK; ++k) vnow[k] = voff[k];
        locate(t + kWaves, page, length, there);
        load_k();
        page = t + 2 * kWaves < t1 ? page_of(table, t + 2 * kWaves) : -1;
#pragma unroll
        for (int k = 0; k < VK; ++k) {
          vnext[k] = voff[k];
          voff[k] = vnow[k];
        }
      }

      float x[RB][KU][4];
#pragma unroll
      for (int q = 0; q < RB; ++q) {
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float slope;
            x[q][u][r] = a.cap > 0.f ? capped.score(s[q][u][r], capped.k3, slope) : s[q][u][r] * mult;
          }
        if (a.table) {
          const int rel0 = j0 - first;   // the first key from the first query
          if (rel0 - (a.Nq - 1) >= a.radius || rel0 + KEYS - 1 <= -a.radius) {
            const float far = rel0 > 0 ? far_hi[q] : far_lo[q];
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
              for (int r = 0; r < 4; ++r) x[q][u][r] += far;
          } else {
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int rel = j0 + 16 * u + 4 * h + r - pos[q];
                x[q][u][r] += table_value(a, min(max(rel, -a.radius), a.radius) + a.radius, head[q]);
              }
          }
        }
        float mx = -kInf;
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int k = 16 * u + 4 * h + r;
            const bool ok = j0 + k < lim[q] && (now >> k & 1);
            x[q][u][r] = ok ? x[q][u][r] : -kInf;
            mx = fmaxf(mx, x[q][u][r]);
          }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
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

      if (now != (KEYS == 32 ? 0xffffffffu : 0xffffu)) {
        // what a key that is not there holds has to count nothing, whatever it is
#pragma unroll
        for (int k = 0; k < VK; ++k)
          if (!(now >> (16 * (k >> 2) + 4 * h + (k & 3)) & 1))
#pragma unroll
            for (int c = 0; c < VC / VL; ++c) vf[k][c] = vvec{};
      }
      if (a.causal && j0 + KEYS > first + 1 && any_not_finite()) {
        // a value that is not finite counts for the queries that see it alone (zero times it is not zero): one query
        // after the other, the last first, with the keys behind each taken away
        for (int qi = (min(row0 + 16 * RB, rows) - 1) / a.G; qi >= row0 / a.G; --qi) {
#pragma unroll
          for (int k = 0; k < VK; ++k)
            if (j0 + 16 * (k >> 2) + 4 * h + (k & 3) > first + qi)
#pragma unroll
              for (int c = 0; c < VC / VL; ++c) vf[k][c] = vvec{};
          bool mine[RB];
#pragma unroll
          for (int q = 0; q < RB; ++q) mine[q] = pos[q] == first + qi;
          add_values<true>(x, acc, mine);
        }
      } else {
        add_values<false>(x, acc, {});
      }
      if (next) {
#pragma unroll
        for (int k = 0; k < VK; ++k) voff[k] = vnext[k];
        load_v();
      }
    }

    // the waves' parts through LDS
    float* sh = reinterpret_cast<float*>(lds);                       // [waves][16 RB][DP]
    float* ml = sh + kWaves * 16 * RB * DP;                          // [waves][16 RB][2]
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
    for (int k = threadIdx.x; k < n_rows * DP; k += 64 * kWaves) {
      const int r = k / DP, d = k - r * DP;
      if (d >= a.D) continue;
      float most = -kInf;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) most = fmaxf(most, ml[2 * (w * 16 * RB + r)]);
      const float to = most == -kInf ? 0.f : most;
      float o = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int at = w * 16 * RB + r;
        const float f = fast_exp2(ml[2 * at] - to);
        o += f * sh[at * DP + d];
        sum += f * ml[2 * at + 1];
      }
      if (slot < 0) {
        const int i = (row0 + r) / a.G, g = row0 + r - i * a.G;
        out[(((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D + d] = (T)over_sum(o, sum);
      } else {
        const int64_t at = slot * min(rows, 16 * RB) + r;
        parts.o[at * a.D + d] = o;
        if (d == 0) {
          parts.ml[2 * at] = sum == 0.f ? -kInf : to;
          parts.ml[2 * at + 1] = sum;
        }
      }
    }
    __syncthreads();
  }
};

// An item is a block of rows of a key head of a sequence.  Without groups a workgroup takes an item; with them the tiles
// of all items, one behind the other, are dealt evenly to the workgroups, whatever the sequences' lengths: a workgroup's
// share of an item is its part (workgroup + item) of the join, or the whole, which is written at once.
template <class T, int DP, int RB, int CAP>
__global__ __launch_bounds__(64 * kWaves) void paged_kernel(const AttnArgs a, const PagedArgs p, T* __restrict__ out,
                                                            Parts parts) {
  constexpr int KEYS = Cache<T>::KEYS;
  __shared__ __attribute__((aligned(16))) char lds[kWaves * 16 * RB * (DP + 2) * 4];
  Walk<T, DP, RB, CAP> walk(a, p);
  const int items = a.Hk * p.blocks;   // of a sequence
  if (p.groups == 0) {
    const int b = blockIdx.x / items, item = blockIdx.x - b * items;
    walk.run(b, item / p.blocks, item % p.blocks * 16 * RB, 0, (length_of(p, b) + KEYS - 1) / KEYS, out, parts, -1, lds);
    return;
  }
  const int64_t total = uniform(tiles_before<KEYS>(p, a.B, items));
  const int64_t n = min((int64_t)p.groups, (total + p.least - 1) / p.least);
  if ((int64_t)blockIdx.x >= n) return;
  int64_t at = total * blockIdx.x / n;
  const int64_t end = total * (blockIdx.x + 1) / n;
  // the sequence that holds tile `at`
  int b = 0;
  int64_t before = 0;
  for (const int lane = threadIdx.x & 63;; b += 64) {
    const int64_t own = b + lane < a.B ? (int64_t)((length_of(p, b + lane) + KEYS - 1) / KEYS) * items : 0;
    int64_t sum = own;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const int64_t o = __shfl_up(sum, m);
      if (lane >= m) sum += o;
    }
    const uint64_t past = __ballot(before + sum > at);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      b += l;
      before = uniform(before + __shfl(sum - own, l));
      break;
    }
    before = uniform(before + __shfl(sum, 63));
    if (b + 64 >= a.B) return;
  }
  for (; at < end && b < a.B; ++b) {
    const int tiles = (length_of(p, b) + KEYS - 1) / KEYS;
    while (at < end && at - before < (int64_t)tiles * items) {
      const int item = (int)((at - before) / tiles), t0 = (int)((at - before) - (int64_t)item * tiles);
      const int t1 = (int)min((int64_t)tiles, t0 + (end - at));
      const int64_t slot = t0 == 0 && t1 == tiles ? -1 : (int64_t)blockIdx.x + (int64_t)b * items + item;
      walk.run(b, item / p.blocks, item % p.blocks * 16 * RB, t0, t1, out, parts, slot, lds);
      at += t1 - t0;
    }
    before += (int64_t)tiles * items;
  }
}

// Adds the parts of a row in a fixed order: wave w takes parts w, w + waves, ..., then the waves are added.  Rows that
// one workgroup had are there already; rows of empty sequences get zeros.
constexpr int kJoinWaves = 8;
template <class T, int KEYS>
__global__ __launch_bounds__(64 * kJoinWaves) void paged_join_kernel(const AttnArgs a, const PagedArgs p,
                                                                     T* __restrict__ out, Parts parts, int block_rows) {
  __shared__ float sh[kJoinWaves][3][64];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = blockIdx.x;   // (b, i, head)
  const int h = (int)(row % a.H), i = (int)(row / a.H % a.Nq), b = (int)(row / a.H / a.Nq);
  const int hk = h / a.G, r = i * a.G + h - hk * a.G, items = a.Hk * p.blocks;
  const int item = hk * p.blocks + r / block_rows;
  const int tiles = (length_of(p, b) + KEYS - 1) / KEYS;
  const int64_t total = uniform(tiles_before<KEYS>(p, a.B, items));
  const int64_t n = min((int64_t)p.groups, (total + p.least - 1) / p.least);
  int64_t w0 = 0, w1 = -1;
  if (tiles > 0) {
    const int64_t at = uniform(tiles_before<KEYS>(p, b, items)) + (int64_t)item * tiles;
    w0 = ((at + 1) * n - 1) / total;
    w1 = ((at + tiles) * n - 1) / total;
    if (w0 == w1) return;
  }
  const int64_t slot0 = (int64_t)b * items + item;
  const int stride = min(a.Nq * a.G, block_rows);
  float top = -kInf;
  for (int64_t w = w0 + lane; w <= w1; w += 64) top = fmaxf(top, parts.ml[2 * ((w + slot0) * stride + r % block_rows)]);
#pragma unroll
  for (int m = 32; m > 0; m /= 2) top = fmaxf(top, __shfl_xor(top, m));
  const float to = top == -kInf ? 0.f : top;
  float o[2] = {0.f, 0.f}, sum = 0.f;
  const int d0 = min(lane, a.D - 1), d1 = min(lane + 64, a.D - 1);
#pragma unroll 4
  for (int64_t w = w0 + wave; w <= w1; w += kJoinWaves) {
    const int64_t at = (w + slot0) * stride + r % block_rows;
    const float f = fast_exp2(parts.ml[2 * at] - to);
    o[0] += f * parts.o[at * a.D + d0];
    o[1] += f * parts.o[at * a.D + d1];
    sum += f * parts.ml[2 * at + 1];
  }
  sh[wave][0][lane] = o[0];
  sh[wave][1][lane] = o[1];
  sh[wave][2][lane] = sum;
  __syncthreads();
  if (wave > 0) return;
  o[0] = o[1] = sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) {
    o[0] += sh[w][0][lane];
    o[1] += sh[w][1][lane];
    sum += sh[w][2][lane];
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.D) out[row * a.D + lane + 64 * e] = (T)over_sum(o[e], sum);
}

struct Plan {
  int rb, blocks, groups, least;
  int64_t items, slots;
};

// Rows in blocks of 16 or 32.  Keys shared out over workgroups unless an item's are few (the join costs what the shorter
// walk gains) or the items many.
Plan plan(const AttnArgs& a, const bioemu_paged_cache& c, bool f32) {
  Plan p{};
  const int rows = a.Nq * a.G;
  p.rb = rows <= 16 ? 1 : 2;
  p.blocks = (rows + 16 * p.rb - 1) / (16 * p.rb);
  p.items = (int64_t)a.B * a.Hk * p.blocks;
  const int64_t most = c.pages > 0 ? c.table_width * c.page_size : 0;
  if (most <= 1024 || p.items >= 16 * attn_units()) return p;
  p.groups = 2 * attn_units();
  p.least = 2 * kWaves;
  p.slots = p.groups + p.items;
  return p;
}

size_t parts_bytes(const AttnArgs& a, const Plan& p) {
  return (size_t)p.slots * std::min(a.Nq * a.G, 16 * p.rb) * (a.D + 2) * sizeof(float);
}

int paged_args(const bioemu_paged_cache* c, const bioemu_attention_args* in, AttnArgs* a, Plan* pl) {
  if (const int rc = attn_args("paged_attention", in, a)) return rc;
  if (in->Nk || in->k || in->v || in->q_segments || in->k_segments || in->prefix || in->lengths)
    return set_error(BIOEMU_ERR_INVALID_ARG, "paged_attention: keys, lengths and masks come from the cache");
  if (const int rc = paged_cache_args("paged_attention", c, a->B, a->Hk, in->f32 != 0)) return rc;
  *pl = plan(*a, *c, in->f32 != 0);
  if (pl->items >= (int64_t(1) << 30) || (int64_t)a->B * a->Nq * a->H >= (int64_t(1) << 31))
    return set_error(BIOEMU_ERR_UNSUPPORTED, "paged_attention: B=%d, Nq=%d, H=%d are too many", a->B, a->Nq, a->H);
  return BIOEMU_OK;
}

template <class T, int DP>
int launch(const AttnArgs& a, const PagedArgs& p, const Plan& pl, T* out, void* ws, hipStream_t stream) {
  const int block_rows = 16 * pl.rb;
  Parts parts{static_cast<float*>(ws), nullptr};
  if (ws) parts.ml = parts.o + pl.slots * std::min(a.Nq * a.G, block_rows) * a.D;
  {
    KernelTimerScope timer("paged_attention", stream);
    const dim3 grid((unsigned)(pl.groups ? pl.groups : pl.items));
    const auto go = [&](auto kernel) { kernel<<<grid, 64 * kWaves, 0, stream>>>(a, p, out, parts); };
    const bool wide = !fast_cap<T>(a);
    if (pl.rb == 1) {
      if (!wide)
        go(paged_kernel<T, DP, 1, kCapped>);
      else if constexpr (sizeof(T) == 2)
        go(paged_kernel<T, DP, 1, kCapWide>);
    } else {
      if (!wide)
        go(paged_kernel<T, DP, 2, kCapped>);
      else if constexpr (sizeof(T) == 2)
        go(paged_kernel<T, DP, 2, kCapWide>);
    }
    if (const int rc = check_launch("paged_attention")) return rc;
  }
  if (!pl.groups) return BIOEMU_OK;
  KernelTimerScope timer("paged_join", stream);
  paged_join_kernel<T, Cache<T>::KEYS><<<dim3((unsigned)((int64_t)a.B * a.Nq * a.H)), 64 * kJoinWaves, 0, stream>>>(
      a, p, out, parts, block_rows);
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
  const PagedArgs p{static_cast<const char*>(cache->keys), static_cast<const char*>(cache->values), ks[0] * item,
                    ks[1] * item, ks[2] * item, vs[0] * item, vs[1] * item, vs[2] * item, cache->page_table,
                    cache->table_stride, cache->lengths, cache->counts, (int)cache->pages, (int)cache->page_size,
                    (int)cache->table_width, pl.blocks, pl.groups, pl.least};
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
