// Rotary positions, alone and on the way into a paged cache, for gfx950.
//
//   a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t),  t = position * frequency
//
// The angle is a 64-bit product in turns, of which whole quarters are taken off before it is rounded to fp32: at
// position 10^6 an fp32 product is off by 0.03 radians, this one by 2^-27 wherever it is.
//
// A workgroup takes a few tokens.  Its threads first request the values that they will turn, then compute cos and sin of
// every (token, pair) once, into LDS, and every head of the token reads them there.  Appending is the same with k's rows
// going to their slots and v's copied beside them.
//
// Reading and writing bounds it (a stream of 2 GB is read at 6.2 TB/s).  In bf16: 16384 tokens of 16/4 heads of 128, 26 us
// (6.4 TB/s: the inputs, 84 MB, fit the last-level cache); 2 x 4096 of 32/8 heads of 128, 32 us (5.3); appending 4 x up to
// 4000 of 32/8 heads of 128, 62 us (4.5 of what there is, 5.1 with the zeros of q's padding).  One token, 2 us.
#include <algorithm>

#include "common.h"
#include "internal.h"

namespace bioemu {
namespace {

constexpr int kThreads = 256;
// pieces a thread holds at once; in the half layout a piece is of both halves
template <bool INTERLEAVED>
constexpr int kUnits = INTERLEAVED ? 8 : 4;
constexpr int kMaxWidth = 512;

// n / d for n below 2^31: n mul >> shift, mul = 2^(31 + l) / d rounded up, l = log2 of d rounded up.
struct Divisor {
  uint32_t mul = 0, shift = 0;
  Divisor() = default;
  explicit Divisor(int64_t d) {
    uint32_t l = 0;
    while ((int64_t(1) << l) < d) ++l;
    mul = (uint32_t)(((uint64_t(1) << (31 + l)) + d - 1) / d);
    shift = 31 + l;
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((uint64_t)(uint32_t)n * mul >> shift); }
};

struct RotaryArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;        // k_out and v_out: the caches where appending
  int64_t q_st[3], k_st[3], v_st[3];   // batch, row, head
  int64_t ko_st[3], vo_st[3];          // page, slot, head
  const int* positions;
  const double* frequencies;
  const int *page_table, *lengths, *counts;
  int64_t table_stride;
  float magnitude;
  int N, H, Hk, D, pairs, tokens, per, interleaved, inverse;
  int pages, page_size, table_width;
  int heads, pieces;                    // rows of a token, pieces of a row
  Divisor by_n, by_heads, by_pieces, by_pairs;
};

// cos and sin of `position` times `frequency` radians.
__device__ __forceinline__ f32x2 cos_sin(int position, double frequency, float magnitude, bool inverse) {
  const double turns = position * (frequency * 0.15915494309189535);   // 1 / (2 pi)
  const double quarters = 4.0 * (turns - floor(turns)), whole = rint(quarters);
  float s, c;
  sincospif(0.5f * (float)(quarters - whole), &s, &c);
  const int n = (int)whole & 3;
  const float co = n == 0 ? c : n == 1 ? -s : n == 2 ? -c : s;
  const float si = n == 0 ? s : n == 1 ? c : n == 2 ? -s : -c;
  return f32x2{co * magnitude, inverse ? -si * magnitude : si * magnitude};
}

// Where a token's rows come from and go to.
struct Token {
  int64_t key, value;   // elements of the caches, or -1
  int b, i, live;
};

// V values at a time; a piece is V values, or in the half layout V of each half, or 2 V of what does not turn.  APPEND:
// with v and a cache.  STREAM: results go past the caches.
template <class T, int V, bool INTERLEAVED, bool APPEND, bool STREAM>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const RotaryArgs a) {
  typedef T vec __attribute__((ext_vector_type(V)));
  extern __shared__ __attribute__((aligned(16))) char lds[];
  Token* tok = reinterpret_cast<Token*>(lds);
  f32x2* turn = reinterpret_cast<f32x2*>(lds + a.per * sizeof(Token));   // [per][pairs]

  const int t0 = blockIdx.x * a.per, n = min(a.per, a.tokens - t0);
  const int turned = INTERLEAVED ? 2 * a.pairs / V : a.pairs / V;   // pieces of a row that turn
  const int q_heads = a.q ? a.H : 0, units = n * a.heads * a.pieces;
  constexpr int U = kUnits<INTERLEAVED>;
  // where the two parts of a piece begin in its row; past it: there is no second
  const int apart = (a.D - 2 * a.pairs + 2 * V - 1) / (2 * V) * V;
  const auto first_of = [&](int p) { return INTERLEAVED || p < turned ? p * V : a.pairs + p * V; };
  const auto second_of = [&](int p, int d) { return d + (p < turned ? a.pairs : apart); };

  for (int u0 = 0; u0 == 0 || u0 < units; u0 += kThreads * U) {
    vec x[U], y[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int u = u0 + e * kThreads + threadIdx.x;
      x[e] = y[e] = vec{};
      if (u >= units) continue;
      const int row = a.by_pieces(u), p = u - row * a.pieces, t = a.by_heads(row), head = row - t * a.heads;
      const int b = a.by_n(t0 + t), i = t0 + t - b * a.N, hk = head - q_heads;
      if (APPEND && a.counts && i >= a.counts[b]) continue;   // padding: nothing to read
      const T* src;
      if (hk < 0)
        src = static_cast<const T*>(a.q) + b * a.q_st[0] + i * a.q_st[1] + head * a.q_st[2];
      else if (!APPEND || hk < a.Hk)
        src = static_cast<const T*>(a.k) + b * a.k_st[0] + i * a.k_st[1] + hk * a.k_st[2];
      else
        src = static_cast<const T*>(a.v) + b * a.v_st[0] + i * a.v_st[1] + (hk - a.Hk) * a.v_st[2];
      if constexpr (INTERLEAVED) {
        x[e] = *reinterpret_cast<const vec*>(src + p * V);
      } else {
        const int d = first_of(p), other = second_of(p, d);
        x[e] = *reinterpret_cast<const vec*>(src + d);
        if (other < a.D) y[e] = *reinterpret_cast<const vec*>(src + other);
      }
    }
    if (u0 == 0) {
      if (APPEND && threadIdx.x < n) {
        const int b = a.by_n(t0 + threadIdx.x), i = t0 + threadIdx.x - b * a.N;
        const int count = a.counts ? min(max(a.counts[b], 0), a.N) : a.N;
        // 64 bits: lengths may hold anything
        const int64_t at = (int64_t)a.lengths[b] - count + i;
        Token to{-1, -1, b, i, i < count};
        if (to.live && at >= 0 && at / a.page_size < a.table_width) {
          const int page = a.page_table[b * a.table_stride + at / a.page_size];
          const int slot = (int)(at % a.page_size);
          if (page >= 0 && page < a.pages) {
            to.key = page * a.ko_st[0] + slot * a.ko_st[1];
            to.value = page * a.vo_st[0] + slot * a.vo_st[1];
          }
        }
        tok[threadIdx.x] = to;
      }
      for (int k = threadIdx.x; k < n * a.pairs; k += kThreads) {
        const int t = a.by_pairs(k), b = a.by_n(t0 + t), i = t0 + t - b * a.N;
        int position = i;
        if (a.positions)
          position = a.positions[t0 + t];
        else if (APPEND)
          position = a.lengths[b] - (a.counts ? min(max(a.counts[b], 0), a.N) : a.N) + i;
        turn[k] = cos_sin(position, a.frequencies[k - t * a.pairs], a.magnitude, a.inverse);
      }
      __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int u = u0 + e * kThreads + threadIdx.x;
      if (u >= units) continue;
      const int row = a.by_pieces(u), p = u - row * a.pieces, t = a.by_heads(row), head = row - t * a.heads;
      const int hk = head - q_heads;
      const bool value = APPEND && hk >= a.Hk;
      const f32x2* cs = turn + t * a.pairs;
      vec r = x[e], w = y[e];
      if (p < turned && !value) {
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const f32x2 c = cs[(p * V + j) / 2];
            const float lo = (float)x[e][j], hi = (float)x[e][j + 1];
            r[j] = (T)(lo * c[0] - hi * c[1]);
            r[j + 1] = (T)(lo * c[1] + hi * c[0]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const f32x2 c = cs[p * V + j];
            const float lo = (float)x[e][j], hi = (float)y[e][j];
            r[j] = (T)(lo * c[0] - hi * c[1]);
            w[j] = (T)(lo * c[1] + hi * c[0]);
          }
        }
      }
      T* dst;
      if (hk < 0) {
        dst = static_cast<T*>(a.q_out) + ((int64_t)(t0 + t) * a.H + head) * a.D;
        if (APPEND && !tok[t].live) r = w = vec{};
      } else if constexpr (APPEND) {
        const int64_t at = value ? tok[t].value : tok[t].key;
        if (at < 0) continue;
        dst = value ? static_cast<T*>(a.v_out) + at + (hk - a.Hk) * a.vo_st[2]
                    : static_cast<T*>(a.k_out) + at + hk * a.ko_st[2];
      } else {
        dst = static_cast<T*>(a.k_out) + ((int64_t)(t0 + t) * a.Hk + hk) * a.D;
      }
      const int d = first_of(p), other = INTERLEAVED ? a.D : second_of(p, d);
      vec *to = reinterpret_cast<vec*>(dst + d), *too = reinterpret_cast<vec*>(dst + other);
      if constexpr (STREAM) {
        __builtin_nontemporal_store(r, to);
        if (other < a.D) __builtin_nontemporal_store(w, too);
      } else {
        *to = r;
        if (other < a.D) *too = w;
      }
    }
  }
}

// Values a piece: as many as 16 bytes hold and the turned part is whole pieces of.
int piece(const RotaryArgs& a, bool f32) {
  const int part = a.interleaved ? 2 * a.pairs : a.pairs;
  int v = f32 ? 4 : 8;
  while (part % v) v /= 2;
  return v;
}

template <class T, int V, bool APPEND, bool STREAM>
void launch(const RotaryArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.tokens - 1) / a.per + 1));
  const size_t lds = a.per * (sizeof(Token) + a.pairs * sizeof(f32x2));
  if (a.interleaved) {
    if constexpr (V > 1) rotary_kernel<T, V, true, APPEND, STREAM><<<grid, kThreads, lds, stream>>>(a);
  } else {
    rotary_kernel<T, V, false, APPEND, STREAM><<<grid, kThreads, lds, stream>>>(a);
  }
}
template <class T, int V, bool APPEND>
void launch(const RotaryArgs& a, hipStream_t stream) {
  // Results that no cache near the CUs holds (they have 4 MB a XCD) pass them by, so as not to drive out what is being
  // read: 16384 tokens of 16/4 heads of 128 in bf16 27 us (6.1 TB/s), 39 the other way.
  if ((int64_t)a.tokens * a.heads * a.D * (int64_t)sizeof(T) >= 32 << 20)
    launch<T, V, APPEND, true>(a, stream);
  else
    launch<T, V, APPEND, false>(a, stream);
}

template <bool APPEND>
int run(const char* what, RotaryArgs& a, bool f32, hipStream_t stream) {
  KernelTimerScope timer(what, stream);
  const int v = piece(a, f32);
  a.heads = (a.q ? a.H : 0) + (a.k ? (APPEND ? 2 : 1) * a.Hk : 0);
  a.pieces = a.interleaved ? a.D / v : a.pairs / v + (a.D - 2 * a.pairs + 2 * v - 1) / (2 * v);
  // a workgroup has as many tokens as its threads hold at once, where that leaves the launch wide enough (16384 tokens of
  // 16/4 heads of 128: 26.1 us, 27.4 with a rest that takes another turn)
  const int64_t held = kThreads * (a.interleaved ? kUnits<true> : kUnits<false>);
  a.per = (int)std::min(std::max(held / ((int64_t)a.heads * a.pieces), (int64_t)1), (int64_t)16);
  while (a.per > 1 && a.tokens / a.per < 1024) a.per /= 2;
  // a launch has fewer than 2^32 threads.  So many tokens fit a GPU only with narrow heads: 128 of them at most, and
  // 40 KB of LDS
  while ((a.tokens - 1) / a.per + 1 >= 1 << 24) a.per *= 2;
  a.by_n = Divisor(a.N);
  a.by_heads = Divisor(a.heads);
  a.by_pieces = Divisor(a.pieces);
  a.by_pairs = Divisor(std::max(a.pairs, 1));
  if (f32) {
    if (v == 4) launch<float, 4, APPEND>(a, stream);
    else if (v == 2) launch<float, 2, APPEND>(a, stream);
    else launch<float, 1, APPEND>(a, stream);
  } else {
    if (v == 8) launch<bf16, 8, APPEND>(a, stream);
    else if (v == 4) launch<bf16, 4, APPEND>(a, stream);
    else if (v == 2) launch<bf16, 2, APPEND>(a, stream);
    else launch<bf16, 1, APPEND>(a, stream);
  }
  return check_launch(what);
}

// Rows of the tensor at 16-byte addresses (strides of dimensions of one entry are of no account).
bool rows_aligned(const void* p, const int64_t* st, int64_t n0, int64_t n1, int64_t n2, int64_t per) {
  return aligned16(p) && (n0 <= 1 || st[0] % per == 0) && (n1 <= 1 || st[1] % per == 0) && (n2 <= 1 || st[2] % per == 0);
}

// Checks what both entry points share and lays it out.
int rotary_args(const char* what, const bioemu_rotary_args* in, RotaryArgs* a) {
  if (!in) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: null arguments", what);
  const int64_t B = in->B, N = in->N, H = in->H, Hk = in->Hk, D = in->D;
  if (B < 0 || N < 0 || (in->q && H < 1) || (in->k && Hk < 1) || D < 1 || in->pairs < 0)
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: B=%ld, N=%ld, H=%ld, Hk=%ld, D=%ld, %ld pairs", what, (long)B, (long)N,
                     (long)H, (long)Hk, (long)D, (long)in->pairs);
  if (D % 8 || D > kMaxWidth)
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: head width %ld (a multiple of 8, at most %d)", what, (long)D, kMaxWidth);
  if (2 * in->pairs > D)
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: %ld pairs in heads of %ld", what, (long)in->pairs, (long)D);
  if (in->pairs && !in->frequencies && B * N > 0) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: null pointer", what);
  if (B >= (int64_t(1) << 31) || N >= (int64_t(1) << 31) || B * N >= (int64_t(1) << 31) - 16 || H > 65536 || Hk > 65536)
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: B=%ld, N=%ld, H=%ld, Hk=%ld are too many", what, (long)B, (long)N,
                     (long)H, (long)Hk);
  const int64_t per = in->f32 ? 4 : 8;
  if ((in->q && !rows_aligned(in->q, in->q_stride, B, N, H, per)) ||
      (in->k && !rows_aligned(in->k, in->k_stride, B, N, Hk, per)))
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: rows of q and k start at 16-byte addresses", what);
  *a = RotaryArgs{};
  a->q = in->q;
  a->k = in->k;
  for (int d = 0; d < 3; ++d) {
    a->q_st[d] = in->q_stride[d];
    a->k_st[d] = in->k_stride[d];
  }
  a->positions = in->positions;
  a->frequencies = in->frequencies;
  a->magnitude = in->magnitude;
  a->N = (int)N;
  a->H = (int)H;
  a->Hk = (int)Hk;
  a->D = (int)D;
  a->pairs = (int)in->pairs;
  a->tokens = (int)(B * N);
  a->interleaved = in->interleaved != 0;
  a->inverse = in->inverse != 0;
  return BIOEMU_OK;
}

}  // namespace

int paged_cache_args(const char* what, const bioemu_paged_cache* c, int64_t B, int64_t Hk, bool f32) {
  if (!c) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: null arguments", what);
  if (c->pages < 0 || c->page_size < 1 || c->table_width < 0)
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: %ld pages of %ld, table of %ld", what, (long)c->pages,
                     (long)c->page_size, (long)c->table_width);
  const int64_t most = int64_t(1) << 27;
  if (c->pages >= (int64_t(1) << 31) || c->page_size > (1 << 20) || c->table_width > most ||
      c->table_width * c->page_size > most)
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: %ld pages of %ld, table of %ld are too many", what, (long)c->pages,
                     (long)c->page_size, (long)c->table_width);
  if (B == 0) return BIOEMU_OK;
  if (!c->lengths || (c->table_width > 0 && !c->page_table) || (c->pages > 0 && (!c->keys || !c->values)))
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: null pointer", what);
  const int64_t per = f32 ? 4 : 8;
  if (!rows_aligned(c->keys, c->keys_stride, c->pages, c->page_size, Hk, per) ||
      !rows_aligned(c->values, c->values_stride, c->pages, c->page_size, Hk, per))
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: rows of keys and values start at 16-byte addresses", what);
  return BIOEMU_OK;
}

}  // namespace bioemu

using namespace bioemu;

extern "C" int bioemu_rotary(const bioemu_rotary_args* args, void* q_out, void* k_out, hipStream_t stream) {
  RotaryArgs a;
  if (const int rc = rotary_args("rotary", args, &a)) return rc;
  if (a.tokens == 0 || (!a.q && !a.k)) return BIOEMU_OK;
  if ((a.q && !q_out) || (a.k && !k_out) || !aligned16(q_out) || !aligned16(k_out))
    return set_error(BIOEMU_ERR_INVALID_ARG, "rotary: outputs must be there and 16-byte aligned");
  a.q_out = q_out;
  a.k_out = k_out;
  return run<false>("rotary", a, args->f32 != 0, stream);
}

extern "C" int bioemu_paged_append(const bioemu_paged_cache* cache, const bioemu_rotary_args* args, const void* v,
                                   const int64_t* v_stride, void* q_out, hipStream_t stream) {
  RotaryArgs a;
  if (const int rc = rotary_args("paged_append", args, &a)) return rc;
  const bool f32 = args->f32 != 0;
  if (const int rc = paged_cache_args("paged_append", cache, args->B, args->Hk, f32)) return rc;
  if (a.tokens == 0) return BIOEMU_OK;
  if (!a.k || !v || !v_stride || !rows_aligned(v, v_stride, args->B, a.N, a.Hk, f32 ? 4 : 8) || (a.q && !q_out) ||
      !aligned16(q_out))
    return set_error(BIOEMU_ERR_INVALID_ARG, "paged_append: k, v and q's output must be there and 16-byte aligned");
  a.inverse = 0;
  a.v = v;
  a.q_out = q_out;
  a.k_out = cache->keys;
  a.v_out = cache->values;
  for (int d = 0; d < 3; ++d) {
    a.v_st[d] = v_stride[d];
    a.ko_st[d] = cache->keys_stride[d];
    a.vo_st[d] = cache->values_stride[d];
  }
  a.page_table = cache->page_table;
  a.table_stride = cache->table_stride;
  a.lengths = cache->lengths;
  a.counts = cache->counts;
  a.pages = (int)cache->pages;
  a.page_size = (int)cache->page_size;
  a.table_width = (int)cache->table_width;
  return run<true>("paged_append", a, f32, stream);
}
