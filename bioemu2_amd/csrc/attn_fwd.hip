// Attention forward, for gfx950 (formulas and layouts: attn.h).
//
// attn_fwd: a workgroup owns 128 queries of one head, a wave 32 of them; 64-key (bf16) or 32-key (fp32) tiles of K and
// V are staged in LDS, double-buffered, and shared by the four waves.  Per wave and 32 keys: S^T = K Q^T (DP / 16
// MFMAs), the running maximum and sum of the softmax per lane (a lane is a query; its other half joins by one
// shuffle), O^T += V^T P^T with P straight from registers.  The maximum moves only when a score exceeds it by 2^8:
// until then weights are at most 256 and nothing is rescaled.
// attn_few: up to 32 (query, head of a group) rows share their keys, as single tokens over a cache do: the rows fill
// one MFMA operand, every wave takes 32-key tiles of its own (K and V read once, bound by HBM), and the waves join.
// Both may split the keys over workgroups (few rows, long axis); attn_join adds the parts.
//
// Measured, attn_fwd, bf16: 8192 causal tokens behind a prefix of 1000, 16/4 heads of 128, 286 to 298 us called on and on
// (936 to 975 TFLOP/s of what is not masked; a large matrix product reaches 1195), 306 to 371 under the profiler, whose
// calls stand apart; 2 x 2048 causal, 16/4 heads of 64, capped, 58 us (300 TFLOP/s):
// the vector instructions of the softmax take longer than the MFMAs there.  fp32: 1000 tokens, 8 heads of 64, 25 us
// (82 TFLOP/s; a large fp32 matrix product 154).  attn_few: 8 single tokens over 8200 to 32768 keys of 8 heads of 128,
// 157 us (4.9 TB/s), over 32768 keys each 259 and in fp32 439; one over 773 keys of 16 heads of 64, 13 us, a walk of 25
// tiles' latencies shared by 8 waves; one over 8192 keys of 8 heads of 128, 19 us, in fp32 (two waves) 45.
//
// A training call in bf16 also writes what the rounding of o took off (o_lo): the backward pass needs do . o, and with
// it from o + o_lo the error of dq and dk falls from 1.50 to 1.46 times what rounding their results alone gives (the
// rest is the rounding of the probabilities and of ds to the operands of the products).
#include <algorithm>
#include <atomic>

#include "attn.h"

namespace bioemu {
namespace {

constexpr int kWaveRows = 32;
constexpr int kGroupRows = 128;
constexpr float kRescale = 8.f;   // log2 of the largest weight before the maximum moves

// Per-row partial results of one split: [rows][D] values and [rows][2] (maximum in log2 units, sum).
struct Parts {
  float *o, *ml;
};

// Four values of a row, rounded, and what that took off.
template <class T>
__device__ __forceinline__ void store_quad(T* out, T* lo, const float (&v)[4]) {
  typedef T quad __attribute__((ext_vector_type(4)));
  quad hi, rest;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    hi[c] = (T)v[c];
    rest[c] = (T)(v[c] - (float)hi[c]);
  }
  *reinterpret_cast<quad*>(out) = hi;
  if (lo) *reinterpret_cast<quad*>(lo) = rest;
}

template <class T, int DP, int CAP>
__global__ __launch_bounds__(kAttnThreads) void attn_fwd_kernel(const AttnArgs a, T* __restrict__ out,
                                                                T* __restrict__ lo, float* __restrict__ lse,
                                                                Parts parts, int splits,
                                                                int qblocks, int total) {
  constexpr int KB = Operand<T>::kBlock, SUB = KB / 32, STEPS = DP / 16, DB = DP / 32;
  typedef Staged<T, DP, KB> KV;
  __shared__ __attribute__((aligned(1024))) char tiles[KV::BUFFERS][2][KV::BYTES];
  __shared__ __attribute__((aligned(16))) int segs[2][64];
  __shared__ float lut[2 * (kMaxRadius + kPad) + 1];
  __shared__ int list[kListBlocks];
  __shared__ uint8_t flags[kListBlocks];
  __shared__ int red[3][4], count;

  const int item = attn_item(total, qblocks);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = wave_id(), ln = lane & 31, lh = lane >> 5;
  const int qblk = qblocks - 1 - item % qblocks;   // long rows of a causal mask first
  const int rest = item / qblocks, split = rest % splits, bh = rest / splits, h = bh % a.H, b = bh / a.H;
  const int hk = h / a.G;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const bool seg = a.q_seg != nullptr;

  const int i = qblk * kGroupRows + wave * kWaveRows + ln;
  const bool live = i < a.Nq;
  const int pos = length - a.Nq + i;
  const int qseg = seg && live ? a.q_seg[(int64_t)b * a.Nq + i] : 0;
  // keys below lim are allowed (their segment aside); rows past the last one restrict nothing
  int lim = a.causal ? min(max(pos + 1, prefix), length) : length;
  if (qseg < 0) lim = 0;
  int seg_lo = live && qseg >= 0 ? qseg : 0x7fffffff, seg_hi = live ? qseg : -1, wg_max = live ? lim : 0;
  const WaveRange own_segs(seg_lo, seg_hi);
  wg_extremes(seg_lo, seg_hi, wg_max, red);
  int wave_min = live ? lim : 0x7fffffff, wave_max = live ? lim : 0;
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    wave_min = min(wave_min, __shfl_xor(wave_min, m));
    wave_max = max(wave_max, __shfl_xor(wave_max, m));
  }
  wave_min = __builtin_amdgcn_readfirstlane(wave_min);
  wave_max = __builtin_amdgcn_readfirstlane(wave_max);
  const int wave_pos = __builtin_amdgcn_readfirstlane(pos);   // of the wave's first row
  if (!live) lim = 0x7fffffff;

  const Capped<T, CAP> capped(a);
  if (a.table) fill_lut(a, h, CAP ? capped.k3 : 0.f, lut);

  Frag<T> qf[STEPS];
  {
    const T* row = static_cast<const T*>(a.q) + b * a.qb + (int64_t)(live ? i : 0) * a.qn + h * a.qh;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[s] = row_operand<T>(row, live, s, lh, a.D);
  }
  const T* kbase = static_cast<const T*>(a.k) + b * a.kb + hk * a.kh;
  const T* vbase = static_cast<const T*>(a.v) + b * a.vb + hk * a.vh;
  KV k_tile(a.kn, a.D), v_tile(a.vn, a.D);
  const int* kseg = seg ? a.k_seg + (int64_t)b * a.Nk : nullptr;

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = zero16();
  // weights are 2^(x - mref); a row starts with its first finite score, then mref moves when one exceeds limit
  float mref = 0.f, limit = -kInf, l = 0.f;
  const float mult = a.scale * kLog2e;
  const auto score = [&](float raw, float add) {
    float slope;
    if constexpr (CAP != kUncapped) return capped.score(raw, add, slope);
    return raw * mult + add;
  };

  auto stage = [&](int entry, int buf) {
    const int k0 = (entry & kBlockMask) * KB;
    char(*to)[KV::BYTES] = tiles[buf % KV::BUFFERS];
    k_tile.fetch(kbase + (int64_t)k0 * a.kn, length - k0, a.kn, a.D, to[0], wave);
    v_tile.fetch(vbase + (int64_t)k0 * a.vn, length - k0, a.vn, a.D, to[1], wave);
    if (seg && wave == 0) copy_ints(kseg + k0, length - k0, segs[buf], lane);
  };

  // a turn walks all blocks, or with segments those that one list can hold
  const int blocks = (wg_max + KB - 1) / KB;
  for (int c0 = 0, c1; c0 < blocks; c0 = c1) {
    c1 = seg ? min(blocks, c0 + kListBlocks) : blocks;
    const int n = seg ? list_blocks<KB>(kseg, length, seg_lo, seg_hi, c0, c1, flags, list, &count) : blocks;
    const int t0 = (int)((int64_t)n * split / splits), t1 = (int)((int64_t)n * (split + 1) / splits);
    auto entry = [&](int t) { return seg ? __builtin_amdgcn_readfirstlane(list[t]) : t; };
    if (t0 < t1) stage(entry(t0), t0 & 1);
    for (int t = t0; t < t1; ++t) {
      const int e = entry(t), buf = t & 1, k0 = (e & kBlockMask) * KB;
      __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's copies landed
      __syncthreads();                       // ... and everyone's; the other buffer is free
      char(*tile)[KV::BYTES] = tiles[buf % KV::BUFFERS];
      if constexpr (KV::BUFFERS == 1) {
        k_tile.store(tile[0]);
        v_tile.store(tile[1]);
        __syncthreads();
      }
      if (t + 1 < t1) stage(entry(t + 1), buf ^ 1);
      if (e & kEntryHoles) {
        // keys in no segment have weight 0, and 0 times what their values hold has to be 0
        const int r = threadIdx.x / (kAttnThreads / KB);
        if (segs[buf][r] < 0) KV::clear(tile[1], r, threadIdx.x % (kAttnThreads / KB), kAttnThreads / KB);
        __syncthreads();
      }
      if (k0 >= wave_max) continue;
      bool all = true;   // every key has the one segment of all queries of this wave
      if (seg && !own_segs.meets<KB>(segs[buf], lane, all)) continue;
      const char *kt = tile[0], *vt = tile[1];
      float x[SUB][16];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        f32x16 s = zero16();
#pragma unroll
        for (int st = 0; st < STEPS; ++st) s = mfma16(KV::rows(kt, 32 * u + ln, st, lh), qf[st], s);
        const int rel0 = k0 + 32 * u - wave_pos;   // of the wave's first query and the first key
        if (a.table && !all_far(a, rel0)) {
          const float* bias = lut + (rel0 + a.radius + kPad + 4 * lh - ln);
#pragma unroll
          for (int r = 0; r < 16; ++r) x[u][r] = score(s[r], bias[8 * (r >> 2) + (r & 3)]);
        } else {
          const float add = a.table ? lut[rel0 > 0 ? 2 * (a.radius + kPad) : 0] : CAP ? capped.k3 : 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) x[u][r] = score(s[r], add);
        }
      }
      if (k0 + KB > wave_min)
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            x[u][r] = k0 + 32 * u + 8 * (r >> 2) + 4 * lh + (r & 3) < lim ? x[u][r] : -kInf;
      if (!all)
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int4 ks = *reinterpret_cast<const int4*>(&segs[buf][32 * u + 8 * q + 4 * lh]);
            x[u][4 * q] = ks.x == qseg ? x[u][4 * q] : -kInf;
            x[u][4 * q + 1] = ks.y == qseg ? x[u][4 * q + 1] : -kInf;
            x[u][4 * q + 2] = ks.z == qseg ? x[u][4 * q + 2] : -kInf;
            x[u][4 * q + 3] = ks.w == qseg ? x[u][4 * q + 3] : -kInf;
          }
      float mx = x[0][0];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[u][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      // against mref only now: scores of the type's lowest value may have come first
      if (__ballot(mx > limit)) {
        const bool begun = limit > -kInf;
        const float to = mx == -kInf ? mref : (begun ? fmaxf(mref, mx) : mx);
        const float f = begun ? fast_exp2(mref - to) : 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        l *= f;
        mref = to;
        if (mx > -kInf || begun) limit = mref + kRescale;
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          x[u][r] = fast_exp2(x[u][r] - mref);
          l += x[u][r];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const Frag<T> p = as_operand<T>(x[u], s);
#pragma unroll
          for (int d = 0; d < DB; ++d) acc[d] = mfma16(KV::cols(vt, 32 * u + 16 * s, 32 * d, lane), p, acc[d]);
        }
      }
    }
    __syncthreads();   // the list and both buffers are free
  }

  l += __shfl_xor(l, 32);
  if (!live) return;
  const int64_t row = ((int64_t)b * a.Nq + i) * a.H + h;
  if (splits == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t at = row * a.D + 32 * d + 8 * r + 4 * lh;
        if (32 * d + 8 * r + 4 * lh < a.D) {
          const float v[4] = {acc[d][4 * r] * inv, acc[d][4 * r + 1] * inv, acc[d][4 * r + 2] * inv,
                              acc[d][4 * r + 3] * inv};
          store_quad(out + at, lo ? lo + at : nullptr, v);
        }
      }
    if (lse && lh == 0)
      store_log_sum(lse, (int64_t)a.B * a.H * a.Nq, ((int64_t)b * a.H + h) * a.Nq + i, mref, l);
  } else {
    const int64_t rows = (int64_t)a.B * a.Nq * a.H, at0 = split * rows + row;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 32 * d + 8 * r + 4 * lh;
        if (at < a.D)
          *reinterpret_cast<f32x4*>(parts.o + at0 * a.D + at) =
              f32x4{acc[d][4 * r], acc[d][4 * r + 1], acc[d][4 * r + 2], acc[d][4 * r + 3]};
      }
    if (lh == 0) {
      parts.ml[2 * at0] = l == 0.f ? -kInf : mref;
      parts.ml[2 * at0 + 1] = l;
    }
  }
}

// Waves of attn_few: each has a K and a V tile of its own, 64 KB of LDS in all at most (two workgroups a CU, so that
// one streams while the other starts or joins: 131 KB with two tiles of each measured 168 us where this takes 157).
template <class T, int DP>
constexpr int few_waves() {
  constexpr int w = 65536 / (2 * Tile<T, DP, 32>::BYTES);
  return w < 8 ? w : 8;
}
constexpr int kLgkm0 = 0xc07f;   // s_waitcnt lgkmcnt(0)
constexpr int vmcnt(int n) { return 0x0f70 | (n & 15) | ((n >> 4) << 14); }

// chunk: 32-key tiles of one split.  Splits are of equal length whatever the sequences' lengths (those past a
// sequence's end do nothing), and workgroups take them in plain order, round the XCDs: no two share a key.
// CAP: kCapped (whether there is a cap is asked at run time, beside the latency of the copies) or kCapWide.
template <class T, int DP, int CAP>
__global__ __launch_bounds__((64 * few_waves<T, DP>())) void attn_few_kernel(const AttnArgs a, T* __restrict__ out,
                                                                           T* __restrict__ lo,
                                                                           float* __restrict__ lse, Parts parts,
                                                                           int splits, int chunk) {
  constexpr int W = few_waves<T, DP>(), STEPS = DP / 16, DB = DP / 32;
  typedef Tile<T, DP, 32> KV;
  constexpr int CP = KV::copies(64);
  __shared__ __attribute__((aligned(1024))) char tiles[W][2][KV::BYTES];
  __shared__ float ml[W][2][32];

  const int lane = threadIdx.x & 63, wave = wave_id(), ln = lane & 31, lh = lane >> 5;
  const int bs = blockIdx.x / a.Hk, hk = blockIdx.x - bs * a.Hk, b = bs / splits, split = bs - b * splits;
  const int rows = a.Nq * a.G;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const bool seg = a.q_seg != nullptr;

  // lane n: query i and head g of the group
  const bool live = ln < rows;
  const int i = live ? ln / a.G : 0, h = hk * a.G + (live ? ln - i * a.G : 0);
  const int pos = length - a.Nq + i;
  const int qseg = seg ? a.q_seg[(int64_t)b * a.Nq + i] : 0;
  int lim = a.causal ? min(max(pos + 1, prefix), length) : length;
  if (qseg < 0 || !live) lim = 0;
  int top = lim, low = live ? lim : 0x7fffffff;
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    top = max(top, __shfl_xor(top, m));
    low = min(low, __shfl_xor(low, m));
  }
  top = __builtin_amdgcn_readfirstlane(top);
  low = __builtin_amdgcn_readfirstlane(low);

  const T* kbase = static_cast<const T*>(a.k) + b * a.kb + hk * a.kh;
  const T* vbase = static_cast<const T*>(a.v) + b * a.vb + hk * a.vh;
  unsigned koff[CP], voff[CP];
  KV::offsets(lane, 64, a.kn, a.D, koff);
  KV::offsets(lane, 64, a.vn, a.D, voff);
  char *kt = tiles[wave][0], *vt = tiles[wave][1];
  auto stage_k = [&](int t) {
    KV::copy(kbase + (int64_t)t * 32 * a.kn, length - t * 32, a.kn, a.D, kt, 0, 64, koff);
  };
  auto stage_v = [&](int t) {
    KV::copy(vbase + (int64_t)t * 32 * a.vn, length - t * 32, a.vn, a.D, vt, 0, 64, voff);
  };
  const int blocks = (top + 31) / 32, t0 = min(split * chunk, blocks), t1 = min(t0 + chunk, blocks);
  if (t0 + wave < t1) {   // before the queries and the bias: it takes longest
    stage_k(t0 + wave);
    stage_v(t0 + wave);
  }

  Frag<T> qf[STEPS];
  {
    const T* row = static_cast<const T*>(a.q) + b * a.qb + (int64_t)i * a.qn + h * a.qh;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[s] = row_operand<T>(row, live, s, lh, a.D);
  }
  const float far_lo = a.table ? table_value(a, 0, h) : 0.f, far_hi = a.table ? table_value(a, 2 * a.radius, h) : 0.f;
  const int* kseg = seg ? a.k_seg + (int64_t)b * a.Nk : nullptr;

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = zero16();
  float m = -kInf, mref = 0.f, l = 0.f;
  const Capped<T, CAP> capped(a);
  const float mult = a.scale * kLog2e;

  // K of the next tile is on its way while V of this one is waited for and used, and V while K is: a tile's copies are
  // made as soon as its reader is done with the one before
  for (int t = t0 + wave; t < t1; t += W) {
    const int k0 = t * 32;
    __builtin_amdgcn_s_waitcnt(vmcnt(CP));   // all but V
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    f32x16 s = zero16();
#pragma unroll
    for (int st = 0; st < STEPS; ++st) s = mfma16(KV::rows(kt, ln, st, lh), qf[st], s);
    __builtin_amdgcn_s_waitcnt(kLgkm0);   // the tile has been read
    if (t + W < t1) stage_k(t + W);
    float x[16];
    if (a.cap > 0.f) {
      float slope;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = capped.score(s[r], capped.k3, slope);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = s[r] * mult;
    }
    if (a.table) {
      const int rel0 = k0 - (length - a.Nq);   // the first key from the first query
      if (rel0 - (a.Nq - 1) >= a.radius || rel0 + 31 <= -a.radius) {
        const float far = rel0 > 0 ? far_hi : far_lo;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] += far;
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int rel = k0 + 8 * (r >> 2) + 4 * lh + (r & 3) - pos;
          x[r] += table_value(a, min(max(rel, -a.radius), a.radius) + a.radius, h);
        }
      }
    }
    if (k0 + 32 > low || seg) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = k0 + 8 * (r >> 2) + 4 * lh + (r & 3);
        bool ok = j < lim;
        if (seg) ok = ok && kseg[min(j, a.Nk - 1)] == qseg;
        x[r] = ok ? x[r] : -kInf;
      }
    }
    float mx = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__ballot(mx > m + kRescale)) {
      const float mn = fmaxf(m, mx), to = mn == -kInf ? 0.f : mn;
      const float f = fast_exp2(m - to);
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= f;
      l *= f;
      m = mn;
      mref = to;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x[r] = fast_exp2(x[r] - mref);
      l += x[r];
    }
    if (t + W < t1)
      __builtin_amdgcn_s_waitcnt(vmcnt(CP));   // all but the next K
    else
      __builtin_amdgcn_s_waitcnt(vmcnt(0));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (seg) {
      // two lanes a key: values of a key in no segment are zeroed (0 times them has to be 0)
      const int r = lane >> 1;
      if (k0 + r < length && kseg[k0 + r] < 0) KV::clear(vt, r, lane & 1, 2);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<T> p = as_operand<T>(x, st);
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[d] = mfma16(KV::cols(vt, 16 * st, 32 * d, lane), p, acc[d]);
    }
    __builtin_amdgcn_s_waitcnt(kLgkm0);
    if (t + W < t1) stage_v(t + W);
  }

  // the waves' parts through LDS (over the tiles: W x 32 x DP floats)
  l += __shfl_xor(l, 32);
  __syncthreads();
  float* sh = reinterpret_cast<float*>(&tiles[0][0][0]);
  if (lh == 0) {
    ml[wave][0][ln] = l == 0.f ? -kInf : mref;
    ml[wave][1][ln] = l;
  }
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f32x4*>(sh + (wave * 32 + ln) * DP + 32 * d + 8 * r + 4 * lh) =
          f32x4{acc[d][4 * r], acc[d][4 * r + 1], acc[d][4 * r + 2], acc[d][4 * r + 3]};
  __syncthreads();
  const int64_t all = (int64_t)a.B * a.Nq * a.H;
  for (int k = threadIdx.x; k < rows * DP; k += 64 * W) {
    const int r = k / DP, d = k - r * DP;
    if (d >= a.D) continue;
    float top_m = -kInf;
#pragma unroll
    for (int w = 0; w < W; ++w) top_m = fmaxf(top_m, ml[w][0][r]);
    const float to = top_m == -kInf ? 0.f : top_m;
    float o = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = fast_exp2(ml[w][0][r] - to);
      o += f * sh[(w * 32 + r) * DP + d];
      sum += f * ml[w][1][r];
    }
    const int qi = r / a.G, qh = hk * a.G + r - qi * a.G;
    const int64_t row = ((int64_t)b * a.Nq + qi) * a.H + qh;
    if (splits == 1) {
      const float v = sum == 0.f ? 0.f : o / sum;
      const T hi = (T)v;
      out[row * a.D + d] = hi;
      if (lo) lo[row * a.D + d] = (T)(v - (float)hi);
      if (lse && d == 0) store_log_sum(lse, all, ((int64_t)b * a.H + qh) * a.Nq + qi, to, sum);
    } else {
      parts.o[(split * all + row) * a.D + d] = o;
      if (d == 0) {
        parts.ml[2 * (split * all + row)] = sum == 0.f ? -kInf : to;
        parts.ml[2 * (split * all + row) + 1] = sum;
      }
    }
  }
}

// The splits' parts of a row added, in a fixed order; a split that saw nothing wrote no values.
// attn_join: few rows of many splits, a workgroup a row: wave w takes splits w, w + 4, ..., then the waves are added.
// Lane d holds values d and 64 + d.
template <class T>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(const AttnArgs a, Parts parts, int splits,
                                                                 T* __restrict__ out, T* __restrict__ lo,
                                                                 float* __restrict__ lse) {
  __shared__ float sh[4][3][64];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t rows = (int64_t)a.B * a.Nq * a.H, row = blockIdx.x;
  float top = -kInf;
  for (int s = lane; s < splits; s += 64) top = fmaxf(top, parts.ml[2 * (s * rows + row)]);
#pragma unroll
  for (int m = 32; m > 0; m /= 2) top = fmaxf(top, __shfl_xor(top, m));
  const float to = top == -kInf ? 0.f : top;
  float o[2] = {0.f, 0.f}, sum = 0.f;
  const int d0 = min(lane, a.D - 1), d1 = min(lane + 64, a.D - 1);
  for (int s0 = wave; s0 < splits; s0 += 16) {
    float f[4], l[4], x0[4], x1[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int s = s0 + 4 * q;
      const int64_t at = (s < splits ? s : s0) * rows + row;
      f[q] = s < splits ? fast_exp2(parts.ml[2 * at] - to) : 0.f;
      l[q] = parts.ml[2 * at + 1];
      x0[q] = parts.o[at * a.D + d0];
      x1[q] = parts.o[at * a.D + d1];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      o[0] += f[q] == 0.f ? 0.f : f[q] * x0[q];
      o[1] += f[q] == 0.f ? 0.f : f[q] * x1[q];
      sum += f[q] == 0.f ? 0.f : f[q] * l[q];
    }
  }
  sh[wave][0][lane] = o[0];
  sh[wave][1][lane] = o[1];
  sh[wave][2][lane] = sum;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) o[h] = (sh[0][h][lane] + sh[1][h][lane]) + (sh[2][h][lane] + sh[3][h][lane]);
  sum = (sh[0][2][lane] + sh[1][2][lane]) + (sh[2][2][lane] + sh[3][2][lane]);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d = lane + 64 * h;
    if (d >= a.D) continue;
    const float v = o[h] * inv;
    const T hi = (T)v;
    out[row * a.D + d] = hi;
    if (lo) lo[row * a.D + d] = (T)(v - (float)hi);
  }
  if (lse && lane == 0) {
    const int64_t bi = row / a.H, h = row - bi * a.H, b = bi / a.Nq, i = bi - b * a.Nq;
    store_log_sum(lse, rows, (b * a.H + h) * a.Nq + i, to, sum);
  }
}

// attn_join_rows: many rows, four values of one a thread.
template <class T>
__global__ __launch_bounds__(kAttnThreads) void attn_join_rows_kernel(const AttnArgs a, Parts parts, int splits,
                                                                      int rows, T* __restrict__ out,
                                                                      T* __restrict__ lo, float* __restrict__ lse) {
  const unsigned quads = a.D / 4, k = blockIdx.x * kAttnThreads + threadIdx.x, row = k / quads, d = (k - row * quads) * 4;
  if ((int)row >= rows) return;
  const f32x2* ml = reinterpret_cast<const f32x2*>(parts.ml) + row;
  float top = -kInf;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[(int64_t)s * rows][0]);
  const float to = top == -kInf ? 0.f : top;
  float o[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const f32x2 w = ml[(int64_t)s * rows];
    const f32x4 x = *reinterpret_cast<const f32x4*>(parts.o + ((int64_t)s * rows + row) * a.D + d);
    const float f = fast_exp2(w[0] - to);
    sum += f == 0.f ? 0.f : f * w[1];
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] += f == 0.f ? 0.f : f * x[c];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  const int64_t at = (int64_t)row * a.D + d;
  store_quad(out + at, lo ? lo + at : nullptr, v);
  if (lse && d == 0) {
    const int64_t bi = row / a.H, h = row - bi * a.H, b = bi / a.Nq, i = bi - b * a.Nq;
    store_log_sum(lse, rows, (b * a.H + h) * a.Nq + i, to, sum);
  }
}

bool few_rows(const AttnArgs& a) { return a.Nq * a.G <= 32; }

// Workgroups that the keys of a query block are split over.  Long rows: as many as bring the launch to two workgroups a
// CU, 256 keys each at least.  Long causal walks (the last rows' takes twice the mean, and nothing is left to start
// beside it): up to four a CU, 1024 keys each at least (1 x 8192, 8 heads of 64, bf16: 109 us with the join, 163 in one
// part; heads of 128: 191 and 212; fp32, 64: 427 and 523), from where the join costs less than that gains (4096 keys,
// heads of 64: 46 and 53; of 128: 79 and 73; 2048, 64: 58 and 59).  So too where more than two run on a CU (bf16, heads
// of up to 32: 4096 x 4096 of 24, all seen: 80 and 90).  Segments: as short as most are, no (4096 in parts of 256: 23
// and 16).
// Few rows: sequences of a cache are of unequal length, so up to sixteen a CU that even out, 512 keys each at least (8
// sequences of 8200 to 32768 keys, 8 heads: 160 us in parts of 2048, 157 in parts of 512), and none for up to 1024 keys,
// where the join costs what the shorter walk gains (773 keys: 18 us in four parts, 13 in one).  Both bounds were measured
// in bf16 at these sizes only; one or two sequences, and fp32, whose waves are fewer, take them as they are.
int key_splits(const AttnArgs& a, bool f32) {
  const bool few = few_rows(a);
  if (few && a.Nk <= 1024) return 1;
  const int64_t base = few ? (int64_t)a.B * a.Hk : (int64_t)a.B * a.H * ((a.Nq + kGroupRows - 1) / kGroupRows);
  const int64_t units = attn_units();
  const auto at_most = [&](int64_t want, int64_t keys) { return std::min(want, (a.Nk + keys - 1) / keys); };
  int64_t s = few ? at_most((16 * units + base - 1) / base, 512) : at_most((2 * units + base - 1) / base, 256);
  const int far = !f32 && a.D <= 64 ? 4096 : 8192;
  if (!few && !a.q_seg && a.Nk >= far && (a.causal || (!f32 && a.D <= 32)))
    s = std::max(s, std::min(4 * units / base, (int64_t)a.Nk / 1024));
  return s < 1 ? 1 : (int)s;
}

size_t parts_bytes(const AttnArgs& a, int splits) {
  return splits == 1 ? 0 : (size_t)splits * a.B * a.Nq * a.H * (a.D + 2) * sizeof(float);
}

template <class T, int DP>
int launch_fwd(const AttnArgs& a, void* o, void* o_lo, float* lse, void* ws, hipStream_t stream) {
  const int splits = key_splits(a, sizeof(T) == 4);
  const int64_t rows = (int64_t)a.B * a.Nq * a.H;
  Parts parts{static_cast<float*>(ws), nullptr};
  parts.ml = parts.o ? parts.o + (int64_t)splits * rows * a.D : nullptr;
  T *out = static_cast<T*>(o), *lo = static_cast<T*>(o_lo);
  if (few_rows(a)) {
    const int tiles = (a.Nk + 31) / 32, chunk = (tiles + splits - 1) / splits;
    KernelTimerScope timer("attn_few", stream);
    const dim3 grid((unsigned)(a.B * a.Hk * splits));
    const auto launch = [&](auto kernel) {
      kernel<<<grid, 64 * few_waves<T, DP>(), 0, stream>>>(a, out, lo, lse, parts, splits, chunk);
    };
    if (fast_cap<T>(a))
      launch(attn_few_kernel<T, DP, kCapped>);
    else if constexpr (sizeof(T) == 2)
      launch(attn_few_kernel<T, DP, kCapWide>);
    if (const int rc = check_launch("attn_few")) return rc;
  } else {
    const int qblocks = (a.Nq + kGroupRows - 1) / kGroupRows;
    const int64_t total = (int64_t)a.B * a.H * splits * qblocks;
    KernelTimerScope timer("attn_fwd", stream);
    const dim3 grid(attn_grid(total));
    const auto launch = [&](auto kernel) {
      kernel<<<grid, kAttnThreads, 0, stream>>>(a, out, lo, lse, parts, splits, qblocks, (int)total);
    };
    if (!(a.cap > 0.f))
      launch(attn_fwd_kernel<T, DP, kUncapped>);
    else if (fast_cap<T>(a))
      launch(attn_fwd_kernel<T, DP, kCapped>);
    else if constexpr (sizeof(T) == 2)
      launch(attn_fwd_kernel<T, DP, kCapWide>);
    if (const int rc = check_launch("attn_fwd")) return rc;
  }
  if (splits == 1) return BIOEMU_OK;
  KernelTimerScope timer("attn_join", stream);
  // 256 rows of 64 splits: 6 us by a workgroup each, 35 by quads; 32000 rows of 2: 5.6 us by quads, 13 by a wave each
  if (rows < 4 * attn_units() && splits > 4)
    attn_join_kernel<T><<<dim3((unsigned)rows), kAttnThreads, 0, stream>>>(a, parts, splits, out, lo, lse);
  else
    attn_join_rows_kernel<T><<<dim3((unsigned)((rows * (a.D / 4) + kAttnThreads - 1) / kAttnThreads)), kAttnThreads, 0,
                               stream>>>(a, parts, splits, (int)rows, out, lo, lse);
  return check_launch("attn_join");
}

}  // namespace

int attn_units() {
  // asking the runtime takes microseconds, as long as a launch
  static std::atomic<int> units[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return compute_units();
  int n = units[dev].load(std::memory_order_relaxed);
  if (n == 0) units[dev].store(n = compute_units(), std::memory_order_relaxed);
  return n;
}

int attn_args(const char* what, const bioemu_attention_args* in, AttnArgs* a) {
  if (!in) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: null arguments", what);
  const int64_t B = in->B, Nq = in->Nq, Nk = in->Nk, H = in->H, Hk = in->Hk, D = in->D;
  if (B < 0 || Nq < 0 || Nk < 0 || H < 1 || Hk < 1 || D < 1)
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: B=%ld, Nq=%ld, Nk=%ld, H=%ld, Hk=%ld, D=%ld", what, (long)B, (long)Nq,
                     (long)Nk, (long)H, (long)Hk, (long)D);
  if (H % Hk) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: %ld heads over %ld key heads", what, (long)H, (long)Hk);
  if (D % 8 || D > 128)
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: head width %ld (a multiple of 8, at most 128)", what, (long)D);
  const int64_t most = int64_t(1) << 27;
  if (Nq > most || Nk > most || B * H > (1 << 20) || B * Nq * H >= (int64_t(1) << 31) ||
      B * H * ((Nq + 127) / 128) * 512 >= (int64_t(1) << 31) || B * H * ((Nk + 127) / 128) * 32 >= (int64_t(1) << 31))
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: B=%ld, H=%ld, Nq=%ld, Nk=%ld are too many", what, (long)B, (long)H,
                     (long)Nq, (long)Nk);
  if (!(in->scale > -kInf && in->scale < kInf) || !(in->cap >= 0.f && in->cap < kInf))
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: scale %g, cap %g", what, (double)in->scale, (double)in->cap);
  if (in->cap > 0.f && (in->cap > 1e5f || !(fabsf(in->scale) / in->cap < 1e30f)))
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: cap %g with scale %g (a cap is at most 1e5)", what, (double)in->cap,
                     (double)in->scale);
  const int64_t per = in->f32 ? 4 : 8, far = int64_t(1) << 23;
  const void* ptr[3] = {in->q, in->k, in->v};
  const int64_t* st[3] = {in->q_stride, in->k_stride, in->v_stride};
  const int64_t len[3] = {Nq, Nk, Nk};
  int64_t row[3];
  for (int t = 0; t < 3; ++t) {
    if (!ptr[t] && B * len[t] > 0) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: null pointer", what);
    row[t] = len[t] > 1 ? st[t][1] : D;   // a single row has none, whatever stands there
    if (!aligned16(ptr[t]) || st[t][0] % per || row[t] % per || st[t][2] % per)
      return set_error(BIOEMU_ERR_INVALID_ARG, "%s: rows of q, k and v start at 16-byte addresses", what);
    if (row[t] > far || row[t] < D)
      return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: row stride %ld (head width to 2^23)", what, (long)row[t]);
  }
  if ((in->q_segments == nullptr) != (in->k_segments == nullptr))
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: segments of queries and of keys come together", what);
  if (in->bias_table) {
    if (!in->bias_buckets) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: null pointer", what);
    if (in->radius < 0 || in->radius > kMaxRadius || in->num_buckets < 1 || in->num_buckets > 256)
      return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: radius %ld (at most %d), %ld buckets (at most 256)", what,
                       (long)in->radius, kMaxRadius, (long)in->num_buckets);
  }
  *a = AttnArgs{in->q, in->k, in->v, in->q_stride[0], row[0], in->q_stride[2], in->k_stride[0],
                row[1], in->k_stride[2], in->v_stride[0], row[2], in->v_stride[2], in->q_segments,
                in->k_segments, in->prefix, in->lengths, in->bias_table, in->bias_buckets, in->scale, in->cap, (int)B,
                (int)Nq, (int)Nk, (int)H, (int)Hk, (int)(H / Hk), (int)D, (int)in->radius, (int)in->num_buckets,
                in->causal, in->table_bf16};
  return BIOEMU_OK;
}

}  // namespace bioemu

using namespace bioemu;

extern "C" size_t bioemu_attention_workspace_bytes(const bioemu_attention_args* args) {
  AttnArgs a;
  if (attn_args("attention", args, &a) || a.B == 0 || a.Nq == 0) return 0;
  return parts_bytes(a, key_splits(a, args->f32 != 0));
}

extern "C" int bioemu_attention_fwd(const bioemu_attention_args* args, void* o, void* o_lo, float* lse,
                                    void* workspace, size_t workspace_bytes, hipStream_t stream) {
  AttnArgs a;
  if (const int rc = attn_args("attention", args, &a)) return rc;
  if (a.B == 0 || a.Nq == 0) return BIOEMU_OK;
  if (!o || !aligned16(o) || !aligned16(o_lo))
    return set_error(BIOEMU_ERR_INVALID_ARG, "attention: o and o_lo must be 16-byte aligned");
  if (o_lo && args->f32) return set_error(BIOEMU_ERR_INVALID_ARG, "attention: o_lo is of bf16 calls");
  const size_t need = parts_bytes(a, key_splits(a, args->f32 != 0));
  if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return set_error(BIOEMU_ERR_WORKSPACE, "attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const int dp = a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128;
#define BIOEMU_FWD(T, P) \
  if (dp == P) return launch_fwd<T, P>(a, o, o_lo, lse, workspace, stream)
  if (args->f32) {
    BIOEMU_FWD(float, 32);
    BIOEMU_FWD(float, 64);
    BIOEMU_FWD(float, 128);
  } else {
    BIOEMU_FWD(bf16, 32);
    BIOEMU_FWD(bf16, 64);
    BIOEMU_FWD(bf16, 128);
  }
#undef BIOEMU_FWD
  return BIOEMU_ERR_UNSUPPORTED;
}
