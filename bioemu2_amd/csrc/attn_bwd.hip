// Attention backward, for gfx950 (formulas and layouts: attn.h).
//
//   dv_j = sum_i p_ij do_i;  dp_ij = do_i . v_j;  ds_ij = p_ij (dp_ij - do_i . o_i);  dtable[t, h] = sum ds over bucket t
//   dqk = ds (1 - tanh^2) scale;  dq_i = sum_j dqk_ij k_j;  dk_j = sum_i dqk_ij q_i
//
// p comes back from q, k and the row's saved log-sum.  Two kernels, no atomics between workgroups: attn_bwd_q owns
// 128 queries of a head and walks the keys (dq; the row sums do . o, which it writes for the other kernel; the table's
// gradient), attn_bwd_kv owns 128 keys of a key head and walks the queries of the group's heads (dk, dv).  The scores
// are so computed twice, 7 products instead of 5; adding dq over workgroups instead would need fp32 atomics (an order
// that changes results) or as many copies of dq.
//
// Measured, bf16: 2 x 2048 causal tokens, 16/4 heads of 64, capped, q 72 us, kv 85 us (the capped softmax's vector
// instructions); 4096 causal tokens, 16/4 heads of 128, q 199, kv 241 (266 and 334 registers: one wave a SIMD); 4096 packed tokens, 16 heads of 24, with the table's gradient, q 56, kv 47 (the walk of the longest
// sequence); fp32: 1000 tokens, 8 heads of 64, q 40, kv 46.
//
// Either may split its walk over workgroups where the rows alone do not fill the chip; attn_bwd_finish adds the parts.
//
// Rows whose scores' reference is at or beyond kWideRow (attn.h) take their weights against it and multiply them by the
// inverse sum; all others have log2 of the sum in the constant that is added to a score.
//
// The table's gradient sums ds along the diagonals of every 32 x 32 block that meets the radius: the block goes to LDS,
// rows 68 values apart with zeros between them, and lane e reads its diagonal (value e + n - 31 of row n) without a
// bound to check, 16 reads of two values.  (One LDS add an element took 45 cycles each, 8 times the whole.)  Every wave
// has a row of sums by offset; blocks wholly at or beyond the radius stay in registers.  Then waves, the offsets of a
// bucket and workgroups are added in fixed orders.
#include <algorithm>

#include "attn.h"

namespace bioemu {
namespace {

constexpr int kGroupRows = 128;

constexpr int kDiagRow = 68, kDiagBlock = 32 + 32 * kDiagRow;   // floats; 32 zeros in front of row 0

// LDS beyond the tiles: bias values by offset, and for the table's gradient, per wave, sums of ds by offset and a block.
inline size_t bias_lds(const AttnArgs& a, bool sums) {
  const size_t n = round_up(2 * (a.radius + kPad) + 1, 4);
  return a.table ? (n + (sums ? 4 * (n + kDiagBlock) : 0)) * sizeof(float) : 0;
}

// A lane's row of an accumulator [DB] of 32-value blocks times `scale`, rounded into `out`, or as fp32 into `part`.
template <class T, int DB>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[DB], float scale, T* out, float* part, int lh, int D) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = 32 * d + 8 * r + 4 * lh;
      if (at >= D) continue;
      if (out) {
        typedef T quad __attribute__((ext_vector_type(4)));
        quad v;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = (T)(acc[d][4 * r + c] * scale);
        *reinterpret_cast<quad*>(out + at) = v;
      } else {
        *reinterpret_cast<f32x4*>(part + at) = f32x4{acc[d][4 * r] * scale, acc[d][4 * r + 1] * scale,
                                                     acc[d][4 * r + 2] * scale, acc[d][4 * r + 3] * scale};
      }
    }
}

// Waves per SIMD that the registers have to allow: two where a few registers more would make it one (attn_bwd_kv at
// D = 64, 2 x 2048 causal tokens: 107 us with 257 registers, 87 with 255).
template <class T, int DP, bool KV>
constexpr int bwd_waves() {
  return sizeof(T) == 2 && KV && DP == 64 ? 2 : 1;
}

template <class T, int DP, int CAP>
__global__ __launch_bounds__(kAttnThreads, (bwd_waves<T, DP, false>())) void attn_bwd_q_kernel(
    const AttnArgs a, const T* __restrict__ o, const T* __restrict__ o_lo, const float* __restrict__ lse, const T*
    __restrict__ dout, int64_t db, int64_t dn, int64_t dh, T* __restrict__ dq, float* __restrict__ stats, float*
    __restrict__ dq_part, float* __restrict__ bias_part, int splits, int qblocks, int total) {
  constexpr int KB = Operand<T>::kBlock, SUB = KB / 32, STEPS = DP / 16, DB = DP / 32;
  typedef Staged<T, DP, KB> KV;
  __shared__ __attribute__((aligned(1024))) char tiles[KV::BUFFERS][2][KV::BYTES];
  __shared__ __attribute__((aligned(16))) int segs[2][64];
  __shared__ int list[kListBlocks];
  __shared__ uint8_t flags[kListBlocks];
  __shared__ int red[3][4], count;
  __shared__ float ends[4][2];
  __shared__ uint8_t which[2 * (kMaxRadius + kPad) + 1];   // buckets by offset
  extern __shared__ __attribute__((aligned(16))) float dyn[];   // bias values, sums by offset [4], blocks [4]

  const int item = attn_item(total, qblocks);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = wave_id(), ln = lane & 31, lh = lane >> 5;
  const int qblk = qblocks - 1 - item % qblocks, rest = item / qblocks, split = rest % splits, bh = rest / splits;
  const int h = bh % a.H, b = bh / a.H, hk = h / a.G;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const bool seg = a.q_seg != nullptr;
  const int nrel = lut_size(a), row4 = (nrel + 3) & ~3;
  float *lut = dyn, *sums = dyn + row4, *own = sums + wave * row4;
  float* diag = sums + 4 * row4 + wave * kDiagBlock + 32;

  const int i = qblk * kGroupRows + wave * 32 + ln;
  const bool live = i < a.Nq;
  const int pos = length - a.Nq + i;
  const int qseg = seg && live ? a.q_seg[(int64_t)b * a.Nq + i] : 0;
  int lim = a.causal ? min(max(pos + 1, prefix), length) : length;
  if (qseg < 0 || !live) lim = 0;
  int seg_lo = live && qseg >= 0 ? qseg : 0x7fffffff, seg_hi = live ? qseg : -1, wg_max = lim;
  const WaveRange own_segs(seg_lo, seg_hi);
  wg_extremes(seg_lo, seg_hi, wg_max, red);
  int wave_min = lim, wave_max = lim;
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    wave_min = min(wave_min, __shfl_xor(wave_min, m));
    wave_max = max(wave_max, __shfl_xor(wave_max, m));
  }
  wave_min = __builtin_amdgcn_readfirstlane(wave_min);
  wave_max = __builtin_amdgcn_readfirstlane(wave_max);
  const int wave_pos = __builtin_amdgcn_readfirstlane(pos);

  const Capped<T, CAP> capped(a);
  if (a.table) {
    fill_lut(a, h, CAP ? capped.k3 : 0.f, lut);
    if (bias_part) {
      for (int e = threadIdx.x; e < nrel; e += kAttnThreads)
        which[e] = (uint8_t)min((int)a.buckets[min(max(e - kPad, 0), 2 * a.radius)], a.nb - 1);
      for (int e = threadIdx.x; e < row4 + kDiagBlock; e += kAttnThreads)   // both are multiples of 4
        reinterpret_cast<f32x4*>(sums)[e] = f32x4{};
    }
  }

  const float mult = a.scale * kLog2e, out_scale = a.scale * (CAP != kUncapped ? Capped<T, CAP>::kSlope : 1.f);
  const auto score = [&](float raw, float add, float& slope) {
    if constexpr (CAP != kUncapped) return capped.score(raw, add, slope);
    return raw * mult + add;
  };

  const int64_t row = ((int64_t)b * a.Nq + (live ? i : 0)) * a.H + h, srow = ((int64_t)b * a.H + h) * a.Nq + i;
  // weights are 2^(x + base) row_inv; row_inv is 1 but for wide rows
  const int64_t plane = (int64_t)a.B * a.H * a.Nq;
  const float row_m = live ? lse[srow] : 0.f, row_l = live ? lse[plane + srow] : kInf;
  // a row that sees nothing, for whatever reason, contributes nothing, whatever it holds
  const bool on = live && lim > 0 && row_l != kInf;
  const bool row_wide = a.table && fabsf(row_m) >= kWideRow && row_l < kInf;
  const float row_inv = row_wide ? fast_exp2(-row_l) : 1.f;
  const bool wide = __ballot(row_wide) != 0;
  Frag<T> qf[STEPS], df[STEPS];
  float dsum = 0.f;
  {
    const T* pq = static_cast<const T*>(a.q) + b * a.qb + (int64_t)(live ? i : 0) * a.qn + h * a.qh;
    const T* pd = dout + b * db + (int64_t)(live ? i : 0) * dn + h * dh;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      qf[s] = row_operand<T>(pq, on, s, lh, a.D);
      df[s] = row_operand<T>(pd, on, s, lh, a.D);
      const Frag<T> of = row_operand<T>(o + row * a.D, on, s, lh, a.D);
#pragma unroll
      for (int t = 0; t < 8; ++t) dsum += (float)of[t] * (float)df[s][t];
      if (o_lo) {
        const Frag<T> ol = row_operand<T>(o_lo + row * a.D, on, s, lh, a.D);
#pragma unroll
        for (int t = 0; t < 8; ++t) dsum += (float)ol[t] * (float)df[s][t];
      }
    }
  }
  dsum += __shfl_xor(dsum, 32);
  // (without a table the constant part of the scores is in it, as it is in the table else)
  const float base = (a.table || !CAP ? 0.f : capped.k3) - (row_wide ? row_m : row_m + row_l);
  if (live && lh == 0 && split == 0) {
    stats[srow] = base;
    stats[plane + srow] = -dsum;
    if (a.table) stats[2 * plane + srow] = row_inv;
  }

  const T* kbase = static_cast<const T*>(a.k) + b * a.kb + hk * a.kh;
  const T* vbase = static_cast<const T*>(a.v) + b * a.vb + hk * a.vh;
  KV k_tile(a.kn, a.D), v_tile(a.vn, a.D);
  const int* kseg = seg ? a.k_seg + (int64_t)b * a.Nk : nullptr;

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = zero16();
  float far_lo = 0.f, far_hi = 0.f;

  auto stage = [&](int entry, int buf) {
    const int k0 = (entry & kBlockMask) * KB;
    char(*to)[KV::BYTES] = tiles[buf % KV::BUFFERS];
    k_tile.fetch(kbase + (int64_t)k0 * a.kn, length - k0, a.kn, a.D, to[0], wave);
    v_tile.fetch(vbase + (int64_t)k0 * a.vn, length - k0, a.vn, a.D, to[1], wave);
    if (seg && wave == 0) copy_ints(kseg + k0, length - k0, segs[buf], lane);
  };

  const int blocks = (wg_max + KB - 1) / KB;
  for (int c0 = 0, c1; c0 < blocks; c0 = c1) {   // one turn, or with segments one for each list
    c1 = seg ? min(blocks, c0 + kListBlocks) : blocks;
    const int n = seg ? list_blocks<KB>(kseg, length, seg_lo, seg_hi, c0, c1, flags, list, &count) : blocks;
    auto entry = [&](int t) { return seg ? __builtin_amdgcn_readfirstlane(list[t]) : t; };
    const int t0 = (int)((int64_t)n * split / splits), t1 = (int)((int64_t)n * (split + 1) / splits);
    if (t0 < t1) stage(entry(t0), t0 & 1);
    for (int t = t0; t < t1; ++t) {
      const int e = entry(t), buf = t & 1, k0 = (e & kBlockMask) * KB;
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
      char(*tile)[KV::BYTES] = tiles[buf % KV::BUFFERS];
      if constexpr (KV::BUFFERS == 1) {
        k_tile.store(tile[0]);
        v_tile.store(tile[1]);
        __syncthreads();
      }
      if (t + 1 < t1) stage(entry(t + 1), buf ^ 1);
      if (e & kEntryHoles) {
        const int r = threadIdx.x / (kAttnThreads / KB);
        if (segs[buf][r] < 0) {
          KV::clear(tile[0], r, threadIdx.x % (kAttnThreads / KB), kAttnThreads / KB);
          KV::clear(tile[1], r, threadIdx.x % (kAttnThreads / KB), kAttnThreads / KB);
        }
        __syncthreads();
      }
      if (k0 >= wave_max) continue;
      bool all = true;   // every key has the one segment of all queries of this wave
      if (seg && !own_segs.meets<KB>(segs[buf], lane, all)) continue;
      const char *kt = tile[0], *vt = tile[1];
#pragma unroll 1
      for (int u = 0; u < SUB; ++u) {
        f32x16 s = zero16(), dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = -dsum;
#pragma unroll
        for (int st = 0; st < STEPS; ++st) s = mfma16(KV::rows(kt, 32 * u + ln, st, lh), qf[st], s);
#pragma unroll
        for (int st = 0; st < STEPS; ++st) dp = mfma16(KV::rows(vt, 32 * u + ln, st, lh), df[st], dp);
        float x[16], slope[16];
        const int rel0 = k0 + 32 * u - wave_pos;   // of the wave's first query and the first key
        const bool far = all_far(a, rel0);
        if (a.table && !far) {
          const float* bias = lut + (rel0 + a.radius + kPad + 4 * lh - ln);
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = score(s[r], bias[8 * (r >> 2) + (r & 3)], slope[r]) + base;
        } else if (a.table) {
          const float add = lut[rel0 > 0 ? nrel - 1 : 0];
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = score(s[r], add, slope[r]) + base;
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = score(s[r], base, slope[r]);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = fast_exp2(x[r]) * dp[r];
        if (wide)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] *= row_inv;
        if (k0 + KB > wave_min)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = k0 + 32 * u + 8 * (r >> 2) + 4 * lh + (r & 3) < lim ? x[r] : 0.f;
        if (!all)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int4 ks = *reinterpret_cast<const int4*>(&segs[buf][32 * u + 8 * q + 4 * lh]);
            x[4 * q] = ks.x == qseg ? x[4 * q] : 0.f;
            x[4 * q + 1] = ks.y == qseg ? x[4 * q + 1] : 0.f;
            x[4 * q + 2] = ks.z == qseg ? x[4 * q + 2] : 0.f;
            x[4 * q + 3] = ks.w == qseg ? x[4 * q + 3] : 0.f;
          }
        if (bias_part) {
          if (far) {
            float v = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) v += x[r];
            if (rel0 > 0)
              far_hi += v;
            else
              far_lo += v;
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<f32x4*>(diag + ln * kDiagRow + 8 * q + 4 * lh) =
                  f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            float v0 = 0.f, v1 = 0.f;
#pragma unroll
            for (int n = 0; n < 32; n += 2) {
              v0 += diag[n * (kDiagRow + 1) + lane - 31];
              v1 += diag[(n + 1) * (kDiagRow + 1) + lane - 31];
            }
            if (lane < 63) own[rel0 + lane - 31 + a.radius + kPad] += v0 + v1;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
        if constexpr (CAP != kUncapped)
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] *= slope[r];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const Frag<T> p = as_operand<T>(x, st);
#pragma unroll
          for (int d = 0; d < DB; ++d) acc[d] = mfma16(KV::cols(kt, 32 * u + 16 * st, 32 * d, lane), p, acc[d]);
        }
      }
    }
    __syncthreads();
  }

  if (live) {
    const int64_t at_row = splits == 1 ? row : split * (int64_t)a.B * a.Nq * a.H + row;
    store_rows<T, DB>(acc, out_scale, splits == 1 ? dq + row * a.D : nullptr, dq_part + at_row * a.D, lh, a.D);
  }
  if (bias_part) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) {
      far_lo += __shfl_xor(far_lo, m);
      far_hi += __shfl_xor(far_hi, m);
    }
    if (lane == 0) {
      ends[wave][0] = far_lo;
      ends[wave][1] = far_hi;
    }
    __syncthreads();
    // waves in order into the first one's row, then each wave a quarter of the offsets into the buckets
    for (int e = threadIdx.x; e < nrel; e += kAttnThreads) {
      float v = (sums[e] + sums[row4 + e]) + (sums[2 * row4 + e] + sums[3 * row4 + e]);
      if (e == 0) v += (ends[0][0] + ends[1][0]) + (ends[2][0] + ends[3][0]);
      if (e == nrel - 1) v += (ends[0][1] + ends[1][1]) + (ends[2][1] + ends[3][1]);
      sums[e] = v;
    }
    __syncthreads();
    float* quarter = sums + 4 * row4 + wave * 256;   // over the blocks
    const int e0 = nrel * wave / 4, e1 = nrel * (wave + 1) / 4;
    for (int t = lane; t < a.nb; t += 64) {
      float v = 0.f;
#pragma unroll 16
      for (int e = e0; e < e1; ++e) v += which[e] == t ? sums[e] : 0.f;
      quarter[t] = v;
    }
    __syncthreads();
    quarter = sums + 4 * row4;
    float* out = bias_part + (((int64_t)b * qblocks + qblk) * splits + split) * a.nb * a.H + h;
    for (int t = threadIdx.x; t < a.nb; t += kAttnThreads)
      out[(int64_t)t * a.H] = (quarter[t] + quarter[256 + t]) + (quarter[512 + t] + quarter[768 + t]);
  }
}

template <class T, int DP, int CAP>
__global__ __launch_bounds__(kAttnThreads, (bwd_waves<T, DP, true>())) void attn_bwd_kv_kernel(
    const AttnArgs a, const float* __restrict__ row_stats, const T* __restrict__ dout, int64_t db, int64_t dn,
    int64_t dh, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part, int splits, int kblocks, int
    total) {
  constexpr int QB = Operand<T>::kBlock, SUB = QB / 32, STEPS = DP / 16, DB = DP / 32;
  typedef Staged<T, DP, QB> QD;
  __shared__ __attribute__((aligned(1024))) char tiles[QD::BUFFERS][2][QD::BYTES];
  __shared__ __attribute__((aligned(16))) int segs[2][64];
  __shared__ __attribute__((aligned(16))) float stats[2][2][64];   // what attn_bwd_q wrote of the rows
  __shared__ float inverse[64];
  __shared__ int list[kListBlocks];
  __shared__ uint8_t flags[kListBlocks];
  __shared__ int red[3][4], count;
  extern __shared__ float lut[];

  const int item = attn_item(total, kblocks);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = wave_id(), ln = lane & 31, lh = lane >> 5;
  const int kblk = item % kblocks, rest = item / kblocks, split = rest % splits, bh = rest / splits;
  const int hk = bh % a.Hk, b = bh / a.Hk;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const bool seg = a.q_seg != nullptr;
  const int first = length - a.Nq;   // position of query 0

  const int j = kblk * kGroupRows + wave * 32 + ln;
  const int kseg = seg && j < length ? a.k_seg[(int64_t)b * a.Nk + j] : 0;
  const bool on = j < length && kseg >= 0;
  // queries from imin on see this key (their segment aside)
  const int imin = !on ? 0x7fffffff : (a.causal && j >= prefix ? max(j - first, 0) : 0);
  int seg_lo = on ? kseg : 0x7fffffff, seg_hi = on ? kseg : -1, wg_min = -imin;
  const WaveRange own_segs(seg_lo, seg_hi);
  wg_extremes(seg_lo, seg_hi, wg_min, red);
  wg_min = -wg_min;
  int wave_min = imin, wave_max = imin;
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    wave_min = min(wave_min, __shfl_xor(wave_min, m));
    wave_max = max(wave_max, __shfl_xor(wave_max, m));
  }
  wave_min = __builtin_amdgcn_readfirstlane(wave_min);
  wave_max = __builtin_amdgcn_readfirstlane(wave_max);
  const int wave_key = kblk * kGroupRows + wave * 32;

  Frag<T> kf[STEPS], vf[STEPS];
  {
    const T* pk = static_cast<const T*>(a.k) + b * a.kb + (int64_t)(on ? j : 0) * a.kn + hk * a.kh;
    const T* pv = static_cast<const T*>(a.v) + b * a.vb + (int64_t)(on ? j : 0) * a.vn + hk * a.vh;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      kf[s] = row_operand<T>(pk, on, s, lh, a.D);
      vf[s] = row_operand<T>(pv, on, s, lh, a.D);
    }
  }
  QD q_tile(a.qn, a.D), d_tile(dn, a.D);
  const int* qseg = seg ? a.q_seg + (int64_t)b * a.Nq : nullptr;

  f32x16 ak[DB], av[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) ak[d] = av[d] = zero16();
  const Capped<T, CAP> capped(a);
  const float mult = a.scale * kLog2e, out_scale = a.scale * (CAP != kUncapped ? Capped<T, CAP>::kSlope : 1.f);
  const auto score = [&](float raw, float add, float& slope) {
    if constexpr (CAP != kUncapped) return capped.score(raw, add, slope);
    return raw * mult + add;
  };

  const int64_t plane = (int64_t)a.B * a.H * a.Nq;
  const T *qbase = nullptr, *dbase = nullptr;   // of the current head, as its row of statistics
  int64_t srow = 0;
  auto stage = [&](int en, int buf) {
    const int i0 = (en & kBlockMask) * QB;
    char(*to)[QD::BYTES] = tiles[buf % QD::BUFFERS];
    q_tile.fetch(qbase + (int64_t)i0 * a.qn, a.Nq - i0, a.qn, a.D, to[0], wave);
    d_tile.fetch(dbase + (int64_t)i0 * dn, a.Nq - i0, dn, a.D, to[1], wave);
    if (wave == 0) copy_ints(row_stats + srow + i0, a.Nq - i0, stats[buf][0], lane);
    if (wave == 1) copy_ints(row_stats + plane + srow + i0, a.Nq - i0, stats[buf][1], lane);
    if (seg && wave == 2) copy_ints(qseg + i0, a.Nq - i0, segs[buf], lane);
  };

  const int blocks = (a.Nq + QB - 1) / QB, first_block = min(wg_min, a.Nq) / QB;
  for (int c0 = first_block, c1; c0 < blocks; c0 = c1) {   // one turn, or with segments one for each list
    c1 = seg ? min(blocks, c0 + kListBlocks) : blocks;
    const int n = seg ? list_blocks<QB>(qseg, a.Nq, seg_lo, seg_hi, c0, c1, flags, list, &count) : blocks - c0;
    auto entry = [&](int t) { return seg ? __builtin_amdgcn_readfirstlane(list[t]) : c0 + t; };
    // the blocks of all heads of the group, one after the other, are dealt to the splits
    const int64_t all = (int64_t)n * a.G;
    const int64_t w0 = all * split / splits, w1 = all * (split + 1) / splits;
    for (int g = n ? (int)(w0 / n) : 0; g < a.G && g * (int64_t)n < w1; ++g) {
      const int t0 = (int)max(w0 - g * (int64_t)n, (int64_t)0), t1 = (int)min(w1 - g * (int64_t)n, (int64_t)n);
      const int h = hk * a.G + g;
      qbase = static_cast<const T*>(a.q) + b * a.qb + h * a.qh;
      dbase = dout + b * db + h * dh;
      srow = ((int64_t)b * a.H + h) * a.Nq;
      if (a.table) fill_lut(a, h, CAP ? capped.k3 : 0.f, lut);
      if (t0 < t1) stage(entry(t0), t0 & 1);
      for (int t = t0; t < t1; ++t) {
        const int e = entry(t), buf = t & 1, i0 = (e & kBlockMask) * QB;
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        char(*tile)[QD::BYTES] = tiles[buf % QD::BUFFERS];
        if constexpr (QD::BUFFERS == 1) {
          q_tile.store(tile[0]);
          d_tile.store(tile[1]);
          __syncthreads();
        }
        if (t + 1 < t1) stage(entry(t + 1), buf ^ 1);
        // rows that see nothing (their constant is -infinity) and those past the last have weight 0, and 0 times what
        // they hold has to be 0; wide rows
        const float row_base = stats[buf][0][lane & (QB - 1)];
        bool wide = false;
        if (i0 + QB > a.Nq || __ballot(fabsf(row_base) >= kWideRow)) {
          wide = a.table && __ballot(fabsf(row_base) >= kWideRow && row_base != -kInf) != 0;
          const int r = threadIdx.x / (kAttnThreads / QB);
          if (stats[buf][0][r] == -kInf) {
            QD::clear(tile[0], r, threadIdx.x % (kAttnThreads / QB), kAttnThreads / QB);
            QD::clear(tile[1], r, threadIdx.x % (kAttnThreads / QB), kAttnThreads / QB);
          }
          __syncthreads();
          if (wave == 0 && lane < QB) {
            if (i0 + lane >= a.Nq) stats[buf][0][lane] = -kInf;
            if (wide) inverse[lane] = i0 + lane < a.Nq ? row_stats[2 * plane + srow + i0 + lane] : 0.f;
          }
          __syncthreads();
        }
        if (i0 + QB <= wave_min) continue;
        bool all_same = true;
        if (seg && !own_segs.meets<QB>(segs[buf], lane, all_same)) continue;
        const char *qt = tile[0], *dt = tile[1];
#pragma unroll 1
        for (int u = 0; u < SUB; ++u) {
          f32x16 s = zero16(), dp;
          float base[16];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int at = 32 * u + 8 * q + 4 * lh;
            const f32x4 vl = *reinterpret_cast<const f32x4*>(&stats[buf][0][at]);
            const f32x4 vd = *reinterpret_cast<const f32x4*>(&stats[buf][1][at]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              base[4 * q + c] = vl[c];
              dp[4 * q + c] = vd[c];
            }
          }
#pragma unroll
          for (int st = 0; st < STEPS; ++st) s = mfma16(QD::rows(qt, 32 * u + ln, st, lh), kf[st], s);
#pragma unroll
          for (int st = 0; st < STEPS; ++st) dp = mfma16(QD::rows(dt, 32 * u + ln, st, lh), vf[st], dp);
          float x[16], slope[16];
          const int rel0 = wave_key - (first + i0 + 32 * u);   // of the first query and the wave's first key
          if (a.table && !all_far(a, rel0)) {
            const float* bias = lut + (rel0 + a.radius + kPad + ln - 4 * lh);
#pragma unroll
            for (int r = 0; r < 16; ++r)
              x[r] = score(s[r], bias[-(8 * (r >> 2) + (r & 3))], slope[r]) + base[r];
          } else if (a.table) {
            const float add = lut[rel0 > 0 ? 2 * (a.radius + kPad) : 0];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = score(s[r], add, slope[r]) + base[r];
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = score(s[r], base[r], slope[r]);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = fast_exp2(x[r]);
          if (wide)
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] *= inverse[32 * u + 8 * (r >> 2) + 4 * lh + (r & 3)];
          if (i0 < wave_max)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              x[r] = i0 + 32 * u + 8 * (r >> 2) + 4 * lh + (r & 3) >= imin ? x[r] : 0.f;
          if (!all_same)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int4 qs = *reinterpret_cast<const int4*>(&segs[buf][32 * u + 8 * q + 4 * lh]);
              x[4 * q] = qs.x == kseg ? x[4 * q] : 0.f;
              x[4 * q + 1] = qs.y == kseg ? x[4 * q + 1] : 0.f;
              x[4 * q + 2] = qs.z == kseg ? x[4 * q + 2] : 0.f;
              x[4 * q + 3] = qs.w == kseg ? x[4 * q + 3] : 0.f;
            }
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const Frag<T> p = as_operand<T>(x, st);
#pragma unroll
            for (int d = 0; d < DB; ++d) av[d] = mfma16(QD::cols(dt, 32 * u + 16 * st, 32 * d, lane), p, av[d]);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            x[r] *= dp[r];
            if constexpr (CAP != kUncapped) x[r] *= slope[r];
          }
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const Frag<T> p = as_operand<T>(x, st);
#pragma unroll
            for (int d = 0; d < DB; ++d) ak[d] = mfma16(QD::cols(qt, 32 * u + 16 * st, 32 * d, lane), p, ak[d]);
          }
        }
      }
      __syncthreads();   // bias values and both buffers are free
    }
  }

  if (j >= a.Nk) return;
  const int64_t row = ((int64_t)b * a.Nk + j) * a.Hk + hk, rows = (int64_t)a.B * a.Nk * a.Hk;
  // parts: dk of every split, then dv
  store_rows<T, DB>(ak, out_scale, splits == 1 ? dk + row * a.D : nullptr, part + (split * rows + row) * a.D, lh, a.D);
  store_rows<T, DB>(av, 1.f, splits == 1 ? dv + row * a.D : nullptr, part + ((splits + split) * rows + row) * a.D, lh,
                    a.D);
}

// out = sum over the splits of part[split][n], four values a thread; up to three arrays (a count of 0: none).
struct JoinOne {
  const float* part;
  void* out;
  int64_t n;   // values of one part, a multiple of 8
  int splits;
};
struct JoinArgs {
  JoinOne of[3];
};
// The table's gradient: dtable[k] = sum over the query blocks' parts of part[g][k] (size 0: none).
struct BiasSum {
  const float* part;
  void* dtable;
  int groups, size, table_bf16;
};
// What is left after both walks, in one launch: workgroups from bias_groups on join, the others sum 16 values of the
// table's gradient each, in 16 slices of the parts.
template <class T>
__global__ __launch_bounds__(kAttnThreads) void attn_bwd_finish_kernel(const JoinArgs j, const BiasSum bias,
                                                                       int bias_groups) {
  if ((int)blockIdx.x < bias_groups) {
    __shared__ float sh[16][17];
    const int k = blockIdx.x * 16 + (threadIdx.x & 15), slice = threadIdx.x >> 4;
    float s = 0.f;
    if (k < bias.size)
#pragma unroll 8
      for (int g = slice; g < bias.groups; g += 16) s += bias.part[(int64_t)g * bias.size + k];
    sh[slice][threadIdx.x & 15] = s;
    __syncthreads();
    for (int m = 8; m > 0; m /= 2) {
      if (slice < m) sh[slice][threadIdx.x & 15] += sh[slice + m][threadIdx.x & 15];
      __syncthreads();
    }
    if (slice == 0 && k < bias.size) {
      if (bias.table_bf16)
        static_cast<bf16*>(bias.dtable)[k] = (bf16)sh[0][threadIdx.x];
      else
        static_cast<float*>(bias.dtable)[k] = sh[0][threadIdx.x];
    }
    return;
  }
  int64_t at = ((int64_t)(blockIdx.x - bias_groups) * kAttnThreads + threadIdx.x) * 4;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    const JoinOne& o = j.of[w];
    if (at >= 0 && at < o.n) {
      f32x4 v = *reinterpret_cast<const f32x4*>(o.part + at);
#pragma unroll 4
      for (int s = 1; s < o.splits; ++s) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(o.part + s * o.n + at);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] += x[c];
      }
      typedef T quad __attribute__((ext_vector_type(4)));
      quad q;
#pragma unroll
      for (int c = 0; c < 4; ++c) q[c] = (T)v[c];
      *reinterpret_cast<quad*>(static_cast<T*>(o.out) + at) = q;
    }
    at -= o.n;
  }
}

// Workgroups that a row block's walk is split over: as many as bring the launch to two workgroups a CU, each with at
// least two blocks of the walk (fp32, 2 x 200 tokens of 16 heads: 21 and 15 us in three parts, 29 and 24 whole).  Long
// causal walks (`far`; the longest takes twice the mean, and nothing is left to start beside it): up to four a CU, 1024
// rows each at least.  q, kv and finish, bf16: 1 x 4096, 8 heads of 64, 128 us and 143 without; 1 x 8192 369 and 451;
// 1 x 16384, 4 heads, 548 and 807; 16/4 heads of 128, 4096: 457 and 460; fp32, 8 heads of 64, 4096: 431 and 473.
int walk_splits(int64_t groups, int64_t walk, int block, bool far) {
  const int64_t want = (2 * (int64_t)attn_units() + groups - 1) / groups, most = walk / (2 * block);
  int64_t s = want < most ? want : most;
  if (far) s = std::max(s, std::min(4 * (int64_t)attn_units() / groups, walk / 1024));
  return s < 1 ? 1 : (int)(s < 16 ? s : 16);
}

struct BwdSpace {
  int q_splits, kv_splits;
  size_t stats, q_part, kv_part, bias, total;   // bytes, in this order
};
BwdSpace bwd_space(const AttnArgs& a, bool f32, bool table) {
  const int64_t qblocks = (a.Nq + kGroupRows - 1) / kGroupRows, kblocks = (a.Nk + kGroupRows - 1) / kGroupRows;
  const int block = f32 ? Operand<float>::kBlock : Operand<bf16>::kBlock;
  const bool far = a.causal && !a.q_seg && a.Nk >= 4096;
  BwdSpace s;
  s.q_splits = walk_splits((int64_t)a.B * a.H * qblocks, a.Nk, block, far);
  s.kv_splits = kblocks ? walk_splits((int64_t)a.B * a.Hk * kblocks, (int64_t)a.Nq * a.G, block, far) : 1;
  s.stats = (size_t)round_up((int64_t)a.B * a.H * a.Nq * (a.table ? 12 : 8), 256);
  s.q_part = s.q_splits == 1 ? 0 : (size_t)round_up((int64_t)s.q_splits * a.B * a.H * a.Nq * a.D * 4, 256);
  s.kv_part = s.kv_splits == 1 ? 0 : (size_t)round_up((int64_t)s.kv_splits * 2 * a.B * a.Hk * a.Nk * a.D * 4, 256);
  s.bias = table ? (size_t)(a.B * qblocks * s.q_splits * a.H * a.nb) * 4 : 0;
  s.total = s.stats + s.q_part + s.kv_part + s.bias;
  return s;
}

template <class T, int DP, int CAP>
int launch_bwd_as(const AttnArgs& a, const void* o, const void* o_lo, const float* lse, const void* dout,
                  const int64_t* ds, void* dq, void* dk, void* dv, void* dtable, void* ws, hipStream_t stream) {
  const BwdSpace sp = bwd_space(a, sizeof(T) == 4, dtable != nullptr);
  char* at = static_cast<char*>(ws);
  float* stats = reinterpret_cast<float*>(at);
  float* q_part = reinterpret_cast<float*>(at + sp.stats);
  float* kv_part = reinterpret_cast<float*>(at + sp.stats + sp.q_part);
  float* bias = dtable ? reinterpret_cast<float*>(at + sp.stats + sp.q_part + sp.kv_part) : nullptr;
  const int qblocks = (a.Nq + kGroupRows - 1) / kGroupRows, kblocks = (a.Nk + kGroupRows - 1) / kGroupRows;
  {
    const int64_t total = (int64_t)a.B * a.H * qblocks * sp.q_splits;
    KernelTimerScope timer("attn_bwd_q", stream);
    attn_bwd_q_kernel<T, DP, CAP><<<dim3(attn_grid(total)), kAttnThreads, bias_lds(a, dtable != nullptr), stream>>>(
        a, static_cast<const T*>(o), static_cast<const T*>(o_lo), lse, static_cast<const T*>(dout), ds[0], ds[1], ds[2],
        static_cast<T*>(dq), stats, q_part, bias, sp.q_splits, qblocks, (int)total);
    if (const int rc = check_launch("attn_bwd_q")) return rc;
  }
  if (kblocks > 0) {
    const int64_t total = (int64_t)a.B * a.Hk * kblocks * sp.kv_splits;
    KernelTimerScope timer("attn_bwd_kv", stream);
    attn_bwd_kv_kernel<T, DP, CAP><<<dim3(attn_grid(total)), kAttnThreads, bias_lds(a, false), stream>>>(
        a, stats, static_cast<const T*>(dout), ds[0], ds[1], ds[2], static_cast<T*>(dk), static_cast<T*>(dv),
        kv_part, sp.kv_splits, kblocks, (int)total);
    if (const int rc = check_launch("attn_bwd_kv")) return rc;
  }
  const int64_t nq = sp.q_splits > 1 ? (int64_t)a.B * a.Nq * a.H * a.D : 0;
  const int64_t nk = sp.kv_splits > 1 ? (int64_t)a.B * a.Nk * a.Hk * a.D : 0;
  const BiasSum sum{bias, dtable, a.B * qblocks * sp.q_splits, dtable ? a.nb * a.H : 0, a.table_bf16};
  const int64_t bias_groups = (sum.size + 15) / 16;
  const int64_t groups = bias_groups + (nq + 2 * nk + 4 * kAttnThreads - 1) / (4 * kAttnThreads);
  if (groups == 0) return BIOEMU_OK;
  const JoinArgs join{{{q_part, dq, nq, sp.q_splits},
                       {kv_part, dk, nk, sp.kv_splits},
                       {kv_part + sp.kv_splits * nk, dv, nk, sp.kv_splits}}};
  KernelTimerScope timer("attn_bwd_finish", stream);
  attn_bwd_finish_kernel<T><<<dim3((unsigned)groups), kAttnThreads, 0, stream>>>(join, sum, (int)bias_groups);
  return check_launch("attn_bwd_finish");
}

template <class T, int DP>
int launch_bwd(const AttnArgs& a, const void* o, const void* o_lo, const float* lse, const void* dout, const int64_t* ds,
               void* dq, void* dk, void* dv, void* dtable, void* ws, hipStream_t stream) {
  if (!(a.cap > 0.f))
    return launch_bwd_as<T, DP, kUncapped>(a, o, o_lo, lse, dout, ds, dq, dk, dv, dtable, ws, stream);
  if constexpr (sizeof(T) == 2)
    if (!fast_cap<T>(a))
      return launch_bwd_as<T, DP, kCapWide>(a, o, o_lo, lse, dout, ds, dq, dk, dv, dtable, ws, stream);
  return launch_bwd_as<T, DP, kCapped>(a, o, o_lo, lse, dout, ds, dq, dk, dv, dtable, ws, stream);
}

}  // namespace
}  // namespace bioemu

using namespace bioemu;

extern "C" size_t bioemu_attention_bwd_workspace_bytes(const bioemu_attention_args* args, int table_gradient) {
  AttnArgs a;
  if (attn_args("attention_bwd", args, &a) || a.B == 0 || a.Nq == 0) return 0;
  return bwd_space(a, args->f32 != 0, table_gradient && a.table).total;
}

extern "C" int bioemu_attention_bwd(const bioemu_attention_args* args, const void* o, const void* o_lo,
                                    const float* lse, const void* dout, const int64_t* dout_stride, void* dq, void* dk,
                                    void* dv, void* dtable, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  AttnArgs a;
  if (const int rc = attn_args("attention_bwd", args, &a)) return rc;
  if (a.B == 0 || a.Nq == 0) return set_error(BIOEMU_ERR_INVALID_ARG, "attention_bwd: no queries");
  if (!o || !lse || !dout || !dout_stride || !dq || (a.Nk > 0 && (!dk || !dv)))
    return set_error(BIOEMU_ERR_INVALID_ARG, "attention_bwd: null pointer");
  const int64_t per = args->f32 ? 4 : 8;
  const int64_t ds[3] = {dout_stride[0], a.Nq > 1 ? dout_stride[1] : a.D, dout_stride[2]};
  if (!aligned16(o) || !aligned16(o_lo) || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
      ds[0] % per || ds[1] % per || ds[2] % per || ds[1] > (int64_t(1) << 23) || ds[1] < a.D)
    return set_error(BIOEMU_ERR_INVALID_ARG,
                     "attention_bwd: rows start at 16-byte addresses, at least a head's width apart");
  if (o_lo && args->f32) return set_error(BIOEMU_ERR_INVALID_ARG, "attention_bwd: o_lo is of bf16 calls");
  if (dtable && !a.table) return set_error(BIOEMU_ERR_INVALID_ARG, "attention_bwd: dtable without a table");
  const size_t need = bwd_space(a, args->f32 != 0, dtable != nullptr).total;
  if (!workspace || !aligned16(workspace) || workspace_bytes < need)
    return set_error(BIOEMU_ERR_WORKSPACE, "attention_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const int dp = a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128;
#define BIOEMU_BWD(T, P)                                                                                            \
  if (dp == P) return launch_bwd<T, P>(a, o, o_lo, lse, dout, ds, dq, dk, dv, dtable, workspace, stream)
  if (args->f32) {
    BIOEMU_BWD(float, 32);
    BIOEMU_BWD(float, 64);
    BIOEMU_BWD(float, 128);
  } else {
    BIOEMU_BWD(bf16, 32);
    BIOEMU_BWD(bf16, 64);
    BIOEMU_BWD(bf16, 128);
  }
#undef BIOEMU_BWD
  return BIOEMU_ERR_UNSUPPORTED;
}
