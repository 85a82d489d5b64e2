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
// The table's gradient: per wave an LDS row of sums by offset, added to with one LDS add an element (a wave's adds are
// in program order, its 32 queries fall on 32 different offsets, its two halves have rows of their own); offsets at or
// beyond the radius stay in registers.  Then waves, workgroups and buckets in fixed orders.
#include "attn.h"

namespace bioemu {
namespace {

constexpr int kGroupRows = 128;

// The probability of a masked or unmasked score, and what the gradient of q . k takes beside ds.
template <class T>
__device__ __forceinline__ float capped(const AttnArgs& a, float raw, float s_scale, float s_cap, float& slope) {
  const float y = raw * s_scale;
  if (a.cap > 0.f) {
    const float t = attn_tanh<T>(y);
    slope = 1.f - t * t;
    return s_cap * t;
  }
  return y;
}

// LDS beyond the tiles: bias values by offset, and sums of ds by offset, 8 rows (4 waves x 2 lane halves).
inline size_t bias_lds(const AttnArgs& a, bool sums) {
  return a.table ? (size_t)(2 * a.radius + 1) * sizeof(float) * (sums ? 9 : 1) : 0;
}

template <class T, int DP>
__global__ __launch_bounds__(kAttnThreads) void attn_bwd_q_kernel(const AttnArgs a, const T* __restrict__ o,
                                                                  const float* __restrict__ lse,
                                                                  const T* __restrict__ dout, int64_t db, int64_t dn,
                                                                  int64_t dh, T* __restrict__ dq,
                                                                  float* __restrict__ delta,
                                                                  float* __restrict__ bias_part, int qblocks,
                                                                  int total) {
  constexpr int KB = Operand<T>::kBlock, SUB = KB / 32, STEPS = DP / 16, DB = DP / 32;
  typedef Tile<T, DP, KB> KV;
  constexpr int CP = KV::copies(kAttnThreads);
  __shared__ __attribute__((aligned(1024))) char tiles[2][2][KV::BYTES];
  __shared__ int segs[2][64];
  __shared__ int list[kListBlocks];
  __shared__ uint8_t flags[kListBlocks];
  __shared__ int red[4];
  __shared__ float ends[4][2];
  extern __shared__ float dyn[];   // bias values [2 R + 1], then the sums [4][2][2 R + 1]

  const int item = attn_item(total);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = wave_id(), ln = lane & 31, lh = lane >> 5;
  const int qblk = qblocks - 1 - item % qblocks, bh = item / qblocks, h = bh % a.H, b = bh / a.H, hk = h / a.G;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const bool seg = a.q_seg != nullptr;
  const int nrel = 2 * a.radius + 1;
  float *lut = dyn, *sums = dyn + nrel;

  const int i = qblk * kGroupRows + wave * 32 + ln;
  const bool live = i < a.Nq;
  const int pos = length - a.Nq + i;
  const int qseg = seg && live ? a.q_seg[(int64_t)b * a.Nq + i] : 0;
  int lim = a.causal ? min(max(pos + 1, prefix), length) : length;
  if (qseg < 0 || !live) lim = 0;
  const int seg_lo = seg ? wg_extreme<false>(live && qseg >= 0 ? qseg : 0x7fffffff, red) : 0;
  const int seg_hi = seg ? wg_extreme<true>(live ? qseg : -1, red) : 0;
  const int wg_max = wg_extreme<true>(lim, red);
  int wave_min = lim, wave_max = lim;
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    wave_min = min(wave_min, __shfl_xor(wave_min, m));
    wave_max = max(wave_max, __shfl_xor(wave_max, m));
  }
  wave_min = __builtin_amdgcn_readfirstlane(wave_min);
  wave_max = __builtin_amdgcn_readfirstlane(wave_max);
  const int wave_pos = __builtin_amdgcn_readfirstlane(pos);

  if (a.table) {
    for (int e = threadIdx.x; e < nrel; e += kAttnThreads) lut[e] = table_value(a, e, h);
    for (int e = threadIdx.x; e < 8 * nrel; e += kAttnThreads) sums[e] = 0.f;
  }

  // a row that sees nothing contributes nothing, whatever it holds
  const bool on = live && lim > 0;
  const int64_t row = ((int64_t)b * a.Nq + (live ? i : 0)) * a.H + h, srow = ((int64_t)b * a.H + h) * a.Nq + i;
  const float row_lse = live ? lse[srow] : kInf;
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
    }
  }
  dsum += __shfl_xor(dsum, 32);
  if (live && lh == 0) delta[srow] = dsum;

  const T* kbase = static_cast<const T*>(a.k) + b * a.kb + hk * a.kh;
  const T* vbase = static_cast<const T*>(a.v) + b * a.vb + hk * a.vh;
  unsigned koff[CP], voff[CP];
  KV::offsets(threadIdx.x, kAttnThreads, a.kn, a.D, koff);
  KV::offsets(threadIdx.x, kAttnThreads, a.vn, a.D, voff);
  const int* kseg = seg ? a.k_seg + (int64_t)b * a.Nk : nullptr;

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = zero16();
  float far_lo = 0.f, far_hi = 0.f;
  const float s_scale = a.cap > 0.f ? a.scale / a.cap : a.scale * kLog2e;
  const float s_cap = a.cap * kLog2e;
  float* own = sums + (wave * 2 + lh) * nrel + a.radius;

  auto stage = [&](int entry, int buf) {
    const int k0 = (entry & kBlockMask) * KB;
    KV::copy(kbase + (int64_t)k0 * a.kn, length - k0, a.kn, a.D, tiles[buf][0], wave, kAttnThreads, koff);
    KV::copy(vbase + (int64_t)k0 * a.vn, length - k0, a.vn, a.D, tiles[buf][1], wave, kAttnThreads, voff);
    if (seg && wave == 0) copy_ints(kseg + k0, length - k0, segs[buf], lane);
  };

  const int blocks = (wg_max + KB - 1) / KB;
  for (int c0 = 0; c0 < blocks; c0 += kListBlocks) {
    const int c1 = seg ? min(blocks, c0 + kListBlocks) : blocks;
    const int n = seg ? list_blocks<KB>(kseg, length, seg_lo, seg_hi, c0, c1, flags, list, red) : blocks;
    auto entry = [&](int t) { return seg ? __builtin_amdgcn_readfirstlane(list[t]) : t | kEntryFull; };
    if (n > 0) stage(entry(0), 0);
    for (int t = 0; t < n; ++t) {
      const int e = entry(t), buf = t & 1, k0 = (e & kBlockMask) * KB;
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
      if (t + 1 < n) stage(entry(t + 1), buf ^ 1);
      if (e & kEntryHoles) {
        const int r = threadIdx.x / (kAttnThreads / KB);
        if (segs[buf][r] < 0) {
          KV::clear(tiles[buf][0], r, threadIdx.x % (kAttnThreads / KB), kAttnThreads / KB);
          KV::clear(tiles[buf][1], r, threadIdx.x % (kAttnThreads / KB), kAttnThreads / KB);
        }
        __syncthreads();
      }
      if (k0 >= wave_max) continue;
      const char *kt = tiles[buf][0], *vt = tiles[buf][1];
      const bool full = k0 + KB <= wave_min && (e & kEntryFull);
#pragma unroll 1
      for (int u = 0; u < SUB; ++u) {
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int st = 0; st < STEPS; ++st) s = mfma16(KV::rows(kt, 32 * u + ln, st, lh), qf[st], s);
#pragma unroll
        for (int st = 0; st < STEPS; ++st) dp = mfma16(KV::rows(vt, 32 * u + ln, st, lh), df[st], dp);
        float x[16], slope[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = capped<T>(a, s[r], s_scale, s_cap, slope[r]);
        const int rel0 = k0 + 32 * u - wave_pos;   // of the wave's first query and the first key
        const bool far = rel0 - 31 >= a.radius || rel0 + 31 <= -a.radius;
        if (a.table) {
          if (far) {
            const float v = lut[rel0 > 0 ? 2 * a.radius : 0];
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] += v;
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int rel = rel0 - ln + 8 * (r >> 2) + 4 * lh + (r & 3);
              x[r] += lut[min(max(rel, -a.radius), a.radius) + a.radius];
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = fast_exp2(x[r] - row_lse) * (dp[r] - dsum);
        if (!full) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int kk = 32 * u + 8 * (r >> 2) + 4 * lh + (r & 3);
            const bool ok = (k0 + kk < lim) & (!seg | (segs[buf][kk] == qseg));
            x[r] = ok ? x[r] : 0.f;
          }
        }
        if (a.table) {
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
            for (int r = 0; r < 16; ++r) {
              const int rel = rel0 - ln + 8 * (r >> 2) + 4 * lh + (r & 3);
              if (rel >= a.radius)
                far_hi += x[r];
              else if (rel <= -a.radius)
                far_lo += x[r];
              else
                __hip_atomic_fetch_add(own + rel, x[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
          }
        }
        if (a.cap > 0.f)
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
    T* po = dq + row * a.D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 32 * d + 8 * r + 4 * lh;
        if (at < a.D) {
          typedef T quad __attribute__((ext_vector_type(4)));
          quad v;
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = (T)(acc[d][4 * r + c] * a.scale);
          *reinterpret_cast<quad*>(po + at) = v;
        }
      }
  }
  if (a.table && bias_part) {
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
    float* out = bias_part + (((int64_t)b * qblocks + qblk) * a.H + h) * nrel;
    for (int e = threadIdx.x; e < nrel; e += kAttnThreads) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += sums[w * nrel + e];
      if (e == 0) v += (ends[0][0] + ends[1][0]) + (ends[2][0] + ends[3][0]);
      if (e == nrel - 1) v += (ends[0][1] + ends[1][1]) + (ends[2][1] + ends[3][1]);
      out[e] = v;
    }
  }
}

template <class T, int DP>
__global__ __launch_bounds__(kAttnThreads) void attn_bwd_kv_kernel(const AttnArgs a, const float* __restrict__ lse,
                                                                   const T* __restrict__ dout, int64_t db, int64_t dn,
                                                                   int64_t dh, const float* __restrict__ delta,
                                                                   T* __restrict__ dk, T* __restrict__ dv,
                                                                   int kblocks, int total) {
  constexpr int QB = Operand<T>::kBlock, SUB = QB / 32, STEPS = DP / 16, DB = DP / 32;
  typedef Tile<T, DP, QB> QD;
  constexpr int CP = QD::copies(kAttnThreads);
  __shared__ __attribute__((aligned(1024))) char tiles[2][2][QD::BYTES];
  __shared__ int segs[2][64];
  __shared__ float stats[2][2][64];   // log-sums, do . o
  __shared__ int list[kListBlocks];
  __shared__ uint8_t flags[kListBlocks];
  __shared__ int red[4];
  extern __shared__ float lut[];

  const int item = attn_item(total);
  if (item < 0) return;
  const int lane = threadIdx.x & 63, wave = wave_id(), ln = lane & 31, lh = lane >> 5;
  const int kblk = item % kblocks, bh = item / kblocks, hk = bh % a.Hk, b = bh / a.Hk;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk;
  const int prefix = a.prefix ? a.prefix[b] : 0;
  const bool seg = a.q_seg != nullptr;
  const int first = length - a.Nq;   // position of query 0
  const int nrel = 2 * a.radius + 1;

  const int j = kblk * kGroupRows + wave * 32 + ln;
  const int kseg = seg && j < length ? a.k_seg[(int64_t)b * a.Nk + j] : 0;
  const bool on = j < length && kseg >= 0;
  // queries from imin on see this key (their segment aside)
  const int imin = !on ? 0x7fffffff : (a.causal && j >= prefix ? max(j - first, 0) : 0);
  const int seg_lo = seg ? wg_extreme<false>(on ? kseg : 0x7fffffff, red) : 0;
  const int seg_hi = seg ? wg_extreme<true>(on ? kseg : -1, red) : 0;
  const int wg_min = wg_extreme<false>(imin, red);
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
  unsigned qoff[CP], doff[CP];
  QD::offsets(threadIdx.x, kAttnThreads, a.qn, a.D, qoff);
  QD::offsets(threadIdx.x, kAttnThreads, dn, a.D, doff);
  const int* qseg = seg ? a.q_seg + (int64_t)b * a.Nq : nullptr;

  f32x16 ak[DB], av[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) ak[d] = av[d] = zero16();
  const float s_scale = a.cap > 0.f ? a.scale / a.cap : a.scale * kLog2e;
  const float s_cap = a.cap * kLog2e;

  const T *qbase = nullptr, *dbase = nullptr;   // of the current head, as its row of statistics
  int64_t srow = 0;
  auto stage = [&](int en, int buf) {
    const int i0 = (en & kBlockMask) * QB;
    QD::copy(qbase + (int64_t)i0 * a.qn, a.Nq - i0, a.qn, a.D, tiles[buf][0], wave, kAttnThreads, qoff);
    QD::copy(dbase + (int64_t)i0 * dn, a.Nq - i0, dn, a.D, tiles[buf][1], wave, kAttnThreads, doff);
    if (wave == 0) copy_ints(lse + srow + i0, a.Nq - i0, stats[buf][0], lane);
    if (wave == 1) copy_ints(delta + srow + i0, a.Nq - i0, stats[buf][1], lane);
    if (seg && wave == 2) copy_ints(qseg + i0, a.Nq - i0, segs[buf], lane);
  };

  const int blocks = (a.Nq + QB - 1) / QB, first_block = min(wg_min, a.Nq) / QB;
  for (int c0 = first_block; c0 < blocks; c0 += kListBlocks) {
    const int c1 = seg ? min(blocks, c0 + kListBlocks) : blocks;
    const int n = seg ? list_blocks<QB>(qseg, a.Nq, seg_lo, seg_hi, c0, c1, flags, list, red) : blocks - c0;
    auto entry = [&](int t) { return seg ? __builtin_amdgcn_readfirstlane(list[t]) : (c0 + t) | kEntryFull; };
    for (int g = 0; g < a.G; ++g) {
      const int h = hk * a.G + g;
      qbase = static_cast<const T*>(a.q) + b * a.qb + h * a.qh;
      dbase = dout + b * db + h * dh;
      srow = ((int64_t)b * a.H + h) * a.Nq;
      if (a.table)
        for (int e = threadIdx.x; e < nrel; e += kAttnThreads) lut[e] = table_value(a, e, h);
      if (n > 0) stage(entry(0), 0);
      for (int t = 0; t < n; ++t) {
        const int e = entry(t), buf = t & 1, i0 = (e & kBlockMask) * QB;
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        if (t + 1 < n) stage(entry(t + 1), buf ^ 1);
        // rows that see nothing (their log-sum is infinite) have weight 0, and 0 times what they hold has to be 0
        if (__ballot(lane < QB && stats[buf][0][lane] == kInf)) {
          const int r = threadIdx.x / (kAttnThreads / QB);
          if (stats[buf][0][r] == kInf) {
            QD::clear(tiles[buf][0], r, threadIdx.x % (kAttnThreads / QB), kAttnThreads / QB);
            QD::clear(tiles[buf][1], r, threadIdx.x % (kAttnThreads / QB), kAttnThreads / QB);
          }
          __syncthreads();
        }
        if (i0 + QB <= wave_min) continue;
        const char *qt = tiles[buf][0], *dt = tiles[buf][1];
        const bool full = i0 >= wave_max && (e & kEntryFull) && (!seg || (seg_lo == seg_hi && wave_max != 0x7fffffff));
#pragma unroll 1
        for (int u = 0; u < SUB; ++u) {
          f32x16 s = zero16(), dp = zero16();
#pragma unroll
          for (int st = 0; st < STEPS; ++st) s = mfma16(QD::rows(qt, 32 * u + ln, st, lh), kf[st], s);
#pragma unroll
          for (int st = 0; st < STEPS; ++st) dp = mfma16(QD::rows(dt, 32 * u + ln, st, lh), vf[st], dp);
          float x[16], slope[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = capped<T>(a, s[r], s_scale, s_cap, slope[r]);
          if (a.table) {
            const int rel0 = wave_key - (first + i0 + 32 * u);   // of the first query and the wave's first key
            if (rel0 - 31 >= a.radius || rel0 + 31 <= -a.radius) {
              const float v = lut[rel0 > 0 ? 2 * a.radius : 0];
#pragma unroll
              for (int r = 0; r < 16; ++r) x[r] += v;
            } else {
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int rel = rel0 + ln - (8 * (r >> 2) + 4 * lh + (r & 3));
                x[r] += lut[min(max(rel, -a.radius), a.radius) + a.radius];
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = fast_exp2(x[r] - stats[buf][0][32 * u + 8 * (r >> 2) + 4 * lh + (r & 3)]);
          if (!full) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int ii = 32 * u + 8 * (r >> 2) + 4 * lh + (r & 3);
              const bool ok = (i0 + ii >= imin) & (!seg | (segs[buf][ii] == kseg));
              x[r] = ok ? x[r] : 0.f;
            }
          }
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const Frag<T> p = as_operand<T>(x, st);
#pragma unroll
            for (int d = 0; d < DB; ++d) av[d] = mfma16(QD::cols(dt, 32 * u + 16 * st, 32 * d, lane), p, av[d]);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            x[r] *= dp[r] - stats[buf][1][32 * u + 8 * (r >> 2) + 4 * lh + (r & 3)];
            if (a.cap > 0.f) x[r] *= slope[r];
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
  const int64_t row = ((int64_t)b * a.Nk + j) * a.Hk + hk;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = 32 * d + 8 * r + 4 * lh;
      if (at < a.D) {
        typedef T quad __attribute__((ext_vector_type(4)));
        quad vk, vv;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          vk[c] = (T)(ak[d][4 * r + c] * a.scale);
          vv[c] = (T)av[d][4 * r + c];
        }
        *reinterpret_cast<quad*>(dk + row * a.D + at) = vk;
        *reinterpret_cast<quad*>(dv + row * a.D + at) = vv;
      }
    }
}

// One workgroup a head: the parts of all query blocks by offset, then the offsets of each bucket, in order.
__global__ __launch_bounds__(1024) void attn_bias_reduce_kernel(const AttnArgs a, const float* __restrict__ part,
                                                                int groups, void* __restrict__ dtable) {
  __shared__ float rel[2 * kMaxRadius + 1], sh[16][64];
  const int h = blockIdx.x, nrel = 2 * a.radius + 1, col = threadIdx.x & 63, slice = threadIdx.x >> 6;
  for (int e0 = 0; e0 < nrel; e0 += 64) {
    const int e = e0 + col;
    float v = 0.f;
    if (e < nrel)
#pragma unroll 4
      for (int g = slice; g < groups; g += 16) v += part[((int64_t)g * a.H + h) * nrel + e];
    sh[slice][col] = v;
    __syncthreads();
    if (slice == 0 && e < nrel) {
      v = 0.f;
#pragma unroll
      for (int s = 0; s < 16; ++s) v += sh[s][col];
      rel[e] = v;
    }
    __syncthreads();
  }
  for (int t = threadIdx.x; t < a.nb; t += 1024) {
    float v = 0.f;
    for (int e = 0; e < nrel; ++e) v += min((int)a.buckets[e], a.nb - 1) == t ? rel[e] : 0.f;
    if (a.table_bf16)
      static_cast<bf16*>(dtable)[(int64_t)t * a.H + h] = (bf16)v;
    else
      static_cast<float*>(dtable)[(int64_t)t * a.H + h] = v;
  }
}

struct BwdSpace {
  size_t delta, bias, total;
};
BwdSpace bwd_space(const AttnArgs& a, bool table) {
  const int64_t qblocks = (a.Nq + kGroupRows - 1) / kGroupRows;
  BwdSpace s;
  s.delta = (size_t)round_up((int64_t)a.B * a.H * a.Nq * 4, 256);
  s.bias = table ? (size_t)(a.B * qblocks * a.H * (2 * a.radius + 1)) * 4 : 0;
  s.total = s.delta + s.bias;
  return s;
}

template <class T, int DP>
int launch_bwd(const AttnArgs& a, const void* o, const float* lse, const void* dout, const int64_t* ds, void* dq,
               void* dk, void* dv, void* dtable, void* ws, hipStream_t stream) {
  const BwdSpace sp = bwd_space(a, dtable != nullptr);
  float* delta = static_cast<float*>(ws);
  float* part = dtable ? reinterpret_cast<float*>(static_cast<char*>(ws) + sp.delta) : nullptr;
  const int qblocks = (a.Nq + kGroupRows - 1) / kGroupRows, kblocks = (a.Nk + kGroupRows - 1) / kGroupRows;
  {
    const int64_t total = (int64_t)a.B * a.H * qblocks;
    KernelTimerScope timer("attn_bwd_q", stream);
    attn_bwd_q_kernel<T, DP><<<dim3(attn_grid(total)), kAttnThreads, bias_lds(a, true), stream>>>(
        a, static_cast<const T*>(o), lse, static_cast<const T*>(dout), ds[0], ds[1], ds[2], static_cast<T*>(dq), delta,
        part, qblocks, (int)total);
    if (const int rc = check_launch("attn_bwd_q")) return rc;
  }
  if (kblocks > 0) {
    const int64_t total = (int64_t)a.B * a.Hk * kblocks;
    KernelTimerScope timer("attn_bwd_kv", stream);
    attn_bwd_kv_kernel<T, DP><<<dim3(attn_grid(total)), kAttnThreads, bias_lds(a, false), stream>>>(
        a, lse, static_cast<const T*>(dout), ds[0], ds[1], ds[2], delta, static_cast<T*>(dk), static_cast<T*>(dv),
        kblocks, (int)total);
    if (const int rc = check_launch("attn_bwd_kv")) return rc;
  }
  if (!dtable) return BIOEMU_OK;
  KernelTimerScope timer("attn_bias_reduce", stream);
  attn_bias_reduce_kernel<<<dim3((unsigned)a.H), 1024, 0, stream>>>(a, part, a.B * qblocks, dtable);
  return check_launch("attn_bias_reduce");
}

}  // namespace
}  // namespace bioemu

using namespace bioemu;

extern "C" size_t bioemu_attention_bwd_workspace_bytes(const bioemu_attention_args* args, int table_gradient) {
  AttnArgs a;
  if (attn_args("attention_bwd", args, &a) || a.B == 0 || a.Nq == 0) return 0;
  return bwd_space(a, table_gradient && a.table).total;
}

extern "C" int bioemu_attention_bwd(const bioemu_attention_args* args, const void* o, const float* lse,
                                    const void* dout, const int64_t* dout_stride, void* dq, void* dk, void* dv,
                                    void* dtable, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  AttnArgs a;
  if (const int rc = attn_args("attention_bwd", args, &a)) return rc;
  if (a.B == 0 || a.Nq == 0) return set_error(BIOEMU_ERR_INVALID_ARG, "attention_bwd: no queries");
  if (!o || !lse || !dout || !dout_stride || !dq || (a.Nk > 0 && (!dk || !dv)))
    return set_error(BIOEMU_ERR_INVALID_ARG, "attention_bwd: null pointer");
  const int64_t per = args->f32 ? 4 : 8;
  if (!aligned16(o) || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
      dout_stride[0] % per || dout_stride[1] % per || dout_stride[2] % per || dout_stride[1] > (int64_t(1) << 23) ||
      (a.Nq > 1 && dout_stride[1] < a.D))
    return set_error(BIOEMU_ERR_INVALID_ARG,
                     "attention_bwd: rows start at 16-byte addresses, at least a head's width apart");
  if (dtable && !a.table) return set_error(BIOEMU_ERR_INVALID_ARG, "attention_bwd: dtable without a table");
  const size_t need = bwd_space(a, dtable != nullptr).total;
  if (!workspace || !aligned16(workspace) || workspace_bytes < need)
    return set_error(BIOEMU_ERR_WORKSPACE, "attention_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const int dp = a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128;
#define BIOEMU_BWD(T, P)                                                                                            \
  if (dp == P) return launch_bwd<T, P>(a, o, lse, dout, dout_stride, dq, dk, dv, dtable, workspace, stream)
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
