// Relative-position embedding of the pair representation, with the gradient of its table, for gfx950.
//
//   t(b, i, j) = chain_i == chain_j ? buckets[clamp(pos_j - pos_i, -R, R) + R] : NB - 1
//   out[b, i, j] = z[b, i, j] + table[t(b, i, j)]          (z may be absent)
//   dtable[t]    = sum over the pairs (b, i, j) of bucket t of dout[b, i, j]
//
// Forward is bound by the bytes of out (and z).  A workgroup takes a piece of one row i: the buckets of its columns
// first (LDS), then 16-byte pieces; table rows come from the L1 and L2 caches.
//
// Backward reads dout once.  The sums by bucket are a matrix product with a 0/1 matrix,
//   dtable^T [channels x buckets] = dout^T [channels x pairs] . onehot [pairs x buckets],
// on the bf16 MFMA: 1 and 0 are exact there, products of bf16 gradients are exact and added in fp32, and an fp32
// gradient goes in as three bf16 parts (hi + mid + lo hold its 24 bits).  So a wave needs no atomics and no table of
// its own in LDS, whatever the order of the buckets, and a 32-bucket block that none of 16 pairs falls into is
// skipped (a row's far pairs share a bucket).  Waves are added in a fixed order through LDS, workgroups by
// relpos_bwd_reduce: the same bits every time.  0 times a gradient that is not finite is not 0: a wave whose sums are not
// finite adds its pairs again one by one.
//
// Measured: 768 x 768 pairs of 128 channels, bf16, forward with z 53 us (5.8 TB/s), backward 48 us (3.1 TB/s; cold,
// 384 x 384 22 us, 768 x 768 50, 1536 x 1536 152, 2304 x 2304 286: 5.1 TB/s and some 20 us of any call, its first loads
// and the sums over waves) and 4 for the partial sums; 200 x 200 fp32, forward without z 7 us.
#include "common.h"
#include "internal.h"

namespace bioemu {
namespace {

constexpr int kThreads = 256;
constexpr int kBwdThreads = 512;
constexpr int kMaxBuckets = 256;
constexpr int kBwdBlocks = 4;            // 32-bucket blocks one backward workgroup holds
constexpr int kBwdChannels = 64;         // channels one backward wave holds
constexpr int64_t kBwdGroups = 256;      // backward workgroups in all, about one a CU

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16_alias __attribute__((may_alias));   // LDS written as 16-bit values and read as words

// Bucket of a pair; every table index is below nb whatever the map holds.
__device__ __forceinline__ int pair_bucket(int pi, int pj, int ci, int cj, const uint8_t* __restrict__ buckets,
                                           int radius, int nb) {
  int64_t d = (int64_t)pj - pi;
  d = d < -radius ? -radius : (d > radius ? radius : d);
  const int t = buckets[(int)d + radius];
  return ci != cj || t > nb - 1 ? nb - 1 : t;
}

template <class T, int VEC>
__global__ __launch_bounds__(kThreads) void relpos_fwd_kernel(const void* __restrict__ table, int table_bf16,
                                                              const uint8_t* __restrict__ buckets,
                                                              const int* __restrict__ pos,
                                                              const int* __restrict__ chains,
                                                              const T* __restrict__ z, T* __restrict__ out, int n,
                                                              int c, int radius, int nb, int jt) {
  __shared__ short sh[kThreads];
  const int row = blockIdx.x, j0 = blockIdx.y * jt;   // row = b * n + i
  const int b = row / n;
  const int cols = min(jt, n - j0);
  if ((int)threadIdx.x < cols) {
    const int j = b * n + j0 + threadIdx.x;
    sh[threadIdx.x] = (short)pair_bucket(pos[row], pos[j], chains ? chains[row] : 0, chains ? chains[j] : 0, buckets,
                                         radius, nb);
  }
  __syncthreads();
  const int cv = c / VEC, step = kThreads / cv, rest = kThreads - step * cv;
  int p = threadIdx.x / cv, ch = threadIdx.x - p * cv;
  const int64_t base = ((int64_t)row * n + j0) * c;
  while (p < cols) {
    const int64_t at = base + (int64_t)p * c + ch * VEC;
    const int64_t src = (int64_t)sh[p] * c + ch * VEC;
    float v[VEC];
    if (table_bf16) {
      const bf16* t = static_cast<const bf16*>(table) + src;
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = (float)t[e];
    } else {
      const float* t = static_cast<const float*>(table) + src;
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = t[e];
    }
    if constexpr (VEC == 1) {
      out[at] = (T)(z ? (float)z[at] + v[0] : v[0]);
    } else {
      typedef T vec __attribute__((ext_vector_type(VEC)));
      vec o;
      if (z) {
        const vec x = *reinterpret_cast<const vec*>(z + at);
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = (T)((float)x[e] + v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = (T)v[e];
      }
      *reinterpret_cast<vec*>(out + at) = o;
    }
    p += step;
    ch += rest;
    if (ch >= cv) {
      ch -= cv;
      ++p;
    }
  }
}

// One lane's channel pair (2n, 2n + 1 of the wave's 64) of one pair (i, j).
template <class T>
struct ChannelPair;
template <>
struct ChannelPair<bf16> {
  typedef bf16x2 type;
};
template <>
struct ChannelPair<float> {
  typedef f32x2 type;
};

// Pairs a backward wave holds (and as many on their way): half as many in fp32, which holds their three parts too.
template <class T>
constexpr int unit_pairs() {
  return sizeof(T) == 2 ? 64 : 32;
}

// The 0/1 operand: element t is 1 where bucket t of bk is `col`.
__device__ __forceinline__ bf16x8 onehot(u32x4 bk, int col) {
  const u16x2 target = {(unsigned short)col, (unsigned short)col}, one = {1, 1}, neg = {0xc080, 0xc080},
              full = {0x3f80, 0x3f80};   // bf16 1.0; x * 0xc080 + 0x3f80 is 0 for x = 1
  u32x4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const u16x2 x = __builtin_bit_cast(u16x2, (uint32_t)bk[w]) ^ target;
    r[w] = __builtin_bit_cast(uint32_t, (u16x2)(__builtin_elementwise_min(x, one) * neg + full));
  }
  return __builtin_bit_cast(bf16x8, r);
}

// Orders this wave's LDS accesses for the compiler; the hardware takes a wave's in order.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// part[blockIdx.x][NB][c]: this workgroup's sums for buckets 128 z .. and channels 64 y ..
template <class T, int NBB>
__global__ __launch_bounds__(kBwdThreads) void relpos_bwd_kernel(const T* __restrict__ dout,
                                                                 const uint8_t* __restrict__ buckets,
                                                                 const int* __restrict__ pos,
                                                                 const int* __restrict__ chains,
                                                                 float* __restrict__ part, int n, int c, int radius,
                                                                 int nb, int units, int cols, int paired) {
  typedef typename ChannelPair<T>::type Two;
  constexpr int Waves = kBwdThreads / 64;
  __shared__ float sum[4][NBB * 32][kBwdChannels + 1];
  __shared__ uint32_t bks[Waves][32];   // the 64 buckets of a wave's unit, two to a word
  const int lane = threadIdx.x & 63, wave = wave_id(), ln = lane & 31, lh = lane >> 5;
  const int c0 = blockIdx.y * kBwdChannels, nb0 = blockIdx.z * (kBwdBlocks * 32);
  // channels past the last read channel 0; nothing of them is stored
  const int ch0 = c0 + 2 * ln < c ? c0 + 2 * ln : 0, ch1 = c0 + 2 * ln + 1 < c ? c0 + 2 * ln + 1 : 0;
  f32x16 acc[NBB][2];
#pragma unroll
  for (int q = 0; q < NBB; ++q) acc[q][0] = acc[q][1] = zero16();

  // a unit is unit_pairs() pairs of one row: unit u = row * cols + piece.  The next one's values and bucket are on their way
  // while one is multiplied.
  constexpr int S = unit_pairs<T>() / 16;
  const auto lane_bucket = [&](int row, int j0) {   // of the lane's pair, from nb0; 0xffff: none of this workgroup's
    if (lane >= 16 * S || j0 + lane >= n) return 0xffff;
    const int j = row / n * n + j0 + lane;
    const int bk =
        pair_bucket(pos[row], pos[j], chains ? chains[row] : 0, chains ? chains[j] : 0, buckets, radius, nb) - nb0;
    return bk < 0 || bk >= kBwdBlocks * 32 ? 0xffff : bk;
  };
  const auto fetch = [&](int u, Two (&g)[S][8], int& bk) {
    const int row = u / cols, j0 = (u - row * cols) * (16 * S);
    const T* base = dout + ((int64_t)row * n + j0) * c;
    bk = lane_bucket(row, j0);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int p = min(16 * s + 8 * lh + t, n - 1 - j0);   // past the row: its last pair, under no bucket
        const T* src = base + (int64_t)p * c;
        if (paired)
          g[s][t] = *reinterpret_cast<const Two*>(src + ch0);
        else
          g[s][t] = Two{src[ch0], src[ch1]};
      }
  };
  const int step = gridDim.x * Waves;
  int u = blockIdx.x * Waves + wave, next_bk = 0xffff;
  Two next[S][8];
  if (u < units) fetch(u, next, next_bk);
  for (; u < units; u += step) {
    Two g[S][8];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int t = 0; t < 8; ++t) g[s][t] = next[s][t];
    const int bk = next_bk;
    if (u + step < units) fetch(u + step, next, next_bk);
    reinterpret_cast<u16_alias*>(bks[wave])[lane] = (unsigned short)bk;
    uint64_t there[NBB];
#pragma unroll
    for (int q = 0; q < NBB; ++q) there[q] = __ballot((bk >> 5) == q);
    wave_fence();   // this wave's own words, which LDS takes in order
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const u32x4 bv = *reinterpret_cast<const u32x4*>(&bks[wave][8 * s + 4 * lh]);
      bf16x8 a[3][2];
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          a[0][0][t] = g[s][t][0];
          a[0][1][t] = g[s][t][1];
        }
      } else {
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = g[s][t][e];
            const bf16 hi = (bf16)x;
            const float r1 = x - (float)hi;
            const bf16 mid = (bf16)r1;
            a[0][e][t] = hi;
            a[1][e][t] = mid;
            a[2][e][t] = (bf16)(r1 - (float)mid);
          }
      }
#pragma unroll
      for (int q = 0; q < NBB; ++q) {
        if (((there[q] >> (16 * s)) & 0xffff) == 0) continue;
        const bf16x8 one = onehot(bv, 32 * q + ln);
#pragma unroll
        for (int part_no = 0; part_no < (sizeof(T) == 2 ? 1 : 3); ++part_no)
#pragma unroll
          for (int e = 0; e < 2; ++e) acc[q][e] = mfma32(a[part_no][e], one, acc[q][e]);
      }
    }
    wave_fence();
  }

  // acc[q][e], lane (ln, lh), register 4 r + k: bucket 32 q + ln, channel 2 (8 r + 4 lh + k) + e
  bool finite = true;
#pragma unroll
  for (int q = 0; q < NBB; ++q)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        finite = finite && (__builtin_bit_cast(uint32_t, (float)acc[q][e][i]) & 0x7f800000u) != 0x7f800000u;
  if (__ballot(!finite)) {
#pragma unroll
    for (int q = 0; q < NBB; ++q) acc[q][0] = acc[q][1] = zero16();
    for (u = blockIdx.x * Waves + wave; u < units; u += step) {
      const int row = u / cols, j0 = (u - row * cols) * (16 * S), bks_here = lane_bucket(row, j0);
      const T* src = dout + ((int64_t)row * n + j0) * c;
#pragma unroll 1
      for (int p = 0; p < min(16 * S, n - j0); ++p, src += c) {
        const int bk = __shfl(bks_here, p);
#pragma unroll
        for (int q = 0; q < NBB; ++q)
          if (bk == 32 * q + ln)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int ch = c0 + 2 * (8 * (i >> 2) + 4 * lh + (i & 3)) + e;
                if (ch < c) acc[q][e][i] += (float)src[ch];
              }
      }
    }
  }
  // waves 0 .. 3 lay theirs down, 4 .. 7 add to them
  for (int w = 0; w < 2; ++w) {
    if (wave / 4 == w) {
#pragma unroll
      for (int q = 0; q < NBB; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float* at = &sum[wave & 3][32 * q + ln][2 * (8 * (i >> 2) + 4 * lh + (i & 3)) + e];
            *at = w == 0 ? acc[q][e][i] : *at + acc[q][e][i];
          }
    }
    __syncthreads();
  }
  for (int k = threadIdx.x; k < NBB * 32 * kBwdChannels; k += kBwdThreads) {
    const int r = k >> 6, q = k & 63, t = nb0 + r, ch = c0 + q;
    if (t < nb && ch < c)
      part[((int64_t)blockIdx.x * nb + t) * c + ch] = (sum[0][r][q] + sum[1][r][q]) + (sum[2][r][q] + sum[3][r][q]);
  }
}

// dtable[k] = sum over groups of part[g][k].  One workgroup: 16 values x 64 slices of groups.
__global__ __launch_bounds__(1024) void relpos_bwd_reduce_kernel(const float* __restrict__ part, int groups,
                                                                 int64_t size, void* __restrict__ dtable,
                                                                 int table_bf16) {
  __shared__ float sh[64][17];
  const int64_t k = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const int slice = threadIdx.x >> 4;
  float s = 0.f;
  if (k < size)
#pragma unroll 4
    for (int g = slice; g < groups; g += 64) s += part[g * size + k];
  sh[slice][threadIdx.x & 15] = s;
  __syncthreads();
  for (int m = 32; m > 0; m /= 2) {
    if (slice < m) sh[slice][threadIdx.x & 15] += sh[slice + m][threadIdx.x & 15];
    __syncthreads();
  }
  if (slice == 0 && k < size) {
    if (table_bf16)
      static_cast<bf16*>(dtable)[k] = (bf16)sh[0][threadIdx.x];
    else
      static_cast<float*>(dtable)[k] = sh[0][threadIdx.x];
  }
}

int check_sizes(const char* what, int64_t B, int64_t N, int64_t C, int64_t radius, int64_t NB) {
  if (B < 0 || N < 0 || C < 1 || radius < 0 || NB < 1)
    return set_error(BIOEMU_ERR_INVALID_ARG, "%s: B=%ld, N=%ld, C=%ld, radius=%ld, buckets=%ld", what, (long)B, (long)N,
                     (long)C, (long)radius, (long)NB);
  if (NB > kMaxBuckets || C > 4096 || radius > (1 << 20) || B * N * ((N + 31) / 32) >= (int64_t(1) << 31) ||
      N > 65535 * 64)
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: %ld buckets (at most %d), %ld channels (at most 4096), B=%ld, N=%ld",
                     what, (long)NB, kMaxBuckets, (long)C, (long)B, (long)N);
  return BIOEMU_OK;
}

// Backward workgroups along the pairs: about kBwdGroups in all, and two units a wave at least.
int64_t bwd_groups(int64_t B, int64_t N, int64_t C, int64_t NB) {
  const int64_t units = B * N * ((N + 63) / 64);
  const int64_t others = ((C + kBwdChannels - 1) / kBwdChannels) * ((NB + kBwdBlocks * 32 - 1) / (kBwdBlocks * 32));
  int64_t g = units / (2 * kBwdThreads / 64);
  const int64_t cap = kBwdGroups / others;
  g = g < cap ? g : cap;
  return g < 1 ? 1 : g;
}

}  // namespace
}  // namespace bioemu

using namespace bioemu;

extern "C" int bioemu_relpos_fwd(const void* table, const uint8_t* buckets, const int32_t* positions,
                                 const int32_t* chains, const void* z, void* out, int64_t B, int64_t N, int64_t C,
                                 int64_t radius, int64_t num_buckets, int f32, int table_bf16, hipStream_t stream) {
  if (const int rc = check_sizes("relpos", B, N, C, radius, num_buckets)) return rc;
  if (B == 0 || N == 0) return BIOEMU_OK;
  if (!table || !buckets || !positions || !out) return set_error(BIOEMU_ERR_INVALID_ARG, "relpos: null pointer");
  KernelTimerScope timer("relpos_fwd", stream);
  // about 8192 channels a workgroup: enough workgroups for one short protein, 64 to 256 columns
  const int jt = (int)(C >= 128 ? 64 : (C >= 64 ? 128 : 256));
  const dim3 grid((unsigned)(B * N), (unsigned)((N + jt - 1) / jt));
  const int vw = f32 ? 4 : 8;
  // 16-byte pieces of z and out (more than threads in a row, a column takes several turns); the table is read by values
  const bool vec = C % vw == 0 && aligned16(out) && (!z || aligned16(z));
  if (!vec && C > kThreads)
    return set_error(BIOEMU_ERR_UNSUPPORTED,
                     "relpos: %ld channels (at most %d where rows are not whole 16-byte pieces at 16-byte addresses)",
                     (long)C, kThreads);
#define BIOEMU_RELPOS(T, V)                                                                                         \
  relpos_fwd_kernel<T, V><<<grid, kThreads, 0, stream>>>(table, table_bf16, buckets, positions, chains,             \
                                                         static_cast<const T*>(z), static_cast<T*>(out), (int)N,    \
                                                         (int)C, (int)radius, (int)num_buckets, jt)
  if (f32) {
    if (vec)
      BIOEMU_RELPOS(float, 4);
    else
      BIOEMU_RELPOS(float, 1);
  } else {
    if (vec)
      BIOEMU_RELPOS(bf16, 8);
    else
      BIOEMU_RELPOS(bf16, 1);
  }
#undef BIOEMU_RELPOS
  return check_launch("relpos_fwd");
}

extern "C" size_t bioemu_relpos_bwd_workspace_bytes(int64_t B, int64_t N, int64_t C, int64_t num_buckets) {
  if (B < 1 || N < 1 || C < 1 || num_buckets < 1) return 0;
  return (size_t)(bwd_groups(B, N, C, num_buckets) * num_buckets * C) * sizeof(float);
}

extern "C" int bioemu_relpos_bwd(const void* dout, const uint8_t* buckets, const int32_t* positions,
                                 const int32_t* chains, void* dtable, void* workspace, size_t workspace_bytes,
                                 int64_t B, int64_t N, int64_t C, int64_t radius, int64_t num_buckets, int f32,
                                 int table_bf16, hipStream_t stream) {
  if (const int rc = check_sizes("relpos_bwd", B, N, C, radius, num_buckets)) return rc;
  if (B == 0 || N == 0) return set_error(BIOEMU_ERR_INVALID_ARG, "relpos_bwd: no pairs");
  if (!dout || !buckets || !positions || !dtable)
    return set_error(BIOEMU_ERR_INVALID_ARG, "relpos_bwd: null pointer");
  if (!workspace || workspace_bytes < bioemu_relpos_bwd_workspace_bytes(B, N, C, num_buckets))
    return set_error(BIOEMU_ERR_WORKSPACE, "relpos_bwd: workspace of %zu bytes, %zu needed", workspace_bytes,
                     bioemu_relpos_bwd_workspace_bytes(B, N, C, num_buckets));
  const int64_t groups = bwd_groups(B, N, C, num_buckets);
  float* part = static_cast<float*>(workspace);
  const int pairs = f32 ? unit_pairs<float>() : unit_pairs<bf16>();
  const int cols = (int)((N + pairs - 1) / pairs), units = (int)(B * N * cols);
  {
    KernelTimerScope timer("relpos_bwd", stream);
    const dim3 grid((unsigned)groups, (unsigned)((C + kBwdChannels - 1) / kBwdChannels),
                    (unsigned)((num_buckets + kBwdBlocks * 32 - 1) / (kBwdBlocks * 32)));
    const int blocks = num_buckets >= kBwdBlocks * 32 ? kBwdBlocks : (int)((num_buckets + 31) / 32);
    const int paired = C % 2 == 0 && (reinterpret_cast<uintptr_t>(dout) & (f32 ? 7u : 3u)) == 0;
#define BIOEMU_RELPOS(T, Q)                                                                                         \
  if (blocks == Q)                                                                                                  \
  relpos_bwd_kernel<T, Q><<<grid, kBwdThreads, 0, stream>>>(static_cast<const T*>(dout), buckets, positions, chains, \
                                                            part, (int)N, (int)C, (int)radius, (int)num_buckets,    \
                                                            units, cols, paired)
    if (f32) {
      BIOEMU_RELPOS(float, 1);
      BIOEMU_RELPOS(float, 2);
      BIOEMU_RELPOS(float, 3);
      BIOEMU_RELPOS(float, 4);
    } else {
      BIOEMU_RELPOS(bf16, 1);
      BIOEMU_RELPOS(bf16, 2);
      BIOEMU_RELPOS(bf16, 3);
      BIOEMU_RELPOS(bf16, 4);
    }
#undef BIOEMU_RELPOS
    if (const int rc = check_launch("relpos_bwd")) return rc;
  }
  KernelTimerScope timer("relpos_bwd_reduce", stream);
  const int64_t size = num_buckets * C;
  relpos_bwd_reduce_kernel<<<dim3((unsigned)((size + 15) / 16)), 1024, 0, stream>>>(part, (int)groups, size, dtable,
                                                                                   table_bf16);
  return check_launch("relpos_bwd_reduce");
}
