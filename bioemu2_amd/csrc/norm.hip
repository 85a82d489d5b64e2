// LayerNorm with its backward pass, for gfx950.
//
//   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh * g + b
//   gy = dy * g;  dx = r (gy - mean gy - xh * mean (gy * xh));  dg = sum_rows dy * xh;  db = sum_rows dy
//
// Bound by HBM: x is read and y written once, and backward x and dy are read and dx written once.  A row lies in the
// registers of LPR lanes (8 to 64 of a wave, or the whole workgroup), so the variance is a second pass over registers
// and not E[x^2] - mu^2, which loses what a large mean leaves.  Statistics, sums and the weight gradients are fp32;
// y and dx are rounded once.  A lane owns the same channels of every row it meets, so the weight gradients are sums in
// its registers; a workgroup adds its row groups in a fixed order and writes one partial row, and norm_bwd_reduce adds
// the partial rows in a fixed order: no atomics, the same bits every time.
//
// Measured: 589824 rows of 128, bf16, forward 59 us (5.1 TB/s), backward 92 us (4.9 TB/s) and 5 for the partial rows;
// 170163 rows of 64, fp32, 17 us (5.1 TB/s), 23 us (5.7 TB/s) and 4; a stream of one read and one write reaches 6.1.
// Cold, rows read by single values: 60000 of 333, bf16 75 + 115 us, fp32 61 + 98 (of 384: 33 + 35, 54 + 56).
#include "common.h"
#include "internal.h"

namespace bioemu {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBwdGroups = 1024;   // workgroups of the backward pass: partial rows of the weight gradients

template <class T, int VEC>
struct Pack;
template <>
struct Pack<bf16, 8> {
  typedef bf16x8 type;
};
template <>
struct Pack<float, 4> {
  typedef f32x4 type;
};
template <class T>
struct Pack<T, 1> {
  typedef T type;
};

template <class T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = (float)*p;
  } else {
    const typename Pack<T, VEC>::type x = *reinterpret_cast<const typename Pack<T, VEC>::type*>(p);
#pragma unroll
    for (int t = 0; t < VEC; ++t) v[t] = (float)x[t];
  }
}

template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  if constexpr (VEC == 1) {
    *p = (T)v[0];
  } else {
    typename Pack<T, VEC>::type x;
#pragma unroll
    for (int t = 0; t < VEC; ++t) x[t] = (T)v[t];
    *reinterpret_cast<typename Pack<T, VEC>::type*>(p) = x;
  }
}

// Sum over the LPR lanes of a row (all of them get it).  LPR = 256: over the workgroup, through LDS; sh holds one
// float per wave and use, a different one for every call between two barriers.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* sh) {
#pragma unroll
  for (int m = 1; m < (LPR < 64 ? LPR : 64); m *= 2) v += __shfl_xor(v, m);
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  }
  return v;
}

// A weight row (fp32 or bf16) as this lane's channels.
template <int VEC, int LPR, int VPL>
__device__ __forceinline__ void load_weight(const void* w, int is_bf16, int c, int lane, float none, float* out) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int at = (i * LPR + lane) * VEC;
#pragma unroll
    for (int t = 0; t < VEC; ++t) {
      const int k = at + t < c ? at + t : c - 1;
      out[i * VEC + t] =
          w == nullptr ? none
                       : (is_bf16 ? (float)static_cast<const bf16*>(w)[k] : static_cast<const float*>(w)[k]);
    }
  }
}

// Rows a lane group works on at a time: two where they are short, so that twice the loads are in flight.
template <int LPR, int E>
constexpr int kRowsAtOnce = LPR <= 64 && E <= 8 ? 2 : 1;

// stats: NULL or [rows][2] (mean, 1 / deviation), what the backward pass reads.
template <class T, int VEC, int LPR, int VPL>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                            const void* __restrict__ w, const void* __restrict__ b,
                                                            int w_bf16, T* __restrict__ y, float* __restrict__ stats,
                                                            int64_t rows, int c, float eps) {
  constexpr int E = VEC * VPL, RPG = kThreads / LPR, U = kRowsAtOnce<LPR, E>;
  __shared__ float sh[2][4];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  float wv[E], bv[E];
  load_weight<VEC, LPR, VPL>(w, w_bf16, c, lane, 1.f, wv);
  load_weight<VEC, LPR, VPL>(b, w_bf16, c, lane, 0.f, bv);
  const float inv_c = 1.f / (float)c;
  // every lane of a workgroup makes the same number of turns (barriers where a row spans waves)
  for (int64_t row0 = (int64_t)blockIdx.x * RPG * U; row0 < rows; row0 += (int64_t)gridDim.x * RPG * U) {
    float v[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * RPG + group;
      const T* px = x + (row < rows ? row : 0) * ldx;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int at = (i * LPR + lane) * VEC;
        if (at < c) {
          load_vec<T, VEC>(px + at, v[u] + i * VEC);
        } else {
#pragma unroll
          for (int t = 0; t < VEC; ++t) v[u][i * VEC + t] = 0.f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * RPG + group;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += v[u][e];
      const float mean = row_sum<LPR>(s, sh[0]) * inv_c;
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if ((i * LPR + lane) * VEC < c)
#pragma unroll
          for (int t = 0; t < VEC; ++t) {
            const float d = v[u][i * VEC + t] - mean;
            v[u][i * VEC + t] = d;
            q += d * d;
          }
      const float var = row_sum<LPR>(q, sh[1]) * inv_c;
      const float r = 1.f / sqrtf(var + eps);
      if (row < rows) {
        T* py = y + row * c;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          const int at = (i * LPR + lane) * VEC;
          if (at < c) {
            float o[VEC];
#pragma unroll
            for (int t = 0; t < VEC; ++t) o[t] = v[u][i * VEC + t] * r * wv[i * VEC + t] + bv[i * VEC + t];
            store_vec<T, VEC>(py + at, o);
          }
        }
        if (stats != nullptr && lane == 0) *reinterpret_cast<f32x2*>(stats + 2 * row) = f32x2{mean, r};
      }
    }
    if constexpr (LPR > 64) __syncthreads();   // sh is read before the next row writes it
  }
}

// part: NULL or [gridDim.x][2][c] fp32, this workgroup's sums of dy * xh and of dy.  A launch of one workgroup writes
// them where they belong instead (dweight, dbias; either may be NULL).
template <class T, int VEC, int LPR, int VPL>
__global__ __launch_bounds__(kThreads) void norm_bwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                            const T* __restrict__ dy, int64_t ldy,
                                                            const float* __restrict__ stats,
                                                            const void* __restrict__ w, int w_bf16,
                                                            T* __restrict__ dx, float* __restrict__ part,
                                                            void* __restrict__ dweight, void* __restrict__ dbias,
                                                            int64_t rows, int c) {
  constexpr int E = VEC * VPL, RPG = kThreads / LPR, U = kRowsAtOnce<LPR, E>;
  __shared__ float sh[2][4];
  __shared__ float acc[LPR < kThreads ? kThreads * E : 1];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  float wv[E], dw[E], db[E];
  load_weight<VEC, LPR, VPL>(w, w_bf16, c, lane, 1.f, wv);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
  const float inv_c = 1.f / (float)c;
  for (int64_t row0 = (int64_t)blockIdx.x * RPG * U; row0 < rows; row0 += (int64_t)gridDim.x * RPG * U) {
    float xh[U][E], g[U][E];
    f32x2 st[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * RPG + group, r0 = row < rows ? row : 0;
      const T *px = x + r0 * ldx, *pd = dy + r0 * ldy;
      st[u] = *reinterpret_cast<const f32x2*>(stats + 2 * r0);
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int at = (i * LPR + lane) * VEC;
        if (at < c) {
          load_vec<T, VEC>(px + at, xh[u] + i * VEC);
          load_vec<T, VEC>(pd + at, g[u] + i * VEC);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = row0 + u * RPG + group;
      const bool live = row < rows;
      const float mean = st[u][0], r = st[u][1];
      float sg = 0.f, sgx = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (live && (i * LPR + lane) * VEC < c)
#pragma unroll
          for (int t = 0; t < VEC; ++t) {
            const int e = i * VEC + t;
            xh[u][e] = (xh[u][e] - mean) * r;
            dw[e] += g[u][e] * xh[u][e];
            db[e] += g[u][e];
            g[u][e] *= wv[e];
            sg += g[u][e];
            sgx += g[u][e] * xh[u][e];
          }
      const float mg = row_sum<LPR>(sg, sh[0]) * inv_c;
      const float mgx = row_sum<LPR>(sgx, sh[1]) * inv_c;
      if (live && dx != nullptr) {
        T* po = dx + row * c;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          const int at = (i * LPR + lane) * VEC;
          if (at < c) {
            float o[VEC];
#pragma unroll
            for (int t = 0; t < VEC; ++t) o[t] = r * (g[u][i * VEC + t] - mg - xh[u][i * VEC + t] * mgx);
            store_vec<T, VEC>(po + at, o);
          }
        }
      }
    }
    if constexpr (LPR > 64) __syncthreads();
  }
  if (part == nullptr && dweight == nullptr && dbias == nullptr) return;
  const auto put = [&](int which, int k, float v) {
    if (part) {
      part[((int64_t)blockIdx.x * 2 + which) * c + k] = v;
      return;
    }
    void* out = which ? dbias : dweight;
    if (out == nullptr) return;
    if (w_bf16)
      static_cast<bf16*>(out)[k] = (bf16)v;
    else
      static_cast<float*>(out)[k] = v;
  };
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float* src = which ? db : dw;
    if constexpr (LPR < kThreads) {
      // acc[group][channel slot]; thread t adds slot t, t + 256, ... over the groups in order
      if (which) __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) acc[group * (LPR * E) + (e / VEC * LPR + lane) * VEC + e % VEC] = src[e];
      __syncthreads();
      for (int k = threadIdx.x; k < LPR * E && k < c; k += kThreads) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < RPG; ++q) s += acc[q * (LPR * E) + k];
        put(which, k, s);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int k = (e / VEC * LPR + lane) * VEC + e % VEC;
        if (k < c) put(which, k, src[e]);
      }
    }
  }
}

// dw[k] = sum over groups of part[g][0][k], db[k] of part[g][1][k].  One workgroup: 16 channels x 64 slices of groups.
__global__ __launch_bounds__(1024) void norm_bwd_reduce_kernel(const float* __restrict__ part, int groups, int c,
                                                               void* __restrict__ dw, void* __restrict__ db,
                                                               int w_bf16) {
  __shared__ float sh[64][17];
  const int k = blockIdx.x * 16 + (threadIdx.x & 15), slice = threadIdx.x >> 4;
  float s = 0.f;
  if (k < 2 * c)
#pragma unroll 4
    for (int g = slice; g < groups; g += 64) s += part[(int64_t)g * 2 * c + k];
  sh[slice][threadIdx.x & 15] = s;
  __syncthreads();
  for (int n = 32; n > 0; n /= 2) {
    if (slice < n) sh[slice][threadIdx.x & 15] += sh[slice + n][threadIdx.x & 15];
    __syncthreads();
  }
  if (slice == 0 && k < 2 * c) {
    void* out = k < c ? dw : db;
    const int at = k < c ? k : k - c;
    if (out != nullptr) {
      if (w_bf16)
        static_cast<bf16*>(out)[at] = (bf16)sh[0][threadIdx.x];
      else
        static_cast<float*>(out)[at] = sh[0][threadIdx.x];
    }
  }
}

// Lanes per row and vectors per lane for a width: the fewest lanes that hold the row in one vector each, the whole
// workgroup once a wave would need more than four (backward: the sums of dy * xh and dy stay in registers too).
template <class F>
int for_width(bool f32, bool vec, int64_t c, F&& f) {
  const int vw = vec ? (f32 ? 4 : 8) : 1;
  const int64_t n = (c + vw - 1) / vw;   // vectors per row
  if (n <= 8) return f(vw, 8, 1);
  if (n <= 16) return f(vw, 16, 1);
  if (n <= 32) return f(vw, 32, 1);
  if (n <= 64) return f(vw, 64, 1);
  if (n <= 128) return f(vw, 64, 2);
  if (n <= 256) return f(vw, 64, 4);
  if (n <= 512) return f(vw, 256, 2);
  if (n <= 1024) return f(vw, 256, 4);
  if (n <= 2048) return f(vw, 256, 8);
  return f(vw, 256, 16);
}

int64_t max_width(bool f32, bool vec) { return vec ? (f32 ? 256 * 16 * 4 : 256 * 8 * 8) : 256 * 16; }

// Workgroups for `rows` rows: one turn each until there are `cap` of them, whole turns for all from then on.
int row_groups(int64_t rows, int lpr, int elems, int64_t cap) {
  const int at_once = (lpr <= 64 && elems <= 8 ? 2 : 1) * (kThreads / lpr);   // kRowsAtOnce
  const int64_t turns = (rows + at_once - 1) / at_once;
  if (turns <= cap) return (int)turns;
  const int64_t each = (turns + cap - 1) / cap;
  return (int)((turns + each - 1) / each);
}

template <class T>
int launch_fwd(const void* x, int64_t ldx, const void* w, const void* b, int w_bf16, void* y, float* stats,
               int64_t rows, int64_t c, float eps, bool vec, hipStream_t stream) {
  constexpr bool f32 = sizeof(T) == 4;
  constexpr int VW = f32 ? 4 : 8;
  return for_width(f32, vec, c, [&](int vw, int lpr, int vpl) {
    // eight workgroups a CU: enough loads in flight, and the weights are read once per workgroup
    const dim3 grid(row_groups(rows, lpr, vw * vpl, (int64_t)compute_units() * 8));
    KernelTimerScope timer("norm_fwd", stream);
#define BIOEMU_CASE(V, L, P)                                                                                        \
  if (vw == V && lpr == L && vpl == P)                                                                              \
    norm_fwd_kernel<T, V, L, P><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(x), ldx, w, b, w_bf16,         \
                                                               static_cast<T*>(y), stats, rows, (int)c, eps);
#define BIOEMU_WIDTHS(V)                                                                                            \
  BIOEMU_CASE(V, 8, 1)                                                                                              \
  BIOEMU_CASE(V, 16, 1)                                                                                             \
  BIOEMU_CASE(V, 32, 1)                                                                                             \
  BIOEMU_CASE(V, 64, 1) BIOEMU_CASE(V, 64, 2) BIOEMU_CASE(V, 64, 4) BIOEMU_CASE(V, 256, 2) BIOEMU_CASE(V, 256, 4)   \
      BIOEMU_CASE(V, 256, 8) if constexpr (V != 8) { BIOEMU_CASE(V, 256, 16) }
    BIOEMU_WIDTHS(VW)
    BIOEMU_WIDTHS(1)
#undef BIOEMU_CASE
    return check_launch("norm_fwd");
  });
}

template <class T>
int launch_bwd(const void* x, int64_t ldx, const void* dy, int64_t ldy, const float* stats, const void* w, int w_bf16,
               void* dx, void* dw, void* db, void* ws, int64_t rows, int64_t c, bool vec, hipStream_t stream) {
  constexpr bool f32 = sizeof(T) == 4;
  constexpr int VW = f32 ? 4 : 8;
  return for_width(f32, vec, c, [&](int vw, int lpr, int vpl) {
    dim3 grid(row_groups(rows, lpr, vw * vpl, kMaxBwdGroups));
    const bool weights = dw != nullptr || db != nullptr;
    if (weights && grid.x <= 4) grid.x = 1;   // four turns of one workgroup take less than the second launch
    float* part = weights && grid.x > 1 ? static_cast<float*>(ws) : nullptr;
    {
      KernelTimerScope timer("norm_bwd", stream);
#define BIOEMU_CASE(V, L, P)                                                                                        \
  if (vw == V && lpr == L && vpl == P)                                                                              \
    norm_bwd_kernel<T, V, L, P><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(x), ldx,                       \
                                                               static_cast<const T*>(dy), ldy, stats, w, w_bf16,    \
                                                               static_cast<T*>(dx), part, dw, db, rows, (int)c);
      BIOEMU_WIDTHS(VW)
      BIOEMU_WIDTHS(1)
#undef BIOEMU_CASE
#undef BIOEMU_WIDTHS
      const int rc = check_launch("norm_bwd");
      if (rc || part == nullptr) return rc;
    }
    KernelTimerScope timer("norm_bwd_reduce", stream);
    norm_bwd_reduce_kernel<<<dim3((unsigned)((2 * c + 15) / 16)), 1024, 0, stream>>>(part, (int)grid.x, (int)c, dw,
                                                                                      db, w_bf16);
    return check_launch("norm_bwd_reduce");
  });
}

int check_width(const char* what, int64_t rows, int64_t c, int f32, bool vec) {
  if (rows < 0 || c < 1) return set_error(BIOEMU_ERR_INVALID_ARG, "%s: rows=%ld, c=%ld", what, (long)rows, (long)c);
  if (c > max_width(f32 != 0, vec))
    return set_error(BIOEMU_ERR_UNSUPPORTED, "%s: width %ld (at most %ld where rows are whole 16-byte vectors, %ld else)",
                     what, (long)c, (long)max_width(f32 != 0, true), (long)max_width(f32 != 0, false));
  return BIOEMU_OK;
}

}  // namespace
}  // namespace bioemu

using namespace bioemu;

extern "C" int bioemu_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y, float* stats,
                                     int64_t rows, int64_t c, int64_t x_stride, float eps, int f32, int weight_bf16,
                                     hipStream_t stream) {
  const int vw = f32 ? 4 : 8;
  const bool vec = c % vw == 0 && x_stride % vw == 0 && aligned16(x) && aligned16(y);
  if (const int rc = check_width("layer_norm", rows, c, f32, vec)) return rc;
  if (rows == 0) return BIOEMU_OK;
  if (!x || !y) return set_error(BIOEMU_ERR_INVALID_ARG, "layer_norm: null pointer");
  return f32 ? launch_fwd<float>(x, x_stride, weight, bias, weight_bf16, y, stats, rows, c, eps, vec, stream)
             : launch_fwd<bf16>(x, x_stride, weight, bias, weight_bf16, y, stats, rows, c, eps, vec, stream);
}

extern "C" size_t bioemu_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t c) {
  if (rows < 1 || c < 1) return 0;
  return (size_t)(rows < kMaxBwdGroups ? rows : kMaxBwdGroups) * 2 * (size_t)c * sizeof(float);
}

extern "C" int bioemu_layer_norm_bwd(const void* x, const void* dy, const float* stats, const void* weight, void* dx,
                                     void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                                     int64_t rows, int64_t c, int64_t x_stride, int64_t dy_stride, int f32,
                                     int weight_bf16, hipStream_t stream) {
  const int vw = f32 ? 4 : 8;
  const bool vec = c % vw == 0 && x_stride % vw == 0 && dy_stride % vw == 0 && aligned16(x) && aligned16(dy) &&
                   (dx == nullptr || aligned16(dx));
  if (const int rc = check_width("layer_norm_bwd", rows, c, f32, vec)) return rc;
  if (rows == 0) return set_error(BIOEMU_ERR_INVALID_ARG, "layer_norm_bwd: no rows");
  if (!x || !dy || !stats) return set_error(BIOEMU_ERR_INVALID_ARG, "layer_norm_bwd: null pointer");
  if ((dweight || dbias) && (!workspace || workspace_bytes < bioemu_layer_norm_bwd_workspace_bytes(rows, c)))
    return set_error(BIOEMU_ERR_WORKSPACE, "layer_norm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes,
                     bioemu_layer_norm_bwd_workspace_bytes(rows, c));
  return f32 ? launch_bwd<float>(x, x_stride, dy, dy_stride, stats, weight, weight_bf16, dx, dweight, dbias,
                                 workspace, rows, c, vec, stream)
             : launch_bwd<bf16>(x, x_stride, dy, dy_stride, stats, weight, weight_bf16, dx, dweight, dbias, workspace,
                                rows, c, vec, stream);
}
