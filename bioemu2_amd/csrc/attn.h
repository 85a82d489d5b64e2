// Shared parts of the attention kernels (attn_fwd.hip, attn_bwd.hip), for gfx950.
//
//   s(i, j) = cap tanh(scale q_i . k_j / cap) + bias[clamp(j - pos_i, -R, R)],   p = softmax over the allowed j
//   pos_i = length - Nq + i;  allowed: j < length, segment_i == segment_j >= 0,
//   and (not causal, or j <= pos_i, or j < prefix)
//
// One code for both types, on v_mfma_f32_32x32x16_bf16 (8 values a lane, 16 of the reduced index).  An fp32 operand is
// three bf16 parts, hi + mid + lo, which hold its 24 bits; of their nine products the six of 2^-16 of the whole and more
// are taken, smallest first: 192 cycles where eight v_mfma_f32_32x32x2_f32 take 512, and the same error (the
// accumulator's rounding).
// Scores are kept transposed to the operand that follows: a 32 x 32 accumulator (lane n = column, register 4 r + c =
// row 8 r + 4 h + c) is, register for register, the B operand of the next product whose reduced index is its rows in
// the order kappa(h, t) = 4 h + t, 8 + 4 h + t - 4; the A operand of that product comes out of LDS in that order by the
// transposing 8-byte read (or by single reads where fp32 lies unsplit).  So probabilities never leave registers.
//
// Tiles (rows of DP values, DP = 32, 64 or 128 >= D) go global -> LDS by buffer loads that write LDS.  Bytes past D and
// rows past the end read as zero through the buffer bound, so no lane reads outside its tensor.  16-byte pieces are
// XOR-swizzled by row.
#pragma once

#include "common.h"
#include "internal.h"

namespace bioemu {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kAttnThreads = 256;
constexpr int kAttnXcds = 8;
constexpr int kMaxRadius = 512;     // of the distance bias
constexpr int kListBlocks = 1024;   // key (or query) blocks listed at a time where segments are given
constexpr float kInf = __builtin_inff();

// The host's view of the arguments (bioemu_attention_args) with 32-bit sizes.
struct AttnArgs {
  const void *q, *k, *v;
  int64_t qb, qn, qh, kb, kn, kh, vb, vn, vh;   // strides in elements
  const int *q_seg, *k_seg, *prefix, *lengths;
  const void* table;
  const uint8_t* buckets;
  float scale, cap;
  int B, Nq, Nk, H, Hk, G, D, radius, nb, causal, table_bf16;
};

template <class T>
struct Operand;
template <>
struct Operand<bf16> {
  typedef bf16x8 frag;
  static constexpr int kBlock = 64;   // rows of a staged tile
};
template <>
struct Operand<float> {
  typedef f32x8 frag;
  static constexpr int kBlock = 32;
};
template <class T>
using Frag = typename Operand<T>::frag;

__device__ __forceinline__ f32x16 mfma16(bf16x8 a, bf16x8 b, f32x16 c) { return mfma32(a, b, c); }
struct Parts3 {
  bf16x8 hi, mid, lo;
};
__device__ __forceinline__ Parts3 parts3(f32x8 x) {
  Parts3 p;
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    p.hi[t] = (bf16)x[t];
    const float r = x[t] - (float)p.hi[t];
    p.mid[t] = (bf16)r;
    p.lo[t] = (bf16)(r - (float)p.mid[t]);
  }
  return p;
}
__device__ __forceinline__ f32x16 mfma16(const Parts3& x, const Parts3& y, f32x16 c) {
  c = mfma32(x.mid, y.mid, c);
  c = mfma32(x.lo, y.hi, c);
  c = mfma32(x.hi, y.lo, c);
  c = mfma32(x.mid, y.hi, c);
  c = mfma32(x.hi, y.mid, c);
  return mfma32(x.hi, y.hi, c);
}
__device__ __forceinline__ f32x16 mfma16(const Parts3& x, f32x8 y, f32x16 c) { return mfma16(x, parts3(y), c); }
__device__ __forceinline__ f32x16 mfma16(f32x8 x, f32x8 y, f32x16 c) { return mfma16(parts3(x), parts3(y), c); }

// Copies from memory into LDS: lane i's BYTES at byte voff of the source go to lds + BYTES i; zeros past its end.
// Written as instructions: the compiler lets every later LDS read wait for a copy that it knows of, and these are to
// land while the tile before them is worked on.  They have no result registers; whoever reads what they bring waits
// for vmcnt first (and for the workgroup's barrier where another wave made the copy).  The LDS address is an operand
// in M0, which the compiler sets (s_nop: the state between that and its use by a copy).
__device__ __forceinline__ u32x4 copy_source(const void* base, unsigned bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  return u32x4{(unsigned)p, (unsigned)(p >> 32) & 0xffffu, bytes, 0x00020000u};
}
template <int BYTES>
__device__ __forceinline__ void copy_to_lds(u32x4 source, unsigned voff, void* lds) {
  const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  if constexpr (BYTES == 16)
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(source), "{m0}"(at) : "memory");
  else
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(source), "{m0}"(at) : "memory");
}

// Row swizzle of 16-byte pieces, by pieces per row (a power of two).  A read of 32 rows' pieces takes rows that differ
// in bits 0 and 1 and two of bits 2 .. 4 at a time; a transposing read takes four rows' 64 neighbouring bytes.  Both
// meet every bank once where bits 0 and 1 of the row choose a 64-byte quarter of 256 bytes of LDS and bits 2 and 3 a
// piece of it (the first row bits are in the address already where rows are 64 or 128 bytes).
template <int CPR>
__device__ __forceinline__ int attn_swz(int r) {
  return CPR == 4 ? (r >> 2) & 3 : CPR == 8 ? ((r >> 1) & 1) * 4 + ((r >> 2) & 3) : (r & 3) * 4 + ((r >> 2) & 3);
}

// A tile in LDS: ROWS rows of DP values of T.
template <class T, int DP, int ROWS>
struct Tile {
  static constexpr int RB = DP * (int)sizeof(T), CPR = RB / 16, BYTES = ROWS * RB;
  __device__ static __forceinline__ int piece(int r, int c) { return r * RB + ((c ^ attn_swz<CPR>(r)) << 4); }

  // Copies of 16 bytes: thread t of `threads` moves pieces t, t + threads, ...; their byte offsets in the source.
  static constexpr int copies(int threads) { return ROWS * CPR / threads; }
  template <int N>
  __device__ static __forceinline__ void offsets(int t, int threads, int64_t stride, int D, unsigned (&voff)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = i * threads + t, r = p / CPR, c = (p % CPR) ^ attn_swz<CPR>(r);
      voff[i] = c * 16 < D * (int)sizeof(T) ? (unsigned)(r * stride * (int)sizeof(T)) + c * 16 : 0xfffffff0u;
    }
  }
  // `rows` (may be <= 0) rows exist behind `base`; wave-uniform arguments apart from voff.
  template <int N>
  __device__ static __forceinline__ void copy(const T* base, int rows, int64_t stride, int D, char* lds, int wave,
                                              int threads, const unsigned (&voff)[N]) {
    const int n = rows < ROWS ? rows : ROWS;
    const unsigned bytes = n <= 0 ? 0 : (unsigned)(((n - 1) * stride + D) * (int64_t)sizeof(T));
    const u32x4 rs = copy_source(base, bytes);
#pragma unroll
    for (int i = 0; i < N; ++i) copy_to_lds<16>(rs, voff[i], lds + (i * threads + wave * 64) * 16);
  }

  // Operand with the tile's rows as its outer index: row `r`, values 16 s + 8 h ..
  __device__ static __forceinline__ Frag<T> rows(const char* lds, int r, int s, int h) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const bf16x8*>(lds + piece(r, 2 * s + h));
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(lds + piece(r, 4 * s + 2 * h));
      const f32x4 b = *reinterpret_cast<const f32x4*>(lds + piece(r, 4 * s + 2 * h + 1));
      return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // Operand with the tile's columns d0 .. d0 + 31 as its outer index and rows r0 .. r0 + 15 in the order kappa.
  __device__ static __forceinline__ Frag<T> cols(const char* lds, int r0, int d0, int lane) {
    if constexpr (sizeof(T) == 2) {
      const int r = r0 + 4 * (lane >> 5) + ((lane & 15) >> 2), d = d0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      const char* p0 = lds + piece(r, d >> 3) + (d & 4) * 2;
      const char* p1 = lds + piece(r + 8, d >> 3) + (d & 4) * 2;
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p0);
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p1);
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(bf16x8, (s16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    } else {
      f32x8 o;
      const int d = d0 + (lane & 31), h = lane >> 5;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int r = r0 + (t < 4 ? 4 * h + t : 4 + 4 * h + t);
        o[t] = *reinterpret_cast<const float*>(lds + piece(r, d >> 2) + (d & 3) * 4);
      }
      return o;
    }
  }
  // Zeroes row r (whoever calls owns the row's 16-byte pieces first, first + step, ...).
  __device__ static __forceinline__ void clear(char* lds, int r, int first, int step) {
    for (int c = first; c < CPR; c += step) *reinterpret_cast<u32x4*>(lds + piece(r, c)) = u32x4{0, 0, 0, 0};
  }
};

// A tile that the waves of a workgroup share, as they read it.  bf16: the tile above, copied while the one before it is
// worked on (two buffers).  fp32: its three bf16 parts in a plane each, split once by the thread that fetched the values
// into registers (else every wave splits every operand it reads: 1000 x 1000 tokens, 8 heads of 64, forward / q / kv
// 30 / 48 / 57 us, so 25 / 40 / 46); one buffer, filled between two barriers.
template <class T, int DP, int ROWS>
struct Staged;
template <int DP, int ROWS>
struct Staged<bf16, DP, ROWS> : Tile<bf16, DP, ROWS> {
  typedef Tile<bf16, DP, ROWS> Base;
  static constexpr int BUFFERS = 2, N = Base::copies(kAttnThreads);
  unsigned off[N];
  __device__ __forceinline__ Staged(int64_t stride, int D) { Base::offsets(threadIdx.x, kAttnThreads, stride, D, off); }
  __device__ __forceinline__ void fetch(const bf16* base, int rows, int64_t stride, int D, char* lds, int wave) {
    Base::copy(base, rows, stride, D, lds, wave, kAttnThreads, off);
  }
};
template <int DP, int ROWS>
struct Staged<float, DP, ROWS> {
  typedef Tile<bf16, DP, ROWS> Plane;
  static constexpr int BUFFERS = 1, BYTES = 3 * Plane::BYTES, PER = DP / 4, N = ROWS * PER / kAttnThreads;
  unsigned off[N];
  f32x4 v[N];
  // thread t holds the 16-byte pieces t, t + 256, ... of the rows
  __device__ __forceinline__ Staged(int64_t stride, int D) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = i * kAttnThreads + threadIdx.x, r = p / PER, c = p % PER;
      off[i] = c * 4 < D ? (unsigned)(r * stride * 4) + c * 16 : 0xfffffff0u;
    }
  }
  __device__ __forceinline__ void fetch(const float* base, int rows, int64_t stride, int D, char*, int) {
    const int n = rows < ROWS ? rows : ROWS;
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(base, n <= 0 ? 0 : (unsigned)(((n - 1) * stride + D) * 4));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off[i], 0, 0));
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = i * kAttnThreads + threadIdx.x, r = p / PER, c = p % PER;
      bf16x4 part[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = v[i][e];
        part[0][e] = (bf16)x;
        const float r1 = x - (float)part[0][e];
        part[1][e] = (bf16)r1;
        part[2][e] = (bf16)(r1 - (float)part[1][e]);
      }
      char* at = lds + Plane::piece(r, c >> 1) + (c & 1) * 8;
#pragma unroll
      for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x4*>(at + q * Plane::BYTES) = part[q];
    }
  }
  __device__ static __forceinline__ Parts3 rows(const char* lds, int r, int s, int h) {
    return Parts3{Plane::rows(lds, r, s, h), Plane::rows(lds + Plane::BYTES, r, s, h),
                  Plane::rows(lds + 2 * Plane::BYTES, r, s, h)};
  }
  __device__ static __forceinline__ Parts3 cols(const char* lds, int r0, int d0, int lane) {
    return Parts3{Plane::cols(lds, r0, d0, lane), Plane::cols(lds + Plane::BYTES, r0, d0, lane),
                  Plane::cols(lds + 2 * Plane::BYTES, r0, d0, lane)};
  }
  __device__ static __forceinline__ void clear(char* lds, int r, int first, int step) {
#pragma unroll
    for (int q = 0; q < 3; ++q) Plane::clear(lds + q * Plane::BYTES, r, first, step);
  }
};

// Eight values of an accumulator as the next product's operand: rows 16 s .. 16 s + 15 in the order kappa.
template <class T>
__device__ __forceinline__ Frag<T> as_operand(const float (&x)[16], int s) {
  Frag<T> f;
#pragma unroll
  for (int t = 0; t < 8; ++t) f[t] = (T)x[8 * s + t];
  return f;
}

// A row's values 16 s + 8 h .. + 7 from memory as the operand whose outer index is rows; zero past D or if !live.
template <class T>
__device__ __forceinline__ Frag<T> row_operand(const T* row, bool live, int s, int h, int D) {
  Frag<T> f;
  const int d = 16 * s + 8 * h;
  if constexpr (sizeof(T) == 2) {
    f = live && d < D ? *reinterpret_cast<const bf16x8*>(row + d) : bf16x8{};
  } else {
    const f32x4 a = live && d < D ? *reinterpret_cast<const f32x4*>(row + d) : f32x4{};
    const f32x4 b = live && d + 4 < D ? *reinterpret_cast<const f32x4*>(row + d + 4) : f32x4{};
    f = f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  return f;
}

// 64 32-bit values into LDS, zero from the n-th on (one wave).
__device__ __forceinline__ void copy_ints(const void* src, int n, void* lds, int lane) {
  copy_to_lds<4>(copy_source(src, n <= 0 ? 0 : (n < 64 ? n : 64) * 4), lane * 4, lds);
}

// How scores are capped.  kCapWide: bf16 with a cap beyond kFastCap.
enum CapForm { kUncapped, kCapped, kCapWide };
constexpr float kFastCap = 4096.f;

// A capped score in log2 units, x = s_cap tanh(y) + add with s_cap = cap log2 e and y = raw scale / cap, and what the
// tanh leaves of a gradient: slope times kSlope is 1 - tanh^2.
// bf16 operands: by r = 1 / (1 + e^2y) of the hardware exponential and reciprocal, tanh = 1 - 2 r, 1 - tanh^2 =
// 4 (r - r^2): six instructions, off by 2e-7 of the cap: 8e-4 of a weight at kFastCap, where rounding it to bf16 takes
// 2e-3.  fp32 and wider caps: tanhf, off by some 2^-22 of the score itself (2 x 2048 causal tokens, 16/4 heads of 64,
// bf16: forward / q / kv 60 / 73 / 86 us fast, 90 / 104 / 119 with tanhf).
template <class T, int CAP>
struct Capped {
  static constexpr bool kFast = sizeof(T) == 2 && CAP != kCapWide;
  float k1, k2, k3;
  static constexpr float kSlope = kFast ? 4.f : 1.f;
  __device__ __forceinline__ explicit Capped(const AttnArgs& a) {
    if constexpr (kFast) {
      k1 = a.scale / a.cap * (2.f * kLog2e);
      k2 = -2.f * a.cap * kLog2e;
    } else {
      k1 = a.scale / a.cap;
      k2 = a.cap * kLog2e;
    }
    k3 = kFast ? a.cap * kLog2e : 0.f;
  }
  // `add` includes k3
  __device__ __forceinline__ float score(float raw, float add, float& slope) const {
    if constexpr (kFast) {
      const float r = fast_rcp(1.f + fast_exp2(raw * k1));
      slope = r - r * r;
      return r * k2 + add;
    } else {
      const float t = tanhf(raw * k1);
      slope = 1.f - t * t;
      return t * k2 + add;
    }
  }
};
template <class T>
inline bool fast_cap(const AttnArgs& a) {
  return sizeof(T) == 4 || a.cap <= kFastCap;
}

// A bias in log2 units.  The type's lowest value stays finite (a row of such scores is a softmax over equal scores);
// -infinity stays what it is.
__device__ __forceinline__ float bias_log2(float b) {
  const float v = b * kLog2e;
  return v == -kInf && b != -kInf ? -__FLT_MAX__ : v;
}

__device__ __forceinline__ float table_value(const AttnArgs& a, int entry, int h) {
  const int64_t at = (int64_t)min((int)a.buckets[entry], a.nb - 1) * a.H + h;
  return bias_log2(a.table_bf16 ? (float)static_cast<const bf16*>(a.table)[at]
                                : static_cast<const float*>(a.table)[at]);
}

// Workgroup minimum of `low`, maxima of `high` and `top` (every thread gets them); red: 12 ints of LDS.
__device__ __forceinline__ void wg_extremes(int& low, int& high, int& top, int (*red)[4]) {
#pragma unroll
  for (int m = 32; m > 0; m /= 2) {
    low = min(low, __shfl_xor(low, m));
    high = max(high, __shfl_xor(high, m));
    top = max(top, __shfl_xor(top, m));
  }
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = low;
    red[1][threadIdx.x >> 6] = high;
    red[2][threadIdx.x >> 6] = top;
  }
  __syncthreads();
  low = __builtin_amdgcn_readfirstlane(min(min(red[0][0], red[0][1]), min(red[0][2], red[0][3])));
  high = __builtin_amdgcn_readfirstlane(max(max(red[1][0], red[1][1]), max(red[1][2], red[1][3])));
  top = __builtin_amdgcn_readfirstlane(max(max(red[2][0], red[2][1]), max(red[2][2], red[2][3])));
}

// The bias by offset in LDS, offsets -R - kPad .. R + kPad (beyond the radius its end values): a 32 x 32 block that
// meets the radius reads it without clamping.  Entry rel + R + kPad.
constexpr int kPad = 64;
__device__ __forceinline__ int lut_size(const AttnArgs& a) { return 2 * (a.radius + kPad) + 1; }
// `add`: what a capped score takes besides.
__device__ __forceinline__ void fill_lut(const AttnArgs& a, int h, float add, float* lut) {
  for (int e = threadIdx.x; e < lut_size(a); e += kAttnThreads)
    lut[e] = table_value(a, min(max(e - kPad, 0), 2 * a.radius), h) + add;
}
// Whether all offsets rel0 - 31 .. rel0 + 31 lie at or beyond the radius.
__device__ __forceinline__ bool all_far(const AttnArgs& a, int rel0) {
  return rel0 - 31 >= a.radius || rel0 + 31 <= -a.radius;
}

// The range of the segments of a wave's rows (low above high: none), against the segments of a staged tile.
struct WaveRange {
  int lo, hi;
  __device__ __forceinline__ WaveRange(int low, int high) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) {
      low = min(low, __shfl_xor(low, m));
      high = max(high, __shfl_xor(high, m));
    }
    lo = __builtin_amdgcn_readfirstlane(low);
    hi = __builtin_amdgcn_readfirstlane(high);
  }
  // Whether some of the tile's N rows is of a segment in the range; `all`: all of them are of the only one.
  template <int N>
  __device__ __forceinline__ bool meets(const int* tile, int lane, bool& all) const {
    const int s = tile[lane & (N - 1)];
    all = lo == hi && __ballot(s != lo) == 0;
    return __ballot(s >= lo && s <= hi) != 0;
  }
};

// Blocks of a segment list that can hold an allowed pair.  An entry is the block's number with a flag.
constexpr int kBlockMask = 0x0fffffff, kEntryHoles = 0x20000000;

// Lists the blocks [c0, c1) of BLOCK rows of `seg` (`n` of them exist) that hold a segment in [lo, hi], in order;
// holes: some row is of no segment (or past n).  All 256 threads; returns the entries.  flags: one byte a block, list:
// one int a block.
template <int BLOCK>
__device__ __forceinline__ int list_blocks(const int* __restrict__ seg, int n, int lo, int hi, int c0, int c1,
                                           uint8_t* flags, int* list, int* count) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  constexpr int PER = 64 / BLOCK;   // blocks one wave reads at a time
  constexpr int AHEAD = 8;          // reads in flight
  for (int b8 = c0 + wave * PER; b8 < c1; b8 += 4 * PER * AHEAD) {
    int got[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int r = (b8 + 4 * PER * q) * BLOCK + lane;
      got[q] = r < n ? seg[r] : -1;
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int b0 = b8 + 4 * PER * q, s = got[q];
      const uint64_t hit = __ballot(s >= 0 && s >= lo && s <= hi), hole = __ballot(s < 0);
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const uint64_t m = BLOCK == 64 ? ~0ull : (uint64_t)0xffffffffu << (32 * p);
        if (lane == 0 && b0 + p < c1)
          flags[b0 + p - c0] = (uint8_t)(((hit & m) != 0 ? 1 : 0) | ((hole & m) != 0 ? 2 : 0));
      }
    }
  }
  __syncthreads();
  if (wave == 0) {
    int at = 0;
    for (int b0 = 0; b0 < c1 - c0; b0 += 64) {
      const int f = b0 + lane < c1 - c0 ? flags[b0 + lane] : 0;
      const uint64_t m = __ballot(f & 1);
      if (f & 1)
        list[at + __popcll(m & ((1ull << lane) - 1))] = (c0 + b0 + lane) | (f & 2 ? kEntryHoles : 0);
      at += __popcll(m);
    }
    if (lane == 0) *count = at;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*count);
}

// XCD-aware order of `total` = rows x `cols` items (a row: the blocks of one head): workgroup w runs on XCD w % 8, each
// XCD gets a contiguous range of the items (so the workgroups that read the same keys share its L2); -1 for padding
// workgroups.  An XCD with whole rows takes them column by column: with the long blocks of a causal mask in the first
// columns, long items start first, whatever their head; and the second 32 of them (it has 32 CUs, two workgroups each)
// go backwards, so that the CU of the longest gets the shortest beside it.
__device__ __forceinline__ int attn_item(int total, int cols) {
  const int w = blockIdx.x, per = (total + kAttnXcds - 1) / kAttnXcds, base = (w % kAttnXcds) * per;
  const int n = min(per, total - base);
  int p = w / kAttnXcds;
  if (p >= n) return -1;
  if (p >= 32 && p < 64) p = 32 + min(64, n) - 1 - p;
  if (n % cols == 0 && base % cols == 0) {
    const int rows = n / cols;
    p = (p % rows) * cols + p / rows;
  }
  return base + p;
}
inline unsigned attn_grid(int64_t total) { return (unsigned)(round_up(total, kAttnXcds)); }

// Compute units of the current device, remembered.
int attn_units();

// log2 of a row's sum of weights in two parts: the reference its weights are taken against, and log2 of their sum by it.
// A bias of the type's lowest value makes a reference in which the second part vanishes, so the backward pass adds them
// only where the reference is below kWideRow (there 2^-14 of the sum is kept).
constexpr float kWideRow = 1024.f;
__device__ __forceinline__ void store_log_sum(float* lse, int64_t plane, int64_t at, float m, float l) {
  lse[at] = l == 0.f ? 0.f : m;
  lse[plane + at] = l == 0.f ? kInf : __log2f(l);   // rows that see nothing
}

// Checks the arguments both directions share and lays them out (attn_fwd.hip).
int attn_args(const char* what, const bioemu_attention_args* in, AttnArgs* out);

}  // namespace bioemu
