// Shared device code of the cached-attention kernels: matrix instructions, the keys
// that a workgroup's queries see, and where they sit in the cache.
#pragma once
#include "attention_launch.h"

namespace fx {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

// D = A B + C.  Lane l holds row (A) or column (B) l % 32 (l % 16), depth elements
// 8 (l / 32).. (8 (l / 16)..); of C column l % 32 and rows (r & 3) + 8 (r >> 2) + 4 (l / 32)
// (column l % 16, rows 4 (l / 16) + r).
template <int DT>
__device__ __forceinline__ f32x16_t mfma32(const u32x4_t& a, const u32x4_t& b, const f32x16_t& c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                   c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                  0, 0, 0);
}
template <int DT>
__device__ __forceinline__ f32x4_t mfma16(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                   c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                  0, 0, 0);
}

constexpr float kLog2e = 1.44269504088896340736f;

// 16-bit p reach 2^room and not 1 at a row's largest score (log2 units), the running maximum
// being that much less: fp16 then holds what lies up to 2^-(14 + room) below it in full and
// loses what lies below 2^-(25 + room), in place of 2^-14 and 2^-25 (a key whose value is small
// may outweigh all that make the output).  Scores so large that a difference of `room` is
// rounded get none: p could leave fp16.
__device__ __forceinline__ float p_room(float top, float room) { return fabsf(top) < 0x1p20f ? room : 0.f; }

// The sum / maximum over the two lanes l and l ^ 32 (every lane gets it).
__device__ __forceinline__ float half_pair_max(float v) {
  const unsigned u = __float_as_uint(v);
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_pair_sum(float v) {
  const unsigned u = __float_as_uint(v);
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The same over the four lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float quarter_max(float v) {
  const unsigned u = __float_as_uint(v);
  const u32x2_t r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return half_pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarter_sum(float v) {
  const unsigned u = __float_as_uint(v);
  const u32x2_t r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return half_pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Two 16-bit values of one word: nonzero iff either is an infinity or a NaN (the exponent
// field, all ones, carries into its sign bit).
template <int DT>
__device__ __forceinline__ unsigned nonfinite_pair(unsigned w) {
  constexpr unsigned e = DT == kBF16 ? 0x7f807f80u : 0x7c007c00u;
  constexpr unsigned one = DT == kBF16 ? 0x00800080u : 0x04000400u;
  return ((w & e) + one) & 0x80008000u;
}
// The word with its infinities and NaNs replaced by zero.
template <int DT>
__device__ __forceinline__ unsigned finite_pair(unsigned w) {
  const unsigned bad = nonfinite_pair<DT>(w);  // bit 15, bit 31
  return w & ~((bad >> 15) * 0xffffu);
}

// The least score (log2 units) whose p is not zero in 16 bits beside the running maximum m.  A
// visible infinity must not meet a zero p: where one lies in a tile, lower scores are raised to
// it (beside a row's largest, 2^7 and more in fp16, what that adds to others is nothing).  A row
// without a score yet keeps its -inf.
template <int DT>
__device__ __forceinline__ float least_score(float m) { return m - (DT == kF16 ? 24.f : 125.f); }

// A sequence's share of the call, and the keys that its query rows see.
struct SequenceSpan {
  int n, m;  // keys, queries
};
__device__ __forceinline__ SequenceSpan sequence_span(const CachedAttentionArgs& a, int b) {
  SequenceSpan s{a.L, a.T};
  if (a.lengths) s.n = min(max(a.lengths[b], 0), a.L);
  if (a.query_lengths) s.m = min(max(a.query_lengths[b], 0), a.T);
  return s;
}

// Key tiles (of KT keys) that queries at positions lo_pos .. hi_pos see: those of the sinks,
// from key 0, then the window's, from its first key on (no tile is cut at its front).  Tile i
// of the list starts at tile_start(i).
struct KeyTiles {
  int sink_tiles, first, count;
  bool joined;  // the sinks lie in the window's tiles
  template <int KT>
  __device__ __forceinline__ int tile_start(int i) const {
    return i < sink_tiles ? i * KT : first + (i - sink_tiles) * KT;
  }
  // the first key behind those that some query sees (a tile of the list may reach past it)
  __device__ __forceinline__ int tile_end(int i, int hi_pos, int sinks) const {
    return i < sink_tiles ? sinks : hi_pos + 1;
  }
};
template <int KT>
__device__ __forceinline__ KeyTiles key_tiles(int lo_pos, int hi_pos, int window, int sinks) {
  KeyTiles k{0, 0, 0, false};
  if (hi_pos < 0) return k;
  const int lo = window > 0 ? max(0, lo_pos - window + 1) : 0;
  // sinks that reach the window, or leave a gap that costs no tile, join it (sinks at or
  // behind lo always do: so the sinks of sink tiles all lie in front of the window's tiles)
  const int s = min(sinks, lo);
  k.sink_tiles = (s + KT - 1) / KT;
  k.first = lo;
  if (s > 0 && (hi_pos + KT) / KT <= k.sink_tiles + (hi_pos - lo + KT) / KT) k.sink_tiles = k.first = 0;
  k.joined = window > 0 && sinks > k.first;
  k.count = k.sink_tiles + (hi_pos - k.first + KT) / KT;
  return k;
}

// The keys of one tile that the query at position p sees.  A tile of the sinks counts those
// alone (its other keys come again in the window's tiles, or no query sees them); elsewhere
// j <= p, and inside the window or among the sinks.
struct TileMask {
  int lo, width;  // window: keys lo .. lo + width - 1
  int sinks, last;
  __device__ __forceinline__ TileMask(int p, int window, int sinks_, bool sink_tile, bool joined) {
    lo = window > 0 ? p - window + 1 : 0;
    width = sink_tile ? 0 : window > 0 ? window : p + 1 > 0 ? p + 1 : 0;
    sinks = sink_tile || joined ? sinks_ : 0;
    last = p;
  }
  __device__ __forceinline__ bool sees_window(int j) const { return unsigned(j - lo) < unsigned(width); }
  __device__ __forceinline__ bool sees(int j) const { return sees_window(j) | ((j < sinks) & (j <= last)); }
};
// Every query at lo_pos .. hi_pos sees all keys j0 .. j1 - 1 of a tile.
__device__ __forceinline__ bool all_see(int lo_pos, int hi_pos, int j0, int j1, int window, int sinks,
                                        bool sink_tile) {
  if (j1 <= sinks && j1 - 1 <= lo_pos) return true;
  return !sink_tile && j1 - 1 <= lo_pos && (window <= 0 || j0 > hi_pos - window);
}

// Buffer resource over `rows` rows of D 16-bit values, `stride` elements apart.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_resource(const uint16_t* base, long long stride, int rows,
                                                               int D) {
  return buffer_resource_2g(base, rows > 0 ? unsigned(rows - 1) * unsigned(stride) * 2u + unsigned(D) * 2u : 0u);
}

// 1 / l of a finished row.  A row that sees no key is zero; one that sees only keys of
// score -inf has no softmax (NaN).
__device__ __forceinline__ float softmax_inverse(float l, int p) {
  if (l > 0.f) return 1.f / l;
  return p < 0 ? 0.f : __builtin_nanf("");
}

}  // namespace fx
