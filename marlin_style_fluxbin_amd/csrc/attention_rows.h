// Cached attention of many query rows (a prompt, a chunk, several drafted tokens): one
// pass over the keys with a running maximum and sum, both products on the matrix cores.
//
// A workgroup of four (eight) waves takes 128 (256) query rows of one KV head, row = token
// * G + head of the group, so every head grouping fills the tile and the waves share each key
// and value tile in LDS.  Per tile of KT keys a wave forms
//   S^T = K Q^T   (32 x 32 x 16 products: column = query, so a query's scores sit in two
//                  lanes: its maximum and sum are register work and one lane swap)
//   P^T = 2^(S^T f - m), f = scale log2(e), rounded to the cache's 16-bit type
//   O^T += V^T P^T (P^T is already in the operand layout: the key order of a product is
//                  free as long as both operands use the same, and V^T is read from LDS
//                  by the transposing read in the order that S^T has left P^T in)
// with S, m, the sum and O in fp32.  O is rescaled only when some query's maximum grew by
// more than 2^8, so that p stays below that (fp16: within 2^7 .. 2^15 at the row's largest,
// p_room).
//
// LDS: rows of D 16-bit values in 16-byte chunks, chunk c of key j at c ^ swizzle(j), keys
// and values each for their reads.  16-bit caches load straight into LDS (the
// swizzle is applied to the global address of each lane), the next tile while this one is
// multiplied; the 4-bit cache is widened in registers and stored.
//
// Bound by the matrix cores, at the clock that their power leaves: 16384 tokens of 32 heads
// on 8 KV heads, D = 128, causal: 2000 to 2130 us on different cards, 1.03 to 1.10 PFLOP/s,
// where a library product of 8192^3 reaches 1.26; the products are issued 59% of the time, the
// exponentials and the maxima, which need the vector pipe, beside them.  D = 256 (4096 tokens,
// 16 heads) 174 us, 0.79 PFLOP/s, and D = 64 (32 heads) 100 us, 0.69: per score as many
// exponentials for half the products.  With a window of 1024 keys (4096 tokens, 32 heads) 80 to
// 91 us: three of 18 tiles (the sinks', both ends') are computed whole for a part, and q and
// the output are 67 MB, 14 us at a copy's rate.  A 4-bit cache (1024 tokens over 9000 keys; two
// splits) 186 us, the join's 14 among them: each row tile of a head widens the keys that it
// reads, a fifth of its time at 128 rows, an eighth at 256.
// Registers: spilled are 13 (D = 128) and, in fp16, 17 to memory (D = 256), outside the loop over
// the tiles; over a 4-bit cache 26 to 30 (D = 128, a few of them in each tile) and 10 (D = 256).
// The others fit.
// 128 rows, so that a key or value read from LDS meets 32 columns a wave, four waves a
// tile: two workgroups a CU, one's exponentials beside the other's products.  256 rows and one
// workgroup where that halves the widening (a 4-bit cache, D <= 128).
#pragma once
#include "attention_core.h"

namespace fx {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

template <int D>
struct RowsShape {
  static constexpr int KT = rows_key_tile(D);
  static constexpr int kChunks = D / 8;         // 16-byte chunks of a row
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTileBytes = KT * kRowBytes;
  static constexpr int kSteps = D / 16;         // depth steps of S^T
  static constexpr int kDims = D / 32;          // 32-row blocks of O^T
  static constexpr int kSub = KT / 32;          // 32-key blocks of a tile
};

// LDS serves 256 bytes a clock, 64 banks: sixteen lanes of a 16-byte read (keys: 16 rows, one
// chunk) or 32 of a transposing one (values: 4 rows, 64 bytes), which have to fall into
// different banks.  Measured 515 and 370 bytes a ns for each CU; with the low three bits of
// the row for both, 279 and 274.
template <int D>
__device__ __forceinline__ int key_swizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int value_swizzle(int row) {
  return D == 64 ? (row & 2) << 1 : (row & 3) << 2;
}

__device__ __forceinline__ u32x4_t lds_b128(const lds_char* p) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(p);
}
// Four 16-bit values of one column from four rows: lane i of 16 gives the address of row
// i / 4, columns 4 (i % 4).., and receives column i of the four rows.
__device__ __forceinline__ u32x2_t lds_transposed(const lds_char* p) {
  return __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p)));
}

// 16 bytes per lane from `resource` at the lane's offset to lds + 16 * lane, asynchronously
// (vmcnt).  The instruction has no result register; written as the builtin, every later LDS
// read of the kernel waits for it, whichever buffer it fills.
__device__ __forceinline__ void load_to_lds(const u32x4_t& resource, int offset, lds_char* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(unsigned(size_t(lds))),
               "v"(offset), "s"(resource)
               : "memory", "m0");
}

// One tile (rows left of it may be fewer than KT: the others become zero) into LDS.
template <int D, bool KEYS>
__device__ __forceinline__ void load_rows_to_lds(const uint16_t* base, long long stride, int rows, lds_char* dst,
                                                 int wave, int lane) {
  using S = RowsShape<D>;
  constexpr int kRowsPerLoad = 1024 / S::kRowBytes;  // one wave load: 64 lanes x 16 bytes
  constexpr int kLoads = S::KT / kRowsPerLoad / 4;   // per wave
  const int live = min(rows, S::KT);
  asm volatile("" : "+v"(lane));  // offsets formed here: kept between calls they cost registers
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    // the scalar part of the address in the resource
    const int first = (wave * kLoads + i) * kRowsPerLoad, left = live - first;
    const size_t address = reinterpret_cast<size_t>(base + first * stride);
    const u32x4_t r = {unsigned(address), unsigned(address >> 32) & 0xffffu,
                       left > 0 ? unsigned(left - 1) * unsigned(stride) * 2u + unsigned(D) * 2u : 0u, 0x00020000u};
    const int row = lane / S::kChunks;
    const int chunk = (lane % S::kChunks) ^ (KEYS ? key_swizzle<D>(first + row) : value_swizzle<D>(first + row));
    load_to_lds(r, row * int(stride) * 2 + chunk * 16, dst + first * S::kRowBytes);
  }
}

// The 4-bit cache's tile: each thread holds 16 bytes of codes (32 columns of one key) and
// the key's (scale, minimum) pairs, widens them to fp16 (code * scale + minimum in one
// rounding, 2^-11 of the value, as a 16-bit cache's own rounding) and stores the columns of
// a chunk in the order a0 b0 a1 b1 a2 b2 a3 b3 of its two 4-column units: q and the output
// are permuted alike (kv4_column), so no lane has to sort them.
template <int D>
struct Kv4Stage {
  using S = RowsShape<D>;
  static constexpr int kGroups = D / 64;
  static constexpr int kPieces = D / 32;                    // 16-byte pieces of a key's codes
  static constexpr int kKeysPerPass = 256 / kPieces;        // keys that the 256 threads take at once
  static constexpr int kPasses = (S::KT + kKeysPerPass - 1) / kKeysPerPass;
  u32x4_t codes[kPasses];
  unsigned scales[kPasses][kGroups];

  __device__ __forceinline__ void load(const uint8_t* c, const uint32_t* sc, int rows, int t) {
    const int live = min(rows, S::KT);
    const auto rc = buffer_resource_2g(c, unsigned(live) * (D / 2));
    const auto rs = buffer_resource_2g(sc, unsigned(live) * (kGroups * 4));
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int key = i * kKeysPerPass + t / kPieces, piece = t % kPieces;
      codes[i] = load_b128(rc, key * (D / 2) + piece * 16, 0);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        scales[i][g] = __builtin_amdgcn_raw_buffer_load_b32(rs, key * (kGroups * 4) + g * 4, 0, 0);
    }
  }

  template <bool KEYS>
  __device__ __forceinline__ void store(lds_char* dst, int t) const {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 bias = {_Float16(1024.f), _Float16(1024.f)};
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int key = i * kKeysPerPass + t / kPieces, piece = t % kPieces;
      if (kKeysPerPass * kPasses > S::KT && key >= S::KT) continue;
      // words (unit, group): unit u of the piece holds kGroups 16-bit words
      constexpr int kUnits = 8 / kGroups;  // units of a piece
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const h2 pair = __builtin_bit_cast(h2, scales[i][g]);
        const h2 sc = {pair.x, pair.x}, mn = {pair.y, pair.y};
#pragma unroll
        for (int u = 0; u < kUnits; u += 2) {
          const int wa = u * kGroups + g, wb = wa + kGroups;  // 16-bit words of the piece
          // both words in one register: lanes (a, b)
          const unsigned xa = codes[i][wa >> 1], xb = codes[i][wb >> 1];
          const unsigned ab = __builtin_amdgcn_perm(xb, xa, ((wb & 1) ? 0x07060000u : 0x05040000u) |
                                                               ((wa & 1) ? 0x0302u : 0x0100u));
          u32x4_t w;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const h2 code = __builtin_bit_cast(h2, ((ab >> (4 * r)) & 0x000f000fu) | 0x64006400u) - bias;
            w[r] = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(code, sc, mn));
          }
          // columns 64 g + 4 (units of the pieces before + u) .. + 7: chunk 8 g + that / 8
          const int chunk = 8 * g + (piece * kUnits + u) / 2;
          *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(
              dst + key * S::kRowBytes + ((chunk ^ (KEYS ? key_swizzle<D>(key) : value_swizzle<D>(key))) * 16)) = w;
        }
      }
    }
  }
};

// Column of position x of a widened 4-bit row.
__device__ __forceinline__ int kv4_column(int x) { return (x & ~7) | ((x & 1) << 2) | ((x >> 1) & 3); }

template <int QDT, int D, bool KV4, int NW>
__global__ __launch_bounds__(64 * NW, D == 256 ? 1 : 2) void attention_rows_kernel(const CachedAttentionArgs a) {
  using S = RowsShape<D>;
  constexpr int CDT = KV4 ? kF16 : QDT;  // the products' type
  constexpr int KT = S::KT, kRows = 32 * NW, kThreads = 64 * NW;
  static_assert(NW == 4 || (NW == 8 && KV4 && kRows <= 4 * KT), "loads by four waves; the output through the tiles' memory");
  __shared__ __attribute__((aligned(1024))) char lds_memory[4 * S::kTileBytes];
  lds_char* const lds = (lds_char*)lds_memory;
  const int t = threadIdx.x, lane = t & 63, wave = wave_index();
  const int half = lane >> 5, l31 = lane & 31;

  // ---- which rows of which KV head, which part of its keys.  Workgroup ids go round the
  // XCDs, so eight heads at a time each keep to one XCD and its L2; within a head the last
  // (longest) row tiles come first.
  const int heads = a.B * a.Hk, items = a.row_tiles * a.splits;
  int id = blockIdx.x, head, item;
  const int full = heads / kXcdCount * kXcdCount;
  if (id < full * items) {
    const int slot = id / kXcdCount;
    head = id % kXcdCount + kXcdCount * (slot / items);
    item = slot % items;
  } else {
    id -= full * items;
    head = full + id % (heads - full);
    item = id / (heads - full);
  }
  const int tile = a.row_tiles - 1 - item / a.splits, split = item % a.splits;
  const int b = head / a.Hk, g = head - b * a.Hk;
  const SequenceSpan span = sequence_span(a, b);
  const int rows = span.m * a.G, r0 = tile * kRows;
  if (r0 >= rows) return;
  const int base_pos = span.n - span.m;
  const int lo_pos = base_pos + r0 / a.G, hi_pos = base_pos + (min(r0 + kRows, rows) - 1) / a.G;
  const KeyTiles tiles = key_tiles<KT>(lo_pos, hi_pos, a.window, a.sinks);
  const int per = (tiles.count + a.splits - 1) / a.splits;
  const int it0 = split * per, it1 = min(tiles.count, it0 + per);

  // ---- this lane's query
  const int wave_row = r0 + wave * 32;
  const bool active = wave_row < rows;  // wave-uniform: the others only help loading
  const int row = min(wave_row + l31, rows - 1);
  const int tok = row / a.G, hq = g * a.G + row - tok * a.G;
  const int p = base_pos + tok;
  u32x4_t qf[S::kSteps];
  float f = a.scale * kLog2e;
  {
    const uint16_t* q = a.q + b * a.q_stride[0] + hq * a.q_stride[1] + tok * a.q_stride[2];
    if constexpr (!KV4) {
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(q + 16 * s + 8 * half);
    } else {
      // in fp16, scaled by a power of two so that the row's largest magnitude lies in
      // [2^9, 2^10): exact for every element within 2^-23 of it
      float mag = 0.f;
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        qf[s] = *reinterpret_cast<const u32x4_t*>(q + 16 * s + 8 * half);
#pragma unroll
        for (int e = 0; e < 8; ++e) mag = fmaxf(mag, fabsf(to_f32<QDT>(uint16_t(qf[s][e >> 1] >> (16 * (e & 1))))));
      }
      mag = half_pair_max(mag);
      const int shift = mag > 0.f && mag < INFINITY ? 10 - __builtin_amdgcn_frexp_expf(mag) : 0;
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ldexpf(to_f32<QDT>(uint16_t(qf[s][e >> 1] >> (16 * (e & 1)))), shift);
        // a widened row's order
        qf[s] = u32x4_t{f32x2_to_f16x2_bits(v[0], v[4]), f32x2_to_f16x2_bits(v[1], v[5]),
                        f32x2_to_f16x2_bits(v[2], v[6]), f32x2_to_f16x2_bits(v[3], v[7])};
      }
      f = ldexpf(f, -shift);
    }
    f = fmaxf(f, 0x1p-126f);  // scores that vanish: not 0, which a hidden score's -inf makes NaN
    // the loads end here: a first use inside the loop would wait, every time round, for
    // the tiles in flight too
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) asm volatile("" : "+v"(qf[s]));
  }

  // ---- LDS read addresses: K chunk 2 s + half of key l31 (+ 32 u); V^T: keys 4 half +
  // (i >> 2) (+ 16 kk + 8), columns 32 dt + 16 dg + 4 (i & 3)
  int xk = key_swizzle<D>(l31) * 16;
  const int kaddr = l31 * S::kRowBytes;
  const int i16 = lane & 15, dg = (lane >> 4) & 1, vkey = 4 * half + (i16 >> 2);
  int xv = value_swizzle<D>(vkey) * 16;
  const int vaddr = vkey * S::kRowBytes + (i16 & 1) * 8;
  const int vcol = (2 * dg + ((i16 & 3) >> 1)) * 16;

  f32x16_t o[S::kDims];
#pragma unroll
  for (int d = 0; d < S::kDims; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -INFINITY, m_use = 0.f, l = 0.f;

  const uint16_t* kb = nullptr;
  const uint16_t* vb = nullptr;
  size_t row_at = 0;  // 4-bit cache: first row of the head
  if constexpr (!KV4) {
    kb = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + g * a.k_stride[1];
    vb = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + g * a.v_stride[1];
  } else {
    row_at = size_t(head) * a.L;
  }
  // four waves: each stages keys and values; eight: four stage keys, four values
  Kv4Stage<D> ks, other;
  Kv4Stage<D>& vs = NW == 8 ? ks : other;
  const bool keys_here = NW == 4 || wave < 4, values_here = NW == 4 || wave >= 4;
  const int ts = t & 255;

  // LDS: keys of tile i at (i % 2) tiles, values at 2 + (i % 2) (i from it0)
  const auto key_tile = [&](int parity) __attribute__((always_inline)) { return lds + parity * S::kTileBytes; };
  const auto value_tile = [&](int parity) __attribute__((always_inline)) { return lds + (2 + parity) * S::kTileBytes; };
  // loads of tile `it` of the list (none past the last): 16-bit rows on their way into LDS,
  // 4-bit ones into registers
  auto fetch_keys = [&](int it, int parity) __attribute__((always_inline)) {
    if (it >= it1) return;
    const int j0 = tiles.tile_start<KT>(it), rows = tiles.tile_end(it, hi_pos, a.sinks) - j0;
    const size_t at = row_at + j0;
    if constexpr (!KV4)
      load_rows_to_lds<D, true>(kb + j0 * a.k_stride[2], a.k_stride[2], rows, key_tile(parity), wave, lane);
    else if (keys_here)
      ks.load(static_cast<const uint8_t*>(a.k) + at * (D / 2), a.k_scales + at * (D / 64), rows, ts);
  };
  auto fetch_values = [&](int it, int parity) __attribute__((always_inline)) {
    if (it >= it1) return;
    const int j0 = tiles.tile_start<KT>(it), rows = tiles.tile_end(it, hi_pos, a.sinks) - j0;
    const size_t at = row_at + j0;
    if constexpr (!KV4)
      load_rows_to_lds<D, false>(vb + j0 * a.v_stride[2], a.v_stride[2], rows, value_tile(parity), wave, lane);
    else if (values_here)
      vs.load(static_cast<const uint8_t*>(a.v) + at * (D / 2), a.v_scales + at * (D / 64), rows, ts);
  };

  // operand n of a tile's S^T products (key block n / kSteps, step n % kSteps) and of its O^T
  // products (16 keys n / kDims, column block n % kDims)
  constexpr int kKeyOps = S::kSteps * S::kSub, kValueOps = 2 * S::kSub * S::kDims;
  auto key_operand = [&](const lds_char* kt, int n) __attribute__((always_inline)) {
    return lds_b128(kt + kaddr + n / S::kSteps * 32 * S::kRowBytes + ((n % S::kSteps * 32 + half * 16) ^ xk));
  };
  auto value_operand = [&](const lds_char* vt, int n) __attribute__((always_inline)) {
    const lds_char* at = vt + vaddr + n / S::kDims * 16 * S::kRowBytes + ((vcol + n % S::kDims * 64) ^ xv);
    const u32x2_t x = lds_transposed(at), y = lds_transposed(at + 8 * S::kRowBytes);
    return u32x4_t{x[0], x[1], y[0], y[1]};
  };
  auto scores = [&](const lds_char* kt, f32x16_t(&s)[S::kSub]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < S::kSub; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int n = 0; n < kKeyOps; ++n)
      s[n / S::kSteps] = mfma32<CDT>(key_operand(kt, n), qf[n % S::kSteps], s[n / S::kSteps]);
  };

  // the largest of a tile's scores; the running maximum takes it in
  auto largest = [&](const f32x16_t(&s)[S::kSub]) __attribute__((always_inline)) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < S::kSub; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    return half_pair_max(top) * f;
  };
  auto raise = [&](float top) __attribute__((always_inline)) {
    constexpr bool kF16P = CDT == kF16;
    if (__builtin_amdgcn_ballot_w64(top > m + (kF16P ? p_room(top, 15.f) : 8.f))) {
      const float mn = fmaxf(m, kF16P ? top - p_room(top, 7.f) : top);
      m_use = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - m_use);  // 0 before the first visible key
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < S::kDims; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
  };

  // scores 2 i, 2 i + 1 of the tile: p in the operand layout of P^T, and its sum
  auto weigh = [&](const f32x16_t(&s)[S::kSub], u32x4_t(&pf)[2 * S::kSub], int i) __attribute__((always_inline)) {
    const int u = i / 8, r = i % 8 * 2;
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], f, -m_use));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r + 1], f, -m_use));
    l += p0 + p1;
    asm volatile("" : "+v"(l));  // here, not behind the products with every p kept until then
    float c0 = p0, c1 = p1;
    pf[2 * u + r / 8][(r & 7) / 2] = round_pair_bits<CDT>(c0, c1);
  };

  // A tile that some query sees only in part: hidden scores become -inf.
  auto partial = [&](int it) __attribute__((always_inline)) {
    const int j0 = tiles.tile_start<KT>(it);
    return !all_see(lo_pos, hi_pos, j0, j0 + KT, a.window, a.sinks, it < tiles.sink_tiles);
  };
  auto hide = [&](int it, f32x16_t(&s)[S::kSub]) __attribute__((always_inline)) {
    const bool sink_tile = it < tiles.sink_tiles;
    const TileMask seen(p, a.window, a.sinks, sink_tile, tiles.joined);
    const int first = tiles.tile_start<KT>(it) + 4 * half;
    const auto each = [&](auto sees) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < S::kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[u][r] = sees(first + 32 * u + (r & 3) + 8 * (r >> 2)) ? s[u][r] : -INFINITY;
    };
    if (sink_tile || tiles.joined) each([&](int j) __attribute__((always_inline)) { return seen.sees(j); });
    else each([&](int j) __attribute__((always_inline)) { return seen.sees_window(j); });
  };
  // Keys that no query of the workgroup sees are zeros in LDS.  One that some see may hold an
  // infinity or a NaN, and a product with a zero p, a hidden query's or one too small for 16
  // bits, would make NaN of it.  The careful round adds such values by hand to the rows that
  // see them and zeroes them; in a tile that every query sees it has the scores raised (true
  // returned; by hand in every tile, 1024 tokens whose values are all NaN took 1422 us for 160).
  auto settle = [&](int it, lds_char* vt) __attribute__((always_inline)) {
    const bool whole = !partial(it);
    if (KV4 && whole) return false;  // NaN alone
    unsigned bad = 0;
    for (int i = t * 16; i < S::kTileBytes; i += kThreads * 16) {
      const u32x4_t w = lds_b128(vt + i);
      bad |= nonfinite_pair<CDT>(w[0]) | nonfinite_pair<CDT>(w[1]) | nonfinite_pair<CDT>(w[2]) |
             nonfinite_pair<CDT>(w[3]);
    }
    if (!__syncthreads_or(bad != 0)) return false;
    if (whole) return true;
    const TileMask seen(p, a.window, a.sinks, it < tiles.sink_tiles, tiles.joined);
    const int j0 = tiles.tile_start<KT>(it);
    int h = half;
    asm volatile("" : "+v"(h));  // no address of this rare path is kept in a register elsewhere
    for (int j = 0; j < KT; ++j) {
      if (!active || !seen.sees(j0 + j)) continue;
#pragma unroll
      for (int d = 0; d < S::kDims; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int x = 32 * d + (r & 3) + 8 * (r >> 2) + 4 * h;
          const uint16_t bits = *reinterpret_cast<const __attribute__((address_space(3))) uint16_t*>(
              vt + j * S::kRowBytes + (((x >> 3) ^ value_swizzle<D>(j)) * 16) + (x & 7) * 2);
          o[d][r] += nonfinite_pair<CDT>(bits) ? to_f32<CDT>(bits) : 0.f;
          if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few values at a time: registers are scarce
        }
    }
    __syncthreads();
    for (int i = t * 16; i < S::kTileBytes; i += kThreads * 16) {
      u32x4_t w = lds_b128(vt + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = finite_pair<CDT>(w[e]);
      *reinterpret_cast<__attribute__((address_space(3))) u32x4_t*>(vt + i) = w;
    }
    __syncthreads();
    return false;
  };
  // Loads asked for one step ago have arrived (every wave waits for its own), and every wave
  // is done with what the next ones overwrite.
  auto arrive = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // Step `it` (it - it0 = parity mod 2): p of this tile's scores s beside the products of the
  // next tile's, sn; then O.  In LDS: this tile's values, the next one's keys; on their way:
  // the next one's values, the keys after.
  auto step = [&](int it, int parity, f32x16_t(&s)[S::kSub], f32x16_t(&sn)[S::kSub])
                  __attribute__((always_inline)) {
    arrive();
    fetch_keys(it + 2, parity);
    fetch_values(it + 1, parity ^ 1);
    // the swizzled addresses are formed anew for each tile (kept, they spill other values, and
    // a reload waits for the tile in flight)
    asm volatile("" : "+v"(xk), "+v"(xv));
    if (active) {
      // One list of products, S^T of the next tile and then O^T of this one, operands read
      // from LDS kAhead products early; between the former the exponentials of this tile,
      // between the latter the maximum of the next.  Fenced product by product: left alone,
      // the compiler orders for fewest registers, every operand read just before its use and
      // all exponentials behind all products.
      const lds_char* kt = key_tile(parity ^ 1);
      const lds_char* vt = value_tile(parity);
      constexpr int kAhead = 4, kOps = kKeyOps + kValueOps, kPairs = 8 * S::kSub;
      u32x4_t pf[2 * S::kSub], ring[kAhead + 1];
      const auto operand = [&](int n) __attribute__((always_inline)) {
        return n < kKeyOps ? key_operand(kt, n) : value_operand(vt, n - kKeyOps);
      };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) ring[n] = operand(n);
#pragma unroll
      for (int u = 0; u < S::kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) sn[u][r] = 0.f;
      float top = -INFINITY;  // as if no score were hidden
#pragma unroll
      for (int n = 0; n < kOps; ++n) {
        if (n + kAhead < kOps) ring[(n + kAhead) % (kAhead + 1)] = operand(n + kAhead);
        const u32x4_t x = ring[n % (kAhead + 1)];
        if (n < kKeyOps) {
          sn[n / S::kSteps] = mfma32<CDT>(x, qf[n % S::kSteps], sn[n / S::kSteps]);
#pragma unroll
          for (int i = n * kPairs / kKeyOps; i < (n + 1) * kPairs / kKeyOps; ++i) weigh(s, pf, i);
        } else {
          const int v = n - kKeyOps;
          o[v % S::kDims] = mfma32<CDT>(x, pf[v / S::kDims], o[v % S::kDims]);
#pragma unroll
          for (int i = v * kPairs / kValueOps; i < (v + 1) * kPairs / kValueOps; ++i)
            top = fmaxf(fmaxf(top, sn[i / 8][i % 8 * 2]), sn[i / 8][i % 8 * 2 + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      top = half_pair_max(top) * f;
      if (partial(it + 1)) {
        hide(it + 1, sn);
        top = largest(sn);
      }
      raise(top);
    }
    if constexpr (KV4) {
      if (keys_here && it + 2 < it1) ks.template store<true>(key_tile(parity), ts);
      if (values_here) vs.template store<false>(value_tile(parity ^ 1), ts);
    }
  };
  auto weigh_values = [&](int parity, f32x16_t(&s)[S::kSub]) __attribute__((always_inline)) {
    u32x4_t pf[2 * S::kSub];
#pragma unroll
    for (int i = 0; i < 8 * S::kSub; ++i) weigh(s, pf, i);
#pragma unroll
    for (int n = 0; n < kValueOps; ++n)
      o[n % S::kDims] = mfma32<CDT>(value_operand(value_tile(parity), n), pf[n / S::kDims], o[n % S::kDims]);
  };

  if (it0 < it1) {
    f32x16_t sa[S::kSub], sb[S::kSub];
    fetch_keys(it0, 0);
    fetch_values(it0, 0);
    if constexpr (KV4) {
      if (keys_here) ks.template store<true>(key_tile(0), ts);
      if (values_here) vs.template store<false>(value_tile(0), ts);
    }
    fetch_keys(it0 + 1, 1);
    if constexpr (KV4) {
      if (keys_here && it0 + 1 < it1) ks.template store<true>(key_tile(1), ts);
    }
    arrive();
    if (active) {
      scores(key_tile(0), sa);
      if (partial(it0)) hide(it0, sa);
      raise(largest(sa));
    }
    int it = it0;
    for (; it + 2 < it1; it += 2) {
      step(it, 0, sa, sb);
      step(it + 1, 1, sb, sa);
    }
    if (it + 1 < it1) {
      step(it, 0, sa, sb);
      arrive();
      if (active) weigh_values(1, sb);
    } else {
      arrive();
      if (active) weigh_values(0, sa);
    }
    // If some row came out infinite or NaN, once more and carefully: such a row may have it
    // from a value that it does not see (and a row that has it by right can wait).
    float probe = 0.f;
#pragma unroll
    for (int d = 0; d < S::kDims; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) probe = __builtin_fmaf(o[d][r], 0.f, probe);
    // (the barrier: every wave is done with the tiles)
    if (__builtin_expect(__syncthreads_or(!(probe == 0.f)), 0)) {
#pragma unroll
      for (int d = 0; d < S::kDims; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
      m = -INFINITY;
      m_use = l = 0.f;
      for (it = it0; it < it1; ++it) {
        fetch_keys(it, 0);
        fetch_values(it, 0);
        if constexpr (KV4) {
          if (keys_here) ks.template store<true>(key_tile(0), ts);
          if (values_here) vs.template store<false>(value_tile(0), ts);
        }
        arrive();
        if (active) {
          scores(key_tile(0), sa);
          if (partial(it)) hide(it, sa);
          raise(largest(sa));
        }
        if (settle(it, value_tile(0))) {
          const float least = least_score<CDT>(m) / f;
#pragma unroll
          for (int u = 0; u < S::kSub; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) sa[u][r] = sa[u][r] < least ? least : sa[u][r];
        }
        if (active) weigh_values(0, sa);
        __syncthreads();  // the next tile's loads overwrite this one
      }
    }
  }

  // ---- out.  (The row's place again: kept through the loop, it would cost the loop registers.)
  if (!active) return;
  int own_row = wave_row + l31;
  asm volatile("" : "+v"(own_row));
  const bool live = own_row < rows;
  l = half_pair_sum(l);
  if (a.splits > 1) {
    if (!live) return;
    const size_t slot = (size_t(head) * a.T * a.G + own_row) * a.splits + split;
    float* po = a.partial + slot * D;
#pragma unroll
    for (int d = 0; d < S::kDims; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int x = 32 * d + 2 * r + 4 * half;
        if constexpr (!KV4) {
          *reinterpret_cast<float4*>(po + x) = make_float4(o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) po[kv4_column(x + e)] = o[d][r + e];
        }
      }
    if (half == 0) {
      float* ml = a.partial + size_t(heads) * a.T * a.G * a.splits * D + slot * 2;
      ml[0] = m;
      ml[1] = l;
    }
    return;
  }
  // rows through LDS (each wave its own 32, the tiles are done with): written as the lanes
  // hold them, 16 bytes of 32 rows at a time, a prompt's output cost 16 times the requests
  const float inv = softmax_inverse(l, base_pos + min(own_row, rows - 1) / a.G);
  lds_char* const mine = lds + wave * 32 * S::kRowBytes;
#pragma unroll
  for (int d = 0; d < S::kDims; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[d][r + e] * inv;
      u32x2_t w;
      if constexpr (!KV4) {
        w = u32x2_t{round_pair_bits<QDT>(v[0], v[1]), round_pair_bits<QDT>(v[2], v[3])};
      } else {
        // this lane holds columns 0 4 1 5 of a chunk, lane + 32 its 2 6 3 7: trade for 0 1 2 3
        // and 4 5 6 7
        w = __builtin_amdgcn_permlane32_swap(round_pair_bits<QDT>(v[0], v[2]), round_pair_bits<QDT>(v[1], v[3]), false,
                                             false);
      }
      const int chunk = 4 * d + r / 4;
      *reinterpret_cast<__attribute__((address_space(3))) u32x2_t*>(
          mine + l31 * S::kRowBytes + ((chunk ^ key_swizzle<D>(l31)) * 16) + half * 8) = w;
    }
  wave_lds_order();
#pragma unroll
  for (int i = 0; i < S::kChunks / 2; ++i) {
    const int at = i * 64 + lane, r = at / S::kChunks, chunk = at % S::kChunks;
    const int rr = wave_row + r;
    const u32x4_t w = lds_b128(mine + r * S::kRowBytes + ((chunk ^ key_swizzle<D>(r)) * 16));
    if (rr < rows) {
      const int tk = rr / a.G, hd = g * a.G + rr - tk * a.G;
      *reinterpret_cast<u32x4_t*>(a.out + b * a.out_stride[0] + hd * a.out_stride[1] + tk * a.out_stride[2] +
                                  chunk * 8) = w;
    }
  }
}

template <int DT, int D, bool KV4>
void launch_attention_rows(const CachedAttentionPlan& plan, const CachedAttentionArgs& a, hipStream_t s) {
  const dim3 blocks(unsigned(a.B) * a.Hk * a.row_tiles * a.splits);
  if constexpr (KV4 && D <= 128) {
    if (plan.waves == 8) {
      hipLaunchKernelGGL((attention_rows_kernel<DT, D, KV4, 8>), blocks, dim3(512), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((attention_rows_kernel<DT, D, KV4, 4>), blocks, dim3(256), 0, s, a);
}

}  // namespace fx
