// Cached attention of few query rows for a KV head (row = token * G + head of the group): a
// decode step, or a few drafted tokens; over a 4-bit cache with fp16 queries any number of
// them.  Bound by reading the cache once: 24 sequences x 4100 keys x 8 heads of 128 16-bit
// columns 74 us (5.4 TB/s; a large copy moves 4.8), 32 x 16384..32768 in 4 bits 190 us
// (4.8 TB/s).  D = 256 on a 16-bit cache spills 33 registers and asks for no tile ahead: 8 x
// 8192 keys of 8 heads 129 us (4.2 TB/s).  Short calls are bound by the two launches and their
// chain of loads: 2000 keys of one sequence 9.5 us.  Several row groups (5 tokens of 7 heads
// over 4101 keys of 8 sequences of 4 KV heads in 4 bits: 20 us, 10 of them for 5 keys too) are
// bound by the vector work on the codes, ~600 instructions for 32 keys and 32 rows.
//
// A wave takes 32 keys at a time straight from memory into operand registers, with the
// next 32 on their way: S^T = K Q^T and O^T += V^T P^T on 16 x 16 x 32 products, column =
// query row, so that a query's scores sit in four lanes and P^T leaves S^T in the operand
// layout (16-key blocks u = 0, 1: lane group h = lane / 16 holds keys 16 u + 4 h .. + 3).
// V is read as the rows lie in memory; the two keys of an operand word meet by a byte
// permute.  A workgroup's waves are row_groups (16 RT rows each) x key waves; the key waves
// of all splits take tiles in turn, those of a workgroup join their (m, l, O) in LDS, and
// the splits' partials meet in attention_combine_kernel.
//
// 4-bit cache: the codes themselves are the operands.  A nibble masked in place is the
// fp16 subnormal code * 2^-24 (low nibble of a byte) or code * 2^-20, exactly, so scale and
// minimum enter outside the products, in fp32: per group of 64 columns
//   s_j = scale_j (codes_j . q) + minimum_j sum(q),
//   O   = sum_j (p_j scale_j) codes_j + sum_j p_j minimum_j,
// with p_j scale_j rounded to fp16 (2^-11).  So that the product fits whatever the scales'
// size, the running maximum is taken over s_j + log2 of the key's largest scale (rounded
// down), less 14: p_j scale_j is 2^14 .. 2^15 at the largest of a row, in full down to 2^-28 of
// that and lost below 2^-39, be it for the key's score or for a group's small scale beside
// its neighbours'.  (The matrix unit cuts the eight terms of a step 24 bits below the largest
// exponent among them, where a subnormal counts as 2^-14: below 2^-14 of a code's worth of the
// largest p_j scale_j, an eighth of that weight's own rounding.)
#pragma once
#include <type_traits>

#include "attention_core.h"

namespace fx {

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

// The tile in registers: what this lane's operands need of 32 keys.
template <int D, bool KV4>
struct FewTile {
  static constexpr int kSteps = D / 32, kGroups = D / 64;
  static constexpr int kValueWords = KV4 ? (D == 256 ? 2 : 1) : D / 32;  // words of a key's value that a lane holds
  u32x4_t k16[KV4 ? 1 : 2][KV4 ? 1 : kSteps];  // 16-bit: keys of the blocks u
  unsigned k[KV4 ? 2 : 1][KV4 ? D / 32 : 1];   // codes of the keys: this lane's quarter row
  unsigned v[8][kValueWords];                  // values of the keys 16 (e / 4) + 4 h4 + e % 4
  unsigned scales[KV4 ? (kGroups == 1 ? 1 : kGroups) : 1];  // (scale, minimum) pairs, spread over the wave
};

template <int QDT, int D, bool KV4, int RT, int NW>
__global__ __launch_bounds__(64 * NW, KV4 && RT == 1 && D <= 128 ? 3 : 2) void attention_few_kernel(const CachedAttentionArgs a) {
  using Tile = FewTile<D, KV4>;
  constexpr int CDT = KV4 ? kF16 : QDT;
  constexpr int kSteps = D / 32;   // depth steps of S^T
  constexpr int kUnit = D / 16;    // columns of O^T that a chunk (lane % 16) holds
  constexpr int kGroups = D / 64;
  constexpr int kValueWords = Tile::kValueWords;
  constexpr int kRows = 16 * RT;   // query rows of a wave
  __shared__ float red_ml[NW][2][kRows];
  // the waves' joins; before them, KV4: each wave's (scale, minimum) pairs of a tile
  __shared__ __attribute__((aligned(16))) float red_o[NW][kRows][D + 4];
  const int t = threadIdx.x, lane = t & 63, wave = wave_index();
  const int l16 = lane & 15, h4 = lane >> 4;
  unsigned(*const pairs)[32 * kGroups] = reinterpret_cast<unsigned(*)[32 * kGroups]>(&red_o[wave][0][0]);

  // ---- workgroup: a KV head, a tile of its query rows, a split of the keys; wave: one of
  // the tile's row groups
  const int heads = a.B * a.Hk;
  int id = blockIdx.x;
  const int head = id % heads;
  id /= heads;
  const int split = id % a.splits, row_tile = id / a.splits;
  const int row_group = wave % a.row_groups, key_wave = wave / a.row_groups, key_waves = NW / a.row_groups;
  const int b = head / a.Hk, g = head - b * a.Hk;
  const SequenceSpan span = sequence_span(a, b);
  const int rows = span.m * a.G;
  const int tile_row = row_tile * a.row_groups * kRows;
  if (tile_row >= rows) return;
  const int row0 = tile_row + row_group * kRows;
  const int base_pos = span.n - span.m;
  KeyTiles tiles{0, 0, 0, false};
  int lo_pos = 0, hi_pos = -1;
  if (row0 < rows) {
    lo_pos = base_pos + row0 / a.G;
    hi_pos = base_pos + (min(row0 + kRows, rows) - 1) / a.G;
    tiles = key_tiles<kFewKeys>(lo_pos, hi_pos, a.window, a.sinks);
  }
  // tiles dealt out in turn over the splits and their waves: all read one stretch of the
  // cache at a time, and ragged lengths fill every wave alike
  const int it0 = split * key_waves + key_wave, it1 = tiles.count, it_step = a.splits * key_waves;

  // ---- this lane's query rows, as the B operands of the depth steps
  int p[RT];
  u32x4_t qf[RT][kSteps];
  float f[RT];
  float qsum[RT][kGroups];  // KV4: f * the sums of q over each group's columns
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = min(row0 + 16 * rt + l16, rows - 1), tok = row / a.G, hq = g * a.G + row - tok * a.G;
    p[rt] = base_pos + tok;
    const uint16_t* q = a.q + b * a.q_stride[0] + hq * a.q_stride[1] + tok * a.q_stride[2];
    f[rt] = a.scale * kLog2e;
    if constexpr (!KV4) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) qf[rt][s] = *reinterpret_cast<const u32x4_t*>(q + 32 * s + 8 * h4);
    } else {
      // columns 64 g + 16 h4 .. + 15 of every group, in fp16 and scaled by a power of two so
      // that the row's largest magnitude lies in [2^9, 2^10) (of fp16 subnormals in [2^6,
      // 2^10)); step (g, half): word r holds nibble r of units 4 h4 + 2 half and the next, odd
      // nibbles 2^-4 for their place in the byte.  On packed halves: every wave prepares its
      // rows, and of a short split's time that is a large part.
      unsigned w[kGroups][8];
      u16x2_t big = {0, 0};
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const u32x4_t x = *reinterpret_cast<const u32x4_t*>(q + 64 * gg + 16 * h4 + 8 * c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[gg][4 * c + i] = x[i];
            big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2_t, x[i] & 0x7fff7fffu));
          }
        }
      const float mag = quarter_max(to_f32<QDT>(max(big[0], big[1])));
      int shift = mag > 0.f && mag < INFINITY ? 10 - __builtin_amdgcn_frexp_expf(mag) : 0;
      if constexpr (QDT == kF16) shift = min(shift, 30);  // two factors of fp16; 2^-24 comes to 2^6 by it
      f[rt] = ldexpf(f[rt], -shift);
      const _Float16 once = _Float16(ldexpf(1.f, shift >> 1)), again = _Float16(ldexpf(1.f, shift - (shift >> 1)));
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f16x2_t v;
          if constexpr (QDT == kF16) {  // shift -6 .. 30: in two steps, exact unless down into the subnormals
            v = __builtin_bit_cast(f16x2_t, w[gg][i]) * once * again;
          } else {
            v = __builtin_convertvector(f32x2_t{ldexpf(__uint_as_float(w[gg][i] << 16), shift),
                                                ldexpf(__uint_as_float(w[gg][i] & 0xffff0000u), shift)},
                                        f16x2_t);
          }
          sum = __builtin_amdgcn_fdot2(v, f16x2_t{1, 1}, sum, false);
          w[gg][i] = __builtin_bit_cast(unsigned, v);
        }
        qsum[rt][gg] = quarter_sum(sum) * f[rt];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const unsigned pair = __builtin_amdgcn_perm(w[gg][4 * half + 2 + r / 2], w[gg][4 * half + r / 2],
                                                        r & 1 ? 0x07060302u : 0x05040100u);
            qf[rt][2 * gg + half][r] =
                r & 1 ? __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2_t, pair) * _Float16(0.0625f)) : pair;
          }
      }
      f[rt] = ldexpf(f[rt], 24);  // the codes' 2^-24
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(qf[rt][s]));  // the loads end before the loop
  }

  // ---- the cache
  const uint16_t* kb = nullptr;
  const uint16_t* vb = nullptr;
  size_t row_at = 0;
  if constexpr (!KV4) {
    kb = static_cast<const uint16_t*>(a.k) + b * a.k_stride[0] + g * a.k_stride[1];
    vb = static_cast<const uint16_t*>(a.v) + b * a.v_stride[0] + g * a.v_stride[1];
  } else {
    row_at = size_t(head) * a.L;
  }
  // (past the last tile nothing is read: a load under a branch would make the waits of both
  // sides those of the shorter one, for the tile just asked for)
  auto fetch = [&](int it, Tile& x) __attribute__((always_inline)) {
    const int j0 = it < it1 ? tiles.tile_start<kFewKeys>(it) : 0;
    const int live = it < it1 ? min(tiles.tile_end(it, hi_pos, a.sinks) - j0, kFewKeys) : 0;  // others: zeros
    if constexpr (!KV4) {
      const int ks = int(a.k_stride[2]) * 2, vs = int(a.v_stride[2]) * 2;
      const auto rk = row_resource(kb + j0 * a.k_stride[2], a.k_stride[2], live, D);
      const auto rv = row_resource(vb + j0 * a.v_stride[2], a.v_stride[2], live, D);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
          x.k16[u][s] = load_b128(rk, (16 * u + l16) * ks + (32 * s + 8 * h4) * 2, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = (16 * (e >> 2) + 4 * h4 + (e & 3)) * vs + l16 * kUnit * 2;
        if constexpr (kValueWords == 2) {
          const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(rv, at, 0, 0);
          x.v[e][0] = w[0];
          x.v[e][1] = w[1];
        } else {
#pragma unroll
          for (int c = 0; c < kValueWords; c += 4) {
            const u32x4_t w = load_b128(rv, at + c * 4, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) x.v[e][c + i] = w[i];
          }
        }
      }
    } else {
      const size_t at = row_at + j0;
      const auto rk = buffer_resource_2g(static_cast<const uint8_t*>(a.k) + at * (D / 2), unsigned(live) * (D / 2));
      const auto rv = buffer_resource_2g(static_cast<const uint8_t*>(a.v) + at * (D / 2), unsigned(live) * (D / 2));
      const auto rks = buffer_resource_2g(a.k_scales + at * kGroups, unsigned(live) * (kGroups * 4));
      const auto rvs = buffer_resource_2g(a.v_scales + at * kGroups, unsigned(live) * (kGroups * 4));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int key = (16 * u + l16) * (D / 2) + h4 * (D / 8);
        if constexpr (D == 64) {
          const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(rk, key, 0, 0);
          x.k[u][0] = w[0];
          x.k[u][1] = w[1];
        } else {
#pragma unroll
          for (int c = 0; c < D / 32; c += 4) {
            const u32x4_t w = load_b128(rk, key + c * 4, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) x.k[u][c + i] = w[i];
          }
        }
      }
      if constexpr (kGroups == 1) {
        // lanes 0 .. 31 the keys' pairs, 32 .. 63 the values'
        const unsigned wk = __builtin_amdgcn_raw_buffer_load_b32(rks, lane < 32 ? lane * 4 : kOutOfRange, 0, 0);
        const unsigned wv = __builtin_amdgcn_raw_buffer_load_b32(rvs, lane < 32 ? kOutOfRange : (lane - 32) * 4, 0, 0);
        x.scales[0] = wk | wv;
      } else if constexpr (kGroups == 2) {
        x.scales[0] = __builtin_amdgcn_raw_buffer_load_b32(rks, lane * 4, 0, 0);
        x.scales[1] = __builtin_amdgcn_raw_buffer_load_b32(rvs, lane * 4, 0, 0);
      } else {
        const u32x2_t wk = __builtin_amdgcn_raw_buffer_load_b64(rks, lane * 8, 0, 0);
        const u32x2_t wv = __builtin_amdgcn_raw_buffer_load_b64(rvs, lane * 8, 0, 0);
        x.scales[0] = wk[0];
        x.scales[1] = wk[1];
        x.scales[2] = wv[0];
        x.scales[3] = wv[1];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = (16 * (e >> 2) + 4 * h4 + (e & 3)) * (D / 2) + l16 * (D / 32);
        if constexpr (D == 64) {
          x.v[e][0] = __builtin_amdgcn_raw_buffer_load_b16(rv, key, 0, 0);
        } else if constexpr (D == 128) {
          x.v[e][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, key, 0, 0);
        } else {
          const u32x2_t w = __builtin_amdgcn_raw_buffer_load_b64(rv, key, 0, 0);
          x.v[e][0] = w[0];
          x.v[e][1] = w[1];
        }
      }
    }
  };

  f32x4_t o[RT][kUnit];
  float omin[RT][kGroups];  // KV4: the part of O outside the product, over this lane's keys
  float m[RT], m_use[RT], l[RT];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < kUnit; ++i) o[rt][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) omin[rt][gg] = 0.f;
      m[rt] = -INFINITY;
      m_use[rt] = l[rt] = 0.f;
    }
  };
  clear();

  auto half_of = [](unsigned w, int i) { return f16_bits_to_f32(uint16_t(i ? w >> 16 : w)); };

  // running maximum of row tile rt: over `bound`, all by `less` too large; p up to 2^room
  auto raise = [&](int rt, const float(&bound)[8], float less, float room) __attribute__((always_inline)) {
    float top = bound[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, bound[e]);
    top = quarter_max(top);
    top -= less + (room > 0.f ? p_room(top, room) : 0.f);
    if (__builtin_amdgcn_ballot_w64(top > m[rt])) {
      const float before = m[rt];
      m[rt] = fmaxf(before, top);
      m_use[rt] = m[rt] == -INFINITY ? 0.f : m[rt];
      const float alpha = __builtin_amdgcn_exp2f(before - m_use[rt]);  // 0 before the first visible key
      l[rt] *= alpha;
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) omin[rt][gg] *= alpha;
#pragma unroll
      for (int i = 0; i < kUnit; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[rt][i][r] *= alpha;
    }
  };
  auto mask = [&](int rt, bool sink_tile) __attribute__((always_inline)) {
    return TileMask(p[rt], a.window, a.sinks, sink_tile, tiles.joined);
  };
  auto hide = [&](int rt, int j0, bool sink_tile, float(&s)[8]) __attribute__((always_inline)) {
    asm volatile("");  // a branch: not worked out for the tiles that every row sees
    const TileMask seen = mask(rt, sink_tile);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = seen.sees(j0 + 16 * (e >> 2) + 4 * h4 + (e & 3)) ? s[e] : -INFINITY;
  };

  // scores in log2 units: s[4 u + r] of key j0 + 16 u + 4 h4 + r
  auto compute16 = [&](Tile& x, int j0, bool whole, bool sink_tile, bool careful) __attribute__((always_inline)) {
    u32x4_t pf[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float s[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f32x4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < kSteps; ++st) c = mfma16<CDT>(x.k16[u][st], qf[rt][st], c);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * u + r] = c[r] * f[rt];
      }
      if (!whole) hide(rt, j0, sink_tile, s);
      raise(rt, s, 0.f, CDT == kF16 ? 15.f : 0.f);
      if (whole && careful) {
        asm volatile("");
        const float least = least_score<CDT>(m[rt]);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = s[e] < least ? least : s[e];
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float p0 = __builtin_amdgcn_exp2f(s[e] - m_use[rt]), p1 = __builtin_amdgcn_exp2f(s[e + 1] - m_use[rt]);
        l[rt] += p0 + p1;
        pf[rt][e / 2] = round_pair_bits<CDT>(p0, p1);
      }
    }
    if (!whole && careful) {
      // a hidden key's infinity or NaN must not meet its zero p: rows that see one take it
      // by hand (every lane reads the rows it needs again), then it counts as zero
      unsigned bad = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int c = 0; c < kValueWords; ++c) bad |= nonfinite_pair<CDT>(x.v[e][c]);
      if (__builtin_amdgcn_ballot_w64(bad != 0)) {
        int first_chunk = 4 * h4;
        asm volatile("" : "+v"(first_chunk));  // no address of this rare path is kept in a register elsewhere
        for (int j = j0; j < min(j0 + kFewKeys, hi_pos + 1); ++j) {
          const uint16_t* vr = vb + j * a.v_stride[2];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            if (!mask(rt, sink_tile).sees(j)) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int i = 0; i < kUnit; ++i) {
                const uint16_t bits = vr[(first_chunk + r) * kUnit + i];
                o[rt][i][r] += nonfinite_pair<CDT>(bits) ? to_f32<CDT>(bits) : 0.f;
              }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int c = 0; c < kValueWords; ++c) x.v[e][c] = finite_pair<CDT>(x.v[e][c]);
      }
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      u32x4_t vf;
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        vf[e / 2] = __builtin_amdgcn_perm(x.v[e + 1][i / 2], x.v[e][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) o[rt][i] = mfma16<CDT>(vf, pf[rt], o[rt][i]);
    }
  };

  auto compute4 = [&](Tile& x, int j0, bool whole, bool sink_tile, bool careful) __attribute__((always_inline)) {
    // ---- the tile's (scale, minimum) pairs through LDS: every lane needs those of its eight
    // keys, a lane loads its share of the tile's
    if constexpr (kGroups == 1) {
      pairs[lane >> 5][lane & 31] = x.scales[0];
    } else if constexpr (kGroups == 2) {
      pairs[0][lane] = x.scales[0];
      pairs[1][lane] = x.scales[1];
    } else {
      *reinterpret_cast<u32x2_t*>(&pairs[0][2 * lane]) = u32x2_t{x.scales[0], x.scales[1]};
      *reinterpret_cast<u32x2_t*>(&pairs[1][2 * lane]) = u32x2_t{x.scales[2], x.scales[3]};
    }
    wave_lds_order();
    float s[RT][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      unsigned ks[4 * kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(&pairs[0][(16 * u + 4 * h4) * kGroups + 4 * i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) ks[4 * i + c] = w[c];
      }
      float acc[RT][4], low[RT][4];
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) {
        u32x4_t kf[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // words (unit, group): units 2 half and 2 half + 1 of this lane's four
          const int wa = 2 * half * kGroups + gg, wb = wa + kGroups;
          const unsigned ab = kGroups == 1 ? x.k[u][half]
                                           : __builtin_amdgcn_perm(x.k[u][wb >> 1], x.k[u][wa >> 1],
                                                                   wa & 1 ? 0x07060302u : 0x05040100u);
          const unsigned hi = ab >> 8;
          kf[half] = u32x4_t{ab & 0x000f000fu, ab & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u};
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          f32x4_t c = {0.f, 0.f, 0.f, 0.f};
          c = mfma16<CDT>(kf[0], qf[rt][2 * gg], c);
          c = mfma16<CDT>(kf[1], qf[rt][2 * gg + 1], c);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const unsigned w = ks[r * kGroups + gg];
            acc[rt][r] = __builtin_fmaf(half_of(w, 0), c[r], gg == 0 ? 0.f : acc[rt][r]);
            low[rt][r] = __builtin_fmaf(half_of(w, 1), qsum[rt][gg], gg == 0 ? 0.f : low[rt][r]);
          }
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[rt][4 * u + r] = __builtin_fmaf(acc[rt][r], f[rt], low[rt][r]);
    }
    unsigned vs[2][4 * kGroups];
    float size[8];  // 2^10 (15 + log2 of the keys' largest value scales, rounded down)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(&pairs[1][(16 * u + 4 * h4) * kGroups + 4 * i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) vs[u][4 * i + c] = w[c];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        u16x2_t big = {0, 0};  // of the low halves, all positive
#pragma unroll
        for (int gg = 0; gg < kGroups; ++gg)
          big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2_t, vs[u][r * kGroups + gg]));
        size[4 * u + r] = float(__builtin_bit_cast(unsigned, big) & 0x7c00u);
      }
    }
    float pr[RT][8];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (!whole) hide(rt, j0, sink_tile, s[rt]);
      float bound[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) bound[e] = __builtin_fmaf(size[e], 0x1p-10f, s[rt][e]);
      raise(rt, bound, 15.f, 14.f);  // p * scale below 2^15
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pr[rt][e] = __builtin_amdgcn_exp2f(s[rt][e] - m_use[rt]);
        l[rt] += pr[rt][e];
      }
    }
    // the groups' weights, of all groups together where registers allow
    constexpr int kAtOnce = kGroups == 2 ? 2 : 1;
    u32x4_t pf[RT][kGroups];
    const auto weigh = [&](int g0, auto all) __attribute__((always_inline)) {
#pragma unroll
      for (int gg = g0; gg < g0 + kAtOnce; ++gg)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const unsigned w0 = vs[e >> 2][(e & 3) * kGroups + gg], w1 = vs[e >> 2][((e & 3) + 1) * kGroups + gg];
            const float p0 = pr[rt][e], p1 = pr[rt][e + 1];
            float s0 = p0 * half_of(w0, 0), s1 = p1 * half_of(w1, 0);
            float low = omin[rt][gg];
            if constexpr (decltype(all)::value) {
              low = __builtin_fmaf(p0, half_of(w0, 1), low);
              low = __builtin_fmaf(p1, half_of(w1, 1), low);
            } else {  // a hidden key's pair may be anything
              s0 = p0 == 0.f ? 0.f : s0;
              low += p0 == 0.f ? 0.f : p0 * half_of(w0, 1);
              s1 = p1 == 0.f ? 0.f : s1;
              low += p1 == 0.f ? 0.f : p1 * half_of(w1, 1);
            }
            const unsigned rounded = f32x2_to_f16x2_bits(s0, s1);
            if constexpr (QDT == kF16) {
              // what the rounding of p * scale took away, at the codes' middle: the rounding
              // then weighs codes - 8, the value's own size, in place of codes (0 .. 15).
              // Below a bf16 output's own rounding either way.
              const float lost = (s0 - half_of(rounded, 0)) + (s1 - half_of(rounded, 1));
              low = __builtin_fmaf(8.f, lost, low);
            }
            pf[rt][gg][e / 2] = rounded;
            omin[rt][gg] = low;
          }
    };
    const auto weigh_from = [&](int g0) __attribute__((always_inline)) {
      if (whole || !careful) {
        asm volatile("");  // two paths, neither worked out for the other
        weigh(g0, std::true_type{});
      } else {
        asm volatile("");
        weigh(g0, std::false_type{});
      }
    };
    if constexpr (kAtOnce > 1) weigh_from(0);
#pragma unroll
    for (int gg = 0; gg < kGroups; ++gg) {
      if constexpr (kAtOnce == 1) weigh_from(gg);
      // this group's four columns of the chunk: nibble i of word gg
      unsigned ab[4], hi[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        ab[e / 2] =
            __builtin_amdgcn_perm(x.v[e + 1][gg >> 1], x.v[e][gg >> 1], gg & 1 ? 0x07060302u : 0x05040100u);
        hi[e / 2] = ab[e / 2] >> 8;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned mask = i & 1 ? 0x00f000f0u : 0x000f000fu;
        u32x4_t vf;
#pragma unroll
        for (int c = 0; c < 4; ++c) vf[c] = (i & 2 ? hi[c] : ab[c]) & mask;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][4 * gg + i] = mfma16<CDT>(vf, pf[rt][gg], o[rt][4 * gg + i]);
      }
    }
    wave_lds_order();  // the pairs are read before the next tile's are written
  };

  auto compute = [&](Tile& x, int it, bool careful) __attribute__((always_inline)) {
    int how = careful;
    asm volatile("" : "+v"(how));  // one copy of the loop serves both rounds
    how = __builtin_amdgcn_readfirstlane(how);
    const int j0 = tiles.tile_start<kFewKeys>(it);
    const bool sink_tile = it < tiles.sink_tiles;
    const bool whole = all_see(lo_pos, hi_pos, j0, j0 + kFewKeys, a.window, a.sinks, sink_tile);
    if constexpr (KV4) compute4(x, j0, whole, sink_tile, how != 0);
    else compute16(x, j0, whole, sink_tile, how != 0);
  };

  // Once, and again carefully if some row came out infinite or NaN: such a row may have it
  // from a key that it does not see (and a row that has it by right can wait).
  bool careful = false;
  while (true) {
    // the next tile's loads ahead of this one's products, where registers allow
    if constexpr (KV4 || D <= 128) {
      Tile cur, nxt;
      fetch(it0, cur);
      for (int it = it0; it < it1; it += it_step) {
        fetch(it + it_step, nxt);
        compute(cur, it, careful);
        cur = nxt;
      }
    } else {
      Tile cur;
      for (int it = it0; it < it1; it += it_step) {
        fetch(it, cur);
        compute(cur, it, careful);
      }
    }
    if (careful) break;
    float probe = 0.f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) probe = __builtin_fmaf(omin[rt][gg], 0.f, probe);
#pragma unroll
      for (int i = 0; i < kUnit; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) probe = __builtin_fmaf(o[rt][i][r], 0.f, probe);
    }
    if (!__builtin_amdgcn_ballot_w64(!(probe == 0.f))) break;
    careful = true;
    clear();
  }

  // ---- the key waves' joins: O^T row 4 h4 + r, index i
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] = quarter_sum(l[rt]);
    if constexpr (KV4) {
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) omin[rt][gg] = quarter_sum(omin[rt][gg]);
    }
    if (h4 == 0) {
      red_ml[wave][0][16 * rt + l16] = m[rt];
      red_ml[wave][1][16 * rt + l16] = l[rt];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < kUnit; i += 4) {
        const int chunk = 4 * h4 + r;
        const int d = KV4 ? 16 * i + 4 * chunk : chunk * kUnit + i;  // KV4: group i / 4
        float4 w;
        if constexpr (KV4) {
          const float low = omin[rt][i / 4];
          w = make_float4(__builtin_fmaf(o[rt][i][r], 0x1p24f, low), __builtin_fmaf(o[rt][i + 1][r], 0x1p20f, low),
                          __builtin_fmaf(o[rt][i + 2][r], 0x1p24f, low), __builtin_fmaf(o[rt][i + 3][r], 0x1p20f, low));
        } else {
          w = make_float4(o[rt][i][r], o[rt][i + 1][r], o[rt][i + 2][r], o[rt][i + 3][r]);
        }
        *reinterpret_cast<float4*>(&red_o[wave][16 * rt + l16][d]) = w;
      }
  }
  __syncthreads();
  const int tile_rows = min(a.row_groups * kRows, rows - tile_row);
  // each row's weights of its key waves (in place of their maxima), and what its sum is
  if (t < tile_rows) {
    const int group = t / kRows, rr = t % kRows;
    float mw[NW], top = -INFINITY, lsum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      mw[w] = red_ml[min(w, key_waves - 1) * a.row_groups + group][0][rr];
      top = fmaxf(top, mw[w]);
    }
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w >= key_waves) break;
      // a wave without a visible key has m = -inf and nothing to add, unless its sum is NaN
      const float c = mw[w] == top ? 1.f : __builtin_amdgcn_exp2f(mw[w] - top);
      lsum += c * red_ml[w * a.row_groups + group][1][rr];
      red_ml[w * a.row_groups + group][0][rr] = c;
    }
    if (a.splits > 1) {
      const size_t slot = (size_t(head) * a.T * a.G + tile_row + t) * a.splits + split;
      float* ml = a.partial + size_t(heads) * a.T * a.G * a.splits * D + slot * 2;
      ml[0] = top;
      ml[1] = lsum;
    } else {
      red_ml[group][1][rr] = softmax_inverse(lsum, base_pos + (tile_row + t) / a.G);
    }
  }
  __syncthreads();
  for (int at = t; at < tile_rows * (D / 4); at += 64 * NW) {
    const int in_tile = at / (D / 4), d = at % (D / 4) * 4, group = in_tile / kRows, rr = in_tile % kRows;
    const int r = tile_row + in_tile;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {  // past the last key wave: the last again, with weight 0
      const int wv = min(w, key_waves - 1) * a.row_groups + group;
      const float c = w < key_waves ? red_ml[wv][0][rr] : 0.f;
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(&red_o[wv][rr][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(c, v[i], sum[i]);
    }
    if (a.splits > 1) {
      const size_t slot = (size_t(head) * a.T * a.G + r) * a.splits + split;
      *reinterpret_cast<f32x4_t*>(a.partial + slot * D + d) = sum;
    } else {
      const int tk = r / a.G;
      const float inv = red_ml[group][1][rr];
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = sum[i] * inv;
      *reinterpret_cast<u32x2_t*>(a.out + b * a.out_stride[0] + (g * a.G + r - tk * a.G) * a.out_stride[1] +
                                  tk * a.out_stride[2] + d) =
          u32x2_t{round_pair_bits<QDT>(v[0], v[1]), round_pair_bits<QDT>(v[2], v[3])};
    }
  }
}

template <int DT, int D, bool KV4>
void launch_attention_few(const CachedAttentionPlan& plan, const CachedAttentionArgs& a, hipStream_t s) {
  const dim3 grid(unsigned(a.B) * a.Hk * a.splits * a.row_tiles);
  if constexpr (KV4) {
    if (plan.waves == 8) {  // several row groups
      hipLaunchKernelGGL((attention_few_kernel<DT, D, KV4, (D <= 128 ? 2 : 1), 8>), grid, dim3(512), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((attention_few_kernel<DT, D, KV4, 1, 4>), grid, dim3(256), 0, s, a);
}

}  // namespace fx
