// Cached attention of at most 16 query rows for a KV head (row = token * G + head of the
// group): a decode step, or a few drafted tokens.  Bound by reading the cache once.
//
// A wave takes 32 keys at a time straight from memory into operand registers, with the
// next 32 on their way: S^T = K Q^T and O^T += V^T P^T on 16 x 16 x 32 products, column =
// query row, so that a query's scores sit in four lanes and P^T leaves S^T in the operand
// layout (16-key blocks u = 0, 1: lane group h = lane / 16 holds keys 16 u + 4 h .. + 3).
// V is read as the rows lie in memory; the two keys of an operand word meet by a byte
// permute.  The four waves of a workgroup take every fourth tile and join their (m, l, O)
// in LDS; workgroups along the keys write partials for attention_combine_kernel.
//
// 4-bit cache: the codes themselves are the operands.  A nibble masked in place is the
// fp16 subnormal code * 2^-24 (low nibble of a byte) or code * 2^-20, exactly, so scale and
// minimum enter outside the products, in fp32: per group of 64 columns
//   s_j = scale_j (codes_j . q) + minimum_j sum(q),
//   O   = sum_j (p_j scale_j) codes_j + sum_j p_j minimum_j,
// with p_j scale_j rounded to fp16 (2^-11).  So that the product neither overflows nor
// sinks into the subnormals whatever the scales' size, the running maximum is taken over
// s_j + log2 of the key's largest scale (rounded down).
#pragma once
#include "attention_core.h"

namespace fx {

template <int QDT, int D, bool KV4>
__global__ __launch_bounds__(256, 2) void attention_few_kernel(const CachedAttentionArgs a) {
  constexpr int CDT = KV4 ? kF16 : QDT;
  constexpr int kSteps = D / 32;   // depth steps of S^T
  constexpr int kUnit = D / 16;    // columns of O^T that a chunk (lane % 16) holds
  constexpr int kGroups = D / 64;
  constexpr int kValueWords = KV4 ? (D == 256 ? 2 : 1) : D / 32;  // words of a key's value that a lane holds
  constexpr bool kAhead = KV4 || D <= 128;                // room for the next tile's registers
  __shared__ float red_ml[4][2][16];
  __shared__ __attribute__((aligned(16))) float red_o[4][16][D + 4];
  const int t = threadIdx.x, lane = t & 63, wave = wave_index();
  const int l16 = lane & 15, h4 = lane >> 4;

  const int heads = a.B * a.Hk;
  const int head = blockIdx.x % heads, split = blockIdx.x / heads;
  const int b = head / a.Hk, g = head - b * a.Hk;
  const SequenceSpan span = sequence_span(a, b);
  const int rows = span.m * a.G;
  if (rows == 0) return;
  const int base_pos = span.n - span.m;
  const int lo_pos = base_pos, hi_pos = span.n - 1;
  const KeyTiles tiles = key_tiles<kFewKeys>(lo_pos, hi_pos, a.window, a.sinks);
  const int per = (tiles.count + a.splits - 1) / a.splits;
  const int it0 = split * per, it1 = min(tiles.count, it0 + per);

  // ---- this lane's query row, as the B operand of the depth steps
  const int row = min(l16, rows - 1), tok = row / a.G, hq = g * a.G + row - tok * a.G;
  const int p = base_pos + tok;
  const uint16_t* q = a.q + b * a.q_stride[0] + hq * a.q_stride[1] + tok * a.q_stride[2];
  u32x4_t qf[kSteps];
  float f = a.scale * kLog2e;
  float qsum[kGroups];  // KV4: f * the sums of q over each group's columns
  if constexpr (!KV4) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(q + 32 * s + 8 * h4);
  } else {
    // columns 64 g + 16 h4 .. + 15 of every group, scaled by a power of two so that the
    // row's largest magnitude lies in [2^9, 2^10); step (g, half): word r holds nibble r of
    // units 4 h4 + 2 half and the next, odd nibbles 2^-4 for their place in the byte
    float v[kGroups][16], mag = 0.f;
#pragma unroll
    for (int gg = 0; gg < kGroups; ++gg)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(q + 64 * gg + 16 * h4 + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[gg][8 * c + e] = to_f32<QDT>(uint16_t(w[e >> 1] >> (16 * (e & 1))));
          mag = fmaxf(mag, fabsf(v[gg][8 * c + e]));
        }
      }
    mag = fmaxf(mag, __shfl_xor(mag, 16, 64));
    mag = fmaxf(mag, __shfl_xor(mag, 32, 64));
    const int shift = mag > 0.f && mag < INFINITY ? 10 - __builtin_amdgcn_frexp_expf(mag) : 0;
    f = ldexpf(f, -shift);
#pragma unroll
    for (int gg = 0; gg < kGroups; ++gg) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        v[gg][e] = f16_bits_to_f32(f32_to_f16_bits(ldexpf(v[gg][e], shift)));
        sum += v[gg][e];
      }
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      qsum[gg] = sum * f;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float place = r & 1 ? 0.0625f : 1.f;
          qf[2 * gg + half][r] = f32x2_to_f16x2_bits(v[gg][8 * half + r] * place, v[gg][8 * half + 4 + r] * place);
        }
    }
    f = ldexpf(f, 24);  // the codes' 2^-24
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(qf[s]));  // the loads end before the loop

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
  struct Tile {
    u32x4_t k16[KV4 ? 1 : 2][KV4 ? 1 : kSteps];  // 16-bit: keys of the blocks u
    unsigned k[KV4 ? 2 : 1][KV4 ? D / 32 : 1];   // codes of the keys: this lane's quarter row
    unsigned v[8][kValueWords];                  // values of the keys 16 (e / 4) + 4 h4 + e % 4
    unsigned ks[KV4 ? 2 : 1][KV4 ? 4 : 1][kGroups], vs[KV4 ? 2 : 1][KV4 ? 4 : 1][kGroups];
  };
  auto fetch = [&](int it, Tile& x) __attribute__((always_inline)) {
    const int j0 = tiles.tile_index(it) * kFewKeys;
    const int live = min(span.n - j0, kFewKeys);  // keys past n read as zeros
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
#pragma unroll
        for (int r = 0; r < 4; r += (kGroups == 1 ? 4 : kGroups == 2 ? 2 : 1)) {
          const int at4 = (16 * u + 4 * h4 + r) * (kGroups * 4);
          const u32x4_t ws = load_b128(rks, at4, 0), wv = load_b128(rvs, at4, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x.ks[u][r + i / kGroups][i % kGroups] = ws[i];
            x.vs[u][r + i / kGroups][i % kGroups] = wv[i];
          }
        }
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

  f32x4_t o[kUnit];
#pragma unroll
  for (int i = 0; i < kUnit; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float omin[kGroups];  // KV4: sum p_j minimum_j, over this lane's keys
#pragma unroll
  for (int gg = 0; gg < kGroups; ++gg) omin[gg] = 0.f;
  float m = -INFINITY, m_use = 0.f, l = 0.f;

  auto half_of = [](unsigned w, int i) { return f16_bits_to_f32(uint16_t(i ? w >> 16 : w)); };

  auto compute = [&](Tile& x, int j0) __attribute__((always_inline)) {
    const bool whole = all_see(lo_pos, hi_pos, j0, j0 + kFewKeys, a.window, a.sinks);
    // ---- scores in log2 units: s[4 u + r] of key j0 + 16 u + 4 h4 + r
    float s[8], bound[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (!KV4) {
        f32x4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < kSteps; ++st) c = mfma16<CDT>(x.k16[u][st], qf[st], c);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * u + r] = c[r] * f;
      } else {
        float acc[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int gg = 0; gg < kGroups; ++gg) {
          f32x4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // words (unit, group): units 2 half and 2 half + 1 of this lane's four
            const int wa = 2 * half * kGroups + gg, wb = wa + kGroups;
            const unsigned ab =
                kGroups == 1 ? x.k[u][half]
                             : __builtin_amdgcn_perm(x.k[u][wb >> 1], x.k[u][wa >> 1], wa & 1 ? 0x07060302u : 0x05040100u);
            const unsigned hi = ab >> 8;
            c = mfma16<CDT>(u32x4_t{ab & 0x000f000fu, ab & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u},
                            qf[2 * gg + half], c);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            acc[r] = __builtin_fmaf(half_of(x.ks[u][r][gg], 0), c[r], acc[r]);
            low[r] = __builtin_fmaf(half_of(x.ks[u][r][gg], 1), qsum[gg], low[r]);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * u + r] = __builtin_fmaf(acc[r], f, low[r]);
      }
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!sees(p, j0 + 16 * (e >> 2) + 4 * h4 + (e & 3), a.window, a.sinks)) s[e] = -INFINITY;
    }
    // ---- running maximum
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bound[e] = s[e];
      if constexpr (KV4) {
        // the exponent of the key's largest value scale (2^-24 .. 2^12; a zero or NaN scale
        // keeps the bound finite too)
        unsigned big = 0;
#pragma unroll
        for (int gg = 0; gg < kGroups; ++gg) big = max(big, x.vs[e >> 2][e & 3][gg] & 0x7fffu);
        bound[e] += float(int(big >> 10) - 15);
      }
      top = fmaxf(top, bound[e]);
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__builtin_amdgcn_ballot_w64(top > m)) {
      const float before = m;
      m = fmaxf(m, top);
      m_use = m == -INFINITY ? 0.f : m;
      const float alpha = __builtin_amdgcn_exp2f(before - m_use);  // 0 before the first visible key
      l *= alpha;
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) omin[gg] *= alpha;
#pragma unroll
      for (int i = 0; i < kUnit; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] *= alpha;
    }
    float pr[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pr[e] = __builtin_amdgcn_exp2f(s[e] - m_use);
      l += pr[e];
    }
    // ---- O^T += V^T P^T
    if constexpr (!KV4) {
      u32x4_t pf;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float p0 = pr[e], p1 = pr[e + 1];
        pf[e / 2] = round_pair_bits<CDT>(p0, p1);
      }
      if (!whole) {
        // a hidden key's infinity or NaN must not meet its zero p: rows that see one take it
        // by hand (every lane reads the rows it needs again), then it counts as zero
        unsigned bad = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int c = 0; c < kValueWords; ++c) bad |= nonfinite_pair<CDT>(x.v[e][c]);
        if (__builtin_amdgcn_ballot_w64(bad != 0)) {
          for (int j = j0; j < min(j0 + kFewKeys, span.n); ++j) {
            if (!sees(p, j, a.window, a.sinks)) continue;
            const uint16_t* vr = vb + j * a.v_stride[2];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int i = 0; i < kUnit; ++i) {
                const uint16_t bits = vr[(4 * h4 + r) * kUnit + i];
                o[i][r] += nonfinite_pair<CDT>(bits) ? to_f32<CDT>(bits) : 0.f;
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
        o[i] = mfma16<CDT>(vf, pf, o[i]);
      }
    } else {
#pragma unroll
      for (int gg = 0; gg < kGroups; ++gg) {
        u32x4_t pf;
        float scaled[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned w = x.vs[e >> 2][e & 3][gg];
          scaled[e] = pr[e] * half_of(w, 0);
          float low = pr[e] * half_of(w, 1);
          if (!whole && pr[e] == 0.f) scaled[e] = low = 0.f;  // a hidden key's scale may be anything
          omin[gg] += low;
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) pf[e / 2] = f32x2_to_f16x2_bits(scaled[e], scaled[e + 1]);
        // this group's four columns of the chunk: nibble i of word gg
        unsigned ab[4], hi[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          ab[e / 2] = __builtin_amdgcn_perm(x.v[e + 1][gg >> 1], x.v[e][gg >> 1],
                                            gg & 1 ? 0x07060302u : 0x05040100u);
          hi[e / 2] = ab[e / 2] >> 8;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned mask = i & 1 ? 0x00f000f0u : 0x000f000fu;
          u32x4_t vf;
#pragma unroll
          for (int c = 0; c < 4; ++c) vf[c] = (i & 2 ? hi[c] : ab[c]) & mask;
          o[4 * gg + i] = mfma16<CDT>(vf, pf, o[4 * gg + i]);
        }
      }
    }
  };

  // every fourth tile, the next one's loads ahead of this one's products
  if constexpr (kAhead) {
    Tile cur, nxt;
    int it = it0 + wave;
    if (it < it1) fetch(it, cur);
    while (it < it1) {
      const int j0 = tiles.tile_index(it) * kFewKeys;
      it += 4;
      if (it < it1) fetch(it, nxt);
      compute(cur, j0);
      cur = nxt;
    }
  } else {
    Tile cur;
    for (int it = it0 + wave; it < it1; it += 4) {
      fetch(it, cur);
      compute(cur, tiles.tile_index(it) * kFewKeys);
    }
  }

  // ---- the four waves' joins: column of O^T row 4 h4 + r, index i
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if constexpr (KV4) {
#pragma unroll
    for (int gg = 0; gg < kGroups; ++gg) {
      omin[gg] += __shfl_xor(omin[gg], 16, 64);
      omin[gg] += __shfl_xor(omin[gg], 32, 64);
    }
  }
  if (h4 == 0) {
    red_ml[wave][0][l16] = m;
    red_ml[wave][1][l16] = l;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < kUnit; i += 4) {
      const int chunk = 4 * h4 + r;
      const int d = KV4 ? 16 * i + 4 * chunk : chunk * kUnit + i;  // KV4: group i / 4
      float4 w;
      if constexpr (KV4) {
        const float low = omin[i / 4];
        w = make_float4(__builtin_fmaf(o[i][r], 0x1p24f, low), __builtin_fmaf(o[i + 1][r], 0x1p20f, low),
                        __builtin_fmaf(o[i + 2][r], 0x1p24f, low), __builtin_fmaf(o[i + 3][r], 0x1p20f, low));
      } else {
        w = make_float4(o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]);
      }
      *reinterpret_cast<float4*>(&red_o[wave][l16][d]) = w;
    }
  __syncthreads();
  for (int at = t; at < rows * D; at += 256) {
    const int r = at / D, d = at % D;
    float mw[4], top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      mw[w] = red_ml[w][0][r];
      top = fmaxf(top, mw[w]);
    }
    float lsum = 0.f, osum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // a wave without a visible key has m = -inf and nothing to add, unless its sum is NaN
      const float c = mw[w] == top ? 1.f : __builtin_amdgcn_exp2f(mw[w] - top);
      lsum += c * red_ml[w][1][r];
      osum += c * red_o[w][r][d];
    }
    if (a.splits > 1) {
      const size_t slot = (size_t(head) * a.T * a.G + r) * a.splits + split;
      a.partial[slot * D + d] = osum;
      if (d == 0) {
        float* ml = a.partial + size_t(heads) * a.T * a.G * a.splits * D + slot * 2;
        ml[0] = top;
        ml[1] = lsum;
      }
    } else {
      const int tk = r / a.G;
      const float v = osum * softmax_inverse(lsum, base_pos + tk);
      a.out[b * a.out_stride[0] + (g * a.G + r - tk * a.G) * a.out_stride[1] + tk * a.out_stride[2] + d] =
          from_f32<QDT>(v);
    }
  }
}

template <int DT, int D, bool KV4>
void launch_attention_few(const CachedAttentionArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((attention_few_kernel<DT, D, KV4>), dim3(unsigned(a.B) * a.Hk * a.splits), dim3(256), 0, s, a);
}

}  // namespace fx
