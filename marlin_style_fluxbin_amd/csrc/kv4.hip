// The 4-bit key/value cache: append (quantize) and restore (widen).
//
// Format, per sequence, KV head and position, for each group of 64 columns:
//   minimum = fp16(lo), scale = fp16(fp32(hi - lo) * fp32(1 / 15)),
//   code = clamp(round(fp32(fp32(x - minimum) * fp32(1 / scale))), 0, 15), ties to even
//   (scale 0: code 0), standing for code * scale + minimum,
// lo and hi the group's extremes; every step is one fp32 operation, so the codes are the
// same wherever they are formed.  A group that holds a value beyond 2^15 in magnitude (where
// code * scale + minimum could leave fp16), an infinity or a NaN stands for NaN: scale 0,
// minimum NaN (the attention sizes its running maximum by the scales).
// Codes: uint16 [16, D / 64] per position; word [c, g] holds columns 64 g + 4 c + k, k < 4,
// in bits 4 k .. 4 k + 3.  (scale, minimum) fp16 [D / 64, 2].  So a lane that holds one word
// of 16 neighbouring lanes' contiguous row has four columns of one group, and two words'
// nibbles are matrix operands after a mask (attention_few.h).
//
// Both kernels move bytes: eight lanes share a group, a lane eight of its columns, four rows
// a thread with their loads ahead.  32 x 32768 tokens of 8 heads of 128 columns append in 898
// us (6.1 TB/s; a large copy 4.8, it writes as much as it reads); 8192 tokens of one sequence
// 12.8 us, and restoring them 8.9 us, of which 2 are the launch.
#include "attention_launch.h"

namespace fx {

constexpr float kKv4Limit = 32768.f;

// rows (b, h, t), t fastest, of k (blockIdx.y 0) or v (1); D / 8 lanes a row, kRowsPerThread
// rows a thread with their loads ahead.
constexpr int kAppendRows = 4;
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_append_kernel(const Kv4AppendArgs a) {
  constexpr int kLanes = D / 8, kGroups = D / 64, kRows = 256 / kLanes;
  const int which = blockIdx.y, t = threadIdx.x;
  const uint16_t* x = a.x[which];
  uint32_t* codes = a.codes[which];
  uint32_t* scales = a.scales[which];
  const long long sb = a.stride[which][0], sh = a.stride[which][1], st = a.stride[which][2];
  const int lane = t % kLanes, g = lane / 8, y = lane % 8;
  const int head = blockIdx.x / ((a.T + kRows * kAppendRows - 1) / (kRows * kAppendRows));
  const int tile = blockIdx.x - head * ((a.T + kRows * kAppendRows - 1) / (kRows * kAppendRows));
  const int b = head / a.Hk;
  const int start = a.start ? a.start[b] : a.start0;
  const int count = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  const uint16_t* src = x + b * sb + (head - b * a.Hk) * sh + lane * 8;
  u32x4_t v[kAppendRows];
  bool live[kAppendRows];
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int tok = (tile * kAppendRows + i) * kRows + t / kLanes;
    const long long pos = (long long)start + tok;
    live[i] = tok < count && pos >= 0 && pos < a.L;
    if (live[i]) v[i] = *reinterpret_cast<const u32x4_t*>(src + tok * st);
  }
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int tok = (tile * kAppendRows + i) * kRows + t / kLanes;
    float f[8];
    float lo = INFINITY, hi = -INFINITY;
    bool odd = false;  // a value that the group cannot hold
    if (live[i]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = to_f32<DT>(uint16_t(v[i][e >> 1] >> (16 * (e & 1))));
        lo = fminf(lo, f[e]);
        hi = fmaxf(hi, f[e]);
        odd |= !(fabsf(f[e]) <= kKv4Limit);
      }
    }
    float bad = odd ? 1.f : 0.f;
    // the eight lanes of a group
    lo = fminf(lo, dpp_move<kDppXor1>(lo));
    hi = fmaxf(hi, dpp_move<kDppXor1>(hi));
    bad = fmaxf(bad, dpp_move<kDppXor1>(bad));
    lo = fminf(lo, dpp_move<kDppXor2>(lo));
    hi = fmaxf(hi, dpp_move<kDppXor2>(hi));
    bad = fmaxf(bad, dpp_move<kDppXor2>(bad));
    lo = fminf(lo, dpp_move<kDppHalfMirror>(lo));
    hi = fmaxf(hi, dpp_move<kDppHalfMirror>(hi));
    bad = fmaxf(bad, dpp_move<kDppHalfMirror>(bad));
    const uint16_t min_bits = f32_to_f16_bits(lo), scale_bits = f32_to_f16_bits((hi - lo) * (1.f / 15.f));
    const float minimum = f16_bits_to_f32(min_bits), scale = f16_bits_to_f32(scale_bits);
    const float inverse = scale > 0.f ? 1.f / scale : 0.f;
    unsigned words = 0;  // units 2 y (low half) and 2 y + 1 of group g
    if (live[i]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float c = rintf((f[e] - minimum) * inverse);
        words |= unsigned(int(fminf(fmaxf(c, 0.f), 15.f))) << (4 * e);
      }
    }
    const unsigned stored = bad > 0.f ? 0x7e000000u : unsigned(scale_bits) | unsigned(min_bits) << 16;
    // a unit's words of neighbouring groups share a dword: trade with the other group's lane
    unsigned dword = words;
    int at = y;
    if constexpr (kGroups > 1) {
      const unsigned other = unsigned(__shfl_xor(int(words), 8, 64));
      dword = g & 1 ? (other >> 16) | (words & 0xffff0000u) : (words & 0xffffu) | (other << 16);
      at = (2 * y + (g & 1)) * (kGroups / 2) + g / 2;
    }
    if (live[i]) {
      const size_t row = size_t(head) * a.L + size_t((long long)start + tok);
      codes[row * (D / 8) + at] = dword;
      if (y == 0) scales[row * kGroups + g] = stored;
    }
  }
}

// [B, Hk, rows, D] 16-bit values of the first `rows` positions; a lane widens the eight
// columns 64 g + 8 y .. of a row.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_restore_kernel(const Kv4RestoreArgs a) {
  constexpr int kLanes = D / 8, kGroups = D / 64, kRows = 256 / kLanes;
  const int which = blockIdx.y, t = threadIdx.x;
  const uint32_t* codes = a.codes[which];
  const uint32_t* scales = a.scales[which];
  uint16_t* out = a.out[which];
  const int lane = t % kLanes, g = lane / 8, y = lane % 8;
  const int tiles = (a.rows + kRows * kAppendRows - 1) / (kRows * kAppendRows);
  const int head = blockIdx.x / tiles, tile = blockIdx.x - head * tiles;
  unsigned words[kAppendRows], pair[kAppendRows];
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int pos = min((tile * kAppendRows + i) * kRows + t / kLanes, a.rows - 1);
    const size_t row = size_t(head) * a.L + pos;
    const uint32_t* c = codes + row * (D / 8);
    if constexpr (kGroups == 1) {
      words[i] = c[y];
    } else {
      const unsigned u0 = c[2 * y * (kGroups / 2) + g / 2], u1 = c[(2 * y + 1) * (kGroups / 2) + g / 2];
      words[i] = g & 1 ? (u0 >> 16) | (u1 & 0xffff0000u) : (u0 & 0xffffu) | (u1 << 16);
    }
    pair[i] = scales[row * kGroups + g];
  }
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int pos = (tile * kAppendRows + i) * kRows + t / kLanes;
    if (pos >= a.rows) continue;
    const float scale = f16_bits_to_f32(uint16_t(pair[i])), minimum = f16_bits_to_f32(uint16_t(pair[i] >> 16));
    u32x4_t w;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      // code * scale is exact in fp32
      float v0 = __builtin_fmaf(float((words[i] >> (4 * e)) & 15u), scale, minimum);
      float v1 = __builtin_fmaf(float((words[i] >> (4 * e + 4)) & 15u), scale, minimum);
      w[e / 2] = round_pair_bits<DT>(v0, v1);
    }
    *reinterpret_cast<u32x4_t*>(out + (size_t(head) * a.rows + pos) * D + lane * 8) = w;
  }
}

template <int DT, int D>
void append_launch(const Kv4AppendArgs& a, hipStream_t s) {
  constexpr int kRows = 256 / (D / 8) * kAppendRows;
  const unsigned tiles = (unsigned(a.T) + kRows - 1) / kRows;
  hipLaunchKernelGGL((kv4_append_kernel<DT, D>), dim3(tiles * a.B * a.Hk, 2), dim3(256), 0, s, a);
}
template <int DT, int D>
void restore_launch(const Kv4RestoreArgs& a, hipStream_t s) {
  constexpr int kRows = 256 / (D / 8) * kAppendRows;
  const unsigned tiles = (unsigned(a.rows) + kRows - 1) / kRows;
  hipLaunchKernelGGL((kv4_restore_kernel<DT, D>), dim3(tiles * a.B * a.Hk, 2), dim3(256), 0, s, a);
}

bool launch_kv4_append(int dt, int D, const Kv4AppendArgs& a, hipStream_t s) {
  const bool bf = dt == kBF16;
  switch (D) {
    case 64: bf ? append_launch<kBF16, 64>(a, s) : append_launch<kF16, 64>(a, s); return true;
    case 128: bf ? append_launch<kBF16, 128>(a, s) : append_launch<kF16, 128>(a, s); return true;
    case 256: bf ? append_launch<kBF16, 256>(a, s) : append_launch<kF16, 256>(a, s); return true;
  }
  return false;
}
bool launch_kv4_restore(int dt, int D, const Kv4RestoreArgs& a, hipStream_t s) {
  const bool bf = dt == kBF16;
  switch (D) {
    case 64: bf ? restore_launch<kBF16, 64>(a, s) : restore_launch<kF16, 64>(a, s); return true;
    case 128: bf ? restore_launch<kBF16, 128>(a, s) : restore_launch<kF16, 128>(a, s); return true;
    case 256: bf ? restore_launch<kBF16, 256>(a, s) : restore_launch<kF16, 256>(a, s); return true;
  }
  return false;
}

}  // namespace fx
