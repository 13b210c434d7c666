// Cached attention: the plan of a call, its dispatch, and the join of key splits.
#include <algorithm>

#include "attention_core.h"

namespace fx {

// grid: one wave per query row (row of all heads, four a workgroup).  o = sum_s w_s o_s /
// sum_s w_s l_s with w_s = 2^(m_s - max m) over the row's splits (<= 64: lane s forms w_s).
template <int DT, int D>
__global__ __launch_bounds__(256) void attention_combine_kernel(const CachedAttentionArgs a) {
  const int per_head = a.T * a.G, heads = a.B * a.Hk;
  const int tiles = (per_head + 3) / 4;
  const int head = blockIdx.x / tiles, lane = threadIdx.x & 63;
  const int row = (blockIdx.x - head * tiles) * 4 + wave_index();
  const int b = head / a.Hk, g = head - b * a.Hk;
  const SequenceSpan span = sequence_span(a, b);
  if (row >= span.m * a.G) return;
  const size_t first = (size_t(head) * per_head + row) * a.splits;
  const float* ml = a.partial + size_t(heads) * per_head * a.splits * D + first * 2;
  const bool live = lane < a.splits;
  const float m = live ? ml[lane * 2] : -INFINITY, ls = live ? ml[lane * 2 + 1] : 0.f;
  const float top = wave_max(m);
  const float w = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
  const float l = wave_total(live ? w * ls : 0.f);
  const float* po = a.partial + first * D + lane;
  constexpr int N = D / 64;
  float o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
    const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] += ws * po[size_t(s) * D + 64 * i];
  }
  const int tok = row / a.G;
  const float inv = softmax_inverse(l, span.n - span.m + tok);
  uint16_t* out = a.out + b * a.out_stride[0] + (g * a.G + row - tok * a.G) * a.out_stride[1] +
                  tok * a.out_stride[2] + lane;
#pragma unroll
  for (int i = 0; i < N; ++i) out[64 * i] = from_f32<DT>(o[i] * inv);
}

CachedAttentionPlan plan_cached_attention(int B, int Hk, int G, int T, int L, int D, int window, int sinks,
                                          bool kv4) {
  CachedAttentionPlan plan;
  const long rows = long(T) * G, heads = long(B) * Hk;
  plan.few = rows <= kFewRows;
  plan.row_tiles = plan.few ? 1 : int((rows + kRowsTile - 1) / kRowsTile);
  // the most key tiles that a row tile can see
  const long tokens = plan.few ? T : (kRowsTile + G - 1) / G + 1;
  long keys = L;
  const int kt = plan.few ? kFewKeys : rows_key_tile(D);
  if (window > 0) keys = std::min<long>(L, long(sinks) + window + std::min<long>(tokens, T) - 1 + 2 * kt);
  const long tiles = (keys + kt - 1) / kt;
  // enough workgroups for two (few rows: four) on each of the 256 CUs, each with at least a
  // tile for every wave (few rows) or four tiles (the first one's latency is not hidden)
  const long target = plan.few ? 1024 : 512;
  const long smallest = 4;
  const long groups = heads * plan.row_tiles;
  long splits = std::min((target + groups - 1) / groups, (tiles + smallest - 1) / smallest);
  plan.splits = int(std::max<long>(1, std::min<long>(splits, kMaxAttentionSplits)));
  return plan;
}

template <int DT, int D>
void launch_combine(const CachedAttentionArgs& a, hipStream_t s) {
  const unsigned tiles = (unsigned(a.T) * a.G + 3) / 4;
  hipLaunchKernelGGL((attention_combine_kernel<DT, D>), dim3(tiles * a.B * a.Hk), dim3(256), 0, s, a);
}

template <int DT, int D>
void launch_for_dim(bool kv4, bool few, const CachedAttentionArgs& a, hipStream_t s) {
  if (few) {
    if (kv4) launch_attention_few<DT, D, true>(a, s);
    else launch_attention_few<DT, D, false>(a, s);
  } else {
    if (kv4) launch_attention_rows<DT, D, true>(a, s);
    else launch_attention_rows<DT, D, false>(a, s);
  }
  if (a.splits > 1) launch_combine<DT, D>(a, s);
}

template <int DT>
bool launch_for_type(int D, bool kv4, bool few, const CachedAttentionArgs& a, hipStream_t s) {
  switch (D) {
    case 64: launch_for_dim<DT, 64>(kv4, few, a, s); return true;
    case 128: launch_for_dim<DT, 128>(kv4, few, a, s); return true;
    case 256: launch_for_dim<DT, 256>(kv4, few, a, s); return true;
  }
  return false;
}

bool launch_cached_attention(int dt, int D, bool kv4, bool few, const CachedAttentionArgs& a, hipStream_t s) {
  if (dt == kBF16) return launch_for_type<kBF16>(D, kv4, few, a, s);
  if (dt == kF16) return launch_for_type<kF16>(D, kv4, few, a, s);
  return false;
}

}  // namespace fx
