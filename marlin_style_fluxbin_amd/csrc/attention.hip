// Cached attention: the plan of a call, its dispatch, and the join of key splits.
#include <algorithm>

#include "attention_core.h"

namespace fx {

// The join of a row's key splits: o = sum_s w_s o_s / sum_s w_s l_s, w_s = 2^(m_s - max m).
// W waves a row (every wave forms the weights: lane s holds split s, splits <= 64), each
// with its share of at most N splits loaded at once; four rows (W = 1) or one a workgroup.
// Bound by the launch and one round trip: 64 splits of 32 rows 4.0 us, with one wave looping
// over them 17.7; many rows by the partials: 2 splits of 32768 rows of 128 columns 14 us.
template <int DT, int D, int N, int W>
__global__ __launch_bounds__(256) void attention_combine_kernel(const CachedAttentionArgs a) {
  constexpr int kRows = 4 / W, kCols = D / 64;
  typedef float cols_t __attribute__((ext_vector_type(kCols)));
  __shared__ float red[W > 1 ? W : 1][W > 1 ? D : 1];
  const int per_head = a.T * a.G, heads = a.B * a.Hk;
  const int tiles = (per_head + kRows - 1) / kRows;
  const int wave = wave_index(), lane = threadIdx.x & 63;
  const int head = blockIdx.x / tiles, part = wave % W;
  const int row = (blockIdx.x - head * tiles) * kRows + wave / W;
  const int b = head / a.Hk, g = head - b * a.Hk;
  const SequenceSpan span = sequence_span(a, b);
  if (row >= span.m * a.G) return;  // W > 1: the whole workgroup
  const size_t first = (size_t(head) * per_head + row) * a.splits;
  const float* ml = a.partial + size_t(heads) * per_head * a.splits * D + first * 2;
  const float* po = a.partial + first * D + lane * kCols;
  cols_t v[N];
#pragma unroll
  for (int i = 0; i < N; ++i)  // splits past the last: the last again, not counted below
    v[i] = *reinterpret_cast<const cols_t*>(po + size_t(min(part + W * i, a.splits - 1)) * D);
  const bool live = lane < a.splits;
  const float m = live ? ml[lane * 2] : -INFINITY, ls = live ? ml[lane * 2 + 1] : 0.f;
  const float top = wave_max(m);
  const float w = !live ? 0.f : m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
  const float l = wave_total(w * ls);
  float o[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) o[c] = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = part + W * i;
    const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), min(s, 63)));
#pragma unroll
    for (int c = 0; c < kCols; ++c)  // (a weight of 0 would make NaN of an infinity)
      o[c] = s < a.splits ? __builtin_fmaf(ws, v[i][c], o[c]) : o[c];
  }
  const int tok = row / a.G;
  const float inv = softmax_inverse(l, span.n - span.m + tok);
  uint16_t* out = a.out + b * a.out_stride[0] + (g * a.G + row - tok * a.G) * a.out_stride[1] +
                  tok * a.out_stride[2];
  if constexpr (W == 1) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) out[lane * kCols + c] = from_f32<DT>(o[c] * inv);
  } else {
#pragma unroll
    for (int c = 0; c < kCols; ++c) red[part][lane * kCols + c] = o[c];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < D) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) sum += red[i][d];
      out[d] = from_f32<DT>(sum * inv);
    }
  }
}

// How many splits of the keys: more shorten every workgroup's way until the chip is full, and
// cost the join's launch and the partial results, written and read.  The constants below (us)
// are fits; of 36 sizes measured with 1 .. 64 splits the choice is within 5% of the best at 30
// and within 17% at all.  Splits until the chip is full, whatever the join costs, take longer:
// 3 x 301 tokens of 14 heads of 64 columns, window 257, 19.1 us (2 splits) for 12.5 (1); 1000
// tokens of 32 heads over their own keys 36.7 (2) for 27.9 (1); 2 x 300 tokens of 16 heads of
// 256 columns over 2000 keys 86 (12) for 46 (3).
struct SplitTimes {
  long groups, tiles;  // workgroups of a split, key tiles
  int waves;           // of a workgroup along the keys
  int slots;           // workgroups that run at once, each at the speed of one alone
  float tile;          // a wave's key tile
  float shared;        // 0: further workgroups wait; else they run beside these, `slots` more in `shared` of their time
  float memory;        // reading the cache once
  float tail;          // how much of a workgroup's time is waited for at the end (no window: lengths that differ)
  float join, join_split;
};
// (the splits' time to *best)
int best_splits(const SplitTimes& t, long most, float* best) {
  int splits = 1;
  for (int s = 1; s <= most; s += s < 8 ? 1 : s < 16 ? 2 : s < 32 ? 4 : 8) {
    const float per = std::max(1.f, float(t.tiles) / float(s * t.waves));
    const long rounds = (t.groups * s + t.slots - 1) / t.slots;
    const float one = t.tile * per;
    const float work = one * (rounds == 1 ? 1.f : t.shared > 0.f ? t.shared * rounds : float(rounds));
    const float time = std::max(work, t.memory) + t.tail * one + (s > 1 ? t.join + t.join_split * s : 0.f) +
                       (s > 16 ? 1.5f : 0.f);  // the join's four-wave form
    if (s == 1 || time < *best) *best = time, splits = s;
    if (per == 1.f) break;
  }
  return splits;
}

// Which kernel: up to 16 query rows of a KV head fit one operand of the few-rows kernel.  A
// 4-bit cache keeps it for up to 64 rows (5 tokens of 7 heads over 4101 keys of 8 sequences
// of 4 KV heads: 20 us, the rows kernel 25 us on half as exact fp16 results), and always for
// fp16 queries: the rows kernel widens the cache to fp16, which a bf16 output does not show
// and an fp16 output does (error of the output 1.5 to 2 times its own rounding's).
//
// `wide`: workgroups of eight waves, 256 rows, in the rows kernel over a 4-bit cache, so that
// half as many of them widen a tile.  1024 tokens of 32 heads over 9000 keys 186 us (four
// waves 201), 4096 tokens of a prompt 169 (188); but 1024 tokens over a window of 1024 keys,
// where it leaves half the chip empty, 54 (39): taken where the estimate of the split times is
// smaller.
CachedAttentionPlan plan_with(bool wide, int dt, int B, int Hk, int G, int T, int L, int D, int window, int sinks,
                              bool kv4, float* time) {
  CachedAttentionPlan plan{};
  const long rows = long(T) * G, heads = long(B) * Hk;
  plan.few = rows <= 16 || (kv4 && (dt == kF16 || rows <= 64));
  const int kt = plan.few ? kFewKeys : rows_key_tile(D);
  plan.waves = wide ? 8 : 4;
  plan.row_blocks = plan.row_groups = 1;
  if (plan.few && rows > 16) {
    plan.waves = 8;
    plan.row_blocks = D <= 128 ? 2 : 1;
    while (plan.row_groups < plan.waves && plan.row_groups * plan.row_blocks * 16 < rows) plan.row_groups *= 2;
  }
  const long tile_rows = plan.few ? 16 * plan.row_blocks * plan.row_groups : 32 * plan.waves;
  plan.row_tiles = int((rows + tile_rows - 1) / tile_rows);
  // the most key tiles that a row tile can see
  const long tokens = std::min<long>(T, (tile_rows + G - 1) / G + 1);
  long keys = L;
  if (window > 0) keys = std::min<long>(L, long(sinks) + window + tokens - 1 + 2 * kt);
  const long tiles = (keys + kt - 1) / kt;
  const long groups = heads * plan.row_tiles;
  SplitTimes t{};
  t.groups = groups;
  t.tiles = tiles;
  t.waves = plan.few ? plan.waves / plan.row_groups : 1;
  t.join = 3.5f;
  t.join_split = float(heads * rows) * D * 8 / 4e6f;
  if (!plan.few) {
    t.tile = (D == 64 ? 1.f : 1.2f) * (kv4 ? 1.25f : 1.f) * (wide ? 1.5f : 1.f);
    t.slots = 256;
    t.shared = wide ? 0.f : 0.83f;
    t.join = 5.f;
  } else if (rows > 16) {
    t.tile = D == 64 ? 1.5f : 2.4f;
    t.slots = 256;
  } else {
    t.tile = D == 64 ? 0.65f : D == 128 ? 1.f : 2.f;
    t.slots = kv4 ? 768 : 512;
    t.memory = float(groups) * tiles * kFewKeys * D * (kv4 ? 1.125f : 4.f) / 4.8e6f;
    if (window == 0 || window > L / 2) t.tail = 0.25f;
  }
  // (workgroups beyond these gained nothing anywhere)
  const long target = !plan.few ? 1024 : rows > 16 ? 512 : kv4 ? 2048 : 1024;
  plan.splits = best_splits(t, std::min<long>((target + groups - 1) / groups, kMaxAttentionSplits), time);
  return plan;
}
CachedAttentionPlan plan_cached_attention(int dt, int B, int Hk, int G, int T, int L, int D, int window, int sinks,
                                          bool kv4) {
  float time = 0.f, wide_time = 0.f;
  const CachedAttentionPlan plan = plan_with(false, dt, B, Hk, G, T, L, D, window, sinks, kv4, &time);
  if (plan.few || !kv4 || D > 128) return plan;
  const CachedAttentionPlan wide = plan_with(true, dt, B, Hk, G, T, L, D, window, sinks, kv4, &wide_time);
  return wide_time < time ? wide : plan;
}

template <int DT, int D>
void launch_combine(const CachedAttentionArgs& a, hipStream_t s) {
  const unsigned rows = unsigned(a.T) * a.G, heads = unsigned(a.B) * a.Hk;
  if (a.splits <= 4)
    hipLaunchKernelGGL((attention_combine_kernel<DT, D, 4, 1>), dim3((rows + 3) / 4 * heads), dim3(256), 0, s, a);
  else if (a.splits <= 16)
    hipLaunchKernelGGL((attention_combine_kernel<DT, D, 16, 1>), dim3((rows + 3) / 4 * heads), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attention_combine_kernel<DT, D, kMaxAttentionSplits / 4, 4>), dim3(rows * heads), dim3(256), 0,
                       s, a);
}

template <int DT, int D>
void launch_for_dim(bool kv4, const CachedAttentionPlan& plan, const CachedAttentionArgs& a, hipStream_t s) {
  if (plan.few) {
    if (kv4) launch_attention_few<DT, D, true>(plan, a, s);
    else launch_attention_few<DT, D, false>(plan, a, s);
  } else if (!kv4) {
    launch_attention_rows<DT, D, false>(plan, a, s);
  } else if constexpr (DT == kBF16) {  // fp16 queries of a 4-bit cache always take the few-rows kernel
    launch_attention_rows<DT, D, true>(plan, a, s);
  }
  if (a.splits > 1) launch_combine<DT, D>(a, s);
}

template <int DT>
bool launch_for_type(int D, bool kv4, const CachedAttentionPlan& plan, const CachedAttentionArgs& a, hipStream_t s) {
  switch (D) {
    case 64: launch_for_dim<DT, 64>(kv4, plan, a, s); return true;
    case 128: launch_for_dim<DT, 128>(kv4, plan, a, s); return true;
    case 256: launch_for_dim<DT, 256>(kv4, plan, a, s); return true;
  }
  return false;
}

bool launch_cached_attention(int dt, int D, bool kv4, const CachedAttentionPlan& plan, const CachedAttentionArgs& a,
                             hipStream_t s) {
  if (dt == kBF16) return launch_for_type<kBF16>(D, kv4, plan, a, s);
  if (dt == kF16) return launch_for_type<kF16>(D, kv4, plan, a, s);
  return false;
}

}  // namespace fx
