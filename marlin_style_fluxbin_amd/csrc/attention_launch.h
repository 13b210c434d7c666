// Launch plumbing of the cached attention (attention*.hip, attention_rows.h,
// attention_few.h) and of the 4-bit key/value cache (kv4.hip).
#pragma once
#include "common.h"

namespace fx {

// One call: B sequences, T query tokens each, Hq query heads over Hk key/value heads.
// Sequence b holds n = clamp(lengths[b], 0, L) keys, the last m = clamp(query_lengths[b], 0, T)
// of which are its queries' own positions: query t < m sits at p = n - m + t.
struct CachedAttentionArgs {
  const uint16_t* q;
  uint16_t* out;
  long long q_stride[3], out_stride[3];  // elements: batch, head, token
  // 16-bit cache: k, v and their strides (batch, head, position); 4-bit cache: the codes
  // [B, Hk, L, D / 2] and the (scale, minimum) pairs [B, Hk, L, D / 64, 2], contiguous
  const void* k;
  const void* v;
  long long k_stride[3], v_stride[3];
  const uint32_t* k_scales;
  const uint32_t* v_scales;
  const int* lengths;        // null: L for every sequence
  const int* query_lengths;  // null: T for every sequence
  float* partial;            // splits > 1: [rows, splits, D] outputs, then [rows, splits, 2] (max, sum)
  int B, Hk, G, T, L;        // G = Hq / Hk
  int window, sinks;         // window 0: none
  int splits, row_tiles, row_groups;  // row_groups: attention_few.h
  float scale;
};

// The kernel and split that a call takes, from its sizes alone.
struct CachedAttentionPlan {
  bool few;        // attention_few.h, else attention_rows.h
  int waves;       // of a workgroup (4, 8); each takes 32 rows in the rows kernel
  int row_blocks;  // few: 16-row blocks of a wave (1, 2),
  int row_groups;  //      waves of a workgroup along the rows; the others take other keys
  int row_tiles;   // workgroups along the T * G query rows of a KV head
  int splits;      // workgroups along the keys
};

constexpr int kFewKeys = 32;    // keys of a wave step of the few-rows kernel
constexpr int kMaxAttentionSplits = 64;
constexpr int rows_key_tile(int D) { return D == 256 ? 32 : 64; }

CachedAttentionPlan plan_cached_attention(int dt, int B, int Hk, int G, int T, int L, int D, int window, int sinks,
                                          bool kv4);
// dt: the type of q and out (and of a 16-bit cache)
bool launch_cached_attention(int dt, int D, bool kv4, const CachedAttentionPlan& plan, const CachedAttentionArgs& a,
                             hipStream_t s);

template <int DT, int D, bool KV4>
void launch_attention_rows(const CachedAttentionPlan& plan, const CachedAttentionArgs& a, hipStream_t s);
template <int DT, int D, bool KV4>
void launch_attention_few(const CachedAttentionPlan& plan, const CachedAttentionArgs& a, hipStream_t s);

// The 4-bit cache (format: kv4.hip).
struct Kv4AppendArgs {
  const uint16_t* x[2];         // k, v
  long long stride[2][3];       // elements: batch, head, token
  uint32_t* codes[2];
  uint32_t* scales[2];
  const int* start;             // null: start0 for every sequence
  const int* counts;            // null: T for every sequence
  int start0, B, Hk, T, L;
};
struct Kv4RestoreArgs {
  const uint32_t* codes[2];
  const uint32_t* scales[2];
  uint16_t* out[2];             // [B, Hk, rows, D] contiguous
  int B, Hk, L, rows;
};
bool launch_kv4_append(int dt, int D, const Kv4AppendArgs& a, hipStream_t s);
bool launch_kv4_restore(int dt, int D, const Kv4RestoreArgs& a, hipStream_t s);

}  // namespace fx
