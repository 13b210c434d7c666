// Products of 8-bit rows (int8_launch.h): the sums in whole numbers on the int8 matrix cores, exact
// in any order, the scales and the bias in fp32, one rounding.  Here: which kernel a product takes,
// and the join of K splits.
#include <algorithm>

#include "int8_gemm_few.h"
#include "int8_gemm_tile_launch.h"

namespace fx {
namespace {

// The sums of the K splits, scaled: 4 columns a thread.  Bound by the launch and the partial sums.
__global__ __launch_bounds__(256) void int8_gemm_join_kernel(const Int8GemmArgs g, int splits) {
  const unsigned quads = unsigned(g.N + 3) / 4;
  const unsigned unit = blockIdx.x * 256u + threadIdx.x;
  const int m = int(unit / quads), n = int(unit - unsigned(m) * quads) * 4;
  if (m >= g.M) return;
  const Columns4 columns = load_columns(g, n);
  const float sa = g.a_scales[m];
  const size_t plane = size_t(g.M) * g.N;
  const int* p = g.partial + size_t(m) * g.N + n;
  i32x4_t total = {0, 0, 0, 0};
  if (n + 4 <= g.N) {
    for (int s = 0; s < splits; ++s) {
      i32x4_t v;
      __builtin_memcpy(&v, p + s * plane, 16);
      total += v;
    }
  } else {
    for (int s = 0; s < splits; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < g.N) total[r] += p[s * plane + r];
  }
  store4(g, m, n, total, sa, columns);
}

// Rows at whatever address copied to whole 16 bytes at 16-byte boundaries, zeros behind them: those of
// the activations, then those of the weight (rows 0: none), a thread 16 bytes at a time.
__global__ __launch_bounds__(256) void int8_align_kernel(const Int8AlignArgs a) {
  const int pieces = a.width / 16;
  const long long first = (long long)(a.rows[0]) * pieces, all = first + (long long)(a.rows[1]) * pieces;
  for (long long unit = (long long)(blockIdx.x) * 256 + threadIdx.x; unit < all; unit += (long long)(gridDim.x) * 256) {
    const int which = unit >= first;
    const long long at = unit - (which ? first : 0), row = at / pieces;
    const int column = int(at - row * pieces) * 16;
    *reinterpret_cast<u32x4_t*>(a.to[which] + row * a.width + column) =
        part_b128(a.from[which] + row * a.stride[which] + column, a.columns - column);
  }
}

constexpr int kFewRows = 32;
constexpr int kMaxSplits = 16;

// Columns of a workgroup of the few-rows kernel.  From 17 rows on 32 of them share what is read of the
// activations, where one workgroup a compute unit would not do (24 rows by 6144 x 4096 10.9 us, with 16
// columns 13.6; 32 rows by 4096 x 4096 9.2 with 16 columns, with 32 11.3).
int few_columns(int M, int N) { return M > 16 && N > 4096 ? 32 : 16; }

}  // namespace

// Which kernel, and how many workgroups along K, by an estimate of the time (us).  Few rows: rounds of
// workgroups on a compute unit, each its rows of the weight (and some of the activations' from L2) at
// 26 bytes a ns, whether the other units are at work or not.  Tiles: rounds of workgroups, each its
// stages of 128 columns at what a stage takes, and the operands' bytes, of which the shorter hides but
// in part; for splits the join's launch and the partial sums written and read.  Fitted to 408 sizes (1
// to 4096 rows, 24 shapes of weights) timed with every tile and 1 to 16 splits: within 5% of the best
// measured choice at 386 of them (fitted to half of the weights, at 195 of the other 204).
//
// Rows at any address (`any`) skip the estimate where they are few: read in place, without K splits, 16
// bytes at a time (32 x 300 x 15999 87 us, where 16000 columns in K splits take 10).
Int8GemmPlan plan_int8_gemm(int M, int N, int K, bool any) {
  if (any && M <= kFewRows) return {kInt8Few, 1, K};
  const int stages = (K + 127) / 128;
  const float bytes = (float(M) + N) * K / 7.4e6f;
  Int8GemmPlan best{kInt8Few, 1, K};
  float least = 1e30f;
  if (M <= kFewRows) {
    const int columns = few_columns(M, N), rounds = N / (columns * 256) + (N % (columns * 256) != 0);
    least = 2.08f + rounds * (0.345f + K * (columns + 0.78f * M) / 26100.f);
  }
  // (32 rows fill half of the smallest tiles; the plan itself is then 0.2 us of a call, and 0.7 of a search)
  for (int tile = 0; tile < (M <= kFewRows ? 2 : kInt8Tiles); ++tile) {
    const Int8Tile& t = kInt8Tile[tile];
    const long tiles = long((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn), slots = 256 * t.places;
    for (int splits = 1; splits <= std::min(stages, kMaxSplits); ++splits) {
      if (splits > 1 && tiles * (splits - 1) >= slots) break;  // the chip was full
      const int per = (stages + splits - 1) / splits;
      if ((stages + per - 1) / per != splits) continue;  // a last split would be empty
      const long groups = tiles * splits, rounds = (groups + slots - 1) / slots;
      const float last = float(groups - (rounds - 1) * slots) / float(slots);
      // (a second workgroup on some compute unit already costs what one on each does)
      const float filled = last <= 0.5f ? 0.f : t.places > 1 ? 1.f : 2.f * last - 1.f;
      const float stage = (rounds - 1) * t.full + t.half + (t.full - t.half) * filled;
      const float work = per * stage + rounds * t.ends;
      float time = 1.25f + std::max(work, bytes) + 0.695f * std::min(work, bytes);
      if (splits > 1) time += 1.73f + 0.3f * splits + 2.f * splits * float(M) * N * 4.f / 7.6e6f;
      if (time < least) least = time, best = {tile, splits, splits == 1 ? K : per * 128};
    }
  }
  return best;
}

// A wave's pieces of 128 columns in flight: two, eight waves of them (2048 columns), so that few loads run
// past the last column; four where one pass of them is all and an eighth of it at most runs past.  One row
// by 24576 x K, with two and with four: K 2560 15.5 and 16.4 us, 3328 18.2 and 18.0, 3584 19.0 and 18.8, 4096
// 20.2 and 19.6, 5120 29.8 and 32.9, 6144 31.2 and 33.9, 8192 37.5 and 37.3 (two there: 4096 x 8192 8.3 and
// 8.7).  Sixteen waves where passes of 4096 columns come out even (one row by 4096 x 12288 11.9 us, with
// eight 12.5; by 4096 x 14336 13.7 and 13.1).
template <int XDT, bool ANY, int MT, int RT>
void launch_few(const Int8GemmArgs& g, const Int8RowsArgs& rows, hipStream_t s) {
  const dim3 grid(unsigned(g.N + 16 * RT - 1) / (16 * RT));
  if constexpr (MT == 1) {
    const int past = -g.K & 4095;
    if (g.K > 8192 && (XDT >= 0 || past <= g.K / 16)) {  // (rows quantized here: at most 16 columns a thread)
      hipLaunchKernelGGL((int8_gemm_few_kernel<XDT, ANY, 1, 1, 16, 2>), grid, dim3(1024), 0, s, g, rows);
      return;
    }
  }
  if (g.K > 3584 && g.K <= 4096) hipLaunchKernelGGL((int8_gemm_few_kernel<XDT, ANY, MT, RT, 8, 4>), grid, dim3(512), 0, s, g, rows);
  else hipLaunchKernelGGL((int8_gemm_few_kernel<XDT, ANY, MT, RT, 8, 2>), grid, dim3(512), 0, s, g, rows);
}

template <bool ANY>
void launch_few_rows(const Int8GemmArgs& g, hipStream_t s) {
  if (g.M <= 16) launch_few<-1, ANY, 1, 1>(g, {}, s);
  else if (few_columns(g.M, g.N) == 16) launch_few<-1, ANY, 2, 1>(g, {}, s);
  else launch_few<-1, ANY, 2, 2>(g, {}, s);
}

// Every workgroup quantizes the rows again, 1.5 us for each and each round of workgroups, where codes
// from a launch of their own cost 2 to 3 us (one row by 4096 x 4096 7.1 us for 8.2, by 1024 x 2000 5.4
// for 6.6, by 12288 x 1536 9.2 for 9.1, by 24576 x 4096 24.3 for 22.8; two rows by 1024 x 2000 6.6 for
// 6.7 and by 4096 x 4096 9.1 for 8.7, by 9728 x 896 11.4 for 9.8; four by 1024 x 2000 9.8 for 7.2).  Where
// the two are near, the rule takes the launch less: the host's part of it, 3 us, bounds such a call.  It
// costs the GPU most where several rounds of workgroups have few columns each (one row by 9728 x 896 8.6
// for 7.8).
bool int8_linear_fuses(int M, int N, int K) {
  return M <= 2 && long(M) * N <= 12288 && long(M) * K <= kFewCodes;
}

void launch_int8_linear_few(int x_dt, const Int8RowsArgs& rows, const Int8GemmArgs& g, hipStream_t s) {
  if (x_dt == kBF16) launch_few<kBF16, false, 1, 1>(g, rows, s);
  else launch_few<kF16, false, 1, 1>(g, rows, s);
}

bool launch_int8_gemm(const Int8GemmPlan& plan, const Int8GemmArgs& g, hipStream_t s) {
  if (plan.tile == kInt8Few) {
    if (g.any) launch_few_rows<true>(g, s);
    else launch_few_rows<false>(g, s);
    return true;
  }
  const Int8Tile& t = kInt8Tile[plan.tile];
  const long groups = long((g.M + t.bm - 1) / t.bm) * ((g.N + t.bn - 1) / t.bn) * plan.splits;
  if (groups >= 1L << 22) return false;  // a launch holds fewer than 2^32 threads
  t.launch(g, unsigned(groups), s);
  if (plan.splits > 1) {
    const unsigned long long units = (unsigned long long)(g.M) * ((g.N + 3) / 4);
    hipLaunchKernelGGL(int8_gemm_join_kernel, dim3(unsigned((units + 255) / 256)), dim3(256), 0, s, g, plan.splits);
  }
  return true;
}

void launch_int8_align(const Int8AlignArgs& a, hipStream_t s) {
  const long long units = (long long)(a.rows[0] + (long long)(a.rows[1])) * (a.width / 16);
  hipLaunchKernelGGL(int8_align_kernel, dim3(unsigned(std::min((units + 255) / 256, 16384LL))), dim3(256), 0, s, a);
}

}  // namespace fx
