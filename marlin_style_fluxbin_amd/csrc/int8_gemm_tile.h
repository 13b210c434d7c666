// Products of 8-bit rows, BM rows of the activations by BN of the weight a workgroup: both in LDS in
// a ring of S stages of 128 columns, filled from memory without passing through registers.
#pragma once
#include "int8_gemm.h"

namespace fx {

typedef int i32x16_t __attribute__((ext_vector_type(16)));
typedef unsigned u32x2v_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) char lds8_t;
typedef unsigned any16_t __attribute__((ext_vector_type(4), aligned(2)));

// D[i, j] += sum_k A[i, k] B[j, k] over 32 bytes of k: lane l gives bytes 16 (l / 32) .. of row
// l % 32 of both and holds D[8 (r / 4) + 4 (l / 32) + r % 4, l % 32], r < 16.
__device__ __forceinline__ i32x16_t mfma_i8_32(const u32x4_t& a, const u32x4_t& b, const i32x16_t& c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

// 16 bytes per lane from `resource` at the lane's offset and `column` to lds + at + 16 * lane,
// asynchronously (vmcnt).  The instruction has no result register; written as the builtin, every later
// LDS read of the kernel waits for it, whichever buffer it fills.
__device__ __forceinline__ void fill_lds(const u32x4_t& resource, int offset, int column, unsigned lds, int at) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds" ::"s"(lds), "i"(at),
               "v"(offset), "s"(resource), "s"(column)
               : "memory", "m0", "scc");
}

template <int N>
__device__ __forceinline__ void tile_wait() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void tile_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A wave's results to memory, 32 rows of them at a time through LDS of its own, so that eight lanes
// and more write a row's neighbours: written from the registers (8 bytes a lane and 32 rows at a time)
// the results of a 256 x 256 tile took 20 us.
// OUT: kBF16, kF16, kF32, or -1 for the sums of a K split.
// (w_scales, bias, a_scales: those of this wave's columns and rows, in LDS)
typedef const __attribute__((address_space(3))) float lds_float_t;
struct TileScales {
  lds_float_t *w_scales, *bias, *a_scales;
};
template <int OUT, int NT, int MT>
__device__ __forceinline__ void tile_store_as(const Int8GemmArgs& g, const i32x16_t (&acc)[NT][MT], int m0, int n0,
                                              int split, lds8_t* lds, int lane, const TileScales& scales) {
  constexpr int kSize = OUT == kBF16 || OUT == kF16 ? 2 : 4, kRow = NT * 32 * kSize + 16;
  constexpr int kLanes = NT * 32 * kSize / 16, kPass = 64 / kLanes;  // lanes of a row, rows of a wave store
  const int half = lane >> 5, low = lane & 31;
  char* out = OUT < 0 ? reinterpret_cast<char*>(g.partial + size_t(split) * g.M * g.N) : static_cast<char*>(g.out);
  const long long stride = OUT < 0 ? g.N : g.out_stride;
  f32x4v_t ws[NT * 4], bias[NT * 4];
  if constexpr (OUT >= 0) {
#pragma unroll
    for (int q = 0; q < NT * 4; ++q) {
      typedef const __attribute__((address_space(3))) f32x4v_t* lds128_t;
      ws[q] = *reinterpret_cast<lds128_t>(scales.w_scales + q * 8 + half * 4);
      bias[q] = *reinterpret_cast<lds128_t>(scales.bias + q * 8 + half * 4);
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = m0 + j * 32;
    const float sa = OUT < 0 ? 0.f : scales.a_scales[j * 32 + low];
    wave_lds_order();
#pragma unroll
    for (int q = 0; q < NT * 4; ++q) {
      lds8_t* at = lds + low * kRow + (q * 8 + half * 4) * kSize;
      const i32x16_t& v = acc[q / 4][j];
      const int r0 = (q & 3) * 4;
      if constexpr (OUT < 0) {
        *reinterpret_cast<__attribute__((address_space(3))) i32x4_t*>(at) = i32x4_t{v[r0], v[r0 + 1], v[r0 + 2], v[r0 + 3]};
      } else {
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = fmaf(float(v[r0 + r]) * sa, ws[q][r], bias[q][r]);
        if constexpr (OUT == kF32) {
          *reinterpret_cast<__attribute__((address_space(3))) f32x4v_t*>(at) = f32x4v_t{y[0], y[1], y[2], y[3]};
        } else {
          u32x2v_t p = {round_pair_bits<OUT>(y[0], y[1]), round_pair_bits<OUT>(y[2], y[3])};
          *reinterpret_cast<__attribute__((address_space(3))) u32x2v_t*>(at) = p;
        }
      }
    }
    wave_lds_order();
#pragma unroll
    for (int p = 0; p < 32 / kPass; ++p) {
      constexpr int kEach = 16 / kSize;
      const int row = p * kPass + lane / kLanes, col = lane % kLanes * kEach, left = g.N - n0 - col;
      if (m + row >= g.M || left <= 0) continue;
      const u32x4_t v = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(lds + row * kRow + col * kSize);
      char* to = out + ((m + row) * stride + n0 + col) * kSize;
      if (left >= kEach) {
        // at whatever address the row begins (301 x 1001 x 2000: element by element 1.8 us more); a result is
        // not read again here (8192 x 12288 x 4096 4% faster than with plain stores)
        if constexpr (OUT < 0) __builtin_memcpy(to, &v, 16);
        else __builtin_nontemporal_store(v, reinterpret_cast<any16_t*>(to));
      } else {
#pragma unroll
        for (int e = 0; e < kEach - 1; ++e) {
          if (e >= left) break;
          if constexpr (kSize == 2) reinterpret_cast<uint16_t*>(to)[e] = uint16_t(v[e >> 1] >> (16 * (e & 1)));
          else reinterpret_cast<unsigned*>(to)[e] = v[e];
        }
      }
    }
  }
}
template <int NT, int MT>
__device__ __forceinline__ void tile_store(const Int8GemmArgs& g, const i32x16_t (&acc)[NT][MT], int m0, int n0,
                                           int split, lds8_t* lds, int lane, const TileScales& scales) {
  if (g.partial) tile_store_as<-1>(g, acc, m0, n0, split, lds, lane, scales);
  else if (g.dt == kBF16) tile_store_as<kBF16>(g, acc, m0, n0, split, lds, lane, scales);
  else if (g.dt == kF16) tile_store_as<kF16>(g, acc, m0, n0, split, lds, lane, scales);
  else tile_store_as<kF32>(g, acc, m0, n0, split, lds, lane, scales);
}
constexpr int tile_store_bytes(int NT) { return 32 * (NT * 32 * 4 + 16); }  // of LDS, a wave

// A stage's rows are whole 128-byte lines: pieces of 64 bytes cost the L2 twice the requests (256 x 256
// tiles of 4096 x 4096 x 16384 with as many bytes in flight 243 us, 228 with 128).
constexpr int kTileK = 128;

// acc[n, m] += w a over the columns, a stage's four steps of 32 from LDS into registers during the
// products of the step before, one barrier a stage: behind it the stage that every wave has read makes
// room for the load of the one S ahead.
//
// What bounds it: of 8192 x 12288 x 4096 (256 x 256, 336 us, 2.4e15 operations a second; the library's
// int8 product takes 385) the matrix cores are busy 60% of the clocks, at 1.9 GHz, where the chip's
// power holds it (2.5 GHz with operands of zeros).  Without its loads 74%; with a third place in the
// ring for one operand 1% faster; with the next tile's first stages under a tile's results slower
// (registers).  Reads of LDS: 26% of the clocks, conflicts 5% of these.  With one wave a SIMD (64 x 64)
// a stage's time is its instructions, 4 clocks each: places in the ring are constants, and a scalar
// offset is all that a load adds up (64 x 4096 x 4096 8.7 us, with descriptors and places formed in
// every stage 10.8).
template <int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(WM* WN * 64) void int8_gemm_tile_kernel(const Int8GemmArgs g) {
  constexpr int kWaves = WM * WN, TM = BM / WM, TN = BN / WN, MT = TM / 32, NT = TN / 32;
  constexpr int kStage = (BM + BN) * kTileK, kRows = 1024 / kTileK, kPlaces = kTileK / 16, kSteps = kTileK / 32;
  constexpr int PW = BN / kRows / kWaves, PA = BM / kRows / kWaves, P = PW + PA;  // wave loads of kRows rows a stage
  static_assert(BN % (2 * kRows * kWaves) == 0 && BM % (2 * kRows * kWaves) == 0 && S >= 2, "waves share a stage's loads evenly");
  constexpr int kResults = kWaves * tile_store_bytes(NT);
  __shared__ __attribute__((aligned(1024))) char ring[S * kStage > kResults ? S * kStage : kResults];
  __shared__ __attribute__((aligned(16))) float side[2 * BN + BM];  // scales of the columns, their bias, scales of the rows
  const int lane = threadIdx.x & 63, wave = wave_index();
  const unsigned lds0 = unsigned(size_t((lds8_t*)ring));

  // the tile: those that one XCD runs at a time are neighbours, eight along M
  const int tiles_m = (g.M + BM - 1) / BM, tiles_n = (g.N + BN - 1) / BN, tiles = tiles_m * tiles_n;
  const int linear = xcd_local_index8(blockIdx.x, gridDim.x);
  const int split = linear / tiles, tile = linear - split * tiles;
  constexpr int kGroup = 8;
  const int group = tile / (kGroup * tiles_n), first = group * kGroup, high = min(kGroup, tiles_m - first);
  const int in_group = tile - group * kGroup * tiles_n;
  const int tn = in_group / high, tm = first + in_group - tn * high;
  const int m0 = tm * BM, n0 = tn * BN;
  const int k_begin = split * g.k_per_split, k_end = min(g.K, k_begin + g.k_per_split);
  const int stages = (k_end - k_begin + kTileK - 1) / kTileK;

  // Scales and bias, on the way during the products (loaded behind them 0.3 us more a workgroup).
  static_assert(WM * WN * 64 >= BN && WM * WN * 64 >= BM, "a thread has one of each");
  const int thread = threadIdx.x;
  float w_scale = 0.f, bias = 0.f, a_scale = 0.f;
  if (!g.partial) {
    w_scale = thread < BN ? g.w_scales[min(n0 + thread, g.N - 1)] : 0.f;
    a_scale = thread < BM ? g.a_scales[min(m0 + thread, g.M - 1)] : 0.f;
    if (g.bias && thread < BN) bias = bias_value(g, min(n0 + thread, g.N - 1));
  }

  // This wave's loads: kRows rows of kTileK bytes each, lane l bytes 16 c .. of row l / kPlaces, where it
  // fills place l % kPlaces: c is that place with swizzle(row) applied, so that 16 lanes that read one c
  // of 16 rows in a row meet 16 places of 16 bytes within 256 bytes (64 banks).
  const auto swizzle = [](int row) { return (row >> 1) & 7; };
  int chunk[2], w_off[PW], a_off[PA];
#pragma unroll
  for (int i = 0; i < 2; ++i) chunk[i] = ((lane % kPlaces) ^ swizzle(i * kRows + lane / kPlaces)) * 16;
  const int w_stride = int(g.w_stride), a_stride = int(g.a_stride);
#pragma unroll
  for (int i = 0; i < PW; ++i) w_off[i] = (i * kRows + lane / kPlaces) * w_stride + chunk[i & 1];
#pragma unroll
  for (int i = 0; i < PA; ++i) a_off[i] = (i * kRows + lane / kPlaces) * a_stride + chunk[i & 1];
  const int columns = k_end - k_begin;
  // A wave's range ends with the last of its rows that there are: no access behind it, zeros.  A wave
  // without any has the matrix's last row, so that every range holds more bytes than `column` below: a
  // lane within `chunk < there` is in bounds, and one behind the rows is not, whether the range check
  // counts `column` or not.
  const auto range = [&](const int8_t* p, long long stride, int first, int rows, int all) {
    const int row = min(first, all - 1), there = min(rows, all - row);
    const size_t at = reinterpret_cast<size_t>(p) + row * stride + k_begin;
    return u32x4_t{unsigned(at), unsigned(at >> 32) & 0xffffu, unsigned((there - 1) * int(stride) + columns), 0x00020000u};
  };
  const u32x4_t rw = range(g.w, g.w_stride, n0 + wave * (PW * kRows), PW * kRows, g.N);
  const u32x4_t ra = range(g.a, g.a_stride, m0 + wave * (PA * kRows), PA * kRows, g.M);
  const unsigned w_dst = lds0 + wave * (PW * 1024), a_dst = lds0 + BN * kTileK + wave * (PA * 1024);
  // The XCDs begin at different columns: they read the same rows at different times, and rows of a
  // power of two apart meet more of the memory's channels at any one (5% of the time in tiles of 256,
  // 11 to 17% in the others at 12288 columns and at 48 rows).
  int unissued = stages, column = int(blockIdx.x % kXcdCount) * stages / kXcdCount * kTileK;
  auto issue = [&](int slot) __attribute__((always_inline)) {
    // (the columns behind the last, and past the last stage: no access, zeros)
    const int left = columns - column, there = unissued > 0 ? left : 0;
#pragma unroll
    for (int i = 0; i < PW; ++i)
      fill_lds(rw, chunk[i & 1] < there ? w_off[i] : kOutOfRange, column, w_dst, slot * kStage + i * 1024);
#pragma unroll
    for (int i = 0; i < PA; ++i)
      fill_lds(ra, chunk[i & 1] < there ? a_off[i] : kOutOfRange, column, a_dst, slot * kStage + i * 1024);
    --unissued;
    column = left <= kTileK ? 0 : column + kTileK;
  };

  const int wm = wave / WN, wn = wave % WN;
  const int w_at = int(lds0) + (wn * TN + (lane & 31)) * kTileK, a_at = int(lds0) + (BN + wm * TM + (lane & 31)) * kTileK;
  const int place = ((lane >> 5) ^ swizzle(lane & 31)) * 16;

  i32x16_t acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  u32x4_t w[2][NT], a[2][MT];
  auto read = [&](int h, int step, int slot) __attribute__((always_inline)) {
    typedef const __attribute__((address_space(3))) u32x4_t* lds128_t;
    const int at = place ^ (step * 32), stage = slot * kStage;
#pragma unroll
    for (int i = 0; i < NT; ++i) w[h][i] = *reinterpret_cast<lds128_t>(w_at + at + (stage + i * 32 * kTileK));
#pragma unroll
    for (int j = 0; j < MT; ++j) a[h][j] = *reinterpret_cast<lds128_t>(a_at + at + (stage + j * 32 * kTileK));
    // (the compiler otherwise reads a step's operands just in front of its products)
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = mfma_i8_32(w[h][i], a[h][j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };

#pragma unroll
  for (int s = 0; s < S; ++s) issue(s);
  tile_wait<(S - 1) * P>();
  tile_barrier();
  read(0, 0, 0);
  for (int s = 0; s < stages;) {
#pragma unroll
    for (int slot = 0; slot < S; ++slot) {
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        if (t < kSteps - 1) {
          read((t + 1) & 1, t + 1, slot);
        } else {
          // this stage is in every wave's registers, and the next one is there
          tile_wait<(S - 2) * P>();
          tile_barrier();
          read(0, 0, (slot + 1) % S);
        }
        multiply(t & 1);
      }
      issue(slot);
      if (++s == stages) break;
    }
  }
  if (thread < BN) {
    side[thread] = w_scale;
    side[BN + thread] = bias;
  }
  if (thread < BM) side[2 * BN + thread] = a_scale;
  tile_wait<0>();  // nothing fills this workgroup's LDS after its last wave has left
  tile_barrier();  // nor does a wave read it any more
  lds_float_t* at = (lds_float_t*)side;
  tile_store(g, acc, m0 + wm * TM, n0 + wn * TN, split, (lds8_t*)ring + wave * tile_store_bytes(NT), lane,
             TileScales{at + wn * TN, at + BN + wn * TN, at + 2 * BN + wm * TM});
}

}  // namespace fx
