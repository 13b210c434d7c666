// Rows of 8-bit codes with a scale each: a row p of values becomes code = round(127 p / a), ties to
// even, and scale = a / 127, a = max|p|.  p is a row as it is, its RMSNorm (after the residual's
// addition) or SiLU(gate) * up, so that no 16-bit copy of it is written and read again.
//
// Up to 16384 columns one pass: a row's values stay in registers between its maximum and its codes.  Bound
// by the bytes of the rows: the norm of 8192 rows of 4096 with the residual 44 us, 5.3 TB/s where a large
// copy reaches 4.7 (results stay in the memory-side cache), the SwiGLU of 4096 rows of 12288 50 us; one row
// 3 us, of which the launch is 2.
//
// Wider rows are formed in 64 bits and read twice (with a residual its sum too), bound by that arithmetic:
// 4096 rows of 18944 columns as they are 111 us, normalised with the residual 164, SwiGLU 328, where their
// bytes take 50, 117 and 83 at a copy's rate; one row 11, 14 and 24 us.
#include "int8_row.h"

namespace fx {
namespace {

// TPR threads a row.
template <int DT, int MODE, int TPR, int CH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void int8_rows_kernel(const Int8RowsArgs a) {
  constexpr int kBlock = TPR < 256 ? 256 : TPR;
  __shared__ double red[kBlock / 64];
  const int tl = threadIdx.x % TPR;
  const int row = int(blockIdx.x) * (kBlock / TPR) + (TPR < 256 ? wave_index() / (TPR / 64) : 0);
  if (row >= a.rows) return;  // a whole row's threads, at most a wave where several rows share a workgroup
  RowPointers p;
  p.x = a.x + row * a.x_stride;
  p.second = a.second ? a.second + row * a.second_stride : nullptr;
  p.sum = a.sum ? a.sum + row * a.sum_stride : nullptr;
  p.codes = a.codes + row * a.code_stride;
  quantize_row<DT, MODE, TPR, CH>(a, p, a.scales + row, tl, red);
}

template <int DT, int MODE>
void launch_rows(const Int8RowsArgs& a, hipStream_t s) {
  const int width = a.code_columns > a.columns ? a.code_columns : a.columns;
  const auto go = [&](auto kernel, int threads, int rows_per_block) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(a.rows + rows_per_block - 1) / rows_per_block), dim3(threads), 0, s, a);
  };
  // The fewest threads whose registers hold the row, eight columns a thread and chunk; wider ones have up
  // to four chunks rather than more threads, whose reductions cost more (norm of 8192 rows: 1024 columns
  // 14.2 us, with 256 threads 18.8; 8192 columns 85, with 1024 threads 91; 12288 columns 127 and 175,
  // 16384 columns 168 and 206; one row of 12288 5.1 and 5.8; SwiGLU of 8192 x 6144 38 us, with 512
  // threads 46).
  if (width <= 512) go(int8_rows_kernel<DT, MODE, 64, 1>, 256, 4);
  else if (width <= 1024) go(int8_rows_kernel<DT, MODE, 64, 2>, 256, 4);
  else if (width <= 2048) go(int8_rows_kernel<DT, MODE, 256, 1>, 256, 1);
  else if (width <= 4096) {
    // a row a compute unit: twice the threads (one row of 4096 columns 3.5 us for 3.9; 8192 rows 42.1 for 39.4)
    if (a.rows <= 256) go(int8_rows_kernel<DT, MODE, 512, 1>, 512, 1);
    else go(int8_rows_kernel<DT, MODE, 256, 2>, 256, 1);
  }
  else if (width <= 6144) go(int8_rows_kernel<DT, MODE, 256, 3>, 256, 1);
  else if (width <= 8192) go(int8_rows_kernel<DT, MODE, 512, 2>, 512, 1);
  else if (width <= 12288) go(int8_rows_kernel<DT, MODE, 512, 3>, 512, 1);
  else if (width <= 16384) go(int8_rows_kernel<DT, MODE, 512, 4>, 512, 1);
  else go(int8_rows_kernel<DT, MODE, 1024, 0>, 1024, 1);  // no registers: 4096 rows of 16384 SwiGLU 64 us, of 18944 328
}

// 16 codes a thread, at whatever address (int8_row.h).
template <int DT>
__global__ __launch_bounds__(256) void int8_restore_kernel(const Int8RestoreArgs a, int pieces) {
  const long long unit = (long long)(blockIdx.x) * 256 + threadIdx.x;
  const long long row = unit / pieces;
  if (row >= a.rows) return;
  const int first = int(unit - row * pieces) * 16, n = a.columns - first;
  const int8_t* src = a.codes + row * a.code_stride + first;
  const float scale = a.scales[row];
  constexpr int kSize = DT == kF32 ? 4 : 2;
  char* out = static_cast<char*>(a.out) + (row * a.out_stride + first) * kSize;
  if (n >= 16) {
    unsigned c[4];
    __builtin_memcpy(c, src, 16);
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = float(int(c[e >> 2] << (24 - 8 * (e & 3))) >> 24) * scale;
    if constexpr (DT == kF32) {
      __builtin_memcpy(out, v, 64);
    } else {
      unsigned o[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) o[w] = round_pair_bits<DT>(v[2 * w], v[2 * w + 1]);
      __builtin_memcpy(out, o, 32);
    }
    return;
  }
  for (int e = 0; e < n; ++e) {
    const float v = float(src[e]) * scale;
    if constexpr (DT == kF32) reinterpret_cast<float*>(out)[e] = v;
    else reinterpret_cast<uint16_t*>(out)[e] = from_f32<DT>(v);
  }
}

}  // namespace

bool launch_int8_rows(int dt, int mode, const Int8RowsArgs& a, hipStream_t s) {
  const auto pick = [&](auto type) {
    constexpr int DT = decltype(type)::value;
    if (mode == kRowsPlain) launch_rows<DT, kRowsPlain>(a, s);
    else if (mode == kRowsNorm) launch_rows<DT, kRowsNorm>(a, s);
    else launch_rows<DT, kRowsSwiglu>(a, s);
  };
  if (dt == kBF16) pick(std::integral_constant<int, kBF16>{});
  else if (dt == kF16) pick(std::integral_constant<int, kF16>{});
  else return false;
  return true;
}

bool launch_int8_restore(int dt, const Int8RestoreArgs& a, hipStream_t s) {
  const int pieces = (a.columns + 15) / 16;
  const dim3 grid(unsigned(((long long)(a.rows) * pieces + 255) / 256));
  if (dt == kBF16) hipLaunchKernelGGL(int8_restore_kernel<kBF16>, grid, dim3(256), 0, s, a, pieces);
  else if (dt == kF16) hipLaunchKernelGGL(int8_restore_kernel<kF16>, grid, dim3(256), 0, s, a, pieces);
  else if (dt == kF32) hipLaunchKernelGGL(int8_restore_kernel<kF32>, grid, dim3(256), 0, s, a, pieces);
  else return false;
  return true;
}

}  // namespace fx
