#include "int8_gemm_tile.h"
#include "int8_gemm_tile_launch.h"

namespace fx {
void launch_int8_tile_64x128(const Int8GemmArgs& g, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((int8_gemm_tile_kernel<64, 128, 2, 2, 3>), dim3(groups), dim3(256), 0, s, g);
}
}  // namespace fx
