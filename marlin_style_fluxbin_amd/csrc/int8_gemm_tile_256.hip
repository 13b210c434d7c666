#include "int8_gemm_tile.h"
#include "int8_gemm_tile_launch.h"

namespace fx {
void launch_int8_tile_256(const Int8GemmArgs& g, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((int8_gemm_tile_kernel<256, 256, 2, 4, 2>), dim3(groups), dim3(512), 0, s, g);
}
}  // namespace fx
