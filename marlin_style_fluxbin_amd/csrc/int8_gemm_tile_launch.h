// The tilings of int8_gemm_tile.h, each compiled in a unit of its own.
#pragma once
#include "int8_launch.h"

namespace fx {

void launch_int8_tile_64(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
void launch_int8_tile_128(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
void launch_int8_tile_128x256(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
void launch_int8_tile_256(const Int8GemmArgs& g, unsigned groups, hipStream_t s);

// `places`: workgroups that share a compute unit.  Times in us, fits (plan_int8_gemm): a stage of 128
// columns with half the chip's places taken and with all of them; a workgroup's first loads and its
// results.
struct Int8Tile {
  int bm, bn, places;
  float half, full, ends;
  void (*launch)(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
};
// (of 2048 x 4096 x 4096 the four take 63, 43.7, 37.6 and 45.5 us; of 1024 x 4096 x 4096 34, 22.6, 32 and 44;
// 128 x 128 tiles with two stages, two workgroups a compute unit: 39.4 and 25.7)
constexpr Int8Tile kInt8Tile[] = {
    {64, 64, 2, 0.24f, 0.475f, 1.45f, launch_int8_tile_64},
    {128, 128, 1, 0.44f, 0.58f, 3.f, launch_int8_tile_128},
    {128, 256, 1, 0.755f, 0.9f, 3.95f, launch_int8_tile_128x256},
    {256, 256, 1, 1.335f, 1.57f, 5.3f, launch_int8_tile_256},
};
constexpr int kInt8Tiles = sizeof(kInt8Tile) / sizeof(kInt8Tile[0]);

}  // namespace fx
