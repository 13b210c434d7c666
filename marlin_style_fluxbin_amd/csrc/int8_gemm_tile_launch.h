// The tilings of int8_gemm_tile.h, each compiled in a unit of its own.
#pragma once
#include "int8_launch.h"

namespace fx {

void launch_int8_tile_64(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
void launch_int8_tile_64x128(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
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
// (of 300 x 4096 x 4096 the five take 13.9, 12.7, 15.0, 23.5 and 40.8 us, of 1024 x 4096 x 4096 28.8, 23.6, 21.4,
// 25.5 and 42.1, of 2048 x 4096 x 4096 54.8, 44.8, 42.2, 35.6 and 42.4; 128 x 128 with two stages, two
// workgroups a compute unit, 22.3, 24.3 and 36.7)
constexpr Int8Tile kInt8Tile[] = {
    {64, 64, 2, 0.19f, 0.389f, 1.91f, launch_int8_tile_64},
    {64, 128, 2, 0.33f, 0.645f, 2.31f, launch_int8_tile_64x128},
    {128, 128, 1, 0.39f, 0.409f, 2.97f, launch_int8_tile_128},
    {128, 256, 1, 0.68f, 0.775f, 3.76f, launch_int8_tile_128x256},
    {256, 256, 1, 1.21f, 1.5f, 4.68f, launch_int8_tile_256},
};
constexpr int kInt8Tiles = sizeof(kInt8Tile) / sizeof(kInt8Tile[0]);

}  // namespace fx
