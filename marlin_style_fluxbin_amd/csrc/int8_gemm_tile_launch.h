// The tilings of int8_gemm_tile.h, each compiled in a unit of its own.
#pragma once
#include "int8_launch.h"

namespace fx {

void launch_int8_tile_64(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
void launch_int8_tile_128(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
void launch_int8_tile_128_deep(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
void launch_int8_tile_256(const Int8GemmArgs& g, unsigned groups, hipStream_t s);

// Times in us, fits (plan_int8_gemm): a stage of 128 columns with one workgroup on its compute unit,
// with `places` of them; a workgroup's first loads and its results.
struct Int8Tile {
  int bm, bn, places;
  float alone, full, ends;
  void (*launch)(const Int8GemmArgs& g, unsigned groups, hipStream_t s);
};
constexpr Int8Tile kInt8Tile[] = {
    {64, 64, 2, 0.27f, 0.45f, 1.5f, launch_int8_tile_64},
    {128, 128, 2, 0.75f, 1.15f, 3.f, launch_int8_tile_128},
    {128, 128, 1, 0.58f, 0.58f, 3.f, launch_int8_tile_128_deep},
    {256, 256, 1, 1.55f, 1.55f, 8.f, launch_int8_tile_256},
};
constexpr int kInt8Tiles = sizeof(kInt8Tile) / sizeof(kInt8Tile[0]);
constexpr int kInt8Few = -1;  // int8_gemm_few.h

}  // namespace fx
