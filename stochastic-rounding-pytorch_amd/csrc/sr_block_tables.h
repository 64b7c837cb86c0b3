// sr_block_tables.h -- kernels of the block-scaled operators by format, and their tile shapes.
#pragma once

#include "sr_tile_product.h"

namespace sr {

using Tile128 = TileShape<128, 128, 2, 2>;
using Tile64 = TileShape<64, 64, 2, 2>;
enum BlockTile { kTile128, kTile64, kBlockTiles };

struct BlockProductKernels {
  const void* rows;                  // at most 16 rows of A
  const void* tile[kBlockTiles][2];  // [shape][rows aligned to 16 bytes]
};
// [A is E5M2][B is E5M2][ProductMode]
using BlockProductTable = BlockProductKernels[2][2][3];
// [FP32, BF16, FP16 input][E4M3 nearest, stochastic, E5M2 nearest, stochastic][square]
using BlockCastTable = const void* [3][4][2];

void register_block_product_e4m3(BlockProductTable& t);
void register_block_product_e5m2(BlockProductTable& t);
void register_block_cast(BlockCastTable& t);

}  // namespace sr
