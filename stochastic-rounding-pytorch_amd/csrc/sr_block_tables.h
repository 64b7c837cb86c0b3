// sr_block_tables.h -- kernels of the block-scaled operators by format, and their tile shapes.
#pragma once

#include <cstdint>

#include "sr_tile_product.h"

namespace sr {

using Tile128 = TileShape<128, 128, 2, 2>;
using Tile64 = TileShape<64, 64, 2, 2>;
using Tile64x2 = TileShape<64, 64, 2, 2, 2>;
using Tile64x4 = TileShape<64, 64, 2, 2, 4>;
enum BlockTile { kTile128, kTile64, kTile64x2, kTile64x4, kBlockTiles };

// The tile of a launch that has tiles(side) tiles of side x side: the larger
// one where it gives the chip's 256 CUs work, and groups of waves where the
// small one leaves them idle (128 KB of LDS for four: one workgroup a CU).
template <class Count>
inline BlockTile tile_by_count(Count&& tiles) {
  if (tiles(128) >= 256) return kTile128;
  const int64_t small = tiles(64);
  return small > 512 ? kTile64 : (small > 256 ? kTile64x2 : kTile64x4);
}

struct BlockProductKernels {
  const void* rows;                  // at most 16 rows of A
  const void* tile[kBlockTiles][2];  // [shape][rows aligned to 16 bytes]; nullptr for groups with unaligned rows
};
// [A is E5M2][B is E5M2][ProductMode]
using BlockProductTable = BlockProductKernels[2][2][3];
enum BlockCastKind { kCastParts, kCastWhole, kCastSquare, kCastKinds };
// [FP32, BF16, FP16 input][E4M3 nearest, stochastic, E5M2 nearest, stochastic][kind]
using BlockCastTable = const void* [3][4][kCastKinds];

void register_block_product_e4m3(BlockProductTable& t);
void register_block_product_e5m2(BlockProductTable& t);
void register_block_cast(BlockCastTable& t);

}  // namespace sr
