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
// small one leaves them idle (128 KB of LDS for four: one workgroup a CU).  FP16
// triangles of 64 x 64 tiles without groups, with two and with four: 78 tiles of 12
// stages 6.1, 5.5, 5.7 us; 253 of 88 stages 43.8, 30.9, 26.4; 465 of 30 18.5, 15.2,
// 23.5; 528 of 32 19.5, 24.3, 30.8; up to six stages groups gain nothing (21
// tiles of 6: 4.4, 4.3, 4.8).  128 x 128 tiles against 64 x 64: 190 of them 28.1 and
// 23.8, 253 32.7 and 37.1.
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

struct GroupedProductKernels {
  const void* rows;                  // tiles of 16 rows
  const void* tile[kBlockTiles][2];  // as above
  const void* contract[kBlockTiles];
  const void* lean[2];               // rows and contract: kExponents only
};
using GroupedProductTable = GroupedProductKernels[2][2][3];
enum GroupedCastKind { kGroupedParts, kGroupedWhole, kStackedParts, kStackedWhole, kStackedSquare, kGroupedCastKinds };
using GroupedCastTable = const void* [3][4][kGroupedCastKinds];

void register_block_product_e4m3(BlockProductTable& t);
void register_block_product_e5m2(BlockProductTable& t);
void register_block_cast(BlockCastTable& t);
void register_grouped_product_e4m3(GroupedProductTable& t);
void register_grouped_product_e5m2(GroupedProductTable& t);
void register_grouped_cast(GroupedCastTable& t);

}  // namespace sr
