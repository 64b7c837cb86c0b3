// sr_block_product.hip -- instantiations of the block-scaled product for one format of A (SR_A_E5M2).
#include "sr_block_scaled.h"
#include "sr_block_tables.h"

#ifndef SR_A_E5M2
#error "define SR_A_E5M2 as 0 or 1"
#endif

namespace sr {
namespace {

constexpr int FA = SR_A_E5M2 ? SR_E5M2 : SR_E4M3;

template <int FB, int MODE>
void fill(BlockProductKernels& k) {
  k.rows = reinterpret_cast<const void*>(&block_product_rows_kernel<MODE, FA, FB>);
  k.tile[kTile128][0] = reinterpret_cast<const void*>(&block_product_kernel<MODE, FA, FB, Tile128, false>);
  k.tile[kTile128][1] = reinterpret_cast<const void*>(&block_product_kernel<MODE, FA, FB, Tile128, true>);
  k.tile[kTile64][0] = reinterpret_cast<const void*>(&block_product_kernel<MODE, FA, FB, Tile64, false>);
  k.tile[kTile64][1] = reinterpret_cast<const void*>(&block_product_kernel<MODE, FA, FB, Tile64, true>);
  k.tile[kTile64x2][1] = reinterpret_cast<const void*>(&block_product_kernel<MODE, FA, FB, Tile64x2, true>);
  k.tile[kTile64x4][1] = reinterpret_cast<const void*>(&block_product_kernel<MODE, FA, FB, Tile64x4, true>);
}

template <int FB>
void fill_modes(BlockProductKernels (&k)[kProductModes]) {
  fill<FB, kExponents>(k[kExponents]);
  fill<FB, kFactors>(k[kFactors]);
  fill<FB, kWide>(k[kWide]);
}

}  // namespace

#if SR_A_E5M2
void register_block_product_e5m2(BlockProductTable& t) {
#else
void register_block_product_e4m3(BlockProductTable& t) {
#endif
  fill_modes<SR_E4M3>(t[SR_A_E5M2][0]);
  fill_modes<SR_E5M2>(t[SR_A_E5M2][1]);
}

}  // namespace sr
