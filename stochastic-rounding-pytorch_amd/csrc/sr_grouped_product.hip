// sr_grouped_product.hip -- instantiations of the grouped products for one format of A (SR_A_E5M2).
#include "sr_block_tables.h"
#include "sr_grouped.h"

#ifndef SR_A_E5M2
#error "define SR_A_E5M2 as 0 or 1"
#endif

namespace sr {
namespace {

constexpr int FA = SR_A_E5M2 ? SR_E5M2 : SR_E4M3;

template <int FB, int MODE, class S>
void fill_tile(GroupedProductKernels& k, BlockTile tile) {
  if constexpr (S::kGroups == 1) k.tile[tile][0] = reinterpret_cast<const void*>(&grouped_product_kernel<MODE, FA, FB, S, false>);
  k.tile[tile][1] = reinterpret_cast<const void*>(&grouped_product_kernel<MODE, FA, FB, S, true>);
  k.contract[tile] = reinterpret_cast<const void*>(&grouped_contract_kernel<MODE, FA, FB, S, true>);
}

template <int FB, int MODE>
void fill(GroupedProductKernels& k) {
  k.rows = reinterpret_cast<const void*>(&grouped_product_rows_kernel<MODE, FA, FB>);
  fill_tile<FB, MODE, Tile128>(k, kTile128);
  fill_tile<FB, MODE, Tile64>(k, kTile64);
  fill_tile<FB, MODE, Tile64x2>(k, kTile64x2);
  fill_tile<FB, MODE, Tile64x4>(k, kTile64x4);
}

template <int FB>
void fill_modes(GroupedProductKernels (&k)[kProductModes]) {
  fill<FB, kExponents>(k[kExponents]);
  k[kExponents].lean[0] = reinterpret_cast<const void*>(&grouped_lean_kernel<FA, FB, false>);
  k[kExponents].lean[1] = reinterpret_cast<const void*>(&grouped_lean_kernel<FA, FB, true>);
  fill<FB, kFactors>(k[kFactors]);
  fill<FB, kWide>(k[kWide]);
}

}  // namespace

#if SR_A_E5M2
void register_grouped_product_e5m2(GroupedProductTable& t) {
#else
void register_grouped_product_e4m3(GroupedProductTable& t) {
#endif
  fill_modes<SR_E4M3>(t[SR_A_E5M2][0]);
  fill_modes<SR_E5M2>(t[SR_A_E5M2][1]);
}

}  // namespace sr
