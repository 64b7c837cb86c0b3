// sr_grouped_cast.hip -- instantiations of the casts of groups and stacks.
#include "sr_block_tables.h"
#include "sr_grouped.h"

namespace sr {
namespace {

template <int XE, int QE>
void fill(const void* (&k)[kGroupedCastKinds]) {
  k[kGroupedParts] = reinterpret_cast<const void*>(&grouped_cast_parts_kernel<XE, QE>);
  k[kGroupedWhole] = reinterpret_cast<const void*>(&grouped_cast_tile_kernel<XE, QE>);
  k[kStackedParts] = reinterpret_cast<const void*>(&stacked_cast_parts_kernel<XE, QE>);
  k[kStackedWhole] = reinterpret_cast<const void*>(&stacked_cast_tile_kernel<XE, QE, false>);
  k[kStackedSquare] = reinterpret_cast<const void*>(&stacked_cast_tile_kernel<XE, QE, true>);
}

template <int XE>
void fill_formats(const void* (&k)[4][kGroupedCastKinds]) {
  fill<XE, ENC_E4M3_RN>(k[0]);
  fill<XE, ENC_E4M3_SR>(k[1]);
  fill<XE, ENC_E5M2_RN>(k[2]);
  fill<XE, ENC_E5M2_SR>(k[3]);
}

}  // namespace

void register_grouped_cast(GroupedCastTable& t) {
  fill_formats<ENC_F32>(t[0]);
  fill_formats<ENC_BF16_RN>(t[1]);
  fill_formats<ENC_F16_RN>(t[2]);
}

}  // namespace sr
