// sr_block_cast.hip -- instantiations of the block-scaled cast.
#include "sr_block_scaled.h"
#include "sr_block_tables.h"

namespace sr {
namespace {

template <int XE, int QE>
void fill(const void* (&k)[kCastKinds]) {
  k[kCastParts] = reinterpret_cast<const void*>(&block_cast_parts_kernel<XE, QE>);
  k[kCastWhole] = reinterpret_cast<const void*>(&block_cast_tile_kernel<XE, QE, false>);
  k[kCastSquare] = reinterpret_cast<const void*>(&block_cast_tile_kernel<XE, QE, true>);
}

template <int XE>
void fill_formats(const void* (&k)[4][kCastKinds]) {
  fill<XE, ENC_E4M3_RN>(k[0]);
  fill<XE, ENC_E4M3_SR>(k[1]);
  fill<XE, ENC_E5M2_RN>(k[2]);
  fill<XE, ENC_E5M2_SR>(k[3]);
}

}  // namespace

void register_block_cast(BlockCastTable& t) {
  fill_formats<ENC_F32>(t[0]);
  fill_formats<ENC_BF16_RN>(t[1]);
  fill_formats<ENC_F16_RN>(t[2]);
}

}  // namespace sr
