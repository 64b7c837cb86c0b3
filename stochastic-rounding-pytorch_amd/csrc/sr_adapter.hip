// sr_adapter.hip -- instantiations of the adapters' kernels for one type (SR_TYPE: an sr_dtype's number).
#include "sr_adapter.h"
#include "sr_adapter_tables.h"

#ifndef SR_TYPE
#error "define SR_TYPE as 0 (FP32), 1 (BF16) or 2 (FP16)"
#endif

namespace sr {
namespace {

constexpr int XE = SR_TYPE == 0 ? ENC_F32 : (SR_TYPE == 1 ? ENC_BF16_RN : ENC_F16_RN);

template <int RC>
void fill(AdapterKernels& k, int at) {
  // A row's eight neighbouring columns where they are 16 bytes and their sums leave registers for the loads.
  constexpr int CJ = enc_bytes(XE) == 4 || RC == 8 ? 4 : 8;
  k.shrink[at] = reinterpret_cast<const void*>(&adapter_shrink_kernel<XE, RC>);
  k.expand[at][0] = reinterpret_cast<const void*>(&adapter_expand_kernel<XE, RC, 1, 1>);
  k.expand[at][1] = reinterpret_cast<const void*>(&adapter_expand_kernel<XE, RC, 4, kExpandTiles>);
  k.few[at] = reinterpret_cast<const void*>(&adapter_few_kernel<XE, RC>);
  k.contract[at] = reinterpret_cast<const void*>(&adapter_contract_kernel<XE, RC, CJ>);
  k.contract_columns[at] = 16 * CJ;
}

}  // namespace

#if SR_TYPE == 0
void register_adapters_f32(AdapterKernels& k) {
#elif SR_TYPE == 1
void register_adapters_bf16(AdapterKernels& k) {
#else
void register_adapters_f16(AdapterKernels& k) {
#endif
  fill<1>(k, 0);
  fill<2>(k, 1);
  fill<4>(k, 2);
  fill<8>(k, 3);
  k.finish = reinterpret_cast<const void*>(&adapter_finish_kernel<XE>);
  k.turn = reinterpret_cast<const void*>(&adapter_turn_kernel<enc_bytes(XE)>);
  k.step = kShrinkStep<XE>;
}

}  // namespace sr
