// sr_adapter_tables.h -- kernels of the adapters by type and rank.
#pragma once

namespace sr {

constexpr int kAdapterRanks = 4;  // up to 16, 32, 64 and 128 ranks
constexpr int kExpandTiles = 4;   // times 16 rows of a workgroup of expand whose waves take 64 columns; else 1 and 16

struct AdapterKernels {
  const void* shrink[kAdapterRanks];
  const void* expand[kAdapterRanks][2];  // [.][1]: 64 columns a wave
  const void* few[kAdapterRanks];        // shrink and expand in one, for few rows
  const void* contract[kAdapterRanks];
  int contract_columns[kAdapterRanks];   // of a workgroup
  const void* finish;
  const void* turn;
  int step;  // values of the contracted axis that a wave of shrink takes at once
};
// [FP32, BF16, FP16]
using AdapterTable = AdapterKernels[3];

void register_adapters_f32(AdapterKernels& k);
void register_adapters_bf16(AdapterKernels& k);
void register_adapters_f16(AdapterKernels& k);

}  // namespace sr
