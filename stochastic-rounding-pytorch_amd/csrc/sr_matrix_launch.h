// sr_matrix_launch.h -- argument checks and the launch that the matrix operators' entry points share.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/sr_matrix_hip.h"
#include "sr_error.h"

namespace sr {

constexpr int64_t kMaxRows = 0x7FFFFFFF - 256;  // row indices of a tile stay in 32 bits
constexpr int64_t kMaxLd = 1 << 24, kMaxScaleLd = 1 << 20;

inline int launch(const void* fn, uint64_t groups, int threads, void* arg, void* stream) {
  if (groups > 0x7FFFFFu) return fail(SR_ERR_ARGUMENT, "%llu workgroups exceed a launch", (unsigned long long)groups);
  void* args[] = {arg};
  const hipError_t err = hipLaunchKernel(fn, dim3(static_cast<uint32_t>(groups)), dim3(threads), args, 0,
                                         static_cast<hipStream_t>(stream));
  return err == hipSuccess ? SR_OK : hip_fail(err, "hipLaunchKernel");
}

inline int64_t blocks(int64_t n) { return (n + SR_BLOCK - 1) / SR_BLOCK; }

inline int check_matrix(const sr_block_matrix* x, const char* name, int64_t k) {
  if (!x) return fail(SR_ERR_ARGUMENT, "null argument");
  if (x->dtype != SR_E4M3 && x->dtype != SR_E5M2) return fail(SR_ERR_ARGUMENT, "%s must be E4M3 or E5M2", name);
  if (x->scale_type != SR_SCALE_E8M0 && x->scale_type != SR_SCALE_F32)
    return fail(SR_ERR_ARGUMENT, "%s: unknown scale type %d", name, x->scale_type);
  if (x->block_rows != 1 && x->block_rows != SR_BLOCK)
    return fail(SR_ERR_ARGUMENT, "%s: scales cover 1 or %d rows, not %d", name, SR_BLOCK, x->block_rows);
  if (x->rows < 0 || x->rows > kMaxRows) return fail(SR_ERR_ARGUMENT, "%s: %lld rows", name, (long long)x->rows);
  if (x->ld > kMaxLd || (x->rows > 1 && x->ld < k))
    return fail(SR_ERR_ARGUMENT, "%s: %lld bytes between rows of %lld", name, (long long)x->ld, (long long)k);
  if (x->ld_scale > kMaxScaleLd || x->ld_scale < 0)
    return fail(SR_ERR_ARGUMENT, "%s: %lld scales between rows", name, (long long)x->ld_scale);
  if (x->rows && k && (!x->data || !x->scale)) return fail(SR_ERR_ARGUMENT, "%s: null pointer", name);
  return SR_OK;
}

inline bool aligned_rows(const sr_block_matrix* x) {
  return reinterpret_cast<uintptr_t>(x->data) % 16 == 0 && x->ld % 16 == 0;
}

}  // namespace sr
