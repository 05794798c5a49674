// The tcgen05 prompt attention's launch, for the FP16 pool and for the 8-bit cache's values.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace pkv {

// Arguments checked by the caller; the query FP16 or, with query_fp32, FP32.  fine: over the
// 8-bit cache's values, behind the kernel that reads them (query_fp32 needs it).
int launch_prefill_attention_tc(const void *pool, int32_t num_blocks, int32_t layer, const void *query,
                                bool query_fp32, bool fine, int64_t query_stride, const int32_t *blocks,
                                int32_t start, int32_t tokens, void *out, int64_t out_stride, int32_t *error_flag,
                                cudaStream_t stream);

}  // namespace pkv
