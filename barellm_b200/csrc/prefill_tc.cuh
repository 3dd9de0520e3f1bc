// Tensor-core (tcgen05) paged prefill: shape support test and launcher.
#pragma once
#include "common.cuh"

namespace bl {

bool prefill_tc_supported(int32_t dtype, int64_t head_dim, int64_t block_size, int64_t hq, int64_t hkv);
// row_order: for the expansion of an 8-bit cache (the kernel before this one on the
// stream), the row that each blockIdx.z works on, a permutation of the batch on the
// device; else null.
int prefill_tc_launch(const bl_prefill_args& a, cudaStream_t s, const int32_t* row_order = nullptr);

}  // namespace bl
