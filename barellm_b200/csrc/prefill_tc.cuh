// Tensor-core (tcgen05) paged prefill: shape support test and launcher.
#pragma once
#include "common.cuh"

namespace bl {

bool prefill_tc_supported(int32_t dtype, int64_t head_dim, int64_t block_size, int64_t hq, int64_t hkv);
// What comes with pools that are the expansion of an 8-bit cache (by the kernel before
// this one on the stream), on the device.
struct Expansion {
  const int32_t* row_order;  // the row that each blockIdx.z works on: a permutation of the batch
  const float* k_unit;       // fp16: [batch, num_kv_heads], K and V are these times what the pools hold (powers of two)
  const float* v_unit;
};
int prefill_tc_launch(const bl_prefill_args& a, cudaStream_t s, const Expansion* x = nullptr);

}  // namespace bl
