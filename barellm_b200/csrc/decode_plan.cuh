// Split-K work plan shared by the decode kernels (16/32-bit and 8-bit pools).
// One CTA lists the (row, chunk) units of a batch, full chunks first and then
// partial chunks by decreasing size (decode.cu, decode_plan_kernel).
#pragma once

#include "common.cuh"

namespace bl {

constexpr int kDecodeChunkTokens = 512;  // split-K chunk; fixed so results are batch-invariant
// The plan kernel stamps its header with this value and the batch size; the
// attention kernel runs a plan only when both match, so a workspace that holds
// no plan (or another batch's) yields an error word, not stray reads.
constexpr int32_t kDecodePlanMagic = 0x4e414c50;

struct DecodePlanArgs {
  const int32_t* seq_lens;
  int32_t batch, bs, chunk_blocks, bt_width, max_units;
  int32_t* hdr;       // [0] total units, [1] magic, [2] batch
  int32_t* row_base;  // [batch + 1]
  int2* exec;         // [max_units] (row, chunk)
  int32_t* err;
};

int launch_decode_plan(const DecodePlanArgs& p, cudaStream_t s);

}  // namespace bl
