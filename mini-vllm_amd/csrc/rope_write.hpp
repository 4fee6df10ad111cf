// Internal launch interface of the rotating append (not part of the C ABI).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mvllm {

struct RopeWriteParams {
  void* q_out;            // [tokens, hq, D]
  void* k_pool;           // [num_blocks, 1 << block_shift, hk, D]
  void* v_pool;
  float* k_scales;        // [num_blocks, hk], fp8 pools only
  float* v_scales;
  const void* q;          // row i of q, k, v at i stride elements, its heads contiguous
  const void* k;
  const void* v;
  const void* positions;  // [tokens]
  const float* cos_t;     // [max_positions, D]
  const float* sin_t;
  const int32_t* slots;   // [tokens]
  int64_t q_stride, k_stride, v_stride;
  int64_t num_blocks;
  int64_t max_positions;
  int tokens, hq, hk, block_shift;
};

// Whether launch_rope_write serves this (input, pool) type pair and head dim.
bool rope_write_supported(int dtype, int pool_dtype, int head_dim);

hipError_t launch_rope_write(const RopeWriteParams& p, int dtype, int pool_dtype, int head_dim,
                             int positions_bytes, hipStream_t stream);

}  // namespace mvllm
