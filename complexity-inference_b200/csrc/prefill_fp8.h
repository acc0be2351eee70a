// Arguments of the 8-bit cache's prefill kernels (mma.sync and tensor-memory).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace muk {

struct PrefillFp8Args {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int bt_stride;
  const int32_t* seq_lens;
  const int32_t* cu_q;
  int num_q_heads, num_kv_heads, num_blocks;
  int num_rows, max_q_len, max_blocks;
  float scale_log2;
  int splits;  // CTAs of a cluster that share the keys of a query tile (tensor-memory kernel)
};

// True for the shapes of the tensor-memory kernel: head_dim 128 and a group that
// divides its 128-row tile.
bool prefill_fp8_tc_supported(int head_dim, int num_q_heads, int num_kv_heads);
int launch_prefill_fp8_tc(PrefillFp8Args a, int num_seqs, int max_q_len, cudaStream_t stream);

}  // namespace muk
