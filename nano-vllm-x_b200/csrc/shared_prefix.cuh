// The tensor-core pass over a prefix shared by a whole batch (kShared mode of
// attention_sm100.cu), as its caller in shared_prefix.cu sees it.
#pragma once

#include "common.cuh"

namespace nvattn {

struct SharedPrefix {
  const void* q;
  int64_t q_stride_tok, q_stride_head;
  const void* k;  // bf16 pages [num_blocks][block_size][num_kv_heads][128]
  const void* v;
  const int32_t* block_table;  // pages of the prefix in order; null: 0, 1, 2, ...
  const int32_t* seqlens;      // (batch): rows with fewer than shared_len keys are skipped
  int32_t num_blocks, block_size, shared_len;  // both sizes multiples of 128
  int32_t batch, num_heads, num_kv_heads;
  int32_t nsplit, split_tiles;  // shared_split()
  float scale_log2;
  float* ws_o;    // [batch][num_heads][nsplit][128]
  float2* ws_ml;  // [batch][num_heads][nsplit]
  int32_t* status;
};

void shared_split(int batch, int num_heads, int num_kv_heads, int shared_len, int* nsplit,
                  int* split_tiles);
int launch_shared_prefix(const SharedPrefix& a, cudaStream_t stream);

// kvcache_fp8.cu (cu_seqlens_k null: one sequence of total_k keys)
int launch_load_kvcache_fp8(const void* k_cache, const void* v_cache, const uint8_t* k_scale,
                            const uint8_t* v_scale, const int32_t* cu_seqlens_k, int num_seqs,
                            const int32_t* block_table, int64_t bt_stride, int max_blocks,
                            int num_blocks, int block_size, int num_kv_heads, int64_t total_k,
                            bool zero_rest, void* k_out, void* v_out, int32_t* status,
                            cudaStream_t stream);

}  // namespace nvattn
