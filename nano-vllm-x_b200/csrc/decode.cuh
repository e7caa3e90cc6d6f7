// Split-K decode: what the bf16 and the fp8 kernel share (tile and split sizes,
// parameters, workspace layout, argument checks) and the merge of partials.
#pragma once

#include "common.cuh"

namespace nvattn {

constexpr int kTile = 64;                      // tokens per pipeline stage
constexpr int kDecConsumerWarps = 4;
constexpr int kDecThreads = (kDecConsumerWarps + 1) * 32;
constexpr int kMaxGroup = 16;                  // query heads per KV head handled per CTA
constexpr int kOPad = 132;                     // fp32 row pitch of the merge buffer

struct DecodeParams {
  const __nv_bfloat16* q;
  int64_t q_stride_tok, q_stride_head;
  __nv_bfloat16* out;
  int64_t o_stride_tok, o_stride_head;
  const int32_t* seqlens;
  const int32_t* block_table;
  int64_t bt_stride;
  int32_t num_blocks, block_size, num_heads, num_kv_heads, group;
  int32_t max_blocks;  // block-table width: keys past max_blocks*block_size are ignored
  int32_t nsplit, split_tiles;
  int32_t key_begin;  // suffix kernels: first key of the split range (a whole number of blocks)
  float scale_log2;
  float* ws_o;    // [batch][num_heads][nsplit][128]
  float2* ws_ml;  // [batch][num_heads][nsplit]  (running max (log2 units), sum)
  int32_t* status;
};

__device__ __forceinline__ float neg_inf() { return -INFINITY; }

// Split size for a batch over tables of max_blocks (see decode.cu).
void choose_split(int batch, int num_kv_heads, int max_blocks, int block_size, int* nsplit,
                  int* split_tiles);
// Bytes of `nsplit` partials a (sequence, query head): fp32 O, then (max, sum).
size_t decode_ws_bytes(int batch, int num_heads, int nsplit);
// Points p.ws_o and p.ws_ml into a workspace of decode_ws_bytes (or to null).
void set_decode_workspace(DecodeParams* p, void* workspace, int batch);
// Argument checks shared by the decode entry points; `who` names the caller.
int check_decode_args(const char* who, const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                      const void* k_cache, const void* v_cache, const void* out,
                      const int32_t* cache_seqlens, const int32_t* block_table,
                      int64_t block_table_stride, int32_t max_blocks_per_seq, int32_t num_blocks,
                      int32_t block_size, int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                      int32_t head_dim);
// Merges partials of up to two key ranges into p.out: `first` (nfirst of them, all
// live in a row with keys; p.key_begin keys together) and p's own nsplit ones.
int launch_merge_partials(const DecodeParams& p, const float* first_o, const float2* first_ml,
                          int nfirst, int batch, cudaStream_t stream);

}  // namespace nvattn
