// Split-K decode: what the bf16 and the fp8 kernel share (tile and split sizes,
// parameters, workspace layout, argument checks) and the merge of partials.
#pragma once

#include "common.cuh"

namespace nvattn {

constexpr int kTile = 64;                      // tokens per pipeline stage
// Smallest split of decode.cu; overridable at build time for tuning sweeps.
#ifndef NVATTN_DEC_MIN_SPLIT_TILES
#define NVATTN_DEC_MIN_SPLIT_TILES 4
#endif
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
  int32_t cluster;   // fp8: splits that one cluster merges before it writes (divides nsplit)
  int32_t key_begin;  // suffix kernels: first key of the split range (a whole number of blocks)
  int32_t shared;  // keys whose pages row 0 of the table holds, for rows with at least as many (0: none)
  float scale_log2;
  float* ws_o;    // [batch][num_heads][nsplit][128]
  float2* ws_ml;  // [batch][num_heads][nsplit]  (running max (log2 units), sum)
  int32_t* status;
};

__device__ __forceinline__ float neg_inf() { return -INFINITY; }

// The keys of a row that the decode kernels own beside a shared prefix of
// p.key_begin keys: from the prefix's end on, p.split_tiles tiles a split. A
// row shorter than the prefix takes no part in the prefix: its keys are all its
// own, in splits long enough for the grid. (key_begin 0: all keys.)
struct KeyRange {
  int begin, split;  // first key, keys a split
};
__device__ __forceinline__ KeyRange own_keys(const DecodeParams& p, int ctx) {
  if (ctx >= p.key_begin) return {p.key_begin, p.split_tiles * kTile};
  const int tiles = (max(ctx, 0) + kTile - 1) / kTile;
  return {0, max(p.split_tiles, (tiles + p.nsplit - 1) / p.nsplit) * kTile};
}

// One CTA of a kernel launched beside the prefix's kernel (its programmatic
// dependent) ends only after that grid has completed, so whatever waits for
// this kernel has the prefix's partials too.
__device__ __forceinline__ void join_prefix_grid() {
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1)
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The table entry of key `tok` of a row with ctx keys.
__device__ __forceinline__ int page_of(const DecodeParams& p, const int32_t* row, int tok, int ctx) {
  return __ldg((tok < p.shared && ctx >= p.shared ? p.block_table : row) + tok / p.block_size);
}

// Split size for a batch over tables of max_blocks, of at least min_tiles (see
// decode.cu).
constexpr int kMinSplitTiles = NVATTN_DEC_MIN_SPLIT_TILES;
void choose_split(int batch, int num_kv_heads, int max_blocks, int block_size, int* nsplit,
                  int* split_tiles, int min_tiles = kMinSplitTiles);
// Splits of the fp8 kernel for rows of up to max_keys, and the cluster that
// merges them (decode_fp8.cu).
void choose_split_fp8(int batch, int num_kv_heads, int64_t max_keys, int* nsplit, int* split_tiles,
                      int* cluster);
int device_sm_count();
// Bytes of `nsplit` partials a (sequence, query head): fp32 O, then (max, sum).
size_t decode_ws_bytes(int batch, int num_heads, int nsplit);
// Points p.ws_o and p.ws_ml into a workspace of decode_ws_bytes (or to null);
// p.nsplit and p.cluster are set.
void set_decode_workspace(DecodeParams* p, void* workspace, int batch);
// Argument checks shared by the decode entry points; `who` names the caller.
int check_decode_args(const char* who, const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                      const void* k_cache, const void* v_cache, const void* out,
                      const int32_t* cache_seqlens, const int32_t* block_table,
                      int64_t block_table_stride, int32_t max_blocks_per_seq, int32_t num_blocks,
                      int32_t block_size, int32_t batch, int32_t num_heads, int32_t num_kv_heads,
                      int32_t head_dim);
// The suffix kernels over p's own keys, as programmatic dependents of the prefix's
// kernel, launched just before on `stream` (bf16: if after_prefix).
int launch_decode_suffix(const DecodeParams& p, const void* k_cache, const void* v_cache, int batch,
                         bool after_prefix, cudaStream_t stream);
// All keys of every row, merged into p.out.
int launch_decode_fp8_whole(const DecodeParams& p, const void* k_cache, const void* v_cache,
                            const uint8_t* k_scale, const uint8_t* v_scale, int batch,
                            cudaStream_t stream);
int launch_decode_fp8_suffix(const DecodeParams& p, const void* k_cache, const void* v_cache,
                             const uint8_t* k_scale, const uint8_t* v_scale, int batch,
                             cudaStream_t stream);
// Checks an fp8 cache's scale pointers.
int check_fp8_scales(const char* who, const void* k_scale, const void* v_scale);
// Key positions are 32-bit: a table may cover up to 2^30 keys.
int check_table_keys(const char* who, int32_t max_blocks_per_seq, int32_t block_size);
// Merges partials of up to two key ranges into p.out: `first` (nfirst of them, all
// live in a row with keys; p.key_begin keys together) and p's own nsplit ones.
int launch_merge_partials(const DecodeParams& p, const float* first_o, const float2* first_ml,
                          int nfirst, int batch, cudaStream_t stream);

}  // namespace nvattn
