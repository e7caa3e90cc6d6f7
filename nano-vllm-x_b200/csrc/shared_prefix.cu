// Decode attention for a batch whose sequences share a long prefix (a system
// prompt, a document): its keys are read once for the whole batch.
//
// For row b with keys [0, P) shared and [P, n_b) its own,
//   o = (sum_r 2^(m_r - m) o_r) / (sum_r 2^(m_r - m) l_r),  m = max_r m_r
// over any partition of its keys into ranges r, each with its running maximum
// m_r, its sum l_r and its unnormalised output o_r. The prefix's ranges are
// matrix products of all batch x group rows against the same keys: the
// tensor-core kernel of attention_sm100.cu (4 * 128 * batch * heads * P flops
// over P * kv_heads * 512 bytes: tensor-bound from a few hundred rows on). The
// own keys are the split-K decode kernels (decode.cu, decode_fp8.cu), bound by
// HBM, launched to run beside the prefix's last CTAs; a last kernel merges the
// fp32 partials of both. Short prefixes of few rows are read once a row instead
// (prefix_apart below). With an fp8 cache the prefix is expanded to bf16 in
// the workspace first: it is read once by that, and the tensor-core kernel
// takes it from L2.
#include <algorithm>
#include <cmath>

#include "decode.cuh"
#include "shared_prefix.cuh"

namespace nvattn {

static size_t round256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// Byte offsets of the workspace's regions and the splits they hold.
struct SharedLayout {
  int np, ptiles;  // splits of the prefix (0: none, or read with the own keys)
  int ns, stiles, cluster;  // splits of the own keys; those that a cluster merges
  size_t prefix_o, prefix_ml, own, k, v, bytes;
};

// The prefix is attended apart from the own keys where reading it once a row
// would cost more than the extra launches and partials: from 32 MB of such reads
// on (bf16; 16/8 heads, 5 rows of 1024: 11.8 us apart, 9.6 in one; 8 rows of 1024,
// 32 MB: 12.6 and 12.7; 8 rows of 2048: 15.5 and 16.3; 32/8 heads, 32 rows of 512,
// 64 MB: 15.7 and 21.2), with an fp8 cache, whose prefix is expanded first, from
// 64 MB on (16 rows of 1024, 32 MB: 17.7 and 11.9; 32/8 heads, 32 rows of 1024, 64
// MB: 20.4 and 20.3; 64 rows of 1024: 25.3 and 32.8). Otherwise the decode kernel
// takes all keys of a row, the shared pages from row 0 of the table. The tensor work
// grows with the heads a KV head, and the cost of a row's own reads with it: at 1, 8
// and 16 heads a KV head the bf16 sides cross at the same bytes (8 rows of 1024 over 8
// KV heads: 11.8 and 12.2, 13.8 and 14.6, 14.1 and 17.2; half as many: 12.3 and 10.1
// with 8), the fp8 sides too with 1 and 8 (32 rows of 512: 17.6 and 14.7, 21.4 and
// 20.1) and at half of them with 16 (16 rows of 1024: 22.4 and 24.4).
// The two sides round differently. Read once a row, a bf16 cache's weights go to the
// tensor cores as bf16 (decode.cu) and an fp8 cache's as f16 (decode_fp8.cu: 0.0017
// from 64 bits, the output's own rounding); the prefix apart takes bf16 weights
// against the bf16 values of either cache (0.0023), its own keys as before. So an fp8
// caller's batch that grows past the rule keeps 2^-8 of a weight instead of 2^-12.
static bool prefix_apart(int batch, int num_kv_heads, int shared_len, bool fp8) {
  const int64_t keys = static_cast<int64_t>(batch) * shared_len * num_kv_heads;
  return fp8 ? keys * 258 > (64 << 20) : keys * 512 > (32 << 20);
}

static SharedLayout shared_layout(int batch, int num_heads, int num_kv_heads, int max_blocks,
                                  int block_size, int shared_len, bool fp8) {
  SharedLayout w{};
  const bool apart = prefix_apart(batch, num_kv_heads, shared_len, fp8);
  if (apart) shared_split(batch, num_heads, num_kv_heads, shared_len, &w.np, &w.ptiles);
  const int own_blocks = std::max(1, max_blocks - (apart ? shared_len / block_size : 0));
  w.cluster = 1;
  if (fp8)
    choose_split_fp8(batch, num_kv_heads, static_cast<int64_t>(own_blocks) * block_size, &w.ns,
                     &w.stiles, &w.cluster);
  else
    // behind a prefix: splits of 8 tiles (64 rows x 8 KV heads of up to 1023
    // own keys 75 us the call, of 4 tiles 79, of 16 76)
    choose_split(batch, num_kv_heads, own_blocks, block_size, &w.ns, &w.stiles,
                 apart ? 8 : kMinSplitTiles);
  const size_t rows = static_cast<size_t>(batch) * num_heads;
  size_t at = 0;
  w.prefix_o = at;
  at += round256(rows * w.np * kHeadDim * sizeof(float));
  w.prefix_ml = at;
  at += round256(rows * w.np * sizeof(float2));
  w.own = at;
  const size_t parts = rows * (w.ns / w.cluster);
  at += round256(parts * kHeadDim * sizeof(float)) + round256(parts * sizeof(float2));
  if (fp8 && apart) {
    const size_t kv = static_cast<size_t>(shared_len) * num_kv_heads * kHeadDim * 2;
    w.k = at;
    at += round256(kv);
    w.v = at;
    at += round256(kv);
  }
  w.bytes = at;
  return w;
}

}  // namespace nvattn

using namespace nvattn;

extern "C" size_t nvattn_shared_prefix_workspace_bytes(int32_t batch, int32_t num_heads,
                                                       int32_t num_kv_heads,
                                                       int32_t max_blocks_per_seq,
                                                       int32_t block_size, int32_t shared_len,
                                                       int32_t fp8) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads ||
      num_heads / num_kv_heads > kMaxGroup || max_blocks_per_seq <= 0 || block_size <= 0 ||
      shared_len < 0 || shared_len % block_size || shared_len / block_size > max_blocks_per_seq)
    return 0;
  return shared_layout(batch, num_heads, num_kv_heads, max_blocks_per_seq, block_size, shared_len,
                       fp8 != 0)
      .bytes;
}

extern "C" int nvattn_shared_prefix_decode(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
    const void* v_cache, const uint8_t* k_scale, const uint8_t* v_scale, void* out,
    int64_t o_stride_tok, int64_t o_stride_head, const int32_t* cache_seqlens,
    const int32_t* block_table, int64_t block_table_stride, int32_t max_blocks_per_seq,
    int32_t num_blocks, int32_t block_size, int32_t shared_len, int32_t batch, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, float softmax_scale, void* workspace,
    size_t workspace_bytes, int32_t* status, void* stream) {
  clear_error();
  if (batch == 0) return NVATTN_OK;
  const char* who = "shared_prefix_decode";
  int rc = check_decode_args(who, q, q_stride_tok, q_stride_head, k_cache, v_cache, out,
                             cache_seqlens, block_table, block_table_stride, max_blocks_per_seq,
                             num_blocks, block_size, batch, num_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  rc = check_table_keys(who, max_blocks_per_seq, block_size);
  if (rc) return rc;
  const bool fp8 = k_scale != nullptr || v_scale != nullptr;
  if (fp8) {
    rc = check_fp8_scales(who, k_scale, v_scale);
    if (rc) return rc;
  }
  const auto msg = [who](const char* what) { return std::string(who) + ": " + what; };
  if (batch > 65535) return fail(NVATTN_ERR_UNSUPPORTED, msg("batch > 65535"));
  if (block_size % 128)
    return fail(NVATTN_ERR_UNSUPPORTED, msg("block_size must be a multiple of 128"));
  if (shared_len < 0 || shared_len % block_size || shared_len / block_size > max_blocks_per_seq)
    return fail(NVATTN_ERR_INVALID, msg("shared_len must be whole blocks of the table"));
  // the tensor-core pass takes the maximum of the scores before it scales them
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return fail(NVATTN_ERR_INVALID, msg("softmax_scale must be finite and > 0"));
  if (!aligned16(q) || (q_stride_tok * 2) % 16 || (q_stride_head * 2) % 16)
    return fail(NVATTN_ERR_UNSUPPORTED, msg("q base and strides must be 16-byte multiples (TMA)"));
  const SharedLayout w = shared_layout(batch, num_heads, num_kv_heads, max_blocks_per_seq,
                                       block_size, shared_len, fp8);
  if (workspace == nullptr || workspace_bytes < w.bytes)
    return fail(NVATTN_ERR_WORKSPACE,
                msg("workspace smaller than nvattn_shared_prefix_workspace_bytes()"));
  if (reinterpret_cast<uintptr_t>(workspace) & 255)
    return fail(NVATTN_ERR_INVALID, msg("workspace must be 256-byte aligned"));
  char* ws = static_cast<char*>(workspace);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);

  DecodeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride_tok = q_stride_tok;
  p.q_stride_head = q_stride_head;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_stride_tok = o_stride_tok;
  p.o_stride_head = o_stride_head;
  p.seqlens = cache_seqlens;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.max_blocks = max_blocks_per_seq;
  p.nsplit = w.ns;
  p.split_tiles = w.stiles;
  p.cluster = w.cluster;
  p.key_begin = w.np > 0 ? shared_len : 0;
  p.shared = w.np > 0 ? 0 : shared_len;
  p.scale_log2 = softmax_scale * kLog2e;
  p.status = status;
  set_decode_workspace(&p, ws + w.own, batch);
  float* prefix_o = reinterpret_cast<float*>(ws + w.prefix_o);
  float2* prefix_ml = reinterpret_cast<float2*>(ws + w.prefix_ml);

  if (w.np > 0) {
    SharedPrefix a{};
    a.q = q;
    a.q_stride_tok = q_stride_tok;
    a.q_stride_head = q_stride_head;
    a.k = k_cache;
    a.v = v_cache;
    a.block_table = block_table;
    a.seqlens = cache_seqlens;
    a.num_blocks = num_blocks;
    a.block_size = block_size;
    a.shared_len = shared_len;
    a.batch = batch;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.nsplit = w.np;
    a.split_tiles = w.ptiles;
    a.scale_log2 = p.scale_log2;
    a.ws_o = prefix_o;
    a.ws_ml = prefix_ml;
    a.status = status;
    if (fp8) {
      rc = launch_load_kvcache_fp8(k_cache, v_cache, k_scale, v_scale, nullptr, 1, block_table,
                                   block_table_stride, shared_len / block_size, num_blocks,
                                   block_size, num_kv_heads, shared_len, false, ws + w.k, ws + w.v,
                                   status, s);
      if (rc) return rc;
      a.k = ws + w.k;
      a.v = ws + w.v;
      a.block_table = nullptr;
      a.num_blocks = shared_len / block_size;
    }
    rc = launch_shared_prefix(a, s);
    if (rc) return rc;
  }
  const bool after = w.np > 0;
  if (fp8 && !after)
    return launch_decode_fp8_whole(p, k_cache, v_cache, k_scale, v_scale, batch, s);
  rc = fp8 ? launch_decode_fp8_suffix(p, k_cache, v_cache, k_scale, v_scale, batch, s)
           : launch_decode_suffix(p, k_cache, v_cache, batch, after, s);
  if (rc) return rc;
  return launch_merge_partials(p, prefix_o, prefix_ml, w.np, batch, s);
}
