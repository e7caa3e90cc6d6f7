// The KV cache in 8-bit floating point: rows quantised as they are scattered
// into the paged cache, and read back as dense bf16 rows for the prefill
// kernels. (The reference keeps its cache in the model's type,
// nanovllm/engine/model_runner.py:115; the scatter's contract is that of
// nanovllm/layers/attention.py:10-40.)
//
// One row = the 128 elements of one (token, KV head). With a = max |x_d| the
// row's scale is the smallest power of two 2^k with a <= 448 * 2^k (448 = the
// largest e4m3 value), k >= -100, and x8_d = e4m3(x_d * 2^-k), rounded to
// nearest even. A power of two costs no accuracy (an e4m3 element is off by at
// most 2^-4 of its value, whatever the scale) and keeps everything but that
// one rounding exact: x * 2^-k is exact in fp32, x8 * 2^k is exact in bf16,
// and the attention over the cache adds integers to its exponents. The scale
// is stored as the byte k + 127; a row holding a value that is not finite is
// stored as NaN elements with byte 255, so it reads back as NaN.
//
// Both kernels are copies with a few instructions an element, bound by HBM:
// 8 lanes own a row, lane i its elements 8i..8i+7 and 64+8i..64+8i+7, so that
// every load and store instruction covers whole 32-byte sectors (a lane's 16
// neighbours instead left each sector to two instructions: reading back 68,600
// keys of 8 heads took 93 us, now 74, 5.7 TB/s; storing 16,384 tokens 15.6, 6.5
// TB/s). Every lane has its K and V loads in flight before its first store, and
// bytes that are read or written once stay out of L1.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "shared_prefix.cuh"

namespace nvattn {

constexpr int kRowLanes = 8;       // lanes of one 128-element row
constexpr int kStoreThreads = 256;
constexpr int kLoadThreads = 256;
constexpr int kMinExp = -100;      // smallest scale exponent written

__device__ __forceinline__ int4 ld_once(const void* p) {
  int4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ int2 ld_once8(const void* p) {
  int2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.s32 {%0, %1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "l"(p));
  return v;
}

// This lane's 16 bf16 elements of a row. kAligned: 16-byte rows; otherwise
// element by element (rows at odd strides).
template <bool kAligned>
__device__ __forceinline__ void load_row16(const __nv_bfloat16* row, int part, uint32_t* w) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __nv_bfloat16* src = row + h * 64 + part * 8;
    if (kAligned) {
      const int4 a = ld_once(src);
      w[4 * h] = a.x, w[4 * h + 1] = a.y, w[4 * h + 2] = a.z, w[4 * h + 3] = a.w;
    } else {
      const unsigned short* s = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[4 * h + i] = static_cast<uint32_t>(__ldg(s + 2 * i)) |
                       (static_cast<uint32_t>(__ldg(s + 2 * i + 1)) << 16);
    }
  }
}

// Quantises the 8-lane row whose 16 elements this lane holds; every lane
// returns the row's exponent byte and its own 16 e4m3 elements.
__device__ __forceinline__ int4 quantise_row(const uint32_t* w, uint32_t* exp_byte) {
  // magnitudes as integers: the order of bf16 bits, with inf and NaN on top
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
#pragma unroll
  for (int o = 1; o < kRowLanes; o <<= 1)
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  const uint32_t a = max(m & 0xffffu, m >> 16);
  if (a >= 0x7f80u) {
    *exp_byte = 255u;
    return make_int4(0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f, 0x7f7f7f7f);
  }
  // a = 1.f * 2^(E-127) with f = 7 bits; 448 = 1.75 * 2^8 and 1.75 is f = 0x60
  const int k = max(kMinExp, static_cast<int>(a >> 7) - 135 + ((a & 0x7fu) > 0x60u ? 1 : 0));
  *exp_byte = static_cast<uint32_t>(k + 127);
  const float inv = __int_as_float((127 - k) << 23);  // 2^-k, k in [-100, 120]
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t half[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t p = w[2 * i + j];
      const float2 x = make_float2(__uint_as_float(p << 16) * inv,
                                   __uint_as_float(p & 0xffff0000u) * inv);
      half[j] = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
    }
    q[i] = half[0] | (half[1] << 16);
  }
  return make_int4(q[0], q[1], q[2], q[3]);
}

// One 8-lane group per (token, KV head): its K row and its V row.
template <bool kAligned>
__global__ void __launch_bounds__(kStoreThreads)
    store_kvcache_fp8_kernel(const __nv_bfloat16* __restrict__ key, int64_t key_stride,
                             const __nv_bfloat16* __restrict__ value, int64_t value_stride,
                             uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
                             uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v_scale,
                             const int32_t* __restrict__ slot_mapping, int64_t num_rows,
                             int num_kv_heads, int block_size, int64_t num_slots,
                             int32_t* status) {
  const int64_t r = (static_cast<int64_t>(blockIdx.x) * kStoreThreads + threadIdx.x) / kRowLanes;
  const int part = threadIdx.x % kRowLanes;
  // all 32 lanes stay for the shuffles; rows past the end repeat the last one
  const int64_t row = min(r, num_rows - 1);
  const int64_t tok = row / num_kv_heads;
  const int g = static_cast<int>(row - tok * num_kv_heads);
  const int64_t in = static_cast<int64_t>(g) * kHeadDim;
  const int64_t slot = __ldg(slot_mapping + tok);
  uint32_t kw[8], vw[8];
  load_row16<kAligned>(key + tok * key_stride + in, part, kw);
  load_row16<kAligned>(value + tok * value_stride + in, part, vw);
  uint32_t ke, ve;
  const int4 kq = quantise_row(kw, &ke);
  const int4 vq = quantise_row(vw, &ve);
  if (r >= num_rows || slot == -1) return;  // attention.py:23
  if (slot < 0 || slot >= num_slots) {
    if (part == 0) set_status(status, NVATTN_STATUS_BAD_SLOT);
    return;
  }
  const int64_t at = (slot * num_kv_heads + g) * kHeadDim + part * 8;
  __stcs(reinterpret_cast<int2*>(k_cache + at), make_int2(kq.x, kq.y));
  __stcs(reinterpret_cast<int2*>(k_cache + at + 64), make_int2(kq.z, kq.w));
  __stcs(reinterpret_cast<int2*>(v_cache + at), make_int2(vq.x, vq.y));
  __stcs(reinterpret_cast<int2*>(v_cache + at + 64), make_int2(vq.z, vq.w));
  if (part == 0) {
    const int64_t blk = slot / block_size;
    const int64_t sc = (blk * num_kv_heads + g) * block_size + (slot - blk * block_size);
    k_scale[sc] = static_cast<uint8_t>(ke);
    v_scale[sc] = static_cast<uint8_t>(ve);
  }
}

// A lane's 16 e4m3 elements times 2^k as bf16, 8 a vector (exact: 4 significant bits; past
// bf16's range, as in fp32, infinite).
__device__ __forceinline__ void expand16(const int4 q, uint32_t exp_byte, int4* out) {
  const float s = exp_byte == 255u ? __int_as_float(0x7fffffff)
                                   : __int_as_float(static_cast<int>(exp_byte) << 23);
  const uint32_t w[4] = {static_cast<uint32_t>(q.x), static_cast<uint32_t>(q.y),
                         static_cast<uint32_t>(q.z), static_cast<uint32_t>(q.w)};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> ((i & 1) * 16)), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    o[i] = pack_bf16x2(f.x * s, f.y * s);
  }
  out[0] = make_int4(o[0], o[1], o[2], o[3]);
  out[1] = make_int4(o[4], o[5], o[6], o[7]);
}

// Rows a thread group handles at stride `rows_step`, their loads in flight
// together.
constexpr int kLoadRows = 4;

// CTA: kLoadRows * kLoadThreads / 8 consecutive (key, KV head) rows of the
// dense output. The sequence of a CTA's first key is found by bisection of
// cu_seqlens_k, the others by walking on from it (cu_k null: one sequence of
// all rows).
__global__ void __launch_bounds__(kLoadThreads)
    load_kvcache_fp8_kernel(const uint8_t* __restrict__ k_cache,
                            const uint8_t* __restrict__ v_cache,
                            const uint8_t* __restrict__ k_scale,
                            const uint8_t* __restrict__ v_scale,
                            const int32_t* __restrict__ cu_k, int num_seqs,
                            const int32_t* __restrict__ block_table, int64_t bt_stride,
                            int max_blocks, int num_blocks, int block_size, int num_kv_heads,
                            int64_t num_rows, bool zero_rest, __nv_bfloat16* __restrict__ k_out,
                            __nv_bfloat16* __restrict__ v_out, int32_t* status) {
  constexpr int kStep = kLoadThreads / kRowLanes;
  const int part = threadIdx.x % kRowLanes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kLoadRows * kStep;
  // last sequence whose start is <= the CTA's first key
  int seq = 0;
  if (cu_k != nullptr) {
    const int64_t key0 = first / num_kv_heads;
    int hi = num_seqs;
    while (hi - seq > 1) {
      const int mid = (seq + hi) >> 1;
      if (__ldg(cu_k + mid) <= key0)
        seq = mid;
      else
        hi = mid;
    }
  }
  int4 kq[kLoadRows], vq[kLoadRows];
  uint32_t ke[kLoadRows], ve[kLoadRows];
  int64_t out_row[kLoadRows];
#pragma unroll
  for (int u = 0; u < kLoadRows; ++u) {
    const int64_t row = first + u * kStep + threadIdx.x / kRowLanes;
    out_row[u] = -1;
    kq[u] = vq[u] = make_int4(0, 0, 0, 0);
    ke[u] = ve[u] = 0u;
    if (row >= num_rows) continue;
    const int64_t key = row / num_kv_heads;
    const int g = static_cast<int>(row - key * num_kv_heads);
    int64_t pos = key;
    if (cu_k != nullptr) {
      while (seq < num_seqs && key >= __ldg(cu_k + seq + 1)) ++seq;
      pos = seq < num_seqs ? key - __ldg(cu_k + seq) : -1;
    }
    if (pos < 0) {  // behind the last sequence, or before the first
      if (zero_rest) out_row[u] = row;
      continue;
    }
    out_row[u] = row;
    const int64_t col = pos / block_size;
    int blk = -1;
    if (col < max_blocks) blk = __ldg(block_table + static_cast<int64_t>(seq) * bt_stride + col);
    if (blk < 0 || blk >= num_blocks) {  // zeros, flagged
      if (part == 0) set_status(status, NVATTN_STATUS_BAD_BLOCK);
      continue;
    }
    const int in = static_cast<int>(pos - col * block_size);
    const int64_t at =
        ((static_cast<int64_t>(blk) * block_size + in) * num_kv_heads + g) * kHeadDim + part * 8;
    const int64_t sc = (static_cast<int64_t>(blk) * num_kv_heads + g) * block_size + in;
    const int2 k0 = ld_once8(k_cache + at), k1 = ld_once8(k_cache + at + 64);
    const int2 v0 = ld_once8(v_cache + at), v1 = ld_once8(v_cache + at + 64);
    kq[u] = make_int4(k0.x, k0.y, k1.x, k1.y);
    vq[u] = make_int4(v0.x, v0.y, v1.x, v1.y);
    ke[u] = __ldg(k_scale + sc);
    ve[u] = __ldg(v_scale + sc);
  }
#pragma unroll
  for (int u = 0; u < kLoadRows; ++u) {
    if (out_row[u] < 0) continue;
    const int64_t at = out_row[u] * kHeadDim + part * 8;
    int4 o[2];
    expand16(kq[u], ke[u], o);
    reinterpret_cast<int4*>(k_out + at)[0] = o[0];
    reinterpret_cast<int4*>(k_out + at + 64)[0] = o[1];
    expand16(vq[u], ve[u], o);
    reinterpret_cast<int4*>(v_out + at)[0] = o[0];
    reinterpret_cast<int4*>(v_out + at + 64)[0] = o[1];
  }
}

int launch_load_kvcache_fp8(const void* k_cache, const void* v_cache, const uint8_t* k_scale,
                            const uint8_t* v_scale, const int32_t* cu_seqlens_k, int num_seqs,
                            const int32_t* block_table, int64_t bt_stride, int max_blocks,
                            int num_blocks, int block_size, int num_kv_heads, int64_t total_k,
                            bool zero_rest, void* k_out, void* v_out, int32_t* status,
                            cudaStream_t stream) {
  const int64_t rows = total_k * num_kv_heads;
  const int64_t per_cta = kLoadRows * (kLoadThreads / kRowLanes);
  const int64_t grid = (rows + per_cta - 1) / per_cta;
  if (grid > 0x7fffffffLL) return fail(NVATTN_ERR_INVALID, "load_kvcache_fp8: too many rows");
  load_kvcache_fp8_kernel<<<static_cast<unsigned>(grid), kLoadThreads, 0, stream>>>(
      static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), k_scale, v_scale,
      cu_seqlens_k, num_seqs, block_table, bt_stride, max_blocks, num_blocks, block_size,
      num_kv_heads, rows, zero_rest, static_cast<__nv_bfloat16*>(k_out),
      static_cast<__nv_bfloat16*>(v_out), status);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? NVATTN_OK : cuda_fail(e, "load_kvcache_fp8 launch");
}

}  // namespace nvattn

using namespace nvattn;

extern "C" int nvattn_store_kvcache_fp8(const void* key, int64_t key_stride, const void* value,
                                        int64_t value_stride, void* k_cache, void* v_cache,
                                        uint8_t* k_scale, uint8_t* v_scale,
                                        const int32_t* slot_mapping, int64_t num_tokens,
                                        int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks,
                                        int32_t block_size, int32_t* status, void* stream) {
  clear_error();
  if (num_tokens < 0) return fail(NVATTN_ERR_INVALID, "store_kvcache_fp8: negative num_tokens");
  if (num_tokens == 0) return NVATTN_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !slot_mapping)
    return fail(NVATTN_ERR_INVALID, "store_kvcache_fp8: NULL pointer");
  if (head_dim != kHeadDim)
    return fail(NVATTN_ERR_UNSUPPORTED, "store_kvcache_fp8: head_dim must be 128");
  if (num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0)
    return fail(NVATTN_ERR_INVALID, "store_kvcache_fp8: bad cache geometry");
  const int64_t D = static_cast<int64_t>(num_kv_heads) * kHeadDim;
  if (num_tokens > 1 && (key_stride < D || value_stride < D))
    return fail(NVATTN_ERR_INVALID, "store_kvcache_fp8: token rows overlap");
  if (!aligned16(k_cache) || !aligned16(v_cache))
    return fail(NVATTN_ERR_INVALID, "store_kvcache_fp8: caches must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(key) & 1) || (reinterpret_cast<uintptr_t>(value) & 1))
    return fail(NVATTN_ERR_INVALID, "store_kvcache_fp8: key/value must be 2-byte aligned");
  const int64_t rows = num_tokens * num_kv_heads;
  const int64_t grid = (rows * kRowLanes + kStoreThreads - 1) / kStoreThreads;
  if (grid > 0x7fffffffLL) return fail(NVATTN_ERR_INVALID, "store_kvcache_fp8: too many rows");
  const bool aligned = aligned16(key) && aligned16(value) && key_stride % 8 == 0 &&
                       value_stride % 8 == 0;
  const auto kernel = aligned ? store_kvcache_fp8_kernel<true> : store_kvcache_fp8_kernel<false>;
  kernel<<<static_cast<unsigned>(grid), kStoreThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(key), key_stride, static_cast<const __nv_bfloat16*>(value),
      value_stride, static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), k_scale, v_scale,
      slot_mapping, rows, num_kv_heads, block_size, static_cast<int64_t>(num_blocks) * block_size,
      status);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? NVATTN_OK : cuda_fail(e, "store_kvcache_fp8 launch");
}

extern "C" int nvattn_load_kvcache_fp8(const void* k_cache, const void* v_cache,
                                       const uint8_t* k_scale, const uint8_t* v_scale,
                                       const int32_t* cu_seqlens_k, int32_t num_seqs,
                                       const int32_t* block_table, int64_t block_table_stride,
                                       int32_t max_blocks_per_seq, int32_t num_blocks,
                                       int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                                       int64_t total_k, int32_t zero_rest, void* k_out, void* v_out,
                                       int32_t* status, void* stream) {
  clear_error();
  if (num_seqs < 0 || total_k < 0) return fail(NVATTN_ERR_INVALID, "load_kvcache_fp8: negative size");
  if (num_seqs == 0 || total_k == 0) return NVATTN_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !cu_seqlens_k || !block_table || !k_out ||
      !v_out)
    return fail(NVATTN_ERR_INVALID, "load_kvcache_fp8: NULL pointer");
  if (head_dim != kHeadDim)
    return fail(NVATTN_ERR_UNSUPPORTED, "load_kvcache_fp8: head_dim must be 128");
  if (num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0 || max_blocks_per_seq <= 0 ||
      block_table_stride < max_blocks_per_seq)
    return fail(NVATTN_ERR_INVALID, "load_kvcache_fp8: bad cache or block table geometry");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out))
    return fail(NVATTN_ERR_INVALID, "load_kvcache_fp8: caches and outputs must be 16-byte aligned");
  return launch_load_kvcache_fp8(k_cache, v_cache, k_scale, v_scale, cu_seqlens_k, num_seqs,
                                 block_table, block_table_stride, max_blocks_per_seq, num_blocks,
                                 block_size, num_kv_heads, total_k, zero_rest != 0, k_out, v_out, status,
                                 reinterpret_cast<cudaStream_t>(stream));
}
