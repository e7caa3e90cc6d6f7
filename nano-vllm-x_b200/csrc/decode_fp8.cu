// Paged split-K decode attention over the fp8 cache (layout and rounding in
// kvcache_fp8.cu): the split, the grid and the roles of decode.cu, half the
// bytes.
//
//   o = sum_j softmax_j(c * 2^kk_j * q.k8_j) * 2^kv_j * v8_j
//
// with k8, v8 the e4m3 elements and kk, kv the rows' exponents. No value is
// rounded on the way into the tensor cores but q (below) and the weights:
// e4m3 converts to f16 exactly, so both products run as f16 MMAs with fp32
// accumulation, the exponents are applied to the fp32 scores, and those of V
// are folded into the softmax: with t_j the score in log2 units, the running
// reference is M = max_j (t_j + kv_j), the weights given to the second product
// are w_j = 2^(t_j + kv_j - M) <= 1 (one rounding, to f16: 2^-12), and the sum
// runs over 2^(t_j - M). q's bf16 elements fit f16's 11 bits; its range is
// brought in by a power of two a row, so only elements below 2^-14 of the
// row's largest lose bits (2^-25 of it).
//
// HBM-bound: 258 bytes a (key, KV head) against 4 * 128 * group flops. The
// cost to hide is the conversion, 2 instructions for 4 elements and one byte
// permute for V: a warp owns whole 64-key tiles (the four warps of a CTA take
// turns), so the row maxima, the barrier waits and the rescale are paid once
// for 64 keys.
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "decode.cuh"

namespace nvattn {

constexpr int kTile8 = kTile * kHeadDim;      // one 64-key e4m3 tile (8 KB)
constexpr int kStages8 = 6;                   // ring depth
constexpr int kStageBytes8 = 2 * kTile8;      // K and V
constexpr int kScaleBytes8 = 2 * kTile;       // their exponent bytes
constexpr int kSmem8 = kStages8 * (kStageBytes8 + kScaleBytes8) + 1024 + 2 * kStages8 * 8 +
                       kDecConsumerWarps * kMaxGroup * 2 * 4;
static_assert(kDecConsumerWarps * kMaxGroup * kOPad * 4 <= kStages8 * kStageBytes8,
              "the merge buffer reuses the ring");

// 1-D bulk copy into shared memory, completion on an mbarrier (16-byte
// aligned addresses, size a multiple of 16).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Two e4m3 elements (low byte first) as two f16: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(static_cast<unsigned short>(two)));
  return d;
}

__device__ __forceinline__ void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^(byte - 127) of a stored exponent (27..247; 255 only beside NaN elements).
__device__ __forceinline__ float exp_byte_scale(uint32_t byte) {
  return __uint_as_float(byte << 23);
}

// byte - 127 as fp32 without a conversion: 2^23 + byte has byte in its low bits.
__device__ __forceinline__ float exp_byte_log2(uint32_t byte) {
  return __uint_as_float(0x4B000000u | byte) - (8388608.f + 127.f);
}

// f16 A fragments of this thread's two query rows (rowa, rowb of the group)
// and the exact power of two they were divided by. A 16-dim step takes dims
// 4q..4q+3 of quad lane q (dims may be summed in any order as long as K's
// fragments agree: one 4-byte word of an e4m3 row holds them).
__device__ __forceinline__ void load_q8(const DecodeParams& p, int b, int h0, int rowa, int rowb,
                                        int quad, uint32_t qa[8][4], float* back_a,
                                        float* back_b) {
  const __nv_bfloat16* qb = p.q + static_cast<int64_t>(b) * p.q_stride_tok;
  const uint32_t* row[2] = {
      reinterpret_cast<const uint32_t*>(qb + static_cast<int64_t>(h0 + rowa) * p.q_stride_head),
      reinterpret_cast<const uint32_t*>(qb + static_cast<int64_t>(h0 + rowb) * p.q_stride_head)};
  const bool live[2] = {rowa < p.group, rowb < p.group};
  float* back[2] = {back_a, back_b};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    uint32_t w[16];
    float mx = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      w[2 * kk] = live[r] ? row[r][kk * 8 + quad * 2] : 0u;
      w[2 * kk + 1] = live[r] ? row[r][kk * 8 + quad * 2 + 1] : 0u;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w[i] << 16)),
                           fabsf(__uint_as_float(w[i] & 0xffff0000u))));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // exponent of the largest element, kept where both 2^e and 2^-e are normal
    const int e = min(max(static_cast<int>(__float_as_uint(mx) >> 23), 1), 253);
    const float down = __int_as_float((254 - e) << 23);
    *back[r] = __int_as_float(e << 23);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        qa[kk][2 * i + r] = pack_f16x2(__uint_as_float(w[2 * kk + i] << 16) * down,
                                       __uint_as_float(w[2 * kk + i] & 0xffff0000u) * down);
    }
  }
}

// kSuffix: the keys from p.key_begin on, as fp32 partials for the merge with
// the keys before (shared_prefix.cu).
template <bool kSuffix>
__global__ void __launch_bounds__(kDecThreads, 2)
    paged_decode_fp8_kernel(const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap,
                            const uint8_t* __restrict__ k_scale,
                            const uint8_t* __restrict__ v_scale, const DecodeParams p) {
  const int split = blockIdx.x;
  const int g = blockIdx.y;
  const int b = blockIdx.z;
  int ctx = p.seqlens[b];
  if (ctx > p.max_blocks * p.block_size) {
    if (split == 0 && threadIdx.x == 0) set_status(p.status, NVATTN_STATUS_BAD_BLOCK);
    ctx = p.max_blocks * p.block_size;
  }
  const KeyRange own = kSuffix ? own_keys(p, ctx) : KeyRange{0, p.split_tiles * kTile};
  const int tok_begin = own.begin + split * own.split;
  const int tok_end = min(ctx, tok_begin + own.split);
  if (tok_end <= tok_begin) {
    if (kSuffix) join_prefix_grid();
    if (!kSuffix && p.nsplit == 1 && split == 0) {  // no merge runs: the empty row's zeros
      for (int e = threadIdx.x; e < p.group * kHeadDim; e += blockDim.x)
        p.out[static_cast<int64_t>(b) * p.o_stride_tok +
              static_cast<int64_t>(g * p.group + e / kHeadDim) * p.o_stride_head + e % kHeadDim] =
            __float2bfloat16_rn(0.f);
    }
    return;
  }
  const int ntiles = (tok_end - tok_begin + kTile - 1) / kTile;
  asm volatile("griddepcontrol.launch_dependents;");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* scales = smem + kStages8 * kStageBytes8;
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + kStages8 * kScaleBytes8);
  uint64_t* empty = full + kStages8;
  float* ml_smem = reinterpret_cast<float*>(empty + kStages8);  // [4][16][2]

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages8; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    fence_barrier_init();
  }
  __syncthreads();

  if (warp == kDecConsumerWarps) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tensor_map(&kmap);
      prefetch_tensor_map(&vmap);
      const int32_t* bt = p.block_table + static_cast<int64_t>(b) * p.bt_stride;
      int issued = 0;
      for (; issued < ntiles; ++issued) {
        const int stage = issued % kStages8;
        if (!mbar_wait(&empty[stage], ((issued / kStages8) & 1) ^ 1)) {
          set_status(p.status, NVATTN_STATUS_TIMEOUT);
          break;
        }
        const int tok0 = tok_begin + issued * kTile;
        int blk = bt[tok0 / p.block_size];
        if (blk < 0 || blk >= p.num_blocks) {
          set_status(p.status, NVATTN_STATUS_BAD_BLOCK);
          blk = 0;  // read a valid block; the result is flagged as invalid
        }
        const int tin = tok0 % p.block_size;
        const int64_t sc =
            (static_cast<int64_t>(blk) * p.num_kv_heads + g) * p.block_size + tin;
        uint8_t* st = smem + stage * kStageBytes8;
        uint8_t* ss = scales + stage * kScaleBytes8;
        mbar_arrive_expect_tx(&full[stage], kStageBytes8 + kScaleBytes8);
        tma_load_4d(st, &kmap, &full[stage], 0, g, tin, blk);
        bulk_load(ss, k_scale + sc, kTile, &full[stage]);
        tma_load_4d(st + kTile8, &vmap, &full[stage], 0, g, tin, blk);
        bulk_load(ss + kTile, v_scale + sc, kTile, &full[stage]);
      }
      // no copy of ours is in flight when this warp ends
      for (int it = std::max(0, issued - kStages8); it < issued; ++it)
        mbar_wait(&full[it % kStages8], (it / kStages8) & 1);
    }
    return;  // the producer warp takes no part in the merge below
  }

  // -------------------------------------------------------------- consumers
  const int quad = lane & 3;   // column pair inside an 8-wide MMA tile
  const int rowa = lane >> 2;  // accumulator rows rowa and rowa + 8
  const int rowb = rowa + 8;
  const int h0 = g * p.group;

  uint32_t qa[8][4];
  float scale_a, scale_b;
  load_q8(p, b, h0, rowa, rowb, quad, qa, &scale_a, &scale_b);
  scale_a *= p.scale_log2;
  scale_b *= p.scale_log2;

  // o[2c + e] holds dims 16c + 4*quad + {0, 2} + e of rows rowa, rowb
  float o[16][4];
#pragma unroll
  for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m_a = neg_inf(), m_b = neg_inf(), l_a = 0.f, l_b = 0.f;

  bool timed_out = false;
  for (int it = warp; it < ntiles; it += kDecConsumerWarps) {
    const int stage = it % kStages8;
    if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], (it / kStages8) & 1))) {
      timed_out = true;
      break;
    }
    const int nvalid = min(kTile, tok_end - (tok_begin + it * kTile));
    uint8_t* st = smem + stage * kStageBytes8;
    const uint8_t* ss = scales + stage * kScaleBytes8;
    const uint32_t kbase = smem_u32(st);
    const uint32_t vbase = kbase + kTile8;
    if (nvalid < kTile) {
      // Keys past the end hold stale bytes (maybe NaN): zero their V rows so
      // that 0 * NaN never reaches the sum. Only a range's last tile has
      // them, so no later copy lands in this stage.
      for (int e = lane; e < (kTile - nvalid) * 8; e += 32)
        *reinterpret_cast<int4*>(st + kTile8 + nvalid * 128 + e * 16) = make_int4(0, 0, 0, 0);
      __syncwarp();
    }
    // ---- S = Q K^T: 8 tiles of 8 keys, 8 steps of 16 dims
    float s[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      const int row = n * 8 + (lane & 7);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[4];  // this lane's 4 bytes of steps 4*half .. 4*half + 3
        ldmatrix_x4(kbase + swz128(row, half * 4 + (lane >> 3)), w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mma_f16_16816(s[n], qa[half * 4 + i], e4m3x2_to_f16x2(w[i]),
                        e4m3x2_to_f16x2(w[i] >> 16));
      }
    }
    // ---- exponents, mask, online softmax
    float mx_a = neg_inf(), mx_b = neg_inf();
    float ve[8][2];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const uint32_t kb = *reinterpret_cast<const uint16_t*>(ss + n * 8 + quad * 2);
      const uint32_t vb = *reinterpret_cast<const uint16_t*>(ss + kTile + n * 8 + quad * 2);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool ok = n * 8 + quad * 2 + j < nvalid;
        const float kf = exp_byte_scale((kb >> (8 * j)) & 0xffu);
        ve[n][j] = ok ? exp_byte_log2((vb >> (8 * j)) & 0xffu) : 0.f;
        s[n][j] = ok ? s[n][j] * (scale_a * kf) : neg_inf();
        s[n][2 + j] = ok ? s[n][2 + j] * (scale_b * kf) : neg_inf();
        mx_a = fmaxf(mx_a, s[n][j] + ve[n][j]);
        mx_b = fmaxf(mx_b, s[n][2 + j] + ve[n][j]);
      }
    }
    mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
    mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
    mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
    mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
    const float mn_a = fmaxf(m_a, mx_a), mn_b = fmaxf(m_b, mx_b);
    if (__any_sync(0xffffffffu, mn_a > m_a || mn_b > m_b)) {
      // l in two half steps: with V rows of very different magnitudes the
      // factor alone can leave fp32's range while its product with l does not
      const float h_a = fast_exp2(0.5f * (m_a - mn_a)), h_b = fast_exp2(0.5f * (m_b - mn_b));
      l_a = l_a * h_a * h_a;
      l_b = l_b * h_b * h_b;
      const float al_a = h_a * h_a, al_b = h_b * h_b;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        o[j][0] *= al_a;
        o[j][1] *= al_a;
        o[j][2] *= al_b;
        o[j][3] *= al_b;
      }
      m_a = mn_a;
      m_b = mn_b;
    }
    // ---- O += W V: 4 steps of 16 keys
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t pa[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = 2 * kk + i;
        float w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float ta = s[n][j] - m_a, tb = s[n][2 + j] - m_b;
          l_a += fast_exp2(ta);
          l_b += fast_exp2(tb);
          w[j] = fast_exp2(ta + ve[n][j]);
          w[2 + j] = fast_exp2(tb + ve[n][j]);
        }
        pa[2 * i] = pack_f16x2(w[0], w[1]);
        pa[2 * i + 1] = pack_f16x2(w[2], w[3]);
      }
      const int row = kk * 16 + (lane & 15);
#pragma unroll
      for (int c = 0; c < 8; c += 2) {
        // keys 2q, 2q+1 (r0, r2) and 2q+8, 2q+9 (r1, r3) of dims 2i, 2i+1 of
        // chunks c (r0, r1) and c+1 (r2, r3), i = lane / 4
        uint32_t r[4];
        ldmatrix_x4_trans(vbase + swz128(row, c + (lane >> 4)), r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __byte_perm(r[i], 0, 0x3120);  // pair the keys
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mma_f16_16816(o[2 * (c + i)], pa, e4m3x2_to_f16x2(r[2 * i]),
                        e4m3x2_to_f16x2(r[2 * i + 1]));
          mma_f16_16816(o[2 * (c + i) + 1], pa, e4m3x2_to_f16x2(r[2 * i] >> 16),
                        e4m3x2_to_f16x2(r[2 * i + 1] >> 16));
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[stage]);
  }
  if (timed_out && lane == 0) set_status(p.status, NVATTN_STATUS_TIMEOUT);

  // ---------------------------------------------------------------- merge
  l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
  l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
  l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
  l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);

  // All consumer warps are past their last ring read: reuse the ring.
  asm volatile("bar.sync 1, %0;" ::"r"(kDecConsumerWarps * 32));
  float* obuf = reinterpret_cast<float*>(smem);  // [4 warps][16 rows][kOPad]
  float* ow = obuf + warp * kMaxGroup * kOPad;
  if (quad == 0) {
    ml_smem[(warp * kMaxGroup + rowa) * 2 + 0] = m_a;
    ml_smem[(warp * kMaxGroup + rowa) * 2 + 1] = l_a;
    ml_smem[(warp * kMaxGroup + rowb) * 2 + 0] = m_b;
    ml_smem[(warp * kMaxGroup + rowb) * 2 + 1] = l_b;
  }
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int d = c * 16 + quad * 4;
    *reinterpret_cast<float4*>(ow + rowa * kOPad + d) =
        make_float4(o[2 * c][0], o[2 * c + 1][0], o[2 * c][1], o[2 * c + 1][1]);
    *reinterpret_cast<float4*>(ow + rowb * kOPad + d) =
        make_float4(o[2 * c][2], o[2 * c + 1][2], o[2 * c][3], o[2 * c + 1][3]);
  }
  asm volatile("bar.sync 1, %0;" ::"r"(kDecConsumerWarps * 32));

  const int d = threadIdx.x;  // 0..127: one head-dim column per thread
  for (int r = 0; r < p.group; ++r) {
    float mw[kDecConsumerWarps];
    float mmax = neg_inf();
#pragma unroll
    for (int w = 0; w < kDecConsumerWarps; ++w) {
      mw[w] = ml_smem[(w * kMaxGroup + r) * 2];
      mmax = fmaxf(mmax, mw[w]);
    }
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kDecConsumerWarps; ++w) {
      // a warp without a tile keeps m = -inf, l = 0, o = 0
      const float h = (mw[w] == neg_inf()) ? 0.f : fast_exp2(0.5f * (mw[w] - mmax));
      L += ml_smem[(w * kMaxGroup + r) * 2 + 1] * h * h;
      acc += obuf[(w * kMaxGroup + r) * kOPad + d] * h * h;
    }
    const int h = h0 + r;
    if (!kSuffix && p.nsplit == 1) {
      p.out[static_cast<int64_t>(b) * p.o_stride_tok + static_cast<int64_t>(h) * p.o_stride_head +
            d] = __float2bfloat16_rn(acc / L);
    } else {
      const int64_t slot = (static_cast<int64_t>(b) * p.num_heads + h) * p.nsplit + split;
      p.ws_o[slot * kHeadDim + d] = acc;
      if (d == 0) p.ws_ml[slot] = make_float2(mmax, L);
    }
  }
  if (kSuffix) join_prefix_grid();
}

// Merges the partials of one (sequence, query head) per warp: lane i owns dims
// 4i..4i+3. Launched as a programmatic dependent of the kernel that writes the
// last partials.
constexpr int kMergeWarps = 4;

__global__ void __launch_bounds__(kMergeWarps * 32)
    merge_partials_kernel(const DecodeParams p, const float* __restrict__ first_o,
                          const float2* __restrict__ first_ml, int nfirst, int rows) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int b = row / p.num_heads, h = row - b * p.num_heads;
  const int ctx = min(p.seqlens[b], p.max_blocks * p.block_size);
  const KeyRange own = own_keys(p, ctx);
  const int nf = own.begin > 0 ? nfirst : 0;
  const int n = nf + min(p.nsplit, (max(ctx - own.begin, 0) + own.split - 1) / own.split);
  // partials 0..nf-1 are the first range's, nf..n-1 the own ones
  const int64_t fbase = static_cast<int64_t>(row) * nfirst;
  const int64_t obase = static_cast<int64_t>(row) * p.nsplit;
  auto ml_at = [&](int s) { return s < nf ? first_ml[fbase + s] : p.ws_ml[obase + s - nf]; };
  float mmax = neg_inf();
  for (int s = lane; s < n; s += 32) mmax = fmaxf(mmax, ml_at(s).x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    mmax = fmaxf(mmax, __shfl_xor_sync(0xffffffffu, mmax, off));
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < n; s0 += 32) {
    float wt = 0.f;
    if (s0 + lane < n) {
      const float2 ml = ml_at(s0 + lane);
      // half steps, as in the kernels: l times the factor stays in range
      const float hw = (ml.x == neg_inf()) ? 0.f : fast_exp2(0.5f * (ml.x - mmax));
      L += ml.y * hw * hw;
      wt = hw * hw;
    }
    const int cnt = min(32, n - s0);
#pragma unroll 4
    for (int i = 0; i < cnt; ++i) {
      const int s = s0 + i;
      const float* src = s < nf ? first_o + (fbase + s) * kHeadDim
                                : p.ws_o + (obase + s - nf) * kHeadDim;
      const float4 o = reinterpret_cast<const float4*>(src)[lane];
      const float w = __shfl_sync(0xffffffffu, wt, i);
      acc.x += o.x * w;
      acc.y += o.y * w;
      acc.z += o.z * w;
      acc.w += o.w * w;
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
  const float inv = n > 0 ? 1.f / L : 0.f;  // a row without keys: zeros
  __nv_bfloat16* out = p.out + static_cast<int64_t>(b) * p.o_stride_tok +
                       static_cast<int64_t>(h) * p.o_stride_head + lane * 4;
  const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
  const __nv_bfloat162 hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
  out[0] = lo.x, out[1] = lo.y, out[2] = hi.x, out[3] = hi.y;
}

int launch_merge_partials(const DecodeParams& p, const float* first_o, const float2* first_ml,
                          int nfirst, int batch, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(batch) * p.num_heads;
  if (rows > 0x7fffffffLL - kMergeWarps) return fail(NVATTN_ERR_INVALID, "decode: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + kMergeWarps - 1) / kMergeWarps));
  cfg.blockDim = dim3(kMergeWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, merge_partials_kernel, p, first_o, first_ml,
                                           nfirst, static_cast<int>(rows));
  return e == cudaSuccess ? NVATTN_OK : cuda_fail(e, "merge_partials launch");
}

static int make_cache8_map(CUtensorMap* map, const void* cache, int num_blocks, int block_size,
                           int num_kv_heads) {
  // the 128 bytes of a row as 64 two-byte elements: dims innermost first
  const uint64_t dims[4] = {kHeadDim / 2, static_cast<uint64_t>(num_kv_heads),
                            static_cast<uint64_t>(block_size), static_cast<uint64_t>(num_blocks)};
  const uint64_t row = static_cast<uint64_t>(num_kv_heads) * kHeadDim;
  const uint64_t strides[3] = {kHeadDim, row, row * block_size};
  const uint32_t box[4] = {kHeadDim / 2, 1, kTile, 1};
  return make_tensor_map(map, cache, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool kSuffix>
static int raise_smem8() {
  static std::mutex mu;
  static bool done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 64 && done[dev]) return NVATTN_OK;
  const cudaError_t e = cudaFuncSetAttribute(paged_decode_fp8_kernel<kSuffix>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem8);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_decode_fp8)");
  if (dev < 64) done[dev] = true;
  return NVATTN_OK;
}

template <bool kSuffix>
static int launch_decode_fp8(const DecodeParams& p, const void* k_cache, const void* v_cache,
                             const uint8_t* k_scale, const uint8_t* v_scale, int batch,
                             bool after_prefix, cudaStream_t stream) {
  CUtensorMap kmap, vmap;
  int rc = make_cache8_map(&kmap, k_cache, p.num_blocks, p.block_size, p.num_kv_heads);
  if (rc) return rc;
  rc = make_cache8_map(&vmap, v_cache, p.num_blocks, p.block_size, p.num_kv_heads);
  if (rc) return rc;
  rc = raise_smem8<kSuffix>();
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.nsplit, p.num_kv_heads, batch);
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = kSmem8;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_prefix ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_fp8_kernel<kSuffix>, kmap, vmap,
                                           k_scale, v_scale, p);
  return e == cudaSuccess ? NVATTN_OK : cuda_fail(e, "paged_decode_fp8 launch");
}

int launch_decode_fp8_suffix(const DecodeParams& p, const void* k_cache, const void* v_cache,
                             const uint8_t* k_scale, const uint8_t* v_scale, int batch,
                             bool after_prefix, cudaStream_t stream) {
  return launch_decode_fp8<true>(p, k_cache, v_cache, k_scale, v_scale, batch, after_prefix,
                                 stream);
}

int check_fp8_scales(const char* who, const void* k_scale, const void* v_scale) {
  if (!k_scale || !v_scale) return fail(NVATTN_ERR_INVALID, std::string(who) + ": NULL scales");
  if (!aligned16(k_scale) || !aligned16(v_scale))
    return fail(NVATTN_ERR_INVALID, std::string(who) + ": scales must be 16-byte aligned");
  return NVATTN_OK;
}

}  // namespace nvattn

using namespace nvattn;

extern "C" int nvattn_paged_decode_fp8(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
    const void* v_cache, const uint8_t* k_scale, const uint8_t* v_scale, void* out,
    int64_t o_stride_tok, int64_t o_stride_head, const int32_t* cache_seqlens,
    const int32_t* block_table, int64_t block_table_stride, int32_t max_blocks_per_seq,
    int32_t num_blocks, int32_t block_size, int32_t batch, int32_t num_heads, int32_t num_kv_heads,
    int32_t head_dim, float softmax_scale, void* workspace, size_t workspace_bytes,
    int32_t* status, void* stream) {
  clear_error();
  if (batch == 0) return NVATTN_OK;
  int rc = check_decode_args("paged_decode_fp8", q, q_stride_tok, q_stride_head, k_cache, v_cache,
                             out, cache_seqlens, block_table, block_table_stride,
                             max_blocks_per_seq, num_blocks, block_size, batch, num_heads,
                             num_kv_heads, head_dim);
  if (rc) return rc;
  rc = check_fp8_scales("paged_decode_fp8", k_scale, v_scale);
  if (rc) return rc;
  if (batch > 65535) return fail(NVATTN_ERR_UNSUPPORTED, "paged_decode_fp8: batch > 65535");

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
  p.scale_log2 = softmax_scale * kLog2e;
  p.status = status;
  choose_split(batch, num_kv_heads, max_blocks_per_seq, block_size, &p.nsplit, &p.split_tiles);
  const size_t need = decode_ws_bytes(batch, num_heads, p.nsplit);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(NVATTN_ERR_WORKSPACE, "paged_decode_fp8: workspace smaller than "
                                      "nvattn_decode_workspace_bytes()");
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(NVATTN_ERR_INVALID, "paged_decode_fp8: workspace must be 256-byte aligned");
  set_decode_workspace(&p, need > 0 ? workspace : nullptr, batch);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  rc = launch_decode_fp8<false>(p, k_cache, v_cache, k_scale, v_scale, batch, false, s);
  if (rc || p.nsplit == 1) return rc;
  return launch_merge_partials(p, nullptr, nullptr, 0, batch, s);
}
