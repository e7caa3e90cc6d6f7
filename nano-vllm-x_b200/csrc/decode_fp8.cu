// Paged split-K decode attention over the fp8 cache (layout and rounding in
// kvcache_fp8.cu): the split and the grid of decode.cu, half the bytes.
//
//   o = sum_j softmax_j(c * 2^kk_j * q.k8_j) * 2^kv_j * v8_j
//
// with k8, v8 the e4m3 elements and kk, kv the rows' exponents. No value is
// rounded on the way into the tensor cores but q (below) and the weights:
// e4m3 converts to f16 exactly, so both products run as f16 MMAs with fp32
// accumulation, the exponents are applied to the fp32 scores, and those of V
// are folded into the softmax: with t_j the score in log2 units, a warp's running
// reference is M = max_j (t_j + max(kv_j, -80)) - 15, the weights given to the
// second product are w_j = 2^(t_j + kv_j - M) <= 2^15, and the sum runs over
// 2^(t_j - M). The weights are rounded to f16, half as wide as the plain form's
// fp32: 2^-12 of a weight from 2^-29 of the reference's on (the 15 bits of f16's
// range above one are for the rows whose V is small beside the largest row's, which
// a single large channel can make: with w_j <= 1 they were off by 2^-12 only down to
// 2^-14), 2^-40 of the reference's below that. The sum's terms lie within 2^-105 and
// 2^95 of one for the keys that set M, so that neither rows of zeros (kv = -100)
// overflow it nor values near bf16's largest (kv = 120) take it below fp32's range.
// q's bf16 elements fit f16's 11 bits; its range is
// brought in by a power of two a row, so only elements below 2^-14 of the
// row's largest lose bits (2^-25 of it).
//
// HBM-bound: 258 bytes a (key, KV head) against 4 * 128 * group flops (256
// sequences of 100 to 2048 keys, 16/8 heads: 88 us, 6.1 TB/s, 0.93 of a copy's
// rate; 32 sequences of 4k to 32k keys, 64/8 heads: 177 us, 6.0 TB/s). What is
// left to hide is the arithmetic around the products, so the keys are the M rows
// of the MMAs and the query heads the 8 columns (S^T = K Q^T, O^T = V^T W^T): inside
// a tile no key is padding, and the conversions (2 a 4-byte word, plus one byte
// permute for V) serve all heads. Columns, and the quad lanes that own them, are
// padding where the heads a KV head are no multiple of 8 (6 of 8 with 2 heads). A
// warp owns whole 64-key tiles, the warps of a CTA taking turns, so maxima, barrier
// waits and rescales are paid once for 64 keys. Each warp is its own producer: it
// has room for one tile of K and one of V, and sends for the next tile's K as soon
// as the scores are out and for its V as soon as the second product is, so that
// either half is in flight while the warp works on the other. Up to 8 consecutive
// splits of a row form a cluster, whose CTAs merge through each other's shared
// memory: with no more splits than that the output is written at once, otherwise
// one fp32 partial a cluster.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "decode.cuh"

namespace nvattn {

namespace cg = cooperative_groups;

constexpr int kTile8 = kTile * kHeadDim;      // one 64-key e4m3 tile (8 KB)
// Warps of a CTA and CTAs of an SM for NB blocks of 8 query heads (registers a
// thread grow with NB). 256 sequences of 100 to 2048 keys: 4 warps x 3 CTAs 88 us;
// 6 x 2 91, 3 x 4 92, 2 x 6 94.
constexpr int kDec8Warps = 4;
constexpr int dec8_ctas(int NB) { return NB == 1 ? 3 : 2; }

// The softmax's reference (top of the file): V exponents count from the first on, and
// the largest weight is 2^ the second.
constexpr float kLowestRef8 = -80.f, kHeadroom8 = 15.f;

// Shared memory of one warp: its K and V tile, their exponent bytes.
constexpr int kWarpBytes8 = 2 * kTile8;
constexpr int kWarpScales8 = 2 * kTile;
constexpr int dec8_smem(int NB) {
  return kDec8Warps * (kWarpBytes8 + kWarpScales8 + 2 * 8 + 8 * NB * 8) + 8 * NB * 8 + 1024;
}
static_assert(16 * kOPad * 4 <= kWarpBytes8, "the merge buffer reuses the tiles");

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

// Transposes an 8 x 8 matrix of 16-bit elements held as one fragment register.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// B fragments of query head `h` (column lane / 4): a 16-dim step takes dims
// 4q..4q+3 of quad lane q (dims may be summed in any order as long as K's
// fragments agree: one 4-byte word of an e4m3 row holds them). Returns the
// exact power of two the row was divided by.
__device__ __forceinline__ float load_q8(const __nv_bfloat16* row, bool live, int quad,
                                         uint32_t qb[8][2]) {
  const uint32_t* src = reinterpret_cast<const uint32_t*>(row);
  uint32_t w[16];
  float mx = 0.f;
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    w[2 * kk] = live ? src[kk * 8 + quad * 2] : 0u;
    w[2 * kk + 1] = live ? src[kk * 8 + quad * 2 + 1] : 0u;
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
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      qb[kk][i] = pack_f16x2(__uint_as_float(w[2 * kk + i] << 16) * down,
                             __uint_as_float(w[2 * kk + i] & 0xffff0000u) * down);
  }
  return __int_as_float(e << 23);
}

// NB: blocks of 8 query heads (group <= 8 * NB). kSuffix: the keys from
// p.key_begin on, as fp32 partials for the merge with the keys before
// (shared_prefix.cu).
template <int NB, bool kSuffix>
__global__ void __launch_bounds__(kDec8Warps * 32, dec8_ctas(NB))
    paged_decode_fp8_kernel(const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap,
                            const uint8_t* __restrict__ k_scale,
                            const uint8_t* __restrict__ v_scale, const DecodeParams p) {
  constexpr int kWarps = kDec8Warps;
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
  if (tok_end <= tok_begin) {  // its cluster's other CTAs do not wait for one that ended
    if (kSuffix) join_prefix_grid();
    if (!kSuffix && p.nsplit == p.cluster && split == 0) {  // no merge runs: the empty row's zeros
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
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint8_t* ktile = smem + warp * kWarpBytes8;
  uint8_t* vtile = ktile + kTile8;
  uint8_t* ss = smem + kWarps * kWarpBytes8 + warp * kWarpScales8;  // K's bytes, then V's
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kWarps * (kWarpBytes8 + kWarpScales8));
  uint64_t* k_full = bars + 2 * warp;  // K and both rows of exponent bytes
  uint64_t* v_full = k_full + 1;
  float2* ml_smem = reinterpret_cast<float2*>(bars + 2 * kWarps);  // [warp][8 * NB heads]
  float2* ml_cta = ml_smem + kWarps * 8 * NB;                      // [8 * NB heads]

  // Lane 0 sends for the warp's tiles; `blk` is the page of the tile to send
  // for next, read from the table one tile ahead.
  const int32_t* bt = p.block_table + static_cast<int64_t>(b) * p.bt_stride;
  auto page = [&](int it) {
    if (it >= ntiles) return 0;
    const int blk = page_of(p, bt, tok_begin + it * kTile, ctx);
    if (blk >= 0 && blk < p.num_blocks) return blk;
    set_status(p.status, NVATTN_STATUS_BAD_BLOCK);
    return 0;  // read a valid block; the result is flagged as invalid
  };
  auto send_k = [&](int it, int blk) {
    const int tin = (tok_begin + it * kTile) % p.block_size;
    const int64_t sc = (static_cast<int64_t>(blk) * p.num_kv_heads + g) * p.block_size + tin;
    mbar_arrive_expect_tx(k_full, kTile8 + kWarpScales8);
    tma_load_4d(ktile, &kmap, k_full, 0, g, tin, blk);
    bulk_load(ss, k_scale + sc, kTile, k_full);
    bulk_load(ss + kTile, v_scale + sc, kTile, k_full);
  };
  auto send_v = [&](int it, int blk) {
    mbar_arrive_expect_tx(v_full, kTile8);
    tma_load_4d(vtile, &vmap, v_full, 0, g, (tok_begin + it * kTile) % p.block_size, blk);
  };
  if (lane == 0 && warp < ntiles) {
    mbar_init(k_full, 1);
    mbar_init(v_full, 1);
    fence_barrier_init();
    const int blk = page(warp);
    send_k(warp, blk);
    send_v(warp, blk);
  }
  __syncwarp();

  // -------------------------------------------------------------- consumers
  const int quad = lane & 3;  // this lane's head columns 2*quad, 2*quad + 1 of each block
  const int sub = lane >> 2;  // its key (or dim pair) inside 8
  const int h0 = g * p.group;

  uint32_t qb[NB][8][2];
  float scale[NB][2];  // of head columns 2*quad, 2*quad + 1
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = nb * 8 + sub;
    const float back =
        load_q8(p.q + static_cast<int64_t>(b) * p.q_stride_tok +
                    static_cast<int64_t>(h0 + min(r, p.group - 1)) * p.q_stride_head,
                r < p.group, quad, qb[nb]);
    scale[nb][0] = __shfl_sync(0xffffffffu, back, quad * 8) * p.scale_log2;
    scale[nb][1] = __shfl_sync(0xffffffffu, back, quad * 8 + 4) * p.scale_log2;
  }

  // o[c][nb][2e + j]: dim 16c + 2*sub + e of head column 2*quad + j
  float o[8][NB][4];
  float m[NB][2], l[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c][nb][0] = o[c][nb][1] = o[c][nb][2] = o[c][nb][3] = 0.f;
    m[nb][0] = m[nb][1] = neg_inf();
    l[nb][0] = l[nb][1] = 0.f;
  }

  // ldmatrix addresses: row lane % 16 of a 16-key step, chunk pair member
  // lane / 16 (128-byte rows, 128-byte swizzle)
  uint32_t off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) off[i] = swz128(lane & 15, 2 * i + (lane >> 4));

  const uint32_t kbase = smem_u32(ktile), vbase = smem_u32(vtile);
  bool timed_out = false;
  uint32_t phase = 0;
  for (int it = warp; it < ntiles; it += kWarps, phase ^= 1) {
    const int next = it + kWarps;
    int next_blk = 0;
    if (lane == 0) next_blk = page(next);
    if (!__all_sync(0xffffffffu, mbar_wait(k_full, phase))) {
      timed_out = true;
      break;
    }
    const int nvalid = min(kTile, tok_end - (tok_begin + it * kTile));
    // ---- S^T = K Q^T: 4 steps of 16 keys, 8 of 16 dims
    float s[4][NB][4];  // [mt][nb][2e + j]: key 16mt + 8e + sub, head column 2*quad + j
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[mt][nb][0] = s[mt][nb][1] = s[mt][nb][2] = s[mt][nb][3] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        uint32_t w[4];  // this lane's 4 bytes: keys 0-7 and 8-15 of steps 2i, 2i + 1
        ldmatrix_x4(kbase + mt * 2048 + off[i], w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t a[4] = {e4m3x2_to_f16x2(w[2 * j]), e4m3x2_to_f16x2(w[2 * j + 1]),
                                 e4m3x2_to_f16x2(w[2 * j] >> 16),
                                 e4m3x2_to_f16x2(w[2 * j + 1] >> 16)};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            mma_f16_16816(s[mt][nb], a, qb[nb][2 * i + j][0], qb[nb][2 * i + j][1]);
        }
      }
    }
    // ---- exponents, mask, online softmax
    float ve[4][2];  // exponents of V, [mt][e]
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = mt * 16 + e * 8 + sub;
        const float kf = exp_byte_scale(ss[t]);
        ve[mt][e] = exp_byte_log2(ss[kTile + t]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          s[mt][nb][2 * e] *= scale[nb][0] * kf;
          s[mt][nb][2 * e + 1] *= scale[nb][1] * kf;
        }
      }
    }
    __syncwarp();  // K and the exponents are read: the next tile's may land
    if (lane == 0 && next < ntiles) send_k(next, next_blk);
    if (nvalid < kTile) {  // keys past the end: stale bytes
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (mt * 16 + e * 8 + sub >= nvalid) {
            ve[mt][e] = 0.f;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[mt][nb][2 * e] = s[mt][nb][2 * e + 1] = neg_inf();
          }
        }
      }
    }
    float mn[NB][2];
    bool grew = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = neg_inf();
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
          mx = fmax3(mx, s[mt][nb][j] + fmaxf(ve[mt][0], kLowestRef8),
                     s[mt][nb][2 + j] + fmaxf(ve[mt][1], kLowestRef8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mn[nb][j] = fmaxf(m[nb][j], mx - kHeadroom8);
        grew |= mn[nb][j] > m[nb][j];
      }
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // l in two half steps: with V rows of very different magnitudes the
          // factor alone can leave fp32's range while its product with l does not
          const float h = fast_exp2(0.5f * (m[nb][j] - mn[nb][j]));
          l[nb][j] = l[nb][j] * h * h;
          const float al = h * h;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            o[c][nb][j] *= al;
            o[c][nb][2 + j] *= al;
          }
          m[nb][j] = mn[nb][j];
        }
      }
    }
    // ---- O^T += V^T W^T: 4 steps of 16 keys
    if (!__all_sync(0xffffffffu, mbar_wait(v_full, phase))) {
      timed_out = true;
      break;
    }
    if (nvalid < kTile) {
      // Zero the V rows past the end (maybe NaN), so that 0 * NaN never reaches
      // the sum. Only a range's last tile has them: no later copy lands here.
      for (int e = lane; e < (kTile - nvalid) * 8; e += 32)
        *reinterpret_cast<int4*>(vtile + nvalid * 128 + e * 16) = make_int4(0, 0, 0, 0);
      __syncwarp();
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      uint32_t wb[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float t0 = s[mt][nb][2 * e] - m[nb][0], t1 = s[mt][nb][2 * e + 1] - m[nb][1];
          l[nb][0] += fast_exp2(t0);
          l[nb][1] += fast_exp2(t1);
          wb[nb][e] = transpose8x8(
              pack_f16x2(fast_exp2(t0 + ve[mt][e]), fast_exp2(t1 + ve[mt][e])));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // keys 2q, 2q+1 of dims 2*sub, 2*sub+1: keys 0-7 and 8-15 of chunks 2i, 2i + 1
        uint32_t r[4];
        ldmatrix_x4_trans(vbase + mt * 2048 + off[i], r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t lo = __byte_perm(r[2 * j], 0, 0x3120);  // pair the keys
          const uint32_t hi = __byte_perm(r[2 * j + 1], 0, 0x3120);
          const uint32_t a[4] = {e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16),
                                 e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16)};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            mma_f16_16816(o[2 * i + j][nb], a, wb[nb][0], wb[nb][1]);
        }
      }
    }
    __syncwarp();
    if (lane == 0 && next < ntiles) send_v(next, next_blk);
  }
  if (timed_out) {  // the copies in flight, again with a limit
    mbar_wait(k_full, phase);
    mbar_wait(k_full, phase ^ 1);
    mbar_wait(v_full, phase);
    if (lane == 0) set_status(p.status, NVATTN_STATUS_TIMEOUT);
  }

  // ---------------------------------------------------------------- merge
  __syncthreads();  // all warps are past their tiles: reuse them
  float* obuf = reinterpret_cast<float*>(smem);  // [warp][8 * NB heads][kOPad]
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = warp * 8 * NB + nb * 8 + quad * 2 + j;
      float sum = l[nb][j];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (sub == 0) ml_smem[r] = make_float2(m[nb][j], sum);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<float2*>(obuf + r * kOPad + c * 16 + sub * 2) =
            make_float2(o[c][nb][j], o[c][nb][2 + j]);
    }
  }
  __syncthreads();

  const int first = split - split % p.cluster;
  const int live = min(p.cluster, (ctx - own.begin + own.split - 1) / own.split - first);
  const int64_t slot0 = (static_cast<int64_t>(b) * p.num_heads + h0) * (p.nsplit / p.cluster) +
                        split / p.cluster;
  auto put = [&](int r, int d, float mmax, float L, float acc) {
    if (!kSuffix && p.nsplit == p.cluster) {
      p.out[static_cast<int64_t>(b) * p.o_stride_tok +
            static_cast<int64_t>(h0 + r) * p.o_stride_head + d] = __float2bfloat16_rn(acc / L);
    } else {
      const int64_t slot = slot0 + static_cast<int64_t>(r) * (p.nsplit / p.cluster);
      p.ws_o[slot * kHeadDim + d] = acc;
      if (d == 0) p.ws_ml[slot] = make_float2(mmax, L);
    }
  };
  // over the CTA's warps, in place: element (r, d) is one thread's
  for (int e = threadIdx.x; e < p.group * kHeadDim; e += kWarps * 32) {
    const int r = e / kHeadDim, d = e % kHeadDim;
    float mmax = neg_inf();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mmax = fmaxf(mmax, ml_smem[w * 8 * NB + r].x);
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      // a warp without a tile keeps m = -inf, l = 0, o = 0
      const float2 ml = ml_smem[w * 8 * NB + r];
      const float h = (ml.x == neg_inf()) ? 0.f : fast_exp2(0.5f * (ml.x - mmax));
      L += ml.y * h * h;
      acc += obuf[(w * 8 * NB + r) * kOPad + d] * h * h;
    }
    if (live == 1) {
      put(r, d, mmax, L, acc);
    } else {
      obuf[r * kOPad + d] = acc;
      if (d == 0) ml_cta[r] = make_float2(mmax, L);
    }
  }
  if (live == 1) {
    if (kSuffix) join_prefix_grid();
    return;
  }
  // over the cluster's splits that have keys: the first ones
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int e = (split - first) * kWarps * 32 + threadIdx.x; e < p.group * kHeadDim;
       e += live * kWarps * 32) {
    const int r = e / kHeadDim, d = e % kHeadDim;
    float mmax = neg_inf();
    for (int c = 0; c < live; ++c) mmax = fmaxf(mmax, cluster.map_shared_rank(ml_cta, c)[r].x);
    float L = 0.f, acc = 0.f;
#pragma unroll 4
    for (int c = 0; c < live; ++c) {
      const float2 ml = cluster.map_shared_rank(ml_cta, c)[r];
      const float h = (ml.x == neg_inf()) ? 0.f : fast_exp2(0.5f * (ml.x - mmax));
      L += ml.y * h * h;
      acc += cluster.map_shared_rank(obuf, c)[r * kOPad + d] * h * h;
    }
    put(r, d, mmax, L, acc);
  }
  cluster.sync();  // no CTA ends while the others read from it
  if (kSuffix) join_prefix_grid();
}

// Merges the partials of one (sequence, query head), W warps a row: lane i owns
// dims 4i..4i+3, a warp every W-th partial. Launched as a programmatic
// dependent of the kernel that writes the last partials. Latency-bound: a warp
// has four partials in flight, so many partials want several warps a row.
constexpr int kMergeThreads = 256;

template <int W>
__global__ void __launch_bounds__(kMergeThreads)
    merge_partials_kernel(const DecodeParams p, const float* __restrict__ first_o,
                          const float2* __restrict__ first_ml, int nfirst, int rows) {
  constexpr int kRows = kMergeThreads / 32 / W;
  __shared__ float4 part[W > 1 ? kMergeThreads : 1];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wr = warp % W;
  const int row = min(static_cast<int>(blockIdx.x) * kRows + warp / W, rows - 1);
  const int b = row / p.num_heads, h = row - b * p.num_heads;
  const int ctx = min(p.seqlens[b], p.max_blocks * p.block_size);
  const KeyRange own = own_keys(p, ctx);
  const int nf = own.begin > 0 ? nfirst : 0;
  const int nparts = p.nsplit / p.cluster, part_keys = own.split * p.cluster;
  const int n = nf + min(nparts, (max(ctx - own.begin, 0) + part_keys - 1) / part_keys);
  // partials 0..nf-1 are the first range's, nf..n-1 the own ones
  const int64_t fbase = static_cast<int64_t>(row) * nfirst;
  const int64_t obase = static_cast<int64_t>(row) * nparts - nf;
  auto ml_at = [&](int s) { return s < nf ? first_ml[fbase + s] : p.ws_ml[obase + s]; };
  float mmax = neg_inf();
  for (int s = lane; s < n; s += 32) mmax = fmaxf(mmax, ml_at(s).x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    mmax = fmaxf(mmax, __shfl_xor_sync(0xffffffffu, mmax, off));
  // half steps, as in the kernels: l times the factor stays in range
  auto half = [&](float m) { return m == neg_inf() ? 0.f : fast_exp2(0.5f * (m - mmax)); };
  float L = 0.f;
  for (int s = lane; s < n; s += 32) {
    const float2 ml = ml_at(s);
    const float hw = half(ml.x);
    L += ml.y * hw * hw;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = wr; s < n; s += W) {
    const float* src = s < nf ? first_o + (fbase + s) * kHeadDim : p.ws_o + (obase + s) * kHeadDim;
    const float4 o = reinterpret_cast<const float4*>(src)[lane];
    const float hw = half(ml_at(s).x), w = hw * hw;
    acc.x += o.x * w;
    acc.y += o.y * w;
    acc.z += o.z * w;
    acc.w += o.w * w;
  }
  if (W > 1) {
    part[threadIdx.x] = acc;
    __syncthreads();
    if (wr != 0) return;
#pragma unroll
    for (int i = 1; i < W; ++i) {
      const float4 o = part[threadIdx.x + 32 * i];
      acc.x += o.x;
      acc.y += o.y;
      acc.z += o.z;
      acc.w += o.w;
    }
  }
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
  if (rows > 0x7fffffffLL - kMergeThreads)
    return fail(NVATTN_ERR_INVALID, "decode: too many rows");
  // Warps a row: eight for many partials (131071 keys, 32 of them); otherwise as
  // many as have two partials each, while all rows run at once, 64 warps an SM
  // (2048 rows of up to 15: the call 183 us with one, 179 with four; 80 rows of
  // 12: 12.9 with one, 11.3 with eight; 6400 rows: 67 with one, 69 with two).
  const int parts = nfirst + p.nsplit / p.cluster;
  const int64_t room = 64 * static_cast<int64_t>(device_sm_count());
  int w = 1;
  while (w < kMergeThreads / 32 && (parts > 16 || (parts >= 2 * w && rows * 2 * w <= room))) w *= 2;
  const int per_cta = kMergeThreads / 32 / w;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + per_cta - 1) / per_cta));
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const auto kernel = w == 8   ? merge_partials_kernel<8>
                      : w == 4 ? merge_partials_kernel<4>
                      : w == 2 ? merge_partials_kernel<2>
                               : merge_partials_kernel<1>;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, kernel, p, first_o, first_ml, nfirst, static_cast<int>(rows));
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

template <int NB, bool kSuffix>
static int raise_smem8() {
  static std::mutex mu;
  static bool done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 64 && done[dev]) return NVATTN_OK;
  const cudaError_t e = cudaFuncSetAttribute(paged_decode_fp8_kernel<NB, kSuffix>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, dec8_smem(NB));
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_decode_fp8)");
  if (dev < 64) done[dev] = true;
  return NVATTN_OK;
}

template <int NB, bool kSuffix>
static int launch_decode_fp8(const DecodeParams& p, const void* k_cache, const void* v_cache,
                             const uint8_t* k_scale, const uint8_t* v_scale, int batch,
                             cudaStream_t stream) {
  CUtensorMap kmap, vmap;
  int rc = make_cache8_map(&kmap, k_cache, p.num_blocks, p.block_size, p.num_kv_heads);
  if (rc) return rc;
  rc = make_cache8_map(&vmap, v_cache, p.num_blocks, p.block_size, p.num_kv_heads);
  if (rc) return rc;
  rc = raise_smem8<NB, kSuffix>();
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.nsplit, p.num_kv_heads, batch);
  cfg.blockDim = dim3(kDec8Warps * 32);
  cfg.dynamicSmemBytes = dec8_smem(NB);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kSuffix ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_fp8_kernel<NB, kSuffix>, kmap, vmap,
                                           k_scale, v_scale, p);
  return e == cudaSuccess ? NVATTN_OK : cuda_fail(e, "paged_decode_fp8 launch");
}

int launch_decode_fp8_whole(const DecodeParams& p, const void* k_cache, const void* v_cache,
                            const uint8_t* k_scale, const uint8_t* v_scale, int batch,
                            cudaStream_t stream) {
  const int rc = p.group <= 8 ? launch_decode_fp8<1, false>(p, k_cache, v_cache, k_scale, v_scale,
                                                            batch, stream)
                              : launch_decode_fp8<2, false>(p, k_cache, v_cache, k_scale, v_scale,
                                                            batch, stream);
  if (rc || p.nsplit == p.cluster) return rc;
  return launch_merge_partials(p, nullptr, nullptr, 0, batch, stream);
}

int launch_decode_fp8_suffix(const DecodeParams& p, const void* k_cache, const void* v_cache,
                             const uint8_t* k_scale, const uint8_t* v_scale, int batch,
                             cudaStream_t stream) {
  return p.group <= 8
             ? launch_decode_fp8<1, true>(p, k_cache, v_cache, k_scale, v_scale, batch, stream)
             : launch_decode_fp8<2, true>(p, k_cache, v_cache, k_scale, v_scale, batch, stream);
}

// Splits of a row, in 64-key tiles: the largest of 32/16/8/4 that gives 8 CTAs
// an SM when every row is at the table's width; a batch too small for that
// keeps 8 where they still cover the SMs once (two tiles a warp), and 4 (one)
// otherwise. A batch whose splits all run at once merges them in clusters of up
// to 8. Depends on host sizes only, so a captured graph keeps its grid.
void choose_split_fp8(int batch, int num_kv_heads, int64_t max_keys, int* nsplit,
                      int* split_tiles, int* cluster) {
  const int sms = device_sm_count();
  const int64_t tiles = std::max<int64_t>(1, (max_keys + kTile - 1) / kTile);
  const int64_t pairs = static_cast<int64_t>(batch) * num_kv_heads;
  int st = 32;
  while (st > 4 && pairs * ((tiles + st - 1) / st) < (st > 8 ? 8 : 1) * static_cast<int64_t>(sms))
    st >>= 1;
  const int64_t ns = (tiles + st - 1) / st;
  // Clusters save the merge's launch and its reads (1 x 777 keys: 6.4 -> 5.6 us),
  // but their CTAs wait for one another: with more CTAs than the SMs hold at
  // once that keeps others from starting (32 long contexts: 179 -> 194 us).
  int c = 1;
  while (pairs * ns <= 2 * static_cast<int64_t>(sms) && c < 8 && c < ns) c *= 2;
  *split_tiles = st;
  *cluster = c;
  *nsplit = static_cast<int>((ns + c - 1) / c * c);
}

int check_fp8_scales(const char* who, const void* k_scale, const void* v_scale) {
  if (!k_scale || !v_scale) return fail(NVATTN_ERR_INVALID, std::string(who) + ": NULL scales");
  if (!aligned16(k_scale) || !aligned16(v_scale))
    return fail(NVATTN_ERR_INVALID, std::string(who) + ": scales must be 16-byte aligned");
  return NVATTN_OK;
}

int check_table_keys(const char* who, int32_t max_blocks_per_seq, int32_t block_size) {
  if (static_cast<int64_t>(max_blocks_per_seq) * block_size > (1 << 30))
    return fail(NVATTN_ERR_UNSUPPORTED, std::string(who) + ": table of more than 2^30 keys");
  return NVATTN_OK;
}

}  // namespace nvattn

using namespace nvattn;

extern "C" size_t nvattn_decode_fp8_workspace_bytes(int32_t batch, int32_t num_heads,
                                                    int32_t num_kv_heads,
                                                    int32_t max_blocks_per_seq,
                                                    int32_t block_size) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || max_blocks_per_seq <= 0 ||
      block_size <= 0)
    return 0;
  int nsplit, split_tiles, cluster;
  choose_split_fp8(batch, num_kv_heads,
                   static_cast<int64_t>(max_blocks_per_seq) * block_size, &nsplit, &split_tiles,
                   &cluster);
  return decode_ws_bytes(batch, num_heads, nsplit / cluster);
}

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
  rc = check_table_keys("paged_decode_fp8", max_blocks_per_seq, block_size);
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
  choose_split_fp8(batch, num_kv_heads,
                   static_cast<int64_t>(max_blocks_per_seq) * block_size, &p.nsplit,
                   &p.split_tiles, &p.cluster);
  const size_t need = decode_ws_bytes(batch, num_heads, p.nsplit / p.cluster);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(NVATTN_ERR_WORKSPACE, "paged_decode_fp8: workspace smaller than "
                                      "nvattn_decode_fp8_workspace_bytes()");
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(NVATTN_ERR_INVALID, "paged_decode_fp8: workspace must be 256-byte aligned");
  set_decode_workspace(&p, need > 0 ? workspace : nullptr, batch);
  return launch_decode_fp8_whole(p, k_cache, v_cache, k_scale, v_scale, batch,
                                 reinterpret_cast<cudaStream_t>(stream));
}
