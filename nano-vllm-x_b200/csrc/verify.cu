// Verification of drafted tokens against the target model's probabilities from
// given random numbers (no counterpart in the reference): the step between
// tree-verification attention and the compaction of the accepted path.
//
// Node 0 is the root (the last committed token); node j > 0 holds a drafted
// token. Row j of `logits` is the target's answer after node j, p_j =
// softmax(logits_j / T). The walk starts at the root; at node a with children
// c1 < c2 < ... (in a chain, the one next node):
//   proposals without probabilities: the tokens are tried in order and c_i is
//   accepted iff u_c * R < p_a(x_c), R = 1 - sum of the p_a of the siblings
//   tried before (a token tried before has no probability left); when none is
//   accepted, one token is drawn from p_a without the rejected ones;
//   proposals from a draft model (a chain), q_a = softmax(draft_a / T): accept
//   iff u_c * q_a(x_c) < p_a(x_c); else draw from max(p_a - q_a, 0).
// At a node without children the draw is from p_a itself. Either rule leaves
// the tokens distributed as the target's. The draw is by inversion: the first
// token whose cumulative weight exceeds u * total. T <= 0: a child is accepted
// iff it is the argmax, the draw is the argmax.
//
// Only the rows on the walked path are read, each once: one cluster of CTAs
// per sequence walks it, every CTA holding its slice of the current row in
// shared memory, and every CTA takes the same decisions from the same
// exchanged sums. HBM-bound while rows stream (two bytes a logit), one cluster
// barrier a node.
//
// The answers are tokens, so sums that decide between neighbours are kept in
// 64 bits: the draw's cumulative weights always (with 151,936 weights of which
// many are near 1e-6, sums in fp32 would move a border past u in about one
// draw in a hundred), an acceptance when the fp32 sums leave its outcome
// within 2^-14 of the border. 2^t in fp64 is table-driven (P. T. P. Tang, ACM
// TOMS 15(2), 1989): t = k/256 + f, |f| <= 1/512, 2^t = 2^(k>>8) * T[k & 255]
// * 2^f with a degree-4 polynomial (error z^5/120 < 4e-17 at z = f ln 2).
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"

namespace nvattn {

namespace cg = cooperative_groups;

constexpr int kVerifyCluster = 8;
constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxNodes = 64;
constexpr int kMaxVocab = 393216;  // a slice of the target's and the draft's row fit shared memory
constexpr int kExpTable = 256;

struct VerifyParams {
  const __nv_bfloat16* logits;
  int64_t l_stride_seq, l_stride_row;
  const __nv_bfloat16* draft;  // null: proposals without probabilities
  int64_t d_stride_seq, d_stride_row;
  const int64_t* tokens;       // (batch, nodes - 1)
  const int32_t* parents;      // null: a chain
  int64_t parents_stride;
  const float* u_accept;       // (batch, nodes - 1)
  const float* u_pick;         // (batch)
  const float* temperatures;   // null: greedy
  const int32_t* num_nodes;    // null: all
  int32_t nodes, vocab, slice;
  int64_t* out_tokens;
  int32_t* out_path;
  int32_t* out_num;
};

// What a CTA tells the others of its slice.
struct VerifySums {
  unsigned long long key;  // largest logit and its first column (pick_key order)
  float qmax;
  double psum, qsum;       // sums of exponentials, or of weights
};

struct VerifyShared {
  VerifySums sums[2];
  double warp_a[kVerifyWarps], warp_b[kVerifyWarps];
  unsigned long long warp_key[kVerifyWarps];
  float warp_q[kVerifyWarps];
  // the cluster's totals
  float pmax, qmax;
  int argmax, owner;
  double psum, qsum, base;
  int32_t parents[kMaxNodes];
  int next, count, nrejected, ambiguous;
  int32_t path[kMaxNodes + 1];
  int64_t rejected[kMaxNodes];
  double table[kExpTable];
};

__device__ __forceinline__ unsigned long long vkey(float s, uint32_t col) {
  uint32_t b = __float_as_uint(s == 0.f ? 0.f : s);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(b) << 32) | (0xFFFFFFFFu - col);
}

__device__ __forceinline__ float vkey_score(unsigned long long key) {
  const uint32_t b = static_cast<uint32_t>(key >> 32);
  return key == 0ull ? -INFINITY : __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

// fp64 value of a bf16 (zero and subnormals become +-2^-127 and above, far
// below any logit's spacing that matters).
__device__ __forceinline__ double bf16_to_f64(uint32_t b) {
  const uint32_t hi = ((b & 0x8000u) << 16) | (((b & 0x7fffu) << 13) + (896u << 20));
  return __hiloint2double(static_cast<int>(hi), 0);
}

// 2^((l - top) * c) in fp64 for a bf16 logit; 0 for NaN and far below.
__device__ __forceinline__ double weight64(uint32_t bits, uint32_t top_bits, double c, double top_c,
                                           const double* __restrict__ table) {
  if (bits == top_bits) return 1.0;  // also where the largest logit is infinite
  const double t = fma(bf16_to_f64(bits), c, -top_c);
  if ((bits & 0x7fffu) > 0x7f80u || !(t > -1000.0)) return 0.0;
  const double shift = 26388279066624.0;  // 1.5 * 2^44: rounds to multiples of 2^-8
  const double s = t + shift;
  const int k = __double2loint(s);
  const double z = (t - (s - shift)) * 0.693147180559945309417;
  double e = fma(z, 1.0 / 24.0, 1.0 / 6.0);
  e = fma(e, z, 0.5);
  e = fma(e, z, 1.0);
  const double tj = table[k & (kExpTable - 1)];
  const double r = fma(e * z, tj, tj);
  return __hiloint2double(__double2hiint(r) + ((k >> 8) << 20), __double2loint(r));
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Columns [x0, x0 + len) of a row into `buf` (16-byte aligned), at the row's
// own alignment: column x0 + i lands at buf[s + i], s = the return value; the
// rest of the first and last 16-byte group is -inf. Each thread folds what it
// loads into its best (score, column).
__device__ __forceinline__ int load_slice(const __nv_bfloat16* row, int x0, int len,
                                          unsigned short* buf, float& best, uint32_t& bcol) {
  const unsigned short* src = reinterpret_cast<const unsigned short*>(row) + x0;
  const int s = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) >> 1);
  const int groups = (s + len + 7) / 8;
  for (int gi = threadIdx.x; gi < groups; gi += kVerifyThreads) {
    const int at = gi * 8 - s;
    uint32_t w[4];
    if (at >= 0 && at + 8 <= len) {
      const int4 v = __ldg(reinterpret_cast<const int4*>(src + at));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = at + 2 * e;
        const uint32_t lo = (i >= 0 && i < len) ? __ldg(src + i) : 0xff80u;
        const uint32_t hi = (i + 1 >= 0 && i + 1 < len) ? __ldg(src + i + 1) : 0xff80u;
        w[e] = lo | (hi << 16);
      }
    }
    reinterpret_cast<int4*>(buf)[gi] = make_int4(w[0], w[1], w[2], w[3]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float l = __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
      if (l > best) {  // columns come in increasing order: the first of equals stays
        best = l;
        bcol = static_cast<uint32_t>(x0 + at + e);
      }
    }
  }
  return s;
}

// Sum over the slice of 2^((l - top) * c), fp32 terms and fp64 totals.
__device__ __forceinline__ double slice_sum32(const unsigned short* buf, int s, int len, float top,
                                              float c) {
  if (top == -INFINITY) return 0.0;  // nothing but -inf and NaN
  const int groups = (s + len + 7) / 8;
  float acc[2] = {0.f, 0.f};
  for (int gi = threadIdx.x; gi < groups; gi += kVerifyThreads) {
    const int4 v = reinterpret_cast<const int4*>(buf)[gi];
    const uint32_t w[4] = {static_cast<uint32_t>(v.x), static_cast<uint32_t>(v.y),
                           static_cast<uint32_t>(v.z), static_cast<uint32_t>(v.w)};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float l = __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
      // NaN compares false; the top itself is 1 even where it is infinite
      acc[e & 1] += l == top ? 1.f : (l < top ? fast_exp2((l - top) * c) : 0.f);
    }
  }
  return static_cast<double>(acc[0]) + static_cast<double>(acc[1]);
}

template <bool kDraft>
__global__ void __cluster_dims__(kVerifyCluster, 1, 1) __launch_bounds__(kVerifyThreads)
    verify_kernel(const VerifyParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / kVerifyCluster;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  extern __shared__ __align__(16) uint8_t smem[];
  VerifyShared& sh = *reinterpret_cast<VerifyShared*>(smem);
  const size_t head = (sizeof(VerifyShared) + 15) & ~size_t(15);
  unsigned short* pbuf = reinterpret_cast<unsigned short*>(smem + head);
  unsigned short* qbuf = pbuf + p.slice + 16;

  const int x0 = min(rank * p.slice, p.vocab);
  const int len = min(p.slice, p.vocab - x0);
  const int n = p.num_nodes ? min(max(p.num_nodes[b], 0), p.nodes) : p.nodes;
  const float temp = p.temperatures ? p.temperatures[b] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double c64 = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(temp);
  const float c32 = static_cast<float>(c64);
  const int64_t* tokens = p.tokens + static_cast<int64_t>(b) * (p.nodes - 1);
  const float* u = p.u_accept + static_cast<int64_t>(b) * (p.nodes - 1);

  if (n == 0) {  // a padding row (uniform over the cluster)
    for (int i = tid; rank == 0 && i < p.nodes; i += kVerifyThreads) {
      p.out_tokens[static_cast<int64_t>(b) * p.nodes + i] = -1;
      p.out_path[static_cast<int64_t>(b) * p.nodes + i] = -1;
    }
    if (rank == 0 && tid == 0) p.out_num[b] = 0;
    return;
  }
  for (int i = tid; i < p.nodes; i += kVerifyThreads)
    sh.parents[i] = p.parents ? p.parents[static_cast<int64_t>(b) * p.parents_stride + i] : i - 1;
  for (int i = tid; i < kExpTable; i += kVerifyThreads)
    sh.table[i] = exp2(static_cast<double>(i) / kExpTable);
  if (tid == 0) {
    sh.count = 0;
    sh.path[0] = 0;
  }
  int parity = 0;

  // Adds up what every CTA of the cluster wrote to its sums[parity]: totals
  // relative to the cluster's largest logit when `scaled` (sums of
  // exponentials), plain totals and the owner of the draw's threshold
  // otherwise. Ends with the totals visible to the whole CTA.
  auto exchange = [&](bool scaled) {
    cluster.sync();
    if (warp == 0) {
      const VerifySums* mine = &sh.sums[parity];
      VerifySums v{0ull, -INFINITY, 0.0, 0.0};
      if (lane < kVerifyCluster) v = *cluster.map_shared_rank(mine, lane);
      unsigned long long key = v.key;
      float qm = v.qmax;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k2 = __shfl_xor_sync(0xffffffffu, key, o);
        key = k2 > key ? k2 : key;
        qm = fmaxf(qm, __shfl_xor_sync(0xffffffffu, qm, o));
      }
      if (scaled) {
        const float pm = vkey_score(key), m = vkey_score(v.key);
        const double ps = warp_sum(m == pm ? v.psum
                                           : (m > -INFINITY ? v.psum * exp2((static_cast<double>(m) - pm) * c64) : 0.0));
        const double qs = warp_sum(v.qmax == qm ? v.qsum
                                                : (v.qmax > -INFINITY ? v.qsum * exp2((static_cast<double>(v.qmax) - qm) * c64) : 0.0));
        if (lane == 0) {
          sh.pmax = pm;
          sh.qmax = qm;
          sh.psum = ps;
          sh.qsum = qs;
          sh.argmax = key ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)) : 0;
        }
      } else {
        // inclusive prefix over the ranks, in rank order
        double run = 0.0, incl = 0.0;
        for (int r = 0; r < kVerifyCluster; ++r) {
          run += __shfl_sync(0xffffffffu, v.psum, r);
          if (lane == r) incl = run;
        }
        const double threshold = static_cast<double>(fmaxf(p.u_pick[b], 0.f)) * run;
        const unsigned over = __ballot_sync(0xffffffffu, lane < kVerifyCluster && incl > threshold);
        const unsigned some = __ballot_sync(0xffffffffu, lane < kVerifyCluster && v.psum > 0.0);
        const int owner = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : 0);
        const double before = __shfl_sync(0xffffffffu, incl - v.psum, owner);
        if (lane == 0) {
          sh.psum = run;
          sh.base = threshold - before;  // what the owner's own weights have to exceed
          sh.owner = owner;
        }
      }
    }
    parity ^= 1;
    __syncthreads();
  };

  int node = 0;
  bool have_draft_row = false;
  int ps = 0, qs = 0;  // where the slices start in their buffers
  while (true) {
    // ---- the row's slice, its largest logit and its sum of exponentials
    const __nv_bfloat16* prow = p.logits + static_cast<int64_t>(b) * p.l_stride_seq +
                                static_cast<int64_t>(node) * p.l_stride_row;
    float best = -INFINITY, qbest = -INFINITY;
    uint32_t bcol = 0, qcol = 0;
    ps = load_slice(prow, x0, len, pbuf, best, bcol);
    const bool has_child = kDraft ? node + 1 < n : true;
    have_draft_row = kDraft && has_child && !greedy;
    const __nv_bfloat16* qrow = nullptr;
    if (have_draft_row) {
      qrow = p.draft + static_cast<int64_t>(b) * p.d_stride_seq +
             static_cast<int64_t>(node) * p.d_stride_row;
      qs = load_slice(qrow, x0, len, qbuf, qbest, qcol);
    }
    unsigned long long key = best > -INFINITY ? vkey(best, bcol) : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k2 = __shfl_xor_sync(0xffffffffu, key, o);
      key = k2 > key ? k2 : key;
      qbest = fmaxf(qbest, __shfl_xor_sync(0xffffffffu, qbest, o));
    }
    if (lane == 0) {
      sh.warp_key[warp] = key;
      sh.warp_q[warp] = qbest;
    }
    __syncthreads();
    key = 0ull;
    qbest = -INFINITY;
    for (int w = 0; w < kVerifyWarps; ++w) {
      key = sh.warp_key[w] > key ? sh.warp_key[w] : key;
      qbest = fmaxf(qbest, sh.warp_q[w]);
    }
    if (!greedy) {
      const double a = warp_sum(slice_sum32(pbuf, ps, len, vkey_score(key), c32));
      const double d = have_draft_row ? warp_sum(slice_sum32(qbuf, qs, len, qbest, c32)) : 0.0;
      if (lane == 0) {
        sh.warp_a[warp] = a;
        sh.warp_b[warp] = d;
      }
      __syncthreads();
    }
    if (tid == 0) {
      VerifySums v{key, qbest, 0.0, 0.0};
      for (int w = 0; !greedy && w < kVerifyWarps; ++w) {
        v.psum += sh.warp_a[w];
        v.qsum += sh.warp_b[w];
      }
      sh.sums[parity] = v;
    }
    exchange(true);

    // ---- which child goes on. Warp 0 of every CTA takes the same decision.
    // exact: the sums are fp64's own; otherwise an outcome within 2^-14 of
    // its border is left open (fp32 terms put the sums off by < 2^-18).
    auto decide = [&](bool exact) {
      if (warp != 0) return;
      const uint32_t top = __float_as_uint(sh.pmax) >> 16;
      const uint32_t qtop = __float_as_uint(sh.qmax) >> 16;
      const double top_c = static_cast<double>(sh.pmax) * c64;
      const double qtop_c = static_cast<double>(sh.qmax) * c64;
      int next = -1, nrej = 0, open = 0;
      double left = 1.0;
      for (int c0 = node + 1; c0 < n && next < 0 && !open; c0 += 32) {
        const int c = c0 + lane;
        const bool mine = c < n && sh.parents[c] == node;
        int64_t tok = mine ? tokens[c - 1] : -1;
        const bool in = mine && tok >= 0 && tok < p.vocab;
        double here = 0.0, against = 0.0;
        if (in && !greedy && sh.psum > 0.0) {
          here = weight64(reinterpret_cast<const unsigned short*>(prow)[tok], top, c64, top_c,
                          sh.table) / sh.psum;
          if (kDraft && sh.qsum > 0.0)
            against = weight64(reinterpret_cast<const unsigned short*>(qrow)[tok], qtop, c64,
                               qtop_c, sh.table) / sh.qsum;
        }
        const double uc = mine ? static_cast<double>(u[c - 1]) : 0.0;
        unsigned todo = __ballot_sync(0xffffffffu, mine);
        while (todo && next < 0 && !open) {
          const int src = __ffs(todo) - 1;
          todo &= todo - 1;
          const int64_t x = __shfl_sync(0xffffffffu, tok, src);
          const bool inside = __shfl_sync(0xffffffffu, static_cast<int>(in), src);
          double hc = __shfl_sync(0xffffffffu, here, src);
          const double uu = __shfl_sync(0xffffffffu, uc, src);
          const double qc = __shfl_sync(0xffffffffu, against, src);
          bool ok;
          if (greedy) {
            ok = inside && x == sh.argmax && sh.pmax > -INFINITY;
          } else {
            if (!kDraft) {  // a token tried before has no probability left
              bool twin = false;
              for (int i = lane; i < nrej; i += 32) twin |= sh.rejected[i] == x;
              if (__any_sync(0xffffffffu, twin)) hc = 0.0;
            }
            const double bar = uu * (kDraft ? qc : left);
            ok = bar < hc && hc > 0.0;
            if (!exact && hc > 0.0 && fabs(bar - hc) <= 0x1p-14 * (hc + (kDraft ? bar : 1.0)))
              open = 1;
          }
          if (ok) {
            next = c0 + src;
          } else {
            left -= hc;
            if (lane == 0 && inside) sh.rejected[nrej] = x;
            if (inside) ++nrej;
            __syncwarp();
          }
        }
      }
      if (lane == 0) {
        sh.next = next;
        sh.nrejected = nrej;
        sh.ambiguous = open;
      }
    };

    // fp64 sums of exponentials of the staged rows, exchanged
    auto sums64 = [&]() {
      const uint32_t top = __float_as_uint(sh.pmax) >> 16, qtop = __float_as_uint(sh.qmax) >> 16;
      const double top_c = static_cast<double>(sh.pmax) * c64;
      const double qtop_c = static_cast<double>(sh.qmax) * c64;
      double a = 0.0, d = 0.0;
      for (int i = tid; i < len; i += kVerifyThreads) {
        a += weight64(pbuf[ps + i], top, c64, top_c, sh.table);
        if (have_draft_row) d += weight64(qbuf[qs + i], qtop, c64, qtop_c, sh.table);
      }
      a = warp_sum(a);
      d = warp_sum(d);
      if (lane == 0) {
        sh.warp_a[warp] = a;
        sh.warp_b[warp] = d;
      }
      const float pm = sh.pmax, qm = sh.qmax;
      __syncthreads();
      if (tid == 0) {
        VerifySums v{pm > -INFINITY ? vkey(pm, static_cast<uint32_t>(sh.argmax)) : 0ull, qm, 0.0,
                     0.0};
        for (int w = 0; w < kVerifyWarps; ++w) {
          v.psum += sh.warp_a[w];
          v.qsum += sh.warp_b[w];
        }
        sh.sums[parity] = v;
      }
      exchange(true);
    };

    decide(false);
    __syncthreads();
    bool exact = false;
    if (sh.ambiguous) {
      sums64();
      exact = true;
      decide(true);
      __syncthreads();
    }
    if (sh.next >= 0) {
      node = sh.next;
      if (tid == 0) sh.path[++sh.count] = node;
      __syncthreads();  // also: the slice may be overwritten
      continue;
    }

    // ---- nothing goes on: draw from what the last row has left
    int64_t pick = -1;
    if (greedy || !(sh.pmax > -INFINITY)) {
      if (rank == 0 && tid == 0) pick = sh.argmax;
    } else {
      const bool residual = have_draft_row;
      if (residual && !exact) sums64();
      const uint32_t top = __float_as_uint(sh.pmax) >> 16, qtop = __float_as_uint(sh.qmax) >> 16;
      const double top_c = static_cast<double>(sh.pmax) * c64;
      const double qtop_c = static_cast<double>(sh.qmax) * c64;
      const double pinv = residual ? 1.0 / sh.psum : 1.0;
      const double qinv = residual && sh.qsum > 0.0 ? 1.0 / sh.qsum : 0.0;
      if (!kDraft) {  // the rejected tokens leave the slice
        for (int i = tid; i < sh.nrejected; i += kVerifyThreads) {
          const int64_t at = sh.rejected[i] - x0;
          if (at >= 0 && at < len) pbuf[ps + at] = 0xff80u;
        }
        __syncthreads();
      }
      bool use_q = residual;
      // the weight of column x0 + i (the largest logit itself may be rejected)
      auto weight = [&](int i) {
        double w = weight64(pbuf[ps + i], top, c64, top_c, sh.table) * pinv;
        if (use_q) w = fmax(w - weight64(qbuf[qs + i], qtop, c64, qtop_c, sh.table) * qinv, 0.0);
        return w;
      };
      // a warp owns consecutive columns, so that sums are in column order
      const int seg = (len + kVerifyWarps - 1) / kVerifyWarps;
      const int i0 = min(warp * seg, len), i1 = min(i0 + seg, len);
      for (int attempt = 0; attempt < 2; ++attempt) {
        double a = 0.0;
        for (int i = i0 + lane; i < i1; i += 32) a += weight(i);
        a = warp_sum(a);
        if (lane == 0) sh.warp_a[warp] = a;
        __syncthreads();
        if (tid == 0) {
          VerifySums v{0ull, -INFINITY, 0.0, 0.0};
          for (int w = 0; w < kVerifyWarps; ++w) v.psum += sh.warp_a[w];
          sh.sums[parity] = v;
        }
        exchange(false);
        if (sh.psum > 0.0 || attempt == 1) break;
        // nothing is left (rounding rejected the last of the mass): draw from p
        use_q = false;
        float ib = -INFINITY;
        uint32_t ic = 0;
        ps = load_slice(prow, x0, len, pbuf, ib, ic);
        __syncthreads();
      }
      if (rank == sh.owner) {
        // the warp whose weights cross the threshold scans its columns in order
        double before = 0.0;
        int ow = -1, last = -1;
        for (int w = 0; w < kVerifyWarps; ++w) {
          if (sh.warp_a[w] > 0.0) last = w;
          if (ow < 0 && before + sh.warp_a[w] > sh.base) ow = w;
          if (ow < 0) before += sh.warp_a[w];
        }
        const bool none = ow < 0;  // u so near 1 that rounding hid the border: the last weight
        if (none) ow = last;
        if (warp == ow) {
          const double want = none ? INFINITY : sh.base - before;
          double run = 0.0;
          int found = -1, lastx = -1;
          for (int j = i0; j < i1 && found < 0; j += 32) {
            const double w = j + lane < i1 ? weight(j + lane) : 0.0;
            double incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double y = __shfl_up_sync(0xffffffffu, incl, o);
              if (lane >= o) incl += y;
            }
            const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && run + incl > want);
            const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
            if (some) lastx = j + 31 - __clz(some);
            if (over) found = j + __ffs(over) - 1;
            run += __shfl_sync(0xffffffffu, incl, 31);
          }
          if (lane == 0) pick = x0 + (found >= 0 ? found : max(lastx, 0));
        }
      }
    }
    const int count = sh.count;
    const int64_t row = static_cast<int64_t>(b) * p.nodes;
    if (pick >= 0) p.out_tokens[row + count] = pick;
    if (rank == 0) {
      for (int i = tid; i < p.nodes; i += kVerifyThreads) {
        p.out_path[row + i] = i <= count ? sh.path[i] : -1;
        if (i != count) p.out_tokens[row + i] = i < count ? tokens[sh.path[i + 1] - 1] : -1;
      }
      if (tid == 0) p.out_num[b] = count;
    }
    break;
  }
  cluster.sync();  // no CTA leaves while its sums may be read
}

static size_t verify_smem(int slice, bool draft) {
  const size_t head = (sizeof(VerifyShared) + 15) & ~size_t(15);
  return head + static_cast<size_t>(slice + 16) * 2 * (draft ? 2 : 1);
}

template <bool kDraft>
static int launch_verify(const VerifyParams& p, int batch, cudaStream_t stream) {
  static std::mutex mu;
  static bool done[64];
  const size_t limit = verify_smem((kMaxVocab / kVerifyCluster + 7) / 8 * 8, kDraft);
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !done[dev]) {
      const cudaError_t e =
          cudaFuncSetAttribute(verify_kernel<kDraft>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(limit));
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(verify_kernel)");
      if (dev < 64) done[dev] = true;
    }
  }
  verify_kernel<kDraft><<<static_cast<unsigned>(batch) * kVerifyCluster, kVerifyThreads,
                          verify_smem(p.slice, kDraft), stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? NVATTN_OK : cuda_fail(e, "verify_kernel launch");
}

}  // namespace nvattn

using namespace nvattn;

extern "C" int nvattn_verify_draft(
    const void* logits, int64_t l_stride_seq, int64_t l_stride_row, const void* draft_logits,
    int64_t d_stride_seq, int64_t d_stride_row, const int64_t* draft_tokens,
    const int32_t* parents, int64_t parents_stride, const float* u_accept, const float* u_pick,
    const float* temperatures, const int32_t* num_nodes, int32_t batch, int32_t nodes,
    int32_t vocab, int64_t* out_tokens, int32_t* out_path, int32_t* out_num, void* stream) {
  clear_error();
  if (batch < 0 || nodes < 0) return fail(NVATTN_ERR_INVALID, "verify_draft: negative size");
  if (batch == 0 || nodes == 0) return NVATTN_OK;
  if (!logits || !u_pick || !out_tokens || !out_path || !out_num ||
      (nodes > 1 && (!draft_tokens || !u_accept)))
    return fail(NVATTN_ERR_INVALID, "verify_draft: NULL pointer");
  if (nodes > kMaxNodes) return fail(NVATTN_ERR_UNSUPPORTED, "verify_draft: at most 64 nodes");
  if (vocab <= 0) return fail(NVATTN_ERR_INVALID, "verify_draft: vocab must be > 0");
  if (vocab > kMaxVocab)
    return fail(NVATTN_ERR_UNSUPPORTED, "verify_draft: at most 393216 vocabulary columns");
  if (draft_logits && parents)
    return fail(NVATTN_ERR_UNSUPPORTED, "verify_draft: draft logits need a chain (no parents)");
  if (l_stride_row < 0 || l_stride_seq < 0 || d_stride_row < 0 || d_stride_seq < 0 ||
      parents_stride < 0)
    return fail(NVATTN_ERR_INVALID, "verify_draft: negative stride");
  if ((reinterpret_cast<uintptr_t>(logits) & 1) || (reinterpret_cast<uintptr_t>(draft_logits) & 1))
    return fail(NVATTN_ERR_INVALID, "verify_draft: logits must be 2-byte aligned");
  if (batch > 0x7fffffff / kVerifyCluster)
    return fail(NVATTN_ERR_INVALID, "verify_draft: batch too large");
  VerifyParams p{};
  p.logits = static_cast<const __nv_bfloat16*>(logits);
  p.l_stride_seq = l_stride_seq;
  p.l_stride_row = l_stride_row;
  p.draft = static_cast<const __nv_bfloat16*>(draft_logits);
  p.d_stride_seq = d_stride_seq;
  p.d_stride_row = d_stride_row;
  p.tokens = draft_tokens;
  p.parents = parents;
  p.parents_stride = parents_stride;
  p.u_accept = u_accept;
  p.u_pick = u_pick;
  p.temperatures = temperatures;
  p.num_nodes = num_nodes;
  p.nodes = nodes;
  p.vocab = vocab;
  p.slice = ((vocab + kVerifyCluster - 1) / kVerifyCluster + 7) / 8 * 8;
  p.out_tokens = out_tokens;
  p.out_path = out_path;
  p.out_num = out_num;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return draft_logits ? launch_verify<true>(p, batch, s) : launch_verify<false>(p, batch, s);
}
