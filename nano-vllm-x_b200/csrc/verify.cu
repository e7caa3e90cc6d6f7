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
// Only the rows on the walked path are read: one cluster of CTAs per sequence
// walks it, a CTA per slice of the columns, and every CTA takes the same
// decisions from the same exchanged sums. Scanning a row costs one MUFU
// exponential and about four other instructions a logit (each thread sums
// against its own maximum, so a row is read once and nothing is staged); the
// exchange is one cluster barrier a node.
//
// The answers are tokens, so sums that decide between neighbours are kept in
// 64 bits: the draw's cumulative weights always (with 151,936 weights of which
// many are near 1e-6, sums in fp32 would move a border past u in about one
// draw in a hundred), an acceptance when the fp32 sums leave its outcome
// within 2^-14 of the border. 2^t in fp64 is table-driven (P. T. P. Tang, ACM
// TOMS 15(2), 1989): t = k/1024 + f, |f| <= 2^-11, 2^t = 2^(k>>10) *
// T[k & 1023] * 2^f with a cubic (error (f ln 2)^4/24 < 6e-16), 8 fp64
// operations. The draw reads its row a second time (from L2) for those sums: a
// lane owns a run of columns, so prefix sums over lanes, warps and CTAs find
// the lane whose run crosses the threshold, and one warp scans that run.
#include <cooperative_groups.h>

#include <mutex>

#include "common.cuh"

namespace nvattn {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kMaxNodes = 64;
constexpr int kMaxVocab = 1 << 20;  // keeps the fp32 sums well inside decide()'s margin
constexpr int kExpTable = 1024;

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
  unsigned long long key;  // largest logit and its first column (vkey order)
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
  int next, count, nrejected, open;
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

// 2^((l - top) * c) in fp64 for a bf16 logit that is not NaN: exactly 1 for the
// largest (also where that is infinite), exactly 0 below 2^-1000.
__device__ __forceinline__ double weight64(uint32_t bits, uint32_t top_bits, double c, double top_c,
                                           const double* __restrict__ table) {
  const double t = fma(bf16_to_f64(bits), c, -top_c);
  const double shift = 6597069766656.0;  // 1.5 * 2^42: rounds to multiples of 2^-10
  const double s = t + shift;
  const int k = __double2loint(s);
  const double f = t - (s - shift);
  double e = fma(f, 0.055504108664821580, 0.24022650695910071);  // (ln 2)^3/6, (ln 2)^2/2
  e = fma(e, f, 0.69314718055994531);
  const double tj = table[k & (kExpTable - 1)];
  const double r = fma(e * f, tj, tj);
  const double w = __hiloint2double(__double2hiint(r) + ((k >> 10) << 20), __double2loint(r));
  // t's high word as an integer: -1000 and below
  const bool none = static_cast<uint32_t>(__double2hiint(t)) >= 0xC08F4000u || bits == 0xff80u;
  return bits == top_bits ? 1.0 : (none ? 0.0 : w);
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two bf16 -inf.
__device__ __forceinline__ __nv_bfloat162 neg_inf2() {
  return __nv_bfloat162(__nv_bfloat162_raw{0xff80u, 0xff80u});
}

// NaN becomes -inf (the maximum of two bf16 skips NaN).
__device__ __forceinline__ uint32_t clean2(uint32_t w) {
  const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w),
                                   neg_inf2());
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Columns [at, at + 8) of a slice of `len` columns as 4 pairs, -inf outside the
// slice and for NaN; one 16-byte load where the address allows.
__device__ __forceinline__ void load8(const unsigned short* src, int at, int len, uint32_t w[4]) {
  if (at >= 0 && at + 8 <= len && (reinterpret_cast<uintptr_t>(src + at) & 15) == 0) {
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
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = clean2(w[e]);
}

__device__ __forceinline__ float scale_to(float m, float top, float c) {
  return m == top ? 1.f : fast_exp2((m - top) * c);  // 0 for m = -inf
}

// This thread's part of a slice: its largest logit m and the sum over its
// logits of 2^((l - m) * c), kRowBatch vectors in flight.
constexpr int kRowBatch = 5;

__device__ __forceinline__ void scan_row(const unsigned short* src, int len, float c, float& m,
                                         float& sum) {
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) >> 1);
  const int groups = (shift + len + 7) / 8;
  m = -INFINITY;
  sum = 0.f;
  for (int g0 = threadIdx.x; g0 < groups; g0 += kRowBatch * kVerifyThreads) {
    uint32_t w[kRowBatch][4];
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) load8(src, (g0 + u * kVerifyThreads) * 8 - shift, len, w[u]);
    __nv_bfloat162 mx = neg_inf2();
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = __hmax2(mx, *reinterpret_cast<__nv_bfloat162*>(&w[u][e]));
    }
    const float top = fmaxf(m, fmaxf(__low2float(mx), __high2float(mx)));
    if (top == -INFINITY) continue;
    if (top == INFINITY) {  // infinite logits share everything
      if (m < INFINITY) sum = 0.f;
#pragma unroll
      for (int u = 0; u < kRowBatch; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum += static_cast<float>((w[u][e] & 0xffffu) == 0x7f80u) +
                 static_cast<float>((w[u][e] >> 16) == 0x7f80u);
      }
      m = top;
      continue;
    }
    sum *= scale_to(m, top, c);
    m = top;
    const uint64_t ntop2 = pack_f32x2(-top, -top), c2 = pack_f32x2(c, c);
    uint64_t acc[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
    const uint64_t zero2 = acc[0];
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t l2 = (static_cast<uint64_t>(w[u][e] & 0xffff0000u) << 32) | (w[u][e] << 16);
        acc[e & 1] = add_f32x2(acc[e & 1],
                               exp2_mufu_f32x2(fma_f32x2(add_f32x2(l2, ntop2), c2, zero2)));
      }
    }
    const float2 a = unpack_f32x2(add_f32x2(acc[0], acc[1]));
    sum += a.x + a.y;
  }
}

// Greedy rows: this thread's best logit of a slice and its first column.
__device__ __forceinline__ unsigned long long scan_best(const unsigned short* src, int x0,
                                                        int len) {
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) >> 1);
  const int groups = (shift + len + 7) / 8;
  float best = -INFINITY;
  uint32_t bcol = 0;
  for (int g0 = threadIdx.x; g0 < groups; g0 += kRowBatch * kVerifyThreads) {
    uint32_t w[kRowBatch][4];
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) load8(src, (g0 + u * kVerifyThreads) * 8 - shift, len, w[u]);
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float l = __uint_as_float((e & 1) ? (w[u][e >> 1] & 0xffff0000u) : (w[u][e >> 1] << 16));
        if (l > best) {  // columns come in increasing order: the first of equals stays
          best = l;
          bcol = static_cast<uint32_t>(x0 + (g0 + u * kVerifyThreads) * 8 - shift + e);
        }
      }
    }
  }
  return best > -INFINITY ? vkey(best, bcol) : 0ull;
}

template <bool kDraft>
__global__ void __launch_bounds__(kVerifyThreads, 3) verify_kernel(const VerifyParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int b = blockIdx.x / ranks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ VerifyShared sh;

  const int x0 = min(rank * p.slice, p.vocab);
  const int len = min(p.slice, p.vocab - x0);
  const int n = p.num_nodes ? min(max(p.num_nodes[b], 0), p.nodes) : p.nodes;
  const float temp = p.temperatures ? p.temperatures[b] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double c64 = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(temp);
  const float c32 = fminf(static_cast<float>(c64), 1e30f);
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
  for (int i = tid; !greedy && i < kExpTable; i += kVerifyThreads)
    sh.table[i] = exp2(static_cast<double>(i) / kExpTable);
  if (tid == 0) {
    sh.count = 0;
    sh.path[0] = 0;
  }
  __syncthreads();
  int parity = 0;

  // Adds up what every CTA of the cluster wrote to its sums[parity]; ends with
  // the totals visible to the whole CTA. scaled: sums of exponentials, each
  // relative to its CTA's largest logit; otherwise weights, and the owner of the
  // draw's threshold.
  auto exchange = [&](bool scaled) {
    cluster.sync();
    if (warp == 0) {
      VerifySums v{0ull, -INFINITY, 0.0, 0.0};
      if (lane < ranks) v = *cluster.map_shared_rank(&sh.sums[parity], lane);
      if (scaled) {
        unsigned long long key = v.key;
        float qm = v.qmax;
#pragma unroll
        for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
          const unsigned long long k2 = __shfl_xor_sync(0xffffffffu, key, o);
          key = k2 > key ? k2 : key;
          qm = fmaxf(qm, __shfl_xor_sync(0xffffffffu, qm, o));
        }
        const float pm = vkey_score(key);
        const double ps = warp_sum(v.psum * static_cast<double>(scale_to(vkey_score(v.key), pm, c32)));
        const double qs = warp_sum(v.qsum * static_cast<double>(scale_to(v.qmax, qm, c32)));
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
        for (int r = 0; r < ranks; ++r) {
          run += __shfl_sync(0xffffffffu, v.psum, r);
          if (lane == r) incl = run;
        }
        const double threshold = static_cast<double>(fmaxf(p.u_pick[b], 0.f)) * run;
        const unsigned over = __ballot_sync(0xffffffffu, lane < ranks && incl > threshold);
        const unsigned some = __ballot_sync(0xffffffffu, lane < ranks && v.psum > 0.0);
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
  while (true) {
    // ---- the row's largest logit and sum of exponentials
    const unsigned short* prow =
        reinterpret_cast<const unsigned short*>(p.logits) +
        static_cast<int64_t>(b) * p.l_stride_seq + static_cast<int64_t>(node) * p.l_stride_row;
    const bool with_q = kDraft && !greedy && node + 1 < n;
    const unsigned short* qrow = nullptr;
    if (with_q)
      qrow = reinterpret_cast<const unsigned short*>(p.draft) +
             static_cast<int64_t>(b) * p.d_stride_seq + static_cast<int64_t>(node) * p.d_stride_row;
    float qm = -INFINITY, qsum = 0.f, pm = -INFINITY, psum = 0.f;
    unsigned long long key;
    if (greedy) {
      key = scan_best(prow + x0, x0, len);
    } else {
      scan_row(prow + x0, len, c32, pm, psum);
      if (with_q) scan_row(qrow + x0, len, c32, qm, qsum);
      key = pm > -INFINITY ? vkey(pm, 0u) : 0ull;  // the column is the greedy rows' alone
    }
    {
      unsigned long long wkey = key;
      float wq = qm;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k2 = __shfl_xor_sync(0xffffffffu, wkey, o);
        wkey = k2 > wkey ? k2 : wkey;
        wq = fmaxf(wq, __shfl_xor_sync(0xffffffffu, wq, o));
      }
      // warp sums of up to 2^14 fp32 terms near 1 and below: fp32 carries them
      // well inside the decisions' 2^-14
      const float a = warp_sum(psum * scale_to(pm, vkey_score(wkey), c32));
      const float d = kDraft ? warp_sum(qsum * scale_to(qm, wq, c32)) : 0.f;
      if (lane == 0) {
        sh.warp_key[warp] = wkey;
        sh.warp_q[warp] = wq;
        sh.warp_a[warp] = a;
        sh.warp_b[warp] = d;
      }
    }
    __syncthreads();
    if (warp == 0) {
      const bool in = lane < kVerifyWarps;
      const unsigned long long k0 = in ? sh.warp_key[lane] : 0ull;
      const float q0 = in ? sh.warp_q[lane] : -INFINITY;
      unsigned long long k = k0;
      float q = q0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k2 = __shfl_xor_sync(0xffffffffu, k, o);
        k = k2 > k ? k2 : k;
        q = fmaxf(q, __shfl_xor_sync(0xffffffffu, q, o));
      }
      const double a = warp_sum(in ? sh.warp_a[lane] * scale_to(vkey_score(k0), vkey_score(k), c32) : 0.0);
      const double d = warp_sum(in ? sh.warp_b[lane] * scale_to(q0, q, c32) : 0.0);
      if (lane == 0) sh.sums[parity] = VerifySums{k, q, a, d};
    }
    exchange(true);

    // ---- which child goes on. Warp 0 of every CTA takes the same decision.
    // exact: the sums are fp64's own; otherwise an outcome within 2^-14 of
    // its border is left open (the fp32 terms put the sums off by < 2^-17).
    auto decide = [&](bool exact) {
      if (warp != 0) return;
      const uint32_t top = __float_as_uint(sh.pmax) >> 16;
      const uint32_t qtop = __float_as_uint(sh.qmax) >> 16;
      const double top_c = static_cast<double>(sh.pmax) * c64;
      const double qtop_c = static_cast<double>(sh.qmax) * c64;
      const bool any = sh.pmax > -INFINITY;
      int next = -1, nrej = 0, open = 0;
      double left = 1.0;
      for (int c0 = node + 1; c0 < n && next < 0 && !open; c0 += 32) {
        const int c = c0 + lane;
        const bool mine = c < n && sh.parents[c] == node;
        const int64_t tok = mine ? tokens[c - 1] : -1;
        const bool in = mine && tok >= 0 && tok < p.vocab;
        double here = 0.0, against = 0.0;
        if (in && !greedy && any) {
          here = weight64(clean2(prow[tok]) & 0xffffu, top, c64, top_c, sh.table) / sh.psum;
          if (with_q && sh.qmax > -INFINITY)
            against = weight64(clean2(qrow[tok]) & 0xffffu, qtop, c64, qtop_c, sh.table) / sh.qsum;
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
            ok = inside && any && x == sh.argmax;
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
        sh.open = open;
      }
    };
    decide(false);
    __syncthreads();

    // ---- fp64: a lane's run of consecutive columns, warps and ranks in order
    const int run = ((len + kVerifyThreads - 1) / kVerifyThreads + 7) / 8 * 8;
    const int i0 = min(tid * run, len), i1 = min(i0 + run, len);
    const uint32_t top = __float_as_uint(sh.pmax) >> 16, qtop = __float_as_uint(sh.qmax) >> 16;
    const double top_c = static_cast<double>(sh.pmax) * c64;
    const double qtop_c = static_cast<double>(sh.qmax) * c64;
    const bool any = sh.pmax > -INFINITY, any_q = with_q && sh.qmax > -INFINITY;
    const unsigned long long pkey = any ? vkey(sh.pmax, static_cast<uint32_t>(sh.argmax)) : 0ull;
    const float qmax = sh.qmax;

    // Sums over the run: a of p's exponentials without the rejected tokens, and
    // with a draft row d of q's and, of the columns where p / psum exceeds q /
    // qsum with the sums as they stand, ra and rd of both.
    auto run_sums = [&](bool skip, double pinv, double qinv, double& a, double& d, double& ra,
                        double& rd) {
      a = d = ra = rd = 0.0;
      bool held = false;  // a rejected token lies in this run
      for (int i = 0; skip && i < sh.nrejected; ++i)
        held |= sh.rejected[i] >= x0 + i0 && sh.rejected[i] < x0 + i1;
      for (int at = i0; at < i1; at += 8) {
        uint32_t w[4], v[4];
        load8(prow + x0, at, len, w);
        if (with_q) load8(qrow + x0, at, len, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t pb = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
          double wp = weight64(pb, top, c64, top_c, sh.table);
          if (held) {
            for (int i = 0; i < sh.nrejected; ++i)
              if (sh.rejected[i] == x0 + at + e) wp = 0.0;
          }
          a += wp;
          if (kDraft && with_q) {
            const uint32_t qb = (e & 1) ? v[e >> 1] >> 16 : v[e >> 1] & 0xffffu;
            const double wq = any_q ? weight64(qb, qtop, c64, qtop_c, sh.table) : 0.0;
            d += wq;
            if (fma(wp, pinv, -wq * qinv) > 0.0) {
              ra += wp;
              rd += wq;
            }
          }
        }
      }
    };
    // fp64 sums of exponentials over the whole rows
    auto sums64 = [&](double a, double d) {
      a = warp_sum(a);
      d = warp_sum(d);
      if (lane == 0) {
        sh.warp_a[warp] = a;
        sh.warp_b[warp] = d;
      }
      __syncthreads();
      if (tid == 0) {
        VerifySums v{pkey, qmax, 0.0, 0.0};
        for (int w = 0; w < kVerifyWarps; ++w) {
          v.psum += sh.warp_a[w];
          v.qsum += sh.warp_b[w];
        }
        sh.sums[parity] = v;
      }
      exchange(true);
    };

    if (sh.open) {
      double a, d, ra, rd;
      run_sums(false, 1.0, 0.0, a, d, ra, rd);
      sums64(a, d);
      decide(true);
      __syncthreads();
    }
    if (sh.next >= 0) {
      node = sh.next;
      if (tid == 0) sh.path[++sh.count] = node;
      __syncthreads();
      continue;
    }

    // ---- nothing goes on: draw from what the last row has left
    int64_t pick = -1;
    if (greedy || !any) {
      if (rank == 0 && tid == 0) pick = sh.argmax;
    } else {
      bool use_q = any_q, skip = !kDraft && sh.nrejected > 0;
      double pinv = 1.0, qinv = 0.0;
      for (int attempt = 0; attempt < 2; ++attempt) {
        double mine, a, d, ra, rd;
        if (use_q) {
          // One pass gives the exact sums and, over the columns that are
          // positive by the sums at hand, the parts of the residual: a column
          // on the wrong side by a rounding of those has a residual of no more
          // than that rounding.
          pinv = 1.0 / sh.psum;
          qinv = 1.0 / sh.qsum;
          __syncthreads();
          run_sums(false, pinv, qinv, a, d, ra, rd);
          sums64(a, d);
          pinv = 1.0 / sh.psum;
          qinv = 1.0 / sh.qsum;
          __syncthreads();
          mine = fmax(ra * pinv - rd * qinv, 0.0);
        } else {
          run_sums(skip, 1.0, 0.0, a, d, ra, rd);
          mine = a;
        }
        // prefix over the lanes, in column order
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        if (lane == 31) sh.warp_a[warp] = incl;
        __syncthreads();
        if (tid == 0) {
          VerifySums v{0ull, -INFINITY, 0.0, 0.0};
          for (int w = 0; w < kVerifyWarps; ++w) v.psum += sh.warp_a[w];
          sh.sums[parity] = v;
        }
        exchange(false);
        if (!(sh.psum > 0.0) && attempt == 0) {
          // nothing is left (rounding rejected the last of the mass): draw from p
          use_q = skip = false;
          pinv = 1.0;
          qinv = 0.0;
          continue;
        }
        if (rank == sh.owner) {
          // the warp, then the lane, whose weights cross the threshold (with u so
          // near 1 that rounding hides the border: the last ones with weight)
          double before = 0.0;
          int ow = -1, last = 0;
          for (int w = 0; w < kVerifyWarps; ++w) {
            if (sh.warp_a[w] > 0.0) last = w;
            if (ow < 0 && before + sh.warp_a[w] > sh.base) ow = w;
            if (ow < 0) before += sh.warp_a[w];
          }
          const bool none = ow < 0;
          if (none) ow = last;
          if (warp == ow) {
            const double want = none ? INFINITY : sh.base - before;
            const unsigned over = __ballot_sync(0xffffffffu, incl > want);
            const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
            const int ol = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : 0);
            double sum = __shfl_sync(0xffffffffu, incl - mine, ol);
            const int j0 = __shfl_sync(0xffffffffu, i0, ol), j1 = __shfl_sync(0xffffffffu, i1, ol);
            int found = -1, lastx = j0;
            for (int j = j0; j < j1 && found < 0; j += 32) {
              const int i = j + lane;
              double w = 0.0;
              if (i < j1) {
                w = weight64(clean2(prow[x0 + i]) & 0xffffu, top, c64, top_c, sh.table) * pinv;
                for (int r = 0; skip && r < sh.nrejected; ++r)
                  if (sh.rejected[r] == x0 + i) w = 0.0;
                if (use_q)
                  w = fmax(w - weight64(clean2(qrow[x0 + i]) & 0xffffu, qtop, c64, qtop_c, sh.table) *
                                   qinv, 0.0);
              }
              double part = w;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, part, o);
                if (lane >= o) part += y;
              }
              const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && sum + part > want);
              const unsigned pos = __ballot_sync(0xffffffffu, w > 0.0);
              if (pos) lastx = j + 31 - __clz(pos);
              if (hit) found = j + __ffs(hit) - 1;
              sum += __shfl_sync(0xffffffffu, part, 31);
            }
            if (lane == 0) pick = x0 + (found >= 0 ? found : lastx);
          }
        }
        break;
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

template <bool kDraft>
static int launch_verify(VerifyParams p, int batch, cudaStream_t stream) {
  static std::mutex mu;
  static bool done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(
          verify_kernel<kDraft>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(verify_kernel)");
      if (dev < 64) done[dev] = true;
    }
  }
#ifndef VCLUSTER
#define VCLUSTER (batch * 16 <= 148 ? 16 : 8)
#endif
  const int ranks = VCLUSTER;
  p.slice = ((p.vocab + ranks - 1) / ranks + 7) / 8 * 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch) * ranks);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<kDraft>, p);
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
    return fail(NVATTN_ERR_UNSUPPORTED, "verify_draft: at most 2^20 vocabulary columns");
  if (draft_logits && parents)
    return fail(NVATTN_ERR_UNSUPPORTED, "verify_draft: draft logits need a chain (no parents)");
  if (l_stride_row < 0 || l_stride_seq < 0 || d_stride_row < 0 || d_stride_seq < 0 ||
      parents_stride < 0)
    return fail(NVATTN_ERR_INVALID, "verify_draft: negative stride");
  if ((reinterpret_cast<uintptr_t>(logits) & 1) || (reinterpret_cast<uintptr_t>(draft_logits) & 1))
    return fail(NVATTN_ERR_INVALID, "verify_draft: logits must be 2-byte aligned");
  if (batch > 0x7fffffff / kMaxCluster)
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
  p.out_tokens = out_tokens;
  p.out_path = out_path;
  p.out_num = out_num;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return draft_logits ? launch_verify<true>(p, batch, s) : launch_verify<false>(p, batch, s);
}
