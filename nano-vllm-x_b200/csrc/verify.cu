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
// Two kernels. The walk reads only the rows on the path: one cluster of CTAs per
// sequence, a CTA per slice of the columns. A row costs one pass with one MUFU
// exponential and about three other instructions a logit (each thread sums
// against its own maximum) and one cluster barrier: every warp writes its sums
// into the shared memory of all CTAs, and after the barrier every warp adds the
// same numbers up and takes the same decision, with nothing to broadcast. The walk
// takes a node's rows after the decision that leads there, so only rows on the path
// are read, but one after another: it is bound by latency (about 5 us a node alone, 7
// beside 63 other sequences). That is this walk's order, not the operator's: the
// sums of all rows could be taken at once and the decisions after. The next node's
// rows are sent for to L2 before it is accepted, and the code of a step is kept short
// (it once overran the instruction cache at twice the time). The draw then goes over
// each sequence's last row, all sequences at once, in fp64 throughout, which an
// answer clear of its border does not need. 64 sequences of 7 drafts, 151,936
// columns: walk 75 us, draw 49 (46 before it noted the columns near the residual's
// border; then both in one kernel, where an early end is drawn at once, took the same
// 120, a step that sums up a node's and its first child's rows together 130, a table
// of weights over the rows' bf16 values for the draw 121).
//
// The answers are tokens, so sums that decide between neighbours are kept in
// 64 bits: the draw's cumulative weights always (with 151,936 weights of which
// many are near 1e-6, sums in fp32 would move a border past u in about one
// draw in a hundred), the sides of max(p - q, 0) where the fp32 sums leave them
// open, an acceptance when they leave its outcome within 2^-14 of the border. 2^t
// in fp64 is table-driven (P. T. P. Tang, ACM TOMS 15(2), 1989): t = k/1024 + f,
// |f| <= 2^-11, 2^t = 2^(k>>10) * T[k & 1023] * 2^f with a cubic (error
// (f ln 2)^4/24 < 6e-16), 8 fp64 operations, whose latency bounds the draw. In it
// a warp owns consecutive columns, its lanes keep the sums of consecutive bins, and
// prefix sums over warps, bins and lanes find the column.
#include <cooperative_groups.h>

#include <mutex>

#include "decode.cuh"

namespace nvattn {

namespace cg = cooperative_groups;

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kMaxNodes = 64;
constexpr int kMaxVocab = 1 << 20;  // keeps the fp32 sums well inside the margin of open decisions
constexpr int kExpTable = 1024;
constexpr uint32_t kNoLogit = 0xff80u;  // bf16 bits of -inf
// Temperatures count up to this (every law is flat long before): a logit of
// -inf is then 2^-980 below any other, and never drawn.
constexpr float kMaxTemperature = 1e30f;

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
  int32_t ahead;  // the walk sends for the first child's rows before it is accepted
  int32_t border;  // near_border, by the walk's batches
  int64_t* out_tokens;
  int32_t* out_path;
  int32_t* out_num;
};

// A sequence's temperature, up to kMaxTemperature; 0 for greedy, NaN among it.
__device__ __forceinline__ float temperature_of(const VerifyParams& p, int b) {
  const float t = p.temperatures ? p.temperatures[b] : 0.f;
  return t > 0.f ? fminf(t, kMaxTemperature) : 0.f;
}

// What a warp tells the cluster: (max, sum) of its part of the target's and the
// draft's row; or a pick key; or two fp64 sums.
union VerifySlot {
  float4 f;
  double2 d;
  unsigned long long key[2];
};

struct VerifyShared {
  VerifySlot slots[2][kMaxCluster * kVerifyWarps];  // of all warps, in column order
};

// What the walk leaves in out_tokens[b][count] for the draw, which overwrites it
// with the token: the largest logits of the last row (bf16 bits) and the ratio
// of its sums of exponentials, target over draft.
struct DrawState {
  uint32_t top, qtop;
  float ratio;
};
__device__ __forceinline__ int64_t pack_state(const DrawState& s) {
  return static_cast<int64_t>((static_cast<uint64_t>(__float_as_uint(s.ratio)) << 32) |
                              (s.qtop << 16) | s.top);
}
__device__ __forceinline__ DrawState unpack_state(int64_t v) {
  const uint64_t u = static_cast<uint64_t>(v);
  return {static_cast<uint32_t>(u) & 0xffffu, (static_cast<uint32_t>(u) >> 16),
          __uint_as_float(static_cast<uint32_t>(u >> 32))};
}

__device__ __forceinline__ unsigned long long vkey(float s, uint32_t col) {
  uint32_t b = __float_as_uint(s == 0.f ? 0.f : s);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(b) << 32) | (0xFFFFFFFFu - col);
}

__device__ __forceinline__ float vkey_score(unsigned long long key) {
  const uint32_t b = static_cast<uint32_t>(key >> 32);
  return key == 0ull ? -INFINITY : __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

// exp2 of j / 1024 for a CTA's table.
__device__ __forceinline__ void fill_table(double* table) {
  for (int i = threadIdx.x; i < kExpTable; i += kVerifyThreads)
    table[i] = exp2(static_cast<double>(i) / kExpTable);
}

// One row's scale in fp64: the weight of a bf16 logit l is 2^((l - top) * c),
// held above 2^-1000 (no draw reaches weights below kNothing). c is at most what
// puts the next bf16 below the top at 2^-2000, and has 45 significant bits
// (changing a weight by 2^-45 of its exponent), so that l * c and top * c are
// exact: the exponent is rounded once, and the top's weight is one. A row whose top
// has no finite bf16 below it (infinite, or the lowest finite one) belongs to the
// logits that equal its top: they are weighed as 0 and any other as -980, with c = 1.
struct RowScale {
  double c, top_c;
  uint32_t top;  // bf16 bits
  bool ties;

  __device__ __forceinline__ RowScale(uint32_t top_bits, double c64) : top(top_bits) {
    const float top_l = __uint_as_float(top_bits << 16);
    ties = top_bits == 0x7f80u || top_bits == 0xff7fu;
    const uint32_t below = (top_bits & 0x7fffu) == 0u ? 0x8001u
                           : (top_bits & 0x8000u)     ? top_bits + 1u
                                                      : top_bits - 1u;
    const double gap =
        static_cast<double>(top_l) - static_cast<double>(__uint_as_float(below << 16));
    c = ties ? 1.0 : (c64 * gap > 2000.0 ? 2000.0 / gap : c64);
    c = __longlong_as_double(__double_as_longlong(c) & ~0xffll);
    top_c = ties ? 0.0 : static_cast<double>(top_l) * c;
  }
  // NaN and -inf become the lowest bf16, which weighs 2^-1000 beside any other top.
  __device__ __forceinline__ uint32_t raise(uint32_t two) const {
    if (ties)
      two = ((two & 0xffffu) == top ? 0u : 0xc475u) |
            ((two >> 16) == top ? 0u : 0xc4750000u);  // -980
    const __nv_bfloat162 lowest(__nv_bfloat162_raw{0xff7fu, 0xff7fu});
    const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&two), lowest);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ double log2_weight(float l) const {
    const double t = fma(static_cast<double>(l), c, -top_c);
    // max(t, -1000) on the high word: as unsigned, further below zero is larger
    const uint32_t hi = min(static_cast<uint32_t>(__double2hiint(t)), 0xC08F4000u);
    return __hiloint2double(static_cast<int>(hi), __double2loint(t));
  }
};

// 2^t for t in [-1001, 1].
__device__ __forceinline__ double exp2_64(double t, const double* __restrict__ table) {
  const double shift = 6597069766656.0;  // 1.5 * 2^42: rounds to multiples of 2^-10
  const double s = t + shift;
  const int k = __double2loint(s);
  const double f = t - (s - shift);
  double e = fma(f, 0.055504108664821580, 0.24022650695910071);  // (ln 2)^3/6, (ln 2)^2/2
  e = fma(e, f, 0.69314718055994531);
  const double tj = table[k & (kExpTable - 1)];
  const double r = fma(e * f, tj, tj);
  return __hiloint2double(__double2hiint(r) + ((k & ~(kExpTable - 1)) << 10), __double2loint(r));
}

// Whether wp may be on the other side of x = wq * ratio by the rows' true sums. The
// ratio is that of the walk's sums, in fp32: a thread takes 40 columns at a time (12
// additions; exp2 is off by 2^-22.5, its argument, in a row of 2^20 columns, by 2e-6
// of the terms that count), scales and adds once a batch (3.3e-7), and then come 20
// additions and scalings over threads, warps and CTAs: 4.5e-6 and 3.3e-7 a batch at
// most, twice that for the quotient. That is 1.5e-5 with kShortBatches and 4.4e-5 with
// the most there are (kMaxVocab columns on 512 threads, 53 batches). `border` is 1.5 *
// 2^-16 or 2^-14 of a mantissa of up to 2 in steps of 2^-20, the high words' last bit,
// and one for the bits below. Weights under 2^-60 are not looked at: all of them
// together move the residual by less than 2^-53.
constexpr int kShortBatches = 9, kBorderShort = 49, kBorderLong = 129;
constexpr int kNears = 8;  // such columns that a thread of the draw notes

__device__ __forceinline__ bool near_border(double wp, double x, int border) {
  const int hi = __double2hiint(wp);
  return static_cast<uint32_t>(hi - __double2hiint(x) + border) <= static_cast<uint32_t>(2 * border) &&
         hi > 0x3C300000;
}

// Weights up to this count as none: above the sum of all that log2_weight held
// up (2^20 columns of 2^-980 at most). Thresholds are raised to it.
constexpr double kNothing = 0x1p-950;

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ T warp_max(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const T w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// Inclusive prefix sum over the lanes.
__device__ __forceinline__ double warp_scan(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
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

// Columns [0, len) of a row at `src`, as 16-byte groups at the row's own
// alignment: group g holds columns 8g - shift .. 8g - shift + 7. Groups [lo, hi)
// lie inside and are one load each; one before and one behind may lie partly
// inside and are read element by element.
struct Slice {
  const unsigned short* src;
  int len, shift, lo, hi, groups;

  __device__ __forceinline__ Slice(const unsigned short* s, int n)
      : src(s),
        len(n),
        shift(static_cast<int>((reinterpret_cast<uintptr_t>(s) & 15) >> 1)),
        lo(shift > 0 ? 1 : 0),
        hi((shift + n) / 8),
        groups((shift + n + 7) / 8) {}

  // Issues group g's load, if it lies inside (-inf otherwise); nothing here
  // depends on the data, so a batch of these is in flight together.
  __device__ __forceinline__ void load(int g, uint32_t w[4]) const {
    int4 v = make_int4(0xff80ff80, 0xff80ff80, 0xff80ff80, 0xff80ff80);
    if (g >= lo && g < hi) v = __ldg(reinterpret_cast<const int4*>(src + (g * 8 - shift)));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
  // Sends the whole groups to L2, one thread's instruction: the registers hold a
  // few vectors a thread in flight, this holds the slice.
  __device__ __forceinline__ void prefetch() const {
    if (hi > lo)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src + (lo * 8 - shift)),
                   "r"((hi - lo) * 16)
                   : "memory");
  }
  __device__ __forceinline__ bool partial(int g) const {
    return g >= 0 && g < groups && (g < lo || g >= hi);
  }
  // Columns at .. at + 7, of which some may lie outside (-inf).
  __device__ __forceinline__ void load_any(int at, uint32_t w[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = at + 2 * e;
      const uint32_t a = (i >= 0 && i < len) ? __ldg(src + i) : 0xff80u;
      const uint32_t b = (i + 1 >= 0 && i + 1 < len) ? __ldg(src + i + 1) : 0xff80u;
      w[e] = a | (b << 16);
    }
  }
};

__device__ __forceinline__ float scale_to(float m, float top, float c) {
  return m == top ? 1.f : fast_exp2((m - top) * c);  // 0 for m = -inf
}

// A thread's running (max, sum of 2^((l - max) * c)) over one row.
struct RowSum {
  float m = -INFINITY, sum = 0.f;

  template <int N>
  __device__ __forceinline__ void add(uint32_t (&w)[N][4], float c) {
    __nv_bfloat162 mx = neg_inf2();
#pragma unroll
    for (int u = 0; u < N; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = __hmax2(mx, *reinterpret_cast<const __nv_bfloat162*>(&w[u][e]));
    }
    const float top = fmaxf(m, fmaxf(__low2float(mx), __high2float(mx)));
    if (top == -INFINITY) return;  // nothing but -inf and NaN
    const float base = top * c;
    if (!(fabsf(base) < 0x1p24f)) {
      // infinite, or so steep that the next bf16 is 2^-65536 below: ties of the
      // largest share everything
      if (m < top) sum = 0.f;
      m = top;
#pragma unroll
      for (int u = 0; u < N; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum += static_cast<float>(__uint_as_float(w[u][e] << 16) == top) +
                 static_cast<float>(__uint_as_float(w[u][e] & 0xffff0000u) == top);
      }
      return;
    }
    sum *= scale_to(m, top, c);
    m = top;
    // l * c - base in one fma each: base is rounded, by r exactly, alike in all
    const uint64_t c2 = pack_f32x2(c, c), nbase2 = pack_f32x2(-base, -base);
    const float r = fmaf(top, c, -base);
    float a = exps(w, c2, nbase2);
    if (a != a) {  // NaN logits have no weight
#pragma unroll
      for (int u = 0; u < N; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[u][e] = clean2(w[u][e]);
      }
      a = exps(w, c2, nbase2);
    }
    sum += a * fast_exp2(-r);
  }

 private:
  template <int N>
  __device__ __forceinline__ static float exps(const uint32_t (&w)[N][4], uint64_t c2,
                                               uint64_t nbase2) {
    uint64_t acc[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
#pragma unroll
    for (int u = 0; u < N; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t l2 = pack_f32x2(__uint_as_float(w[u][e] << 16),
                                       __uint_as_float(w[u][e] & 0xffff0000u));
        acc[e & 1] = add_f32x2(acc[e & 1], exp2_mufu_f32x2(fma_f32x2(l2, c2, nbase2)));
      }
    }
    const float2 a = unpack_f32x2(add_f32x2(acc[0], acc[1]));
    return a.x + a.y;
  }
};

// This thread's part of a slice of one row (kRowBatch vectors in flight), or of
// the target's and the draft's row together (that many of each).
constexpr int kRowBatch = 5;

// The partial groups of a slice, one on each of two threads.
__device__ __forceinline__ int edge_group(const Slice& s) {
  const int g = threadIdx.x == 0 ? 0 : (threadIdx.x == 1 ? s.groups - 1 : -1);
  return (threadIdx.x == 1 && g == 0) || !s.partial(g) ? -1 : g;
}

template <bool kTwo>
__device__ __forceinline__ void scan_rows(const Slice& s, const Slice& s2, float c, RowSum& r,
                                          RowSum& r2) {
  const int hi = kTwo ? max(s.hi, s2.hi) : s.hi;
#pragma unroll 1
  for (int g0 = threadIdx.x; g0 < hi; g0 += kRowBatch * kVerifyThreads) {
    uint32_t w[kRowBatch][4], v[kTwo ? kRowBatch : 1][4];
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) s.load(g0 + u * kVerifyThreads, w[u]);
    if constexpr (kTwo) {
#pragma unroll
      for (int u = 0; u < kRowBatch; ++u) s2.load(g0 + u * kVerifyThreads, v[u]);
    }
    r.add(w, c);
    if constexpr (kTwo) r2.add(v, c);
  }
  if (threadIdx.x < 2) {
    uint32_t w[1][4];
    const int g = edge_group(s), g2 = kTwo ? edge_group(s2) : -1;
    if (g >= 0) {
      s.load_any(g * 8 - s.shift, w[0]);
      r.add(w, c);
    }
    if (kTwo && g2 >= 0) {
      s2.load_any(g2 * 8 - s2.shift, w[0]);
      r2.add(w, c);
    }
  }
}

// Greedy rows: this thread's best logit of a slice and its first column.
__device__ __forceinline__ unsigned long long scan_best(const Slice& s, int x0) {
  unsigned long long key = 0ull;
  auto take = [&](const uint32_t w[4], int g) {
    const __nv_bfloat162 m = __hmax2(
        __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]),
                *reinterpret_cast<const __nv_bfloat162*>(&w[1])),
        __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w[2]),
                *reinterpret_cast<const __nv_bfloat162*>(&w[3])));
    const float best = fmaxf(__low2float(m), __high2float(m));  // NaN: all NaN
    if (!(best > -INFINITY) || vkey(best, 0u) <= key) return;
    int first = 7;
#pragma unroll
    for (int e = 7; e >= 0; --e) {
      const float l = __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
      if (l == best) first = e;
    }
    const unsigned long long k = vkey(best, static_cast<uint32_t>(x0 + g * 8 - s.shift + first));
    key = k > key ? k : key;
  };
#pragma unroll 1
  for (int g0 = threadIdx.x; g0 < s.hi; g0 += kRowBatch * kVerifyThreads) {
    uint32_t w[kRowBatch][4];
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) s.load(g0 + u * kVerifyThreads, w[u]);
#pragma unroll
    for (int u = 0; u < kRowBatch; ++u) take(w[u], g0 + u * kVerifyThreads);
  }
  if (threadIdx.x < 2) {
    const int g = edge_group(s);
    if (g >= 0) {
      uint32_t w[4];
      s.load_any(g * 8 - s.shift, w);
      take(w, g);
    }
  }
  return key;
}

// Every warp's slot to every CTA of the cluster. After the barrier this CTA has
// all of them, in column order; a buffer is written again two exchanges later,
// when all have read it. No CTA's shared memory is written before it runs: its
// arrival is in the constructor, the wait for the others' in the first call.
struct Exchange {
  VerifyShared& sh;
  int rank, ranks, warp, lane, parity = 0;
  bool started = false;

  __device__ __forceinline__ explicit Exchange(VerifyShared& s)
      : sh(s),
        rank(static_cast<int>(cg::this_cluster().block_rank())),
        ranks(static_cast<int>(cg::this_cluster().num_blocks())),
        warp(threadIdx.x >> 5),
        lane(threadIdx.x & 31) {}
  __device__ __forceinline__ void arrive() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
  __device__ __forceinline__ const VerifySlot* operator()(const VerifySlot& mine) {
    if (!started) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    started = true;
    VerifySlot* at = &sh.slots[parity][rank * kVerifyWarps + warp];
    if (lane < ranks) *cg::this_cluster().map_shared_rank(at, lane) = mine;
    cg::this_cluster().sync();
    const VerifySlot* all = sh.slots[parity];
    parity ^= 1;
    return all;
  }
};

__device__ __forceinline__ const unsigned short* row_of(const __nv_bfloat16* base, int64_t b,
                                                        int64_t stride_seq, int64_t row,
                                                        int64_t stride_row) {
  return reinterpret_cast<const unsigned short*>(base) + b * stride_seq + row * stride_row;
}

template <bool kDraft>
__global__ void __launch_bounds__(kVerifyThreads, 3) verify_walk_kernel(const VerifyParams p) {
  __shared__ VerifyShared sh;
  __shared__ double table[kExpTable];
  __shared__ int32_t parents[kMaxNodes];
  __shared__ int32_t path[kMaxNodes + 1];
  Exchange exchange(sh);
  const int rank = exchange.rank, ranks = exchange.ranks, lane = exchange.lane;
  const int b = blockIdx.x / ranks;
  const int tid = threadIdx.x;
  const int nslots = ranks * kVerifyWarps;
  // the draw may start beside this grid's last CTAs: it waits for their results
  asm volatile("griddepcontrol.launch_dependents;");

  const int x0 = min(rank * p.slice, p.vocab);
  const int len = min(p.slice, p.vocab - x0);
  const int n = p.num_nodes ? min(max(p.num_nodes[b], 0), p.nodes) : p.nodes;
  const float temp = temperature_of(p, b);
  const bool greedy = !(temp > 0.f);
  const double c64 = greedy ? 1.0 : 1.4426950408889634074 / static_cast<double>(temp);
  const float c32 = fminf(static_cast<float>(c64), 1e30f);
  const int64_t* tokens = p.tokens + static_cast<int64_t>(b) * (p.nodes - 1);
  const float* u = p.u_accept + static_cast<int64_t>(b) * (p.nodes - 1);
  const int64_t out_row = static_cast<int64_t>(b) * p.nodes;

  if (n == 0) {  // a padding row (uniform over the cluster)
    for (int i = tid; rank == 0 && i < p.nodes; i += kVerifyThreads) {
      p.out_tokens[out_row + i] = -1;
      p.out_path[out_row + i] = -1;
    }
    if (rank == 0 && tid == 0) p.out_num[b] = 0;
    return;
  }
  exchange.arrive();
  for (int i = tid; i < p.nodes; i += kVerifyThreads)
    parents[i] = p.parents ? p.parents[static_cast<int64_t>(b) * p.parents_stride + i] : i - 1;
  if (!greedy) fill_table(table);
  if (tid == 0) path[0] = 0;
  __syncthreads();

  int node = 0, count = 0;
  while (true) {
    const unsigned short* prow = row_of(p.logits, b, p.l_stride_seq, node, p.l_stride_row);
    const bool with_q = kDraft && !greedy && node + 1 < n;
    const unsigned short* qrow =
        with_q ? row_of(p.draft, b, p.d_stride_seq, node, p.d_stride_row) : prow;
    const Slice ps(prow + x0, len), qs(qrow + x0, with_q ? len : 0);
    if (tid == 0) {
      if (count == 0) {  // later rows were sent for at the node before
        ps.prefetch();
        qs.prefetch();
      }
      // the rows of the likeliest next node, the first child
      int c = node + 1;
      while (c < n && parents[c] != node) ++c;
      if (c < n && p.ahead) {
        Slice(row_of(p.logits, b, p.l_stride_seq, c, p.l_stride_row) + x0, len).prefetch();
        if (kDraft && !greedy && c + 1 < n)
          Slice(row_of(p.draft, b, p.d_stride_seq, c, p.d_stride_row) + x0, len).prefetch();
      }
    }

    // ---- a candidate child a lane: its token and what the rows say of it
    struct Child {
      int64_t tok;
      float u;
      uint32_t pbits, qbits;
      bool mine, in;
    };
    auto child = [&](int c) {
      Child k{-1, 0.f, 0xff80u, 0xff80u, c < n && parents[min(c, kMaxNodes - 1)] == node, false};
      if (k.mine) {
        k.tok = tokens[c - 1];
        k.u = u[c - 1];
        k.in = k.tok >= 0 && k.tok < p.vocab;
        if (k.in) k.pbits = __ldg(prow + k.tok);
        if (k.in && with_q) k.qbits = __ldg(qrow + k.tok);
      }
      return k;
    };
    const Child first = child(node + 1 + lane);

    // ---- the row's largest logit and sum of exponentials
    float pmax, qmax = -INFINITY;
    double psum = 1.0, qsum = 1.0;
    int argmax = 0;
    if (greedy) {
      VerifySlot v;
      v.key[0] = warp_max(scan_best(ps, x0));
      v.key[1] = 0ull;
      const VerifySlot* all = exchange(v);
      unsigned long long key = 0ull;
      for (int i = lane; i < nslots; i += 32) key = all[i].key[0] > key ? all[i].key[0] : key;
      key = warp_max(key);
      pmax = vkey_score(key);
      argmax = key ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)) : 0;
    } else {
      RowSum r, r2;
      scan_rows<kDraft>(ps, qs, c32, r, r2);
      VerifySlot v;
      v.f.x = warp_max(r.m);
      v.f.y = warp_sum(r.sum * scale_to(r.m, v.f.x, c32));
      v.f.z = kDraft ? warp_max(r2.m) : -INFINITY;
      v.f.w = kDraft ? warp_sum(r2.sum * scale_to(r2.m, v.f.z, c32)) : 0.f;
      const VerifySlot* all = exchange(v);
      float pm = -INFINITY, qm = -INFINITY;
      for (int i = lane; i < nslots; i += 32) {
        pm = fmaxf(pm, all[i].f.x);
        if (kDraft) qm = fmaxf(qm, all[i].f.z);
      }
      pmax = warp_max(pm);
      if (kDraft) qmax = warp_max(qm);
      float a = 0.f, d = 0.f;
      for (int i = lane; i < nslots; i += 32) {
        const float4 f = all[i].f;
        a += f.y * scale_to(f.x, pmax, c32);
        if (kDraft) d += f.w * scale_to(f.z, qmax, c32);
      }
      psum = static_cast<double>(warp_sum(a));
      if (kDraft) qsum = static_cast<double>(warp_sum(d));
    }
    // bf16 bits of the largest logits, kNoLogit where there is none
    const uint32_t top = __float_as_uint(pmax) >> 16;
    const uint32_t qtop = with_q ? __float_as_uint(qmax) >> 16 : kNoLogit;
    const bool any = top != kNoLogit, any_q = qtop != kNoLogit;

    // ---- which child goes on: every warp of the cluster takes this decision
    // alike. With the fp32 sums (off by 2.2e-5 at most, see near_border) an outcome
    // within 2^-14 of its border is left open, and taken again with fp64 sums.
    int next = -1;
#pragma unroll 1
    for (int exact = 0; exact < 2; ++exact) {
      if (exact) {
        const RowScale scale(any ? top : 0u, c64), qscale(any_q ? qtop : 0u, c64);
        double a = 0.0, d = 0.0;
#pragma unroll 4
        for (int i = tid; i < len; i += kVerifyThreads) {
          const uint32_t pb = __ldg(ps.src + i), qb = any_q ? __ldg(qs.src + i) : 0u;
          a += exp2_64(scale.log2_weight(__uint_as_float(scale.raise(pb) << 16)), table);
          if (any_q) d += exp2_64(qscale.log2_weight(__uint_as_float(qscale.raise(qb) << 16)), table);
        }
        VerifySlot v;
        v.d = make_double2(warp_sum(a), warp_sum(d));
        const VerifySlot* all = exchange(v);
        a = d = 0.0;
        for (int i = lane; i < nslots; i += 32) {
          a += all[i].d.x;
          d += all[i].d.y;
        }
        psum = warp_sum(a);
        qsum = warp_sum(d);
      }
      // a logit's weight beside psum; none for NaN and -inf. In fp32 at least
      // 2^-100, so that a live logit is told from none.
      auto weight = [&](uint32_t bits, uint32_t top_bits, float top_l, bool live) {
        const float l = __uint_as_float(bits << 16);
        double w = fmax(static_cast<double>(scale_to(l, top_l, c32)), 0x1p-100);
        if (exact) {
          const RowScale sc(live ? top_bits : 0u, c64);
          w = exp2_64(sc.log2_weight(__uint_as_float(sc.raise(bits) << 16)), table);
        }
        return live && l > -INFINITY && w > kNothing ? w : 0.0;
      };
      double left = psum;  // of p's weights
      int nrej = 0;  // rejected tokens: lane i holds the i-th and the 32+i-th
      int64_t rej0 = -1, rej1 = -1;
      bool open = false;
      next = -1;
      for (int c0 = node + 1; c0 < n && next < 0 && !open; c0 += 32) {
        const Child k = c0 == node + 1 ? first : child(c0 + lane);
        double here = 0.0, against = 0.0;
        if (!greedy) {  // uniform
          here = weight(k.pbits, top, pmax, k.in && any);
          if (kDraft) against = weight(k.qbits, qtop, qmax, k.in && any_q);
        }
        unsigned todo = __ballot_sync(0xffffffffu, k.mine);
        while (todo && next < 0 && !open) {
          const int src = __ffs(todo) - 1;
          todo &= todo - 1;
          const int64_t x = __shfl_sync(0xffffffffu, k.tok, src);
          const bool inside = __shfl_sync(0xffffffffu, static_cast<int>(k.in), src);
          double hc = __shfl_sync(0xffffffffu, here, src);
          const double uu = static_cast<double>(__shfl_sync(0xffffffffu, k.u, src));
          const double qc = kDraft ? __shfl_sync(0xffffffffu, against, src) : 0.0;
          bool ok;
          if (greedy) {
            ok = inside && any && x == argmax;
          } else {
            if (!kDraft && __any_sync(0xffffffffu, inside && (rej0 == x || rej1 == x)))
              hc = 0.0;  // a token tried before has no probability left
            // u q < p over the common denominator; without q: u R < p times psum
            const double side = kDraft && any_q ? hc * qsum : hc;
            const double bar = uu * (kDraft ? qc * psum : left);
            ok = bar < side;
            open = !exact && hc > 0.0 &&
                   (fabs(bar - side) <= 0x1p-14 * (side + (kDraft ? bar : psum)) ||
                    fmax(bar, side) < 0x1p-60);
          }
          if (ok) {
            next = c0 + src;
          } else {
            left -= hc;
            if (!kDraft && inside) {
              if (lane == (nrej & 31)) (nrej < 32 ? rej0 : rej1) = x;
              ++nrej;
            }
          }
        }
      }
      if (!open) break;
    }
    if (next >= 0) {
      node = next;
      ++count;
      if (tid == 0) path[count] = node;
      continue;
    }
    if (rank == 0) {
      __syncthreads();  // path
      for (int i = tid; i < p.nodes; i += kVerifyThreads) {
        p.out_path[out_row + i] = i <= count ? path[i] : -1;
        int64_t t = i < count ? tokens[path[i + 1] - 1] : -1;
        if (i == count)
          t = greedy || !any ? argmax
                             : pack_state({top, qtop, static_cast<float>(psum / qsum)});
        p.out_tokens[out_row + i] = t;
      }
      // !any, told to the draw by the sign, is a pick already
      if (tid == 0) p.out_num[b] = greedy || any ? count : ~count;
    }
    return;
  }
}

// The draw of every sequence's next token from the row of its last node: p, or p
// without its rejected children's tokens, or (a draft row) max(p - q, 0).
template <bool kDraft>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_draw_kernel(const VerifyParams p) {
  __shared__ VerifyShared sh;
  __shared__ double table[kExpTable];
  __shared__ uint16_t near_at[kDraft ? kNears : 1][kVerifyThreads];  // step * 8 + element
  Exchange exchange(sh);
  const int rank = exchange.rank, ranks = exchange.ranks;
  const int lane = exchange.lane, warp = exchange.warp;
  const int b = blockIdx.x / ranks;
  const int nslots = ranks * kVerifyWarps;
  fill_table(table);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the walk is done
  const int n = p.num_nodes ? min(max(p.num_nodes[b], 0), p.nodes) : p.nodes;
  const float temp = temperature_of(p, b);
  const int num = p.out_num[b];
  cg::this_cluster().sync();  // all have read num, and run
  exchange.started = true;
  if (num < 0) {
    if (rank == 0 && threadIdx.x == 0) p.out_num[b] = ~num;
    return;
  }
  if (n == 0 || !(temp > 0.f)) return;

  const int64_t out_row = static_cast<int64_t>(b) * p.nodes;
  const int node = p.out_path[out_row + num];
  const DrawState st = unpack_state(p.out_tokens[out_row + num]);
  const int x0 = min(rank * p.slice, p.vocab);
  const int len = min(p.slice, p.vocab - x0);
  const double c64 = 1.4426950408889634074 / static_cast<double>(temp);
  const RowScale scale(st.top, c64), qscale(st.qtop == kNoLogit ? 0u : st.qtop, c64);
  double ratio = static_cast<double>(st.ratio);
  bool use_q = kDraft && st.qtop != kNoLogit;
  const Slice ps(row_of(p.logits, b, p.l_stride_seq, node, p.l_stride_row) + x0, len);
  const Slice qs(
      (use_q ? row_of(p.draft, b, p.d_stride_seq, node, p.d_stride_row) + x0 : ps.src), len);

  // the rejected tokens: the node's children. Lane i holds the i-th and 32+i-th.
  int64_t rej[2] = {-1, -1};
  if (!kDraft) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = h * 32 + lane;
      const int parent = c >= p.nodes ? -1
                         : p.parents  ? p.parents[static_cast<int64_t>(b) * p.parents_stride + c]
                                      : c - 1;
      if (c > node && c < n && parent == node)
        rej[h] = p.tokens[static_cast<int64_t>(b) * (p.nodes - 1) + c - 1];
    }
  }

  // A warp owns `steps` steps of 32 16-byte groups, in column order; bin i (lane
  // i's) is steps [i * per, (i + 1) * per).
  const int steps = (ps.groups + kVerifyThreads - 1) / kVerifyThreads;
  const int per = (steps + 31) / 32;
  auto group = [&](int step) { return (warp * steps + step) * 32 + lane; };
  // those of the rejected tokens that lie among this warp's columns
  uint32_t mask[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t x = rej[h] - x0 - (warp * steps * 256 - ps.shift);
    mask[h] = __ballot_sync(0xffffffffu, rej[h] >= 0 && x >= 0 && x < steps * 256);
  }
  bool skip = __any_sync(0xffffffffu, rej[0] >= 0 || rej[1] >= 0);
  // Loads of a step's 8 columns: issue() sends for what needs no look at the
  // data, finish() reads partial groups and draft rows at another alignment.
  const bool same = qs.shift == ps.shift;
  auto issue = [&](int g, uint32_t w[4], uint32_t v[4]) {
    ps.load(g, w);
    if (kDraft && use_q && same) qs.load(g, v);
  };
  auto finish = [&](int g, uint32_t w[4], uint32_t v[4]) {
    if (ps.partial(g)) ps.load_any(g * 8 - ps.shift, w);
    if (kDraft && use_q && (!same || ps.partial(g))) qs.load_any(g * 8 - ps.shift, v);
    if (!kDraft && skip) {  // rejected columns have no weight
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll 1
        for (uint32_t m = mask[h]; m; m &= m - 1) {
          const int64_t x =
              __shfl_sync(0xffffffffu, rej[h], __ffs(m) - 1) - x0 - (g * 8 - ps.shift);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (x == e) w[e >> 1] |= (e & 1) ? 0xffff0000u : 0xffffu;  // NaN
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = scale.raise(w[e]);
      if (kDraft && use_q) v[e] = qscale.raise(v[e]);
    }
  };
  auto logit = [](const uint32_t w[4], int e) {
    return __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
  };

  double pinv = 1.0, qinv = 0.0;
  bool exact = false, again = false;  // ratio is that of the exact sums; a second draw, from p
#pragma unroll 1
  while (true) {
    // ---- one pass. With a draft row it gives the exact sums a, d and, over the
    // columns where p exceeds q by the sums of the walk, the parts ra, rd of the
    // residual. A thread notes the columns that those sums may have on the wrong
    // side: of ordinary rows none, a few or, where the rows' logits are on a grid
    // that meets the border, some hundred of 151,936. Otherwise ra is p's.
    double a = 0.0, d = 0.0, ra = 0.0, rd = 0.0, sa = 0.0, sd = 0.0;
    int nears = 0;
    uint32_t w[4], v[4] = {0u, 0u, 0u, 0u}, wn[4], vn[4];
    issue(group(0), w, v);
#pragma unroll 1
    for (int step = 0, in_bin = 0, bin = 0; step < steps; ++step) {
      if (step + 1 < steps) issue(group(step + 1), wn, vn);  // before this step's arithmetic
      finish(group(step), w, v);
      uint32_t near = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double wp = exp2_64(scale.log2_weight(logit(w, e)), table);
        if (kDraft && use_q) {
          const double wq = exp2_64(qscale.log2_weight(logit(v, e)), table), x = wq * ratio;
          a += wp;
          d += wq;
          if (wp > x) {
            sa += wp;
            sd += wq;
          }
          near |= static_cast<uint32_t>(near_border(wp, x, p.border)) << e;
        } else {
          sa += wp;
        }
      }
      if (kDraft && near) {
#pragma unroll 1
        for (; near; near &= near - 1, ++nears)
          if (nears < kNears) near_at[nears][threadIdx.x] = step * 8 + __ffs(near) - 1;
      }
      if (++in_bin == per || step + 1 == steps) {
        const double ta = warp_sum(sa);
        if (lane == bin) ra = ta;
        if (kDraft && use_q) {
          const double td = warp_sum(sd);
          if (lane == bin) rd = td;
        }
        sa = sd = 0.0;
        in_bin = 0;
        ++bin;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = wn[e];
        v[e] = vn[e];
      }
    }
    double mine = ra;  // the weight of this lane's bin
    if (kDraft && use_q) {
      // a thread with more columns near the border than it notes: told by the sign of d
      const bool many = __any_sync(0xffffffffu, !exact && nears > kNears);
      VerifySlot s;
      s.d = make_double2(warp_sum(a), warp_sum(d));
      if (many) s.d.y = -s.d.y;
      const VerifySlot* all = exchange(s);
      bool retake = false;
      a = d = 0.0;
      for (int i = lane; i < nslots; i += 32) {
        a += all[i].d.x;
        d += fabs(all[i].d.y);
        retake |= all[i].d.y < 0.0;
      }
      a = warp_sum(a);
      d = warp_sum(d);
      if (__any_sync(0xffffffffu, retake)) {
        // columns of a common quotient, as where the rows agree but for a few
        // columns: another pass with the sides by the exact sums
        ratio = a / d;
        exact = true;
        continue;
      }
      pinv = 1.0 / a;
      qinv = 1.0 / d;
      double fix = 0.0;  // of this lane's bin: what its near columns' true sides change
      if (exact) nears = 0;
#pragma unroll 1
      for (int k = 0; __any_sync(0xffffffffu, k < nears); ++k) {
        double change = 0.0;
        int bin = 0;
        if (k < nears) {
          const int noted = near_at[k][threadIdx.x], step = noted >> 3;
          const int x = group(step) * 8 - ps.shift + (noted & 7);
          const double wp = exp2_64(
              scale.log2_weight(__uint_as_float(scale.raise(__ldg(ps.src + x)) << 16)), table);
          const double wq = exp2_64(
              qscale.log2_weight(__uint_as_float(qscale.raise(__ldg(qs.src + x)) << 16)), table);
          const double has = wp * pinv - wq * qinv;
          change = fmax(has, 0.0) - (wp > wq * ratio ? has : 0.0);
          bin = step / per;
        }
#pragma unroll 1
        for (unsigned who = __ballot_sync(0xffffffffu, k < nears); who; who &= who - 1) {
          const int from = __ffs(who) - 1;
          const double c = __shfl_sync(0xffffffffu, change, from);
          if (__shfl_sync(0xffffffffu, bin, from) == lane) fix += c;
        }
      }
      mine = fmax(ra * pinv - rd * qinv + fix, 0.0);
    }
    VerifySlot s;
    s.d = make_double2(warp_sum(mine), 0.0);
    const VerifySlot* all = exchange(s);
    // prefix over the warps in column order, `each` consecutive ones a lane
    const int each = (nslots + 31) / 32;
    double own = 0.0;
    for (int i = 0; i < each; ++i)
      own += lane * each + i < nslots ? all[lane * each + i].d.x : 0.0;
    const double incl = warp_scan(own, lane);
    const double total = __shfl_sync(0xffffffffu, incl, 31);
    if (kDraft && use_q && !exact && !(total > 0x1p-12)) {
      // rows that almost agree: the weights that near_border leaves out would
      // count, so another pass with the sides by the exact sums
      ratio = a / d;
      exact = true;
      continue;
    }
    if (!(total > kNothing) && !again) {
      use_q = skip = false;  // rounding rejected the last of the mass: draw from p
      pinv = 1.0;
      qinv = 0.0;
      again = true;
      continue;
    }
    const double threshold =
        fmax(static_cast<double>(fmaxf(p.u_pick[b], 0.f)) * total, kNothing);
    // the first warp whose weights cross the threshold (with u so near 1 that
    // rounding hides the border: the last one with weight)
    const unsigned over = __ballot_sync(0xffffffffu, incl > threshold);
    const unsigned some = __ballot_sync(0xffffffffu, own > kNothing);
    const int ol = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : 0);
    double before = __shfl_sync(0xffffffffu, incl - own, ol);
    int owner = -1, last = 0;
    for (int i = ol * each; i < min((ol + 1) * each, nslots) && owner < 0; ++i) {
      const double t = all[i].d.x;
      if (t > kNothing) last = i;
      if (over && before + t > threshold)
        owner = i;
      else
        before += t;
    }
    const double want = owner >= 0 ? threshold - before : INFINITY;
    if (owner < 0) owner = last;
    if (owner != rank * kVerifyWarps + warp) return;

    // ---- the owner's bin, step, lane and column
    const double bins = warp_scan(mine, lane);
    const unsigned obin = __ballot_sync(0xffffffffu, bins > want);
    const unsigned pbin = __ballot_sync(0xffffffffu, mine > kNothing);
    const int bin = obin ? __ffs(obin) - 1 : (pbin ? 31 - __clz(pbin) : 0);
    double sum = __shfl_sync(0xffffffffu, bins - mine, bin);
    int found = -1, lastx = -1;
#pragma unroll 1
    for (int step = bin * per; step < min((bin + 1) * per, steps) && found < 0; ++step) {
      const int g = group(step), at = g * 8 - ps.shift;
      issue(g, w, v);
      finish(g, w, v);
      double wp[8], t = 0.0;
      int lx = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        wp[e] = exp2_64(scale.log2_weight(logit(w, e)), table) * pinv;
        if (kDraft && use_q)
          wp[e] = fmax(wp[e] - exp2_64(qscale.log2_weight(logit(v, e)), table) * qinv, 0.0);
        t += wp[e];
        if (wp[e] > kNothing) lx = at + e;
      }
      const double upto = warp_scan(t, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, lx >= 0 && sum + upto > want);
      const unsigned pos = __ballot_sync(0xffffffffu, lx >= 0);
      if (hit) {
        int x = -1;  // in that lane, the first column that crosses
        double run = sum + (upto - t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          run += wp[e];
          if (x < 0 && wp[e] > kNothing && run > want) x = at + e;
        }
        found = __shfl_sync(0xffffffffu, x < 0 ? lx : x, __ffs(hit) - 1);
      }
      if (pos) lastx = __shfl_sync(0xffffffffu, lx, 31 - __clz(pos));
      sum += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0)  // weights lie inside the slice
      p.out_tokens[out_row + num] = x0 + min(max(found >= 0 ? found : lastx, 0), len - 1);
    return;
  }
}

// Columns of a CTA of a cluster, in whole 16-byte groups.
static int slice_of(int vocab, int ranks) { return ((vocab + ranks - 1) / ranks + 7) / 8 * 8; }

static cudaError_t launch_cluster(void (*kernel)(VerifyParams), VerifyParams p, int batch, int ranks,
                                  bool dependent, cudaStream_t stream) {
  p.slice = slice_of(p.vocab, ranks);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch) * ranks);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[3];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeClusterSchedulingPolicyPreference;
  attr[1].val.clusterSchedulingPolicyPreference = cudaClusterSchedulingPolicySpread;
  attr[2].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[2].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 3 : 2;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// CTAs an SM that size the clusters (fit below). The walk's rows are a chain, so
// more CTAs a sequence shorten it until they queue for the SMs: 64 sequences of 7
// drafts take 142, 120 and 138 us with 4, 8 and 16 CTAs each. The draw is bound by
// fp64: what the SMs hold at once (64 sequences: 4 CTAs each 120 us for both
// kernels, 8 each 127).
constexpr int kWalkPerSm = 6, kDrawPerSm = 2;

template <bool kDraft>
static int launch_verify(VerifyParams p, int batch, cudaStream_t stream) {
  static std::mutex mu;
  static bool done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !done[dev]) {
      cudaError_t e = cudaFuncSetAttribute(verify_walk_kernel<kDraft>,
                                           cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(verify_draw_kernel<kDraft>,
                                 cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(verify)");
      if (dev < 64) done[dev] = true;
    }
  }
  // CTAs a sequence, from the batch alone
  const int64_t sms = device_sm_count();
  auto fit = [&](int per_sm) {
    int ranks = kMaxCluster;
    while (ranks > 2 && static_cast<int64_t>(batch) * ranks > per_sm * sms) ranks /= 2;
    return ranks;
  };
  const int ranks = fit(kWalkPerSm);
  p.ahead = static_cast<int64_t>(batch) * ranks <= kWalkPerSm * sms;
  // of a thread of the walk: whole groups in batches, then one at a slice's edge
  const int groups = slice_of(p.vocab, ranks) / 8 + 1, step = kRowBatch * kVerifyThreads;
  p.border = (groups + step - 1) / step + 1 <= kShortBatches ? kBorderShort : kBorderLong;
  cudaError_t e = launch_cluster(verify_walk_kernel<kDraft>, p, batch, ranks, false, stream);
  if (e != cudaSuccess) return cuda_fail(e, "verify_walk_kernel launch");
  if (p.temperatures == nullptr) return NVATTN_OK;  // all greedy: nothing to draw
  e = launch_cluster(verify_draw_kernel<kDraft>, p, batch, fit(kDrawPerSm), true, stream);
  return e == cudaSuccess ? NVATTN_OK : cuda_fail(e, "verify_draw_kernel launch");
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
