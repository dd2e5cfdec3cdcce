// Speculative decoding around the attention kernel: verification of a drafted token tree against the target's probabilities,
// and the commit of the accepted path's keys and values into the paged cache.
//
// Verification.  Sequence b owns the nodes cu[b] .. cu[b + 1] - 1; logits[n] are the target's logits AFTER node n, and
// p_n = softmax(logits[n] / temperature[b]) (temperature 0: all mass on the largest logit, the lowest index of a tie).  The walk
// starts at the sequence's first node with r = p.  The children of the current node are tried in the order of their
// positions: child x with draft probability q(x) is accepted when u_accept[x] * q(x) < r(x); otherwise r becomes
// max(r - q, 0), normalised (unchanged if nothing is left).  An accepted child becomes the current node.  Without draft
// probabilities a child is a point mass (q(x) = 1): a rejected token leaves r.  When no child is left the last token is drawn
// from r: the first token whose cumulative sum exceeds u_sample[b] times the total.  So every emitted token is distributed
// as the target's own sample, whatever was drafted.
//
// Four kernels.  verify_stats_kernel reads every node's logits once - that is the cost of the whole: 2 bytes for each logit, at
// 16 exponentials a cycle and SM about 0.7 of the time that HBM needs for them - and leaves the maximum and the sum of
// exponentials of every 2048-column piece of a row.  verify_walk_kernel gathers the probabilities of all nodes' tokens and walks
// every tree out of shared memory (with draft probabilities a cluster of eight CTAs, which sums the residuals between siblings).
// verify_sums_kernel sums what is left in every 8192-column chunk of the row in which a walk ended, verify_pick_kernel finds the
// token in the chunk where the sum passes the coin's share.
//
// A sum that decides a token needs more than fp32, though its terms exp((z - max) / temperature) are fp32: a vocabulary of 10^5
// tokens has bins of 10^-5 and less, and fp32 partial sums would move their borders by a share of that.  The last draw's and the
// residuals' sums are held as unevaluated sums of two fp32 numbers in every thread (about 48 bits, six additions a term), threads
// and chunks are joined in fp64.
//
// The rows' totals from the statistics are sums of fp32 numbers with exponentials from the special-function unit, off by less
// than 2^-17 of themselves: an exponential 2^x by 2^-22 and by 2^-22 |x| for its argument (|x| <= 18 where it counts, since a row
// has less than 2^18 terms), the additions by 2^-20.  Probabilities, acceptances with draft probabilities and log-probabilities
// carry that error.  With certain drafts it would land in full in the mass that rejections leave (1 minus the rejected ones),
// however small that is, and a token that is all that is left could be rejected.  So an acceptance whose two sides lie closer
// together than twice their error is settled by the row's own weights: what is left of the row is summed as for the last draw.  With
// ordinary coins that is one test in 2^15 or fewer, and takes one CTA 28 us for 152064 logits.
#include "common.cuh"

#include <cooperative_groups.h>

namespace b200 {

constexpr int SP_PAGE = 64;
constexpr int SP_DH = 128;
constexpr int SP_MAX_NODES = 64;
constexpr int SP_LOADS = 8;                          // 16-byte loads of a lane for one piece of a row
constexpr int SP_PIECE = SP_LOADS * 32;              // granules of a piece (2048 logits), the work of one warp at a time
constexpr int SP_STAT_THREADS = 256;
constexpr int SP_STAT_CTAS = 2;                      // resident on an SM
constexpr int SP_SUM_THREADS = 256;
constexpr int SP_CHUNK = 1024;                       // granules of a chunk of the last draw (8192 logits)
constexpr int SP_CLUSTER = 8;
constexpr int SP_THREADS = 512;                      // of a walking CTA with draft probabilities; 256 without
constexpr float SP_LOG2E = 1.4426950408889634f;
// Certain drafts: u rest and r are off by less than 2^-17 of r and of the rejected mass (the totals' error); this is twice that.
constexpr double SP_CLOSE = 1.0 / 65536;

// A row of logits as aligned 16-byte granules of eight: rows of an odd vocabulary start anywhere, so a row begins `skip` elements
// into its first granule.  Granules are read whole; what lies outside of the row is replaced by -inf.
struct LogitRow {
  const uint4* granules;
  int skip, count, V;
  __device__ __forceinline__ LogitRow(const __nv_bfloat16* row, int V_) : V(V_) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    granules = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
    skip = static_cast<int>(at & 15) / 2;
    count = (skip + V + 7) / 8;
  }
  __device__ __forceinline__ uint4 load(int g) const {
    if (g >= count) return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    return __ldg(granules + g);
  }
  // the first and the last granule of the row, cut to it
  __device__ __forceinline__ void trim(uint4& v, int g) const {
    if (g == 0 || g == count - 1) {
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = g * 8 - skip + k;
        if (e < 0 || e >= V) w[k / 2] = k & 1 ? (w[k / 2] & 0xffffu) | 0xff800000u : (w[k / 2] & 0xffff0000u) | 0xff80u;
      }
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// What verify_walk_kernel leaves for the last draw of a sequence.
struct WalkEnd {
  double total;              // sum of exp((z - top) / temperature) over the row
  float2 inv_total;          // its reciprocal, as two fp32 numbers
  float2 rz[SP_MAX_NODES];   // reciprocals of the residuals' sums (draft probabilities given)
  int gone[SP_MAX_NODES];    // rejected tokens (point-mass drafts)
  float top;                 // largest z of the row
  int node;                  // batch row in which the walk ended, -1: nothing is left to draw
  int k, nz, ngone, less;    // tokens emitted so far; residuals, rejected tokens; whether one more rejection has to be taken off
};

struct VerifyArgs {
  const __nv_bfloat16* logits;
  long long ld;
  int V;
  const float* draft;
  long long draft_ld;
  const long long* tokens;
  const int* parents;
  const int* cu;
  int B, N, max_nodes, pieces, chunks;
  const float* temperature;
  const float* u_accept;
  const float* u_sample;
  int* count;
  long long* out_tokens;
  int* path;
  float* logprobs;
  float2* part;   // [N][pieces]: maximum, sum of exponentials relative to it
  int* first;     // [N][pieces]: its first column (rows at temperature 0 only)
  WalkEnd* end;   // [B]
  double* sums;   // [B][chunks]: what is left in a chunk
};

// A number as the unevaluated sum of two fp32 numbers, |lo| <= half a step of hi; about 48 bits.
struct Two {
  float hi, lo;
};
__device__ __forceinline__ Two two_sum(float x, float y) {  // exact (Knuth)
  const float s = __fadd_rn(x, y), t = __fsub_rn(s, x);
  return {s, __fadd_rn(__fsub_rn(x, __fsub_rn(s, t)), __fsub_rn(y, t))};
}
__device__ __forceinline__ Two two_norm(float x, float y) {  // |x| >= |y|
  const float s = __fadd_rn(x, y);
  return {s, __fsub_rn(y, __fsub_rn(s, x))};
}
__device__ __forceinline__ Two two_mul(const Two& x, const Two& y) {
  const float p = __fmul_rn(x.hi, y.hi);
  return two_norm(p, __fadd_rn(__fmaf_rn(x.hi, y.hi, -p), __fmaf_rn(x.hi, y.lo, __fmul_rn(x.lo, y.hi))));
}
__device__ __forceinline__ Two two_minus(const Two& x, float y) {
  const Two s = two_sum(x.hi, -y);
  return two_norm(s.hi, __fadd_rn(s.lo, x.lo));
}
__device__ __forceinline__ void two_add(Two& sum, const Two& x) {  // the running sum: hi exact, what it drops goes to lo
  const Two s = two_sum(sum.hi, x.hi);
  sum.hi = s.hi;
  sum.lo = __fadd_rn(sum.lo, __fadd_rn(s.lo, x.lo));
}
__device__ __forceinline__ Two two_of(double x) {
  const float hi = static_cast<float>(x);
  return {hi, static_cast<float>(x - static_cast<double>(hi))};
}
// Two running sums side by side, one instruction for both.
struct TwoPair {
  uint64_t hi, lo;
  __device__ __forceinline__ void add(uint64_t x) {
    const uint64_t s = add2(hi, x), t = sub2(s, hi);
    lo = add2(lo, add2(sub2(hi, sub2(s, t)), sub2(x, t)));
    hi = s;
  }
  __device__ __forceinline__ Two sum() const {
    float h0, h1, l0, l1;
    unpair2(hi, h0, h1);
    unpair2(lo, l0, l1);
    Two s = {h0, l0};
    const Two x = two_sum(s.hi, h1);
    return {x.hi, __fadd_rn(x.lo, __fadd_rn(l0, l1))};
  }
};
__device__ __forceinline__ double two_double(const Two& x) { return static_cast<double>(x.hi) + static_cast<double>(x.lo); }

// log of a positive sum: the exponent's share in fp64, the logarithm of the mantissa in fp32 (off by less than 2^-23)
__device__ __forceinline__ double sp_log(double x) {
  const float f = static_cast<float>(x);
  const int bits = __float_as_int(f), e = (bits >> 23) - 127;
  const float m = __int_as_float((bits & 0x7fffff) | 0x3f800000);  // 1 .. 2
  return static_cast<double>(e) * 0.69314718055994530942 + (static_cast<double>(logf(m)) + (x - static_cast<double>(f)) / static_cast<double>(f));
}

// A token's exponent.  The difference first: of two bf16 numbers near one another it is exact, where z / temp and top / temp would
// each be rounded at their own size (logits of 20 at temperature 0.05: 400, off by 2^-16, and so would the weight be).
__device__ __forceinline__ float sp_exponent(float z, float temp, float top) {
  const float d = __fsub_rn(z, top);
  return temp == 1.f ? d : __fdiv_rn(d, temp);
}
__device__ __forceinline__ float sp_weight(float z, float temp, float top) { return expf(sp_exponent(z, temp, top)); }
__device__ __forceinline__ float sp_logit(const uint4& v, int e) {
  const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
  return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
}
__device__ __forceinline__ void sp_span(const VerifyArgs& a, int b, int& n0, int& T) {
  n0 = min(max(a.cu[b], 0), a.N);
  T = min(min(max(a.cu[b + 1] - n0, 0), a.max_nodes), a.N - n0);
}

// Every warp has a run of pieces of its own (rows in order) and asks for the next piece before it works on this one.  Bound by HBM:
// 4096 rows of 152064 logits, 1246 MB, in 223 us = 5.6 TB/s; 289 rows of 50281, which start anywhere, 9.6 us.
__global__ void __launch_bounds__(SP_STAT_THREADS, SP_STAT_CTAS) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (SP_STAT_THREADS / 32);
  const long long me = static_cast<long long>(blockIdx.x) * (SP_STAT_THREADS / 32) + (threadIdx.x >> 5);
  const long long items = static_cast<long long>(a.N) * a.pieces;
  long long item = items * me / warps;
  const long long end = items * (me + 1) / warps;
  if (item >= end) return;
  int n = static_cast<int>(item / a.pieces), piece = static_cast<int>(item % a.pieces);
  // the sequence of the first row: the last b with cu[b] <= n, 32 candidates at a time
  int lo = 0, hi = a.B;  // cu[lo] <= n (or lo = 0), cu[hi] > n (or hi = B)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && (lane == 0 || a.cu[at] <= n));
    const int k = 31 - __clz(static_cast<int>(below));
    hi = min(hi, lo + (k + 1) * step);
    lo += k * step;
  }
  int b = lo, next_start = a.cu[b + 1];
  auto settle = [&] {  // the sequence of row n; rows of no sequence take any temperature, nobody reads them
    while (n >= next_start && b + 1 < a.B) next_start = a.cu[++b + 1];
    return a.temperature[b];
  };
  float temp = settle();
  LogitRow row(a.logits + n * a.ld, a.V);
  uint4 v[SP_LOADS], w[SP_LOADS];
#pragma unroll
  for (int i = 0; i < SP_LOADS; ++i) v[i] = row.load(piece * SP_PIECE + i * 32 + lane);
  while (true) {
    const int n_now = n, piece_now = piece;
    const LogitRow row_now = row;
    const float temp_now = temp;
    const bool more = ++item < end;
    if (more) {
      if (++piece == a.pieces) {
        piece = 0;
        ++n;
        row = LogitRow(a.logits + n * a.ld, a.V);
      }
#pragma unroll
      for (int i = 0; i < SP_LOADS; ++i) w[i] = row.load(piece * SP_PIECE + i * 32 + lane);
      if (piece == 0) temp = settle();
    }
    const int g0 = piece_now * SP_PIECE + lane;
    if (piece_now == 0 || (piece_now + 1) * SP_PIECE >= row_now.count) {
#pragma unroll
      for (int i = 0; i < SP_LOADS; ++i)
        if (g0 + i * 32 < row_now.count) row_now.trim(v[i], g0 + i * 32);
    }
    const bool greedy = !(temp_now > 0.f);
    const float k = SP_LOG2E / (greedy ? 1.f : temp_now);
    __nv_bfloat162 top2 = *reinterpret_cast<const __nv_bfloat162*>(&v[0].x);
#pragma unroll
    for (int i = 0; i < SP_LOADS; ++i) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v[i]);
      top2 = __hmax2(top2, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    }
    float top = fmaxf(__low2float(top2), __high2float(top2));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top;  // a piece without a finite logit sums to zero
    const uint64_t minus = pair2(-base, -base), scale = pair2(k, k);
    uint64_t s2[2] = {0ull, 0ull};
#pragma unroll
    for (int i = 0; i < SP_LOADS; ++i) {
      const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float p0, p1;
        unpair2(mul2(add2(pair2(__uint_as_float(x[e] << 16), __uint_as_float(x[e] & 0xffff0000u)), minus), scale), p0, p1);
        s2[e & 1] = add2(s2[e & 1], pair2(ex2_approx(p0), ex2_approx(p1)));
      }
    }
    float s0, s1;
    unpair2(add2(s2[0], s2[1]), s0, s1);
    float sum = s0 + s1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const long long at = static_cast<long long>(n_now) * a.pieces + piece_now;
    if (greedy) {
      int first = 0x7fffffff;
#pragma unroll
      for (int i = SP_LOADS - 1; i >= 0; --i)
#pragma unroll
        for (int e = 7; e >= 0; --e)
          if (sp_logit(v[i], e) == top) first = (g0 + i * 32) * 8 - row_now.skip + e;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      if (lane == 0) a.first[at] = first;
    }
    if (lane == 0) a.part[at] = make_float2(top, sum);
    if (!more) break;
#pragma unroll
    for (int i = 0; i < SP_LOADS; ++i) v[i] = w[i];
  }
}

struct WalkSmem {
  double total[SP_MAX_NODES];          // sum of exp((z - top) / temperature) over a node's row
  double p[SP_MAX_NODES];              // probability of a node's token in its parent's row
  double q[SP_MAX_NODES];              // draft probability of the same
  float2 rz[SP_MAX_NODES];             // reciprocals of the residuals' sums so far (draft probabilities given), as two fp32 numbers
  double warp_sum[SP_THREADS / 32];
  double cta_sum[2][SP_CLUSTER];       // partial sums of the cluster's CTAs, two passes in turn
  double rest;                         // mass that rejected point-mass drafts have left of the current node's row
  float top[SP_MAX_NODES];             // largest z of a node's row
  float u[SP_MAX_NODES];
  int best[SP_MAX_NODES];
  int parent[SP_MAX_NODES];
  int token[SP_MAX_NODES];             // -1: not in the vocabulary
  int gone[SP_MAX_NODES];              // rejected tokens of the current node (point-mass drafts)
  int ngone, nz, cur, k, next, step, pending;
  int settled;                         // rest is what the row's weights add up to, not what a subtraction left
  int accepted[SP_MAX_NODES];          // positions of the accepted nodes
};

// What is left of a token's probability after nz residuals, and one more if `less`.
__device__ __forceinline__ Two sp_residual(Two p, float q, const float2* rz, int nz, bool less) {
  for (int j = 0; j < nz; ++j) {
    p = two_minus(p, q);
    p = p.hi > 0.f ? two_mul(p, Two{rz[j].x, rz[j].y}) : Two{0.f, 0.f};
  }
  if (less) {
    p = two_minus(p, q);
    if (!(p.hi > 0.f)) p = Two{0.f, 0.f};
  }
  return p;
}

// What is left of the tokens of one row at some point of a walk: weights (point-mass drafts) or probabilities.
template <bool DRAFT>
struct LeftRow {
  LogitRow row;
  const float* q;
  const float2* rz;
  const int* gone;
  float temp, top;
  Two inv;
  int nz, ngone;
  bool q4;  // granules of q are 16-byte aligned
  __device__ __forceinline__ LeftRow(const VerifyArgs& a, int n, float temperature, float top_, Two inv_, const float2* rz_, int nz_, const int* gone_,
                                     int ngone_)
      : row(a.logits + n * a.ld, a.V), q(DRAFT ? a.draft + n * a.draft_ld : nullptr), rz(rz_), gone(gone_), temp(temperature), top(top_), inv(inv_),
        nz(nz_), ngone(ngone_) {
    q4 = DRAFT && ((reinterpret_cast<uintptr_t>(q) - 4 * row.skip) & 15) == 0;
  }
  // tokens of granule g that are outside of the row or rejected, as bits
  __device__ __forceinline__ uint32_t dropped(int g) const {
    const int e0 = g * 8 - row.skip;
    uint32_t drop = 0;
    if (g == 0 || g >= row.count - 1) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e0 + k < 0 || e0 + k >= row.V) drop |= 1u << k;
    }
    if (!DRAFT)
      for (int j = 0; j < ngone; ++j) {
        const int d = gone[j] - e0;
        if (d >= 0 && d < 8) drop |= 1u << d;
      }
    return drop;
  }
  __device__ __forceinline__ void draft(int g, uint32_t drop, float (&qs)[8]) const {
    const int e0 = g * 8 - row.skip;
    if (q4 && !drop) {
      const float4 lo = __ldg(reinterpret_cast<const float4*>(q + e0)), hi = __ldg(reinterpret_cast<const float4*>(q + e0) + 1);
      qs[0] = lo.x, qs[1] = lo.y, qs[2] = lo.z, qs[3] = lo.w, qs[4] = hi.x, qs[5] = hi.y, qs[6] = hi.z, qs[7] = hi.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) qs[k] = (drop >> k & 1u) ? 0.f : __ldg(q + e0 + k);
    }
  }
  __device__ __forceinline__ void weights(const uint4& v, uint32_t drop, float (&w)[8]) const {
    if (temp == 1.f) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = expf(__fsub_rn(sp_logit(v, k), top));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = expf(__fdiv_rn(__fsub_rn(sp_logit(v, k), top), temp));
    }
    if (drop) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (drop >> k & 1u) w[k] = 0.f;
    }
  }
  // what is left of the eight tokens of granule g
  __device__ __forceinline__ void left(const uint4& v, int g, bool less, Two (&r)[8]) const {
    const uint32_t drop = dropped(g);
    float qs[8], w[8];
    if (DRAFT) draft(g, drop, qs);
    weights(v, drop, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = DRAFT ? two_mul(inv, Two{w[k], 0.f}) : Two{w[k], 0.f};
    if (!DRAFT) return;
    for (int j = 0; j <= nz; ++j) {  // the residuals so far, then one more if `less`: one body for all of them
      if (j == nz && !less) break;
      const Two z = j < nz ? Two{rz[j].x, rz[j].y} : Two{1.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const Two d = two_minus(r[k], qs[k]);
        r[k] = d.hi > 0.f ? two_mul(d, z) : Two{0.f, 0.f};
      }
    }
  }
  // the granule's share of a running sum
  __device__ __forceinline__ void add(const uint4& v, int g, bool less, TwoPair& sum) const {
    if (DRAFT) {
      Two r[8];
      left(v, g, less, r);
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        sum.lo = add2(sum.lo, pair2(r[k].lo, r[k + 1].lo));
        sum.add(pair2(r[k].hi, r[k + 1].hi));
      }
    } else {
      float w[8];
      weights(v, dropped(g), w);
#pragma unroll
      for (int k = 0; k < 8; k += 2) sum.add(pair2(w[k], w[k + 1]));
    }
  }
};

// One CTA for a sequence, with draft probabilities a cluster of eight whose CTAs all take the same walk.  Latency: 256 trees of 16
// nodes 10 us, 64 drafted chains of up to 6 nodes over 128256 tokens 13 us (each rejection sums a residual row).
template <bool DRAFT>
__device__ __forceinline__ void verify_walk(const VerifyArgs& a, WalkSmem& sm) {
  namespace cg = cooperative_groups;
  griddep_launch_dependents();
  griddep_wait();
  const int b = DRAFT ? blockIdx.x / SP_CLUSTER : blockIdx.x, rank = DRAFT ? blockIdx.x % SP_CLUSTER : 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  int n0, T;
  sp_span(a, b, n0, T);
  const float t_in = a.temperature[b];
  const bool greedy = !(t_in > 0.f);
  const float temp = greedy ? 1.f : t_in, k2 = SP_LOG2E / temp;
  const long long o0 = static_cast<long long>(b) * a.max_nodes;
  if (T == 0) {
    if (rank == 0) {
      for (int i = tid; i < a.max_nodes; i += threads) {
        a.out_tokens[o0 + i] = -1;
        a.path[o0 + i] = -1;
        a.logprobs[o0 + i] = 0.f;
      }
      if (tid == 0) {
        a.count[b] = 0;
        a.end[b].node = -1;
      }
    }
    return;
  }
  if (DRAFT && !greedy) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA runs: its shared memory may be written to

  // ---- every node's row statistics and the probability of every node's token, whether the walk will need it or not
  if (tid < T) {
    const long long x = a.tokens[n0 + tid];
    sm.parent[tid] = a.parents[n0 + tid];
    sm.token[tid] = x >= 0 && x < a.V ? static_cast<int>(x) : -1;
    sm.u[tid] = a.u_accept[n0 + tid];
  }
  for (int j = warp; j < T; j += threads / 32) {
    const long long at = static_cast<long long>(n0 + j) * a.pieces;
    float m = -INFINITY, s = 0.f;  // this lane's pieces, relative to their maximum
    for (int c = lane; c < a.pieces; c += 32) {
      const float2 f = a.part[at + c];
      const float to = fmaxf(m, f.x);
      if (to > -INFINITY) s = s * ex2_approx((m - to) * k2) + f.y * ex2_approx((f.x - to) * k2);
      m = to;
    }
    float all = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    double d = s != 0.f ? static_cast<double>(s) * static_cast<double>(ex2_approx((m - all) * k2)) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    int first = 0x7fffffff;
    if (greedy) {
      for (int c = lane; c < a.pieces; c += 32)
        if (a.part[at + c].x == all) first = min(first, a.first[at + c]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    }
    if (lane == 0) {
      sm.top[j] = all;
      sm.total[j] = d;
      sm.best[j] = first >= 0 && first < a.V ? first : 0;
    }
  }
  __syncthreads();
  if (tid > 0 && tid < T) {
    const int up = sm.parent[tid], x = sm.token[tid];
    double p = 0.0, q = 0.0;
    if (up >= 0 && up < tid && x >= 0) {
      p = greedy ? (x == sm.best[up] ? 1.0 : 0.0)
                 : static_cast<double>(sp_weight(__bfloat162float(a.logits[(n0 + up) * a.ld + x]), temp, sm.top[up])) / sm.total[up];
      q = DRAFT ? static_cast<double>(a.draft[(n0 + up) * a.draft_ld + x]) : 1.0;
    }
    sm.p[tid] = p;
    sm.q[tid] = q;
  }
  if (tid == 0) sm.cur = sm.k = sm.ngone = sm.nz = sm.pending = sm.settled = 0, sm.next = 1, sm.rest = 1.0;
  __syncthreads();

  int pass = 0;
  // What is left at the current node.  Draft probabilities: the sum of max(r - q, 0) over the vocabulary, the same in every CTA of
  // the cluster.  Certain drafts: the sum of the weights of all tokens that were not rejected.
  auto residual_sum = [&] {
    constexpr int CTAS = DRAFT ? SP_CLUSTER : 1;
    const int node = sm.cur;
    const LeftRow<DRAFT> row(a, n0 + node, temp, sm.top[node], two_of(1.0 / sm.total[node]), sm.rz, DRAFT ? sm.nz : 0, sm.gone, DRAFT ? 0 : sm.ngone);
    TwoPair part = {0ull, 0ull};
    for (int g = rank * threads + tid; g < row.row.count; g += CTAS * threads) row.add(row.row.load(g), g, DRAFT, part);
    double mine = two_double(part.sum());
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sm.warp_sum[warp] = mine;
    __syncthreads();
    double all = 0.0;
    for (int w = 0; w < threads / 32; ++w) all += sm.warp_sum[w];
    if constexpr (!DRAFT) return all;
    cg::cluster_group cluster = cg::this_cluster();
    if (pass == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < SP_CLUSTER) cluster.map_shared_rank(&sm, tid)->cta_sum[pass & 1][rank] = all;
    cluster.sync();
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < SP_CLUSTER; ++c) sum += sm.cta_sum[pass & 1][c];
    ++pass;
    return sum;
  };

  // ---- the walk: one warp, until the nodes run out or something has to be summed
  while (true) {
    if (warp == 0) {
      int cur = sm.cur, k = sm.k, ngone = sm.ngone, next = sm.next, pending = sm.pending;
      double rest = sm.rest;
      bool settled = sm.settled, sum_first = false;
      while (next < T) {
        // the next child of the current node
        const bool lo = lane >= next && lane < T && sm.parent[lane] == cur;
        const bool hi = lane + 32 >= next && lane + 32 < T && sm.parent[lane + 32] == cur;
        const unsigned long long kids = __ballot_sync(0xffffffffu, lo) | static_cast<unsigned long long>(__ballot_sync(0xffffffffu, hi)) << 32;
        if (kids == 0ull) {
          next = T;
          break;
        }
        const int j = __ffsll(static_cast<long long>(kids)) - 1;
        if (pending) {  // draft probabilities, a sibling was rejected: its residual's sum first
          sum_first = true;
          next = j;
          break;
        }
        const int x = sm.token[j];
        double r = sm.p[j];
        if (DRAFT) {
          r = two_double(sp_residual(two_of(r), static_cast<float>(sm.q[j]), sm.rz, sm.nz, false));
        } else {
          for (int i = 0; i < ngone; ++i)
            if (sm.gone[i] == x) r = 0.0;
        }
        const double need = static_cast<double>(sm.u[j]) * (DRAFT ? sm.q[j] : rest);
        if (!DRAFT && !greedy && !settled && r > 0.0 && fabs(need - r) < SP_CLOSE * (r + (1.0 - rest))) {  // too close for these sums
          sum_first = true;
          next = j;
          break;
        }
        next = j + 1;
        __syncwarp();
        if (x >= 0 && need < r) {
          if (lane == 0) {
            sm.accepted[k] = j;
            sm.nz = 0;
          }
          ++k;
          cur = j;
          ngone = 0;
          rest = 1.0;
          settled = false;
        } else if (DRAFT) {
          pending = 1;
        } else if (x >= 0 && r > 0.0) {
          if (lane == 0) sm.gone[ngone] = x;
          ++ngone;
          rest -= r;
          settled = false;
        }
        __syncwarp();
      }
      if (lane == 0) {
        sm.cur = cur;
        sm.k = k;
        sm.ngone = ngone;
        sm.next = next;
        sm.pending = pending;
        sm.rest = rest;
        sm.settled = settled;
        sm.step = sum_first;
      }
    }
    __syncthreads();
    if (!sm.step) break;
    // at temperature 0 all mass is on one token and stays there, whatever is taken off
    const double sum = greedy ? 0.0 : residual_sum();
    __syncthreads();
    if (tid == 0) {
      if (!DRAFT) {
        sm.rest = sum / sm.total[sm.cur];
        sm.settled = 1;
      } else if (sum > 0.0) {  // else nothing is left: the residual stays what it was
        const Two r = two_of(1.0 / sum);
        sm.rz[sm.nz++] = make_float2(r.hi, r.lo);
      }
      sm.pending = 0;
    }
    __syncthreads();
  }
  if (DRAFT && !greedy && pass == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  if (rank != 0) return;
  const int node = sm.cur, k = sm.k;
  auto logprob = [&](int at, int x) {
    const float z = __bfloat162float(a.logits[(n0 + at) * a.ld + x]);
    return static_cast<float>(static_cast<double>(sp_exponent(z, temp, sm.top[at])) - sp_log(sm.total[at]));
  };
  for (int i = tid; i < a.max_nodes; i += threads) {
    const bool last = greedy && i == k;  // an accepted draft, or at temperature 0 the last token
    const int j = i < k ? sm.accepted[i] : 0, at = last ? node : sm.parent[j], x = last ? sm.best[node] : sm.token[j];
    a.out_tokens[o0 + i] = i < k || last ? x : -1;
    a.logprobs[o0 + i] = i < k || last ? logprob(at, x) : 0.f;
    a.path[o0 + i] = i == 0 ? n0 : i <= k ? n0 + sm.accepted[i - 1] : -1;
  }
  WalkEnd& e = a.end[b];
  if (tid == 0) {
    a.count[b] = k + 1;
    e.node = greedy ? -1 : n0 + node;
    e.k = k;
    e.nz = sm.nz;
    e.ngone = sm.ngone;
    e.less = sm.pending;
    e.top = sm.top[node];
    e.total = sm.total[node];
    const Two inv = two_of(1.0 / sm.total[node]);
    e.inv_total = make_float2(inv.hi, inv.lo);
  }
  if (tid < (DRAFT ? sm.nz : sm.ngone)) {
    if (DRAFT) e.rz[tid] = sm.rz[tid];
    else e.gone[tid] = sm.gone[tid];
  }
}

__global__ void __launch_bounds__(SP_THREADS / 2) verify_walk_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ WalkSmem sm;
  verify_walk<false>(a, sm);
}
__global__ void __cluster_dims__(SP_CLUSTER, 1, 1) __launch_bounds__(SP_THREADS) verify_walk_draft_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ WalkSmem sm;
  verify_walk<true>(a, sm);
}

// Bound by the instructions of the long sums: 39 million terms (256 rows of 152064) in 37 us; with draft probabilities, whose
// residuals take a dozen more instructions a term, 8 million in 19 us.
template <bool DRAFT>
__global__ void __launch_bounds__(SP_SUM_THREADS) verify_sums_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int PER = SP_CHUNK / SP_SUM_THREADS;
  __shared__ uint4 held[PER][SP_SUM_THREADS];
  __shared__ double ssum[SP_SUM_THREADS / 32];
  griddep_launch_dependents();
  griddep_wait();
  const int c = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
  const WalkEnd& e = a.end[b];
  if (e.node < 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const LeftRow<DRAFT> last(a, e.node, a.temperature[b], e.top, Two{e.inv_total.x, e.inv_total.y}, e.rz, e.nz, e.gone, e.ngone);
  // all loads first, the work on them in a loop (unrolled, it was ten times slower: it did not fit the instruction cache)
#pragma unroll
  for (int i = 0; i < PER; ++i) held[i][tid] = last.row.load(c * SP_CHUNK + i * SP_SUM_THREADS + tid);
  const bool less = e.less != 0;
  TwoPair part = {0ull, 0ull};
#pragma unroll 1
  for (int i = 0; i < PER; ++i) last.add(held[i][tid], c * SP_CHUNK + i * SP_SUM_THREADS + tid, less, part);
  double sum = two_double(part.sum());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) ssum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < SP_SUM_THREADS / 32; ++w) sum += ssum[w];
    a.sums[static_cast<long long>(b) * a.chunks + c] = sum;
  }
}

// One CTA per sequence, a thread has consecutive granules of a chunk: two, so that two CTAs fit on an SM and 256 sequences are
// one wave (16 -> 10 us), with draft probabilities one (two make the code too long for the instruction cache: 11 -> 20 us).
__host__ __device__ constexpr int sp_pick_threads(bool draft) { return draft ? SP_CHUNK : SP_CHUNK / 2; }
template <bool DRAFT>
__global__ void __launch_bounds__(sp_pick_threads(DRAFT), DRAFT ? 1 : 2) verify_pick_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int THREADS = sp_pick_threads(DRAFT), PER = SP_CHUNK / THREADS;
  __shared__ double ssum[THREADS / 32];
  __shared__ int pick, tail;
  griddep_launch_dependents();
  griddep_wait();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const WalkEnd& e = a.end[b];
  if (e.node < 0) return;
  const float temp = a.temperature[b];
  const double u = static_cast<double>(a.u_sample[b]);
  const double* sums = a.sums + static_cast<long long>(b) * a.chunks;
  LeftRow<DRAFT> last(a, e.node, temp, e.top, Two{e.inv_total.x, e.inv_total.y}, e.rz, e.nz, e.gone, e.ngone);
  bool less = e.less != 0;
  if (tid == 0) {
    pick = a.V;
    tail = -1;
  }
  // One chunk: the token in which the cumulative sum (`before` at the chunk's beginning) passes `target`, if it does, to
  // `pick`, the last token with weight to `tail`.  Returns the cumulative sum at the chunk's end.
  auto look = [&](int chunk, double before, double target) {
    const int g = chunk * SP_CHUNK + tid * PER;
    Two r[PER][8];
    Two part = {0.f, 0.f};
    int mine_last = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      last.left(last.row.load(g + i), g + i, less, r[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        two_add(part, r[i][k]);
        if (r[i][k].hi > 0.f) mine_last = (g + i) * 8 - last.row.skip + k;
      }
    }
    const double mine = two_double(part);
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    __syncthreads();
    if (lane == 31) ssum[warp] = incl;
    __syncthreads();
    double warps = lane < THREADS / 32 ? ssum[lane] : 0.0, upto = warps;  // the warps' sums, added up by every warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const double all = __shfl_sync(0xffffffffu, upto, 31);
    const double from = before + (__shfl_sync(0xffffffffu, upto - warps, warp) + (incl - mine));
    if (mine_last >= 0) atomicMax(&tail, mine_last);
    if (from <= target && from + mine > target) {
      int found = -1;
      const Two room = two_of(target - from);  // what the sum may grow by
      Two c = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (r[i][k].hi > 0.f && __fadd_rn(__fsub_rn(c.hi, room.hi), __fsub_rn(c.lo, room.lo)) <= 0.f) found = (g + i) * 8 - last.row.skip + k;
          two_add(c, r[i][k]);
          c = two_norm(c.hi, c.lo);
        }
      if (found >= 0) atomicMin(&pick, found);  // one thread, or two at a border that rounding moved
    }
    __syncthreads();
    return before + all;
  };
  double sum = 0.0;
  for (int c = lane; c < a.chunks; c += 32) sum += sums[c];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const double target = u * sum;
  // the chunk in which the sum passes the coin's share: every warp adds the chunks up, 32 at a time
  double before = 0.0;
  int chunk = -1;
  for (int c0 = 0; c0 < a.chunks && chunk < 0; c0 += 32) {
    const double x = c0 + lane < a.chunks ? sums[c0 + lane] : 0.0;
    double upto = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const unsigned over = __ballot_sync(0xffffffffu, before + upto > target);
    if (over) {
      const int at = __ffs(static_cast<int>(over)) - 1;
      chunk = c0 + at;
      before += __shfl_sync(0xffffffffu, upto - x, at);
    } else {
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  __syncthreads();
  // That chunk.  Rare, where it does not settle the matter (nothing is left: then what was there before the last rejection
  // counts, the residual or the rejected token itself; a coin of the last share): all chunks for their sum, then one after the other.
  const bool settled = sum > 0.0 && chunk >= 0;
  double total = 0.0;
  for (int round = settled ? 0 : 1; round < 3; ++round) {
    if (round == 1 && !(sum > 0.0)) {
      less = false;
      if (!DRAFT && last.ngone > 0) --last.ngone;
    }
    double upto = round == 0 ? before : 0.0;
    const double goal = round == 0 ? target : round == 1 ? INFINITY : u * total;
    for (int c = round == 0 ? chunk : 0; c < (round == 0 ? chunk + 1 : a.chunks); ++c) {
      upto = look(c, upto, goal);
      if (pick < a.V) break;
    }
    if (pick < a.V || (round == 0 && tail >= 0)) break;
    total = upto;
    __syncthreads();
  }
  if (tid == 0) {
    const int x = pick < a.V ? pick : max(tail, 0);
    const float z = __bfloat162float(a.logits[e.node * a.ld + x]);
    const long long o = static_cast<long long>(b) * a.max_nodes + e.k;
    a.out_tokens[o] = x;
    a.logprobs[o] = static_cast<float>(static_cast<double>(sp_exponent(z, temp, e.top)) - sp_log(e.total));
  }
}

// ------------------------------------------------------------------ commit of the accepted path
// path[b, j] >= 0 names the batch row whose K and V go to position ctx[b] + j of sequence b, in every layer.  The layers' qkv
// tensors are separate allocations: their addresses travel in the kernel's parameters.
constexpr int COMMIT_LAYERS = 128;
struct CommitLayers {
  const __nv_bfloat16* qkv[COMMIT_LAYERS];
};

// A CTA takes one token through COMMIT_STEP layers: the token's page is looked up once, and its rows of all these layers are
// in flight before the first is stored (one layer a CTA: 34 us for the 576 tokens of a batch in 32 layers, 75 MB each way; eight: 27 us).
constexpr int COMMIT_STEP = 8;

__global__ void __launch_bounds__(256)
kv_commit_kernel(const __grid_constant__ CommitLayers layers, int L, long long ld, int N, __nv_bfloat16* __restrict__ kc,
                 __nv_bfloat16* __restrict__ vc, long long layer_stride, int num_blocks, const int* __restrict__ table, long long table_ld,
                 int max_blocks, const int* __restrict__ ctx, const int* __restrict__ path, int P, int Hq, int Hkv) {
  griddep_launch_dependents();
  griddep_wait();
  const int bj = blockIdx.x, b = bj / P, j = bj % P, l0 = blockIdx.y * COMMIT_STEP;
  const int node = path[bj];
  const int pos = ctx[b] + j;
  if (node < 0 || node >= N || pos < 0 || pos / SP_PAGE >= max_blocks) return;
  const long long blk = table[b * table_ld + pos / SP_PAGE];
  if (blk < 0 || blk >= num_blocks) return;
  const long long from = node * ld + static_cast<long long>(Hq) * SP_DH;
  const long long base = l0 * layer_stride + (blk * Hkv * SP_PAGE + pos % SP_PAGE) * SP_DH;
  const int half = Hkv * (SP_DH / 8);
  for (int i = threadIdx.x; i < 2 * half; i += blockDim.x) {
    const int v = i < half ? i : i - half;
    __nv_bfloat16* dst = (i < half ? kc : vc) + base + static_cast<long long>(v / (SP_DH / 8)) * (SP_PAGE * SP_DH) + v % (SP_DH / 8) * 8;
    uint4 row[COMMIT_STEP];
#pragma unroll
    for (int l = 0; l < COMMIT_STEP; ++l)
      if (l0 + l < L) row[l] = __ldg(reinterpret_cast<const uint4*>(layers.qkv[l0 + l] + from) + i);
#pragma unroll
    for (int l = 0; l < COMMIT_STEP; ++l)
      if (l0 + l < L) *reinterpret_cast<uint4*>(dst + l * layer_stride) = row[l];
  }
}

}  // namespace b200

using namespace b200;

// pieces (statistics) and chunks (last draw) of a row that may begin anywhere in its first granule
static int sp_parts(int V, int granules) { return ((V + 14) / 8 + granules - 1) / granules; }

struct VerifyScratch {
  long long part, first, end, sums, total;  // offsets in bytes
  VerifyScratch(int B, int N, int V) {
    const long long pieces = static_cast<long long>(N) * sp_parts(V, SP_PIECE), chunks = static_cast<long long>(B) * sp_parts(V, SP_CHUNK);
    auto take = [&](long long bytes) {
      const long long at = total;
      total += (bytes + 15) / 16 * 16;
      return at;
    };
    total = 0;
    part = take(pieces * 8);
    first = take(pieces * 4);
    end = take(B * static_cast<long long>(sizeof(WalkEnd)));
    sums = take(chunks * 8);
  }
};

// bytes of workspace that b200_verify_tree needs
extern "C" long long b200_verify_tree_scratch(int B, int N, int V) {
  if (B < 0 || N < 0 || V < 1) return -1;
  return VerifyScratch(B, N, V).total;
}

extern "C" int b200_verify_tree(const void* logits, long long ld, int V, const float* draft, long long draft_ld, const long long* tokens,
                                const int* parents, const int* cu, int B, int N, int max_nodes, const float* temperature,
                                const float* u_accept, const float* u_sample, int* count, long long* out_tokens, int* path, float* logprobs,
                                void* scratch, void* stream) {
  if (B <= 0) return 0;
  if (V <= 0 || V > (1 << 30) || max_nodes < 1 || max_nodes > SP_MAX_NODES) return -1;
  VerifyArgs a;
  a.logits = reinterpret_cast<const __nv_bfloat16*>(logits);
  a.ld = ld;
  a.V = V;
  a.draft = draft;
  a.draft_ld = draft_ld;
  a.tokens = tokens;
  a.parents = parents;
  a.cu = cu;
  a.B = B;
  a.N = N;
  a.max_nodes = max_nodes;
  a.pieces = sp_parts(V, SP_PIECE);
  a.chunks = sp_parts(V, SP_CHUNK);
  a.temperature = temperature;
  a.u_accept = u_accept;
  a.u_sample = u_sample;
  a.count = count;
  a.out_tokens = out_tokens;
  a.path = path;
  a.logprobs = logprobs;
  const VerifyScratch at(B, N, V);
  unsigned char* ws = reinterpret_cast<unsigned char*>(scratch);
  a.part = reinterpret_cast<float2*>(ws + at.part);
  a.first = reinterpret_cast<int*>(ws + at.first);
  a.end = reinterpret_cast<WalkEnd*>(ws + at.end);
  a.sums = reinterpret_cast<double*>(ws + at.sums);
  if (static_cast<double>(B) * a.chunks >= 2147483648.0 || static_cast<double>(B) * SP_CLUSTER >= 2147483648.0) return -3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (N > 0) {
    // a warp for every piece until the GPU is full of them
    const long long items = static_cast<long long>(N) * a.pieces, warps = SP_STAT_THREADS / 32, most = 148 * SP_STAT_CTAS;
    const long long ctas = (items + warps - 1) / warps < most ? (items + warps - 1) / warps : most;
    e = launch_pdl(verify_stats_kernel, dim3(static_cast<unsigned>(ctas)), dim3(SP_STAT_THREADS), 0, st, a);
  }
  if (e == cudaSuccess)
    e = draft ? launch_pdl(verify_walk_draft_kernel, dim3(B * SP_CLUSTER), dim3(SP_THREADS), 0, st, a)
              : launch_pdl(verify_walk_kernel, dim3(B), dim3(SP_THREADS / 2), 0, st, a);
  const auto sums = draft ? verify_sums_kernel<true> : verify_sums_kernel<false>;
  const auto pick = draft ? verify_pick_kernel<true> : verify_pick_kernel<false>;
  if (e == cudaSuccess) e = launch_pdl(sums, dim3(static_cast<unsigned>(B) * a.chunks), dim3(SP_SUM_THREADS), 0, st, a);
  if (e == cudaSuccess) e = launch_pdl(pick, dim3(B), dim3(sp_pick_threads(draft != nullptr)), 0, st, a);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

// qkv: host array of L device pointers
extern "C" int b200_kv_commit(const void* const* qkv, int L, long long ld, int N, void* k_cache, void* v_cache, long long layer_stride,
                              int num_blocks, const int* table, long long table_ld, int max_blocks, const int* ctx, const int* path, int B,
                              int P, int Hq, int Hkv, int Dh, void* stream) {
  if (B <= 0 || P <= 0 || L <= 0 || N <= 0) return 0;
  if (Dh != SP_DH || Hkv <= 0) return -1;
  for (int l0 = 0; l0 < L; l0 += COMMIT_LAYERS) {
    CommitLayers layers;
    const int n = L - l0 < COMMIT_LAYERS ? L - l0 : COMMIT_LAYERS;
    for (int i = 0; i < COMMIT_LAYERS; ++i) layers.qkv[i] = reinterpret_cast<const __nv_bfloat16*>(qkv[l0 + (i < n ? i : 0)]);
    const cudaError_t e = launch_pdl(kv_commit_kernel, dim3(B * P, (n + COMMIT_STEP - 1) / COMMIT_STEP), dim3(256), 0,
                                     reinterpret_cast<cudaStream_t>(stream), layers, n, ld, N, reinterpret_cast<__nv_bfloat16*>(k_cache) + l0 * layer_stride,
                                     reinterpret_cast<__nv_bfloat16*>(v_cache) + l0 * layer_stride, layer_stride, num_blocks, table, table_ld,
                                     max_blocks, ctx, path, P, Hq, Hkv);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
}
