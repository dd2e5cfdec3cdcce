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
// Two kernels.  verify_stats_kernel reads every node's logits once (that is the whole cost: 2 bytes for each logit) and leaves the
// maximum and the sum of exponentials of every 16384-column chunk of a row.  verify_walk_kernel has a cluster of eight CTAs for
// each sequence: all of them take the same walk (the probabilities of all nodes' tokens are gathered before it, so it runs out of
// shared memory), then each has an eighth of the vocabulary of the last node's row for the final draw.
//
// A sum that decides a token is held in fp64, its terms exp(z / temperature - max) in fp32: a vocabulary of 10^5 tokens has
// bins of 10^-5 and less, and fp32 partial sums would move their borders by a share of that.  The statistics' exponentials
// come from the special-function unit (2^-22 of themselves, like the log-probabilities that leave through fp32).
#include "common.cuh"

#include <cooperative_groups.h>

namespace b200 {

constexpr int SP_PAGE = 64;
constexpr int SP_DH = 128;
constexpr int SP_MAX_NODES = 64;
constexpr int SP_LOADS = 8;                               // 16-byte loads of a thread of the statistics kernel
constexpr int SP_STAT_THREADS = 256;
constexpr int SP_CHUNK = SP_LOADS * SP_STAT_THREADS;      // 16-byte granules of a chunk (16384 logits)
constexpr int SP_CLUSTER = 8;
constexpr int SP_THREADS = 512;
constexpr float SP_LOG2E = 1.4426950408889634f;

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
    uint4 v = __ldg(granules + g);
    if (g == 0 || g == count - 1) {
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = g * 8 - skip + k;
        if (e < 0 || e >= V) w[k / 2] = k & 1 ? (w[k / 2] & 0xffffu) | 0xff800000u : (w[k / 2] & 0xffff0000u) | 0xff80u;
      }
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
  }
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
  int B, N, max_nodes, chunks;
  const float* temperature;
  const float* u_accept;
  const float* u_sample;
  int* count;
  long long* out_tokens;
  int* path;
  float* logprobs;
  float4* part;  // [N][chunks]: maximum, sum of exponentials relative to it, its first column (temperature 0)
};

// One CTA per (sequence, node, chunk).
__global__ void __launch_bounds__(SP_STAT_THREADS, 4) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ float smax[SP_STAT_THREADS / 32], ssum[SP_STAT_THREADS / 32];
  __shared__ int sidx[SP_STAT_THREADS / 32];
  griddep_launch_dependents();
  griddep_wait();
  const int c = blockIdx.x % a.chunks, bj = blockIdx.x / a.chunks, j = bj % a.max_nodes, b = bj / a.max_nodes;
  const int n0 = min(max(a.cu[b], 0), a.N), T = min(min(max(a.cu[b + 1] - n0, 0), a.max_nodes), a.N - n0);
  const float temp = a.temperature[b];
  if (j >= T) return;
  const bool greedy = !(temp > 0.f);
  const float k = SP_LOG2E / (greedy ? 1.f : temp);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const LogitRow row(a.logits + (n0 + j) * a.ld, a.V);
  const int g0 = c * SP_CHUNK + tid;
  uint4 v[SP_LOADS];
#pragma unroll
  for (int i = 0; i < SP_LOADS; ++i) v[i] = row.load(g0 + i * SP_STAT_THREADS);
  __nv_bfloat162 top2 = *reinterpret_cast<const __nv_bfloat162*>(&v[0].x);
#pragma unroll
  for (int i = 0; i < SP_LOADS; ++i) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v[i]);
    top2 = __hmax2(top2, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  }
  float top = fmaxf(__low2float(top2), __high2float(top2));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.f : top;  // a warp without a finite logit sums to zero
  float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < SP_LOADS; ++i) {
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s4[e] += ex2_approx((__uint_as_float(w[e] << 16) - base) * k);
      s4[e] += ex2_approx((__uint_as_float(w[e] & 0xffff0000u) - base) * k);
    }
  }
  float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    smax[warp] = top;
    ssum[warp] = sum;
  }
  __syncthreads();
  float m = smax[0];
#pragma unroll
  for (int w = 1; w < SP_STAT_THREADS / 32; ++w) m = fmaxf(m, smax[w]);
  int first = 0x7fffffff;
  if (greedy) {
#pragma unroll
    for (int i = SP_LOADS - 1; i >= 0; --i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 7; e >= 0; --e) {
        const float z = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        if (z == m) first = (g0 + i * SP_STAT_THREADS) * 8 - row.skip + e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    if (lane == 0) sidx[warp] = first;
    __syncthreads();
    first = sidx[0];
#pragma unroll
    for (int w = 1; w < SP_STAT_THREADS / 32; ++w) first = min(first, sidx[w]);
  }
  if (tid == 0) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < SP_STAT_THREADS / 32; ++w)
      if (ssum[w] != 0.f) s += ssum[w] * ex2_approx((smax[w] - m) * k);
    a.part[static_cast<long long>(n0 + j) * a.chunks + c] = make_float4(m, s, __int_as_float(first), 0.f);
  }
}

struct WalkSmem {
  double total[SP_MAX_NODES];          // sum of exp(z / temperature - top) over a node's row
  double p[SP_MAX_NODES];              // probability of a node's token in its parent's row
  double q[SP_MAX_NODES];              // draft probability of the same
  double rz[SP_MAX_NODES];             // reciprocals of the residuals' sums so far (draft probabilities given)
  double warp_sum[SP_THREADS / 32];
  double cta_sum[2][SP_CLUSTER];       // partial sums of the cluster's CTAs, two passes in turn
  int cta_last[2][SP_CLUSTER];
  float top[SP_MAX_NODES];             // largest z / temperature of a node's row
  float u[SP_MAX_NODES];
  int best[SP_MAX_NODES];
  int parent[SP_MAX_NODES];
  int token[SP_MAX_NODES];             // -1: not in the vocabulary
  int gone[SP_MAX_NODES];              // rejected tokens of the current node (point-mass drafts)
  int warp_last[SP_THREADS / 32];
  int ngone, nz, cur, k, next, step, pending;
  int accepted[SP_MAX_NODES];          // positions of the accepted nodes
};

__global__ void __cluster_dims__(SP_CLUSTER, 1, 1) __launch_bounds__(SP_THREADS) verify_walk_kernel(const __grid_constant__ VerifyArgs a) {
  namespace cg = cooperative_groups;
  __shared__ WalkSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  griddep_launch_dependents();
  griddep_wait();
  const int b = blockIdx.x / SP_CLUSTER, rank = blockIdx.x % SP_CLUSTER;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n0 = min(max(a.cu[b], 0), a.N), T = min(min(max(a.cu[b + 1] - n0, 0), a.max_nodes), a.N - n0);
  const float t_in = a.temperature[b];
  const bool greedy = !(t_in > 0.f);
  const float temp = greedy ? 1.f : t_in, k2 = SP_LOG2E / temp;
  const long long o0 = static_cast<long long>(b) * a.max_nodes;
  if (T == 0) {
    if (rank == 0) {
      for (int i = tid; i < a.max_nodes; i += SP_THREADS) {
        a.out_tokens[o0 + i] = -1;
        a.path[o0 + i] = -1;
        a.logprobs[o0 + i] = 0.f;
      }
      if (tid == 0) a.count[b] = 0;
    }
    return;
  }

  if (!greedy) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA runs: its shared memory may be written to

  // ---- every node's row statistics and the probability of every node's token, whether the walk will need it or not
  if (tid < T) {
    const long long x = a.tokens[n0 + tid];
    sm.parent[tid] = a.parents[n0 + tid];
    sm.token[tid] = x >= 0 && x < a.V ? static_cast<int>(x) : -1;
    sm.u[tid] = a.u_accept[n0 + tid];
  }
  for (int j = warp; j < T; j += SP_THREADS / 32) {
    const float4* part = a.part + static_cast<long long>(n0 + j) * a.chunks;
    float m = -INFINITY;
    for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, part[c].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    double s = 0.0;
    int first = 0x7fffffff;
    for (int c = lane; c < a.chunks; c += 32) {
      const float4 f = part[c];
      if (f.y != 0.f) s += static_cast<double>(f.y) * static_cast<double>(ex2_approx((f.x - m) * k2));
      if (f.x == m) first = min(first, __float_as_int(f.z));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    }
    if (lane == 0) {
      sm.top[j] = __fdiv_rn(m, temp);
      sm.total[j] = s;
      sm.best[j] = first >= 0 && first < a.V ? first : 0;
    }
  }
  __syncthreads();
  auto weight = [&](float z, float top) { return expf(__fsub_rn(temp == 1.f ? z : __fdiv_rn(z, temp), top)); };
  if (tid > 0 && tid < T) {
    const int up = sm.parent[tid], x = sm.token[tid];
    double p = 0.0, q = 0.0;
    if (up >= 0 && up < tid && x >= 0) {
      p = greedy ? (x == sm.best[up] ? 1.0 : 0.0)
                 : static_cast<double>(weight(__bfloat162float(a.logits[(n0 + up) * a.ld + x]), sm.top[up])) / sm.total[up];
      q = a.draft ? static_cast<double>(a.draft[(n0 + up) * a.draft_ld + x]) : 1.0;
    }
    sm.p[tid] = p;
    sm.q[tid] = q;
  }
  if (tid == 0) sm.cur = sm.k = sm.ngone = sm.nz = sm.pending = 0, sm.next = 1;
  __syncthreads();

  // Sum over the vocabulary of what is left at the current node: with draft probabilities the residual after sm.nz
  // rejections, less q once more if `less`; without them the weights of the tokens that are not gone.  Returns the cluster's sum;
  // a thread's own share (consecutive tokens) in `mine`, the sum of everything before it in `before`, its last token with
  // weight and the cluster's last one.
  const double* rz = sm.rz;
  int pass = 0;
  auto left_of = [&](double w, double inv_total, float q, int nz, bool less) {
    double r = w * inv_total;
    for (int j = 0; j < nz; ++j) r = fmax(r - static_cast<double>(q), 0.0) * rz[j];
    return less ? fmax(r - static_cast<double>(q), 0.0) : r;
  };
  const int per = ((a.V + 14) / 8 + SP_CLUSTER * SP_THREADS - 1) / (SP_CLUSTER * SP_THREADS);  // granules of a thread
  const int g0 = (rank * SP_THREADS + tid) * per;
  auto visit = [&](bool less, auto&& f) {  // f(token, what is left of it) over this thread's tokens in their order, until it says so
    const int node = sm.cur, nz = sm.nz, ngone = sm.ngone;
    const LogitRow row(a.logits + (n0 + node) * a.ld, a.V);
    const float* q = a.draft ? a.draft + (n0 + node) * a.draft_ld : nullptr;
    const float top = sm.top[node];
    const double inv = 1.0 / sm.total[node];
    for (int g = g0; g < g0 + per && g < row.count; ++g) {
      const uint4 v = row.load(g);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      const int e0 = g * 8 - row.skip;
      uint32_t drop = 0;
      for (int j = 0; j < ngone; ++j) {
        const int d = sm.gone[j] - e0;
        if (d >= 0 && d < 8) drop |= 1u << d;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e0 + e < 0 || e0 + e >= a.V) continue;
        const float z = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        const double x = static_cast<double>(weight(z, top));
        const double r = q ? left_of(x, inv, __ldg(q + e0 + e), nz, less) : (drop >> e & 1u) ? 0.0 : x;
        if (!f(e0 + e, r)) return;
      }
    }
  };
  auto cluster_sum = [&](bool less, double& mine, double& before, int& last) {
    mine = 0.0;
    int my_last = -1;
    visit(less, [&](int e, double r) {
      mine += r;
      if (r > 0.0) my_last = e;
      return true;
    });
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) my_last = max(my_last, __shfl_xor_sync(0xffffffffu, my_last, o));
    __syncthreads();
    if (lane == 31) {
      sm.warp_sum[warp] = incl;
      sm.warp_last[warp] = my_last;
    }
    __syncthreads();
    double below = 0.0, all = 0.0;
    int cta_last = -1;
#pragma unroll
    for (int w = 0; w < SP_THREADS / 32; ++w) {
      if (w < warp) below += sm.warp_sum[w];
      all += sm.warp_sum[w];
      cta_last = max(cta_last, sm.warp_last[w]);
    }
    if (pass == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < SP_CLUSTER) {
      WalkSmem* other = cluster.map_shared_rank(&sm, tid);
      other->cta_sum[pass & 1][rank] = all;
      other->cta_last[pass & 1][rank] = cta_last;
    }
    cluster.sync();
    double lower = 0.0, sum = 0.0;
    last = -1;
#pragma unroll
    for (int c = 0; c < SP_CLUSTER; ++c) {
      if (c < rank) lower += sm.cta_sum[pass & 1][c];
      sum += sm.cta_sum[pass & 1][c];
      last = max(last, sm.cta_last[pass & 1][c]);
    }
    before = lower + below + (incl - mine);
    ++pass;
    return sum;
  };

  // ---- the walk: one warp, until the tokens run out or a residual has to be summed
  while (true) {
    if (warp == 0) {
      int cur = sm.cur, k = sm.k, ngone = sm.ngone, next = sm.next, pending = sm.pending;
      double rest = 1.0;  // mass that rejected point-mass drafts have left
      bool sum_first = false;
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
        if (a.draft) {
          for (int i = 0; i < sm.nz; ++i) r = fmax(r - sm.q[j], 0.0) * rz[i];
        } else {
          for (int i = 0; i < ngone; ++i)
            if (sm.gone[i] == x) r = 0.0;
        }
        const double need = static_cast<double>(sm.u[j]) * (a.draft ? sm.q[j] : rest);
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
        } else if (a.draft) {
          pending = 1;
        } else if (x >= 0 && r > 0.0) {
          if (lane == 0) sm.gone[ngone] = x;
          ++ngone;
          rest -= r;
        }
        __syncwarp();
      }
      if (lane == 0) {
        sm.cur = cur;
        sm.k = k;
        sm.ngone = ngone;
        sm.next = next;
        sm.pending = pending;
        sm.step = sum_first;
      }
    }
    __syncthreads();
    if (!sm.step) break;
    double mine, before;
    int last;
    const double sum = greedy ? (sm.nz == 0 ? 1.0 : 0.0) : cluster_sum(true, mine, before, last);
    __syncthreads();
    if (tid == 0) {
      if (!greedy && sum > 0.0) sm.rz[sm.nz++] = 1.0 / sum;
      sm.pending = 0;
    }
    __syncthreads();
  }

  const int node = sm.cur, k = sm.k;
  auto logprob = [&](int at, int x) {
    const float z = __bfloat162float(a.logits[(n0 + at) * a.ld + x]);
    return static_cast<float>(static_cast<double>(__fsub_rn(__fdiv_rn(z, temp), sm.top[at])) - log(sm.total[at]));
  };
  auto finish = [&](int x) {
    a.out_tokens[o0 + k] = x;
    a.logprobs[o0 + k] = logprob(node, x);
  };
  if (rank == 0) {
    for (int i = tid; i < a.max_nodes; i += SP_THREADS) {
      const int j = i < k ? sm.accepted[i] : 0;
      if (i != k) {
        a.out_tokens[o0 + i] = i < k ? sm.token[j] : -1;
        a.logprobs[o0 + i] = i < k ? logprob(sm.parent[j], sm.token[j]) : 0.f;
      }
      a.path[o0 + i] = i == 0 ? n0 : i <= k ? n0 + sm.accepted[i - 1] : -1;
    }
    if (tid == 0) a.count[b] = k + 1;
  }
  if (greedy) {  // all mass is on one token, and it stays there: its draft would have been accepted
    if (rank == 0 && tid == 0) finish(sm.best[node]);
    return;
  }
  // ---- the last token: the first whose cumulative sum exceeds the coin's share of what is left
  double mine, before;
  int last;
  bool less = sm.pending != 0;
  double sum = cluster_sum(less, mine, before, last);
  if (less && !(sum > 0.0)) {  // nothing is left: the residual before this rejection
    less = false;
    sum = cluster_sum(less, mine, before, last);
  }
  const double target = static_cast<double>(a.u_sample[b]) * sum;
  if (before <= target && before + mine > target) {
    double c = before;
    int pick = -1;
    visit(less, [&](int e, double r) {
      c += r;
      if (r > 0.0) pick = e;
      return !(c > target);
    });
    finish(pick);
  } else if (rank == 0 && tid == 0 && !(sum > target)) {
    finish(max(last, 0));  // a coin of the last share, or a row without weight
  }
}

// ------------------------------------------------------------------ commit of the accepted path
// path[b, j] >= 0 names the batch row whose K and V go to position ctx[b] + j of sequence b, in every layer.  The layers' qkv
// tensors are separate allocations: their addresses travel in the kernel's parameters.
constexpr int COMMIT_LAYERS = 128;
struct CommitLayers {
  const __nv_bfloat16* qkv[COMMIT_LAYERS];
};

__global__ void __launch_bounds__(256)
kv_commit_kernel(const __grid_constant__ CommitLayers layers, int L, long long ld, int N, __nv_bfloat16* __restrict__ kc,
                 __nv_bfloat16* __restrict__ vc, long long layer_stride, int num_blocks, const int* __restrict__ table, long long table_ld,
                 int max_blocks, const int* __restrict__ ctx, const int* __restrict__ path, int B, int P, int Hq, int Hkv) {
  const int bj = blockIdx.x, b = bj / P, j = bj % P, l = blockIdx.y;
  const int node = path[bj];
  if (node < 0 || node >= N) return;
  const int pos = ctx[b] + j;
  if (pos < 0 || pos / SP_PAGE >= max_blocks) return;
  const long long blk = table[b * table_ld + pos / SP_PAGE];
  if (blk < 0 || blk >= num_blocks) return;
  const __nv_bfloat16* src = layers.qkv[l] + node * ld + static_cast<long long>(Hq) * SP_DH;
  const long long base = l * layer_stride + (blk * Hkv * SP_PAGE + pos % SP_PAGE) * SP_DH;
  const int half = Hkv * (SP_DH / 8);
  for (int i = threadIdx.x; i < 2 * half; i += blockDim.x) {
    const int v = i < half ? i : i - half;
    __nv_bfloat16* dst = (i < half ? kc : vc) + base + static_cast<long long>(v / (SP_DH / 8)) * (SP_PAGE * SP_DH) + v % (SP_DH / 8) * 8;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src + static_cast<long long>(i) * 8);
  }
}

}  // namespace b200

using namespace b200;

// columns of the statistics' chunks, and how many a row has
static int sp_chunks(int V) { return ((V + 14) / 8 + SP_CHUNK - 1) / SP_CHUNK; }

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
  a.chunks = sp_chunks(V);
  a.temperature = temperature;
  a.u_accept = u_accept;
  a.u_sample = u_sample;
  a.count = count;
  a.out_tokens = out_tokens;
  a.path = path;
  a.logprobs = logprobs;
  a.part = reinterpret_cast<float4*>(scratch);
  const double ctas = static_cast<double>(B) * max_nodes * a.chunks;
  if (ctas >= 2147483648.0 || static_cast<double>(B) * SP_CLUSTER >= 2147483648.0) return -3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (N > 0) {
    const cudaError_t e = launch_pdl(verify_stats_kernel, dim3(static_cast<unsigned>(ctas)), dim3(SP_STAT_THREADS), 0, st, a);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  const cudaError_t e = launch_pdl(verify_walk_kernel, dim3(B * SP_CLUSTER), dim3(SP_THREADS), 0, st, a);
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
    kv_commit_kernel<<<dim3(B * P, n), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        layers, n, ld, N, reinterpret_cast<__nv_bfloat16*>(k_cache) + l0 * layer_stride,
        reinterpret_cast<__nv_bfloat16*>(v_cache) + l0 * layer_stride, layer_stride, num_blocks, table, table_ld, max_blocks, ctx, path, B, P,
        Hq, Hkv);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
}
