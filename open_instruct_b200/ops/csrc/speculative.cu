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
// Weights exp(z - max) are evaluated in fp32, sums over the vocabulary and everything that decides an outcome is held in fp64:
// a vocabulary of 10^5 tokens has bins of 10^-5 and less, and fp32 partial sums would move their borders by that much.
#include "common.cuh"

namespace b200 {

constexpr int SP_PAGE = 64;
constexpr int SP_DH = 128;
constexpr int SP_MAX_NODES = 64;
constexpr int SP_THREADS = 512;

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T none, Op op, T* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < nw ? red[lane] : none;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One CTA per sequence: statistics of a row are taken when the walk arrives at it.
__global__ void __launch_bounds__(SP_THREADS)
verify_tree_kernel(const __nv_bfloat16* __restrict__ logits, long long ld, int V, const float* __restrict__ draft, long long draft_ld,
                   const long long* __restrict__ tokens, const int* __restrict__ parents, const int* __restrict__ cu, int N, int max_nodes,
                   const float* __restrict__ temperature, const float* __restrict__ u_accept, const float* __restrict__ u_sample,
                   int* __restrict__ count, long long* __restrict__ out_tokens, int* __restrict__ path, float* __restrict__ logprobs) {
  __shared__ double redd[32];
  __shared__ float redf[32];
  __shared__ int redi[32];
  __shared__ double zs[SP_MAX_NODES];      // normalisers of the residuals so far (draft probabilities given)
  __shared__ int gone[SP_MAX_NODES];       // rejected tokens (point-mass drafts)
  __shared__ double warp_sum[32];
  __shared__ int pick;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n0 = min(max(cu[b], 0), N), T = min(min(max(cu[b + 1] - n0, 0), max_nodes), N - n0);
  const long long o0 = static_cast<long long>(b) * max_nodes;
  for (int i = tid; i < max_nodes; i += blockDim.x) {
    out_tokens[o0 + i] = -1;
    path[o0 + i] = (i == 0 && T > 0) ? n0 : -1;
    logprobs[o0 + i] = 0.f;
  }
  if (tid == 0) count[b] = 0;
  if (T == 0) return;
  const float t_in = temperature[b];
  const bool greedy = !(t_in > 0.f);
  const float temp = greedy ? 1.f : t_in;
  int cur = 0, k = 0, nrej = 0, best = 0;
  float top = 0.f;
  double total = 0.0;
  const __nv_bfloat16* row = nullptr;
  const float* q = nullptr;
  auto fmax_ = [](float a, float c) { return fmaxf(a, c); };
  auto add_ = [](double a, double c) { return a + c; };
  auto min_ = [](int a, int c) { return min(a, c); };
  auto weight = [&](int i) { return expf(__fsub_rn(__fdiv_rn(__bfloat162float(row[i]), temp), top)); };
  auto prob = [&](int i) { return greedy ? (i == best ? 1.0 : 0.0) : static_cast<double>(weight(i)) / total; };
  auto residual = [&](int i) {
    double r = prob(i);
    if (draft) {
      for (int j = 0; j < nrej; ++j) r = fmax(r - static_cast<double>(q[i]), 0.0) / zs[j];
    } else {
      for (int j = 0; j < nrej; ++j)
        if (gone[j] == i) r = 0.0;
    }
    return r;
  };
  auto arrive = [&](int node) {
    cur = node;
    nrej = 0;
    row = logits + static_cast<long long>(n0 + node) * ld;
    q = draft ? draft + static_cast<long long>(n0 + node) * draft_ld : nullptr;
    float m = -INFINITY;
    for (int i = tid; i < V; i += blockDim.x) m = fmaxf(m, __bfloat162float(row[i]));
    m = block_reduce(m, -INFINITY, fmax_, redf);
    top = __fdiv_rn(m, temp);
    int at = V;
    double s = 0.0;
    for (int i = tid; i < V; i += blockDim.x) {
      s += static_cast<double>(weight(i));
      if (greedy && __bfloat162float(row[i]) == m) at = min(at, i);
    }
    total = block_reduce(s, 0.0, add_, redd);
    best = greedy ? block_reduce(at, V, min_, redi) : 0;
    if (best >= V) best = 0;
  };
  auto emit = [&](int tok) {
    if (tid == 0) {
      out_tokens[o0 + k] = tok;
      logprobs[o0 + k] =
          static_cast<float>(static_cast<double>(__fsub_rn(__fdiv_rn(__bfloat162float(row[tok]), temp), top)) - log(total));
    }
  };
  arrive(0);
  double rest = 1.0;  // mass that rejected point-mass drafts have left
  for (int j = 1; j < T; ++j) {
    if (parents[n0 + j] != cur) continue;
    const long long x = tokens[n0 + j];
    const bool known = x >= 0 && x < V;
    const int xi = known ? static_cast<int>(x) : 0;
    const double r = known ? residual(xi) : 0.0, u = static_cast<double>(u_accept[n0 + j]);
    const double left_side = draft ? u * (known ? static_cast<double>(q[xi]) : 0.0) : u * rest;
    if (left_side < r) {
      emit(xi);
      ++k;
      if (tid == 0) path[o0 + k] = n0 + j;
      arrive(j);
      rest = 1.0;
      continue;
    }
    __syncthreads();
    if (draft) {
      double s = 0.0;
      for (int i = tid; i < V; i += blockDim.x) s += fmax(residual(i) - static_cast<double>(q[i]), 0.0);
      s = block_reduce(s, 0.0, add_, redd);
      if (s > 0.0) {
        if (tid == 0) zs[nrej] = s;
        ++nrej;
      }
    } else if (known && r > 0.0) {
      if (tid == 0) gone[nrej] = xi;
      ++nrej;
      rest -= r;
    }
    __syncthreads();
  }
  // draw the last token from r: contiguous shares of the vocabulary, prefix sums over the threads
  const int per = (V + blockDim.x - 1) / blockDim.x, i0 = min(V, tid * per), i1 = min(V, i0 + per);
  double mine = 0.0;
  int last = -1;
  for (int i = i0; i < i1; ++i) {
    const double r = residual(i);
    mine += r;
    if (r > 0.0) last = i;
  }
  double incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  last = -block_reduce(-last, 1, min_, redi);
  if (tid == 0) pick = V;
  __syncthreads();
  double before = 0.0, all = 0.0;
  for (int w = 0; w < SP_THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  double c = before + incl - mine;
  const double target = static_cast<double>(u_sample[b]) * all;
  if (c + mine > target) {
    for (int i = i0; i < i1; ++i) {
      c += residual(i);
      if (c > target) {
        atomicMin(&pick, i);
        break;
      }
    }
  }
  __syncthreads();
  const int tok = pick < V ? pick : max(last, 0);
  emit(tok);
  if (tid == 0) count[b] = k + 1;
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

extern "C" int b200_verify_tree(const void* logits, long long ld, int V, const float* draft, long long draft_ld, const long long* tokens,
                                const int* parents, const int* cu, int B, int N, int max_nodes, const float* temperature,
                                const float* u_accept, const float* u_sample, int* count, long long* out_tokens, int* path, float* logprobs,
                                void* stream) {
  if (B <= 0) return 0;
  if (V <= 0 || max_nodes < 1 || max_nodes > SP_MAX_NODES) return -1;
  verify_tree_kernel<<<B, SP_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const __nv_bfloat16*>(logits), ld, V, draft, draft_ld, tokens, parents, cu, N, max_nodes, temperature, u_accept,
      u_sample, count, out_tokens, path, logprobs);
  return static_cast<int>(cudaGetLastError());
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
