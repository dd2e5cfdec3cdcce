// Attention of drafted token trees over the paged KV cache (speculative decoding), GQA, head_dim 128.
//
// Sequence b owns the nodes cu[b] .. cu[b + 1] - 1 of the batch (rows of the fused qkv, RoPE applied).  Node n attends to the
// ctx[b] tokens of the sequence that are in the cache, to its ancestors in the tree and to itself:
//     o[n, h] = sum_j softmax_j(scale * q[n, h] . k[j]) v[j],   j in {0 .. ctx[b] - 1} and {n, parent(n), parent(parent(n)), ...}.
// Keys and values of the nodes come from their qkv rows, so nothing of a draft is in the cache before it is accepted.
// parents[n] is the parent's position inside the sequence (smaller than the node's own), -1 for a root, -2 for padding (a
// padding row gives zeros).
#include "common.cuh"

namespace b200 {

constexpr int TA_DH = 128;
constexpr int TA_PAGE = 64;
constexpr int TA_MAX_NODES = 64;

// Ancestors (the node itself included) of the node at position t as a bit set; 0 for padding.  Parents come before their
// children, anything else ends the walk, so it takes at most t steps whatever the table holds.
__device__ __forceinline__ unsigned long long tree_ancestors(const int* __restrict__ parents, int t) {
  int up = parents[t];
  if (up < -1) return 0ull;
  unsigned long long seen = 1ull << t;
  while (up >= 0 && up < t) {
    t = up;
    seen |= 1ull << t;
    up = parents[t];
  }
  return seen;
}

// One warp per (node, query head); a lane holds four of the 128 dimensions, every key costs one reduction over the warp.
__global__ void __launch_bounds__(128)
tree_attn_kernel(const __nv_bfloat16* __restrict__ qkv, long long ld, const __nv_bfloat16* __restrict__ kc, const __nv_bfloat16* __restrict__ vc,
                 const int* __restrict__ table, long long table_ld, int max_blocks, int num_blocks, const int* __restrict__ ctx,
                 const int* __restrict__ cu, const int* __restrict__ parents, int B, int N, int max_nodes, int Hq, int Hkv, float scale,
                 __nv_bfloat16* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int n0 = min(max(cu[b], 0), N), T = min(min(max(cu[b + 1] - n0, 0), max_nodes), N - n0);
  const int t = blockIdx.z;
  if (t >= T || h >= Hq) return;
  const int kvh = h / (Hq / Hkv);
  const int C = min(max(ctx[b], 0), max_blocks * TA_PAGE);
  const unsigned long long sees = tree_ancestors(parents + n0, t);
  auto load4 = [&](const __nv_bfloat16* p, float (&f)[4]) {
    const uint2 u = *reinterpret_cast<const uint2*>(p + lane * 4);
    f[0] = __uint_as_float(u.x << 16);
    f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16);
    f[3] = __uint_as_float(u.y & 0xffff0000u);
  };
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  load4(qkv + (n0 + t) * ld + static_cast<long long>(h) * TA_DH, q);
  auto key = [&](const __nv_bfloat16* kp, const __nv_bfloat16* vp, bool there) {
    float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (there) {
      load4(kp, k);
      load4(vp, v);
    }
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= scale;
    const float mn = fmaxf(m, s), a = __expf(m - mn), p = __expf(s - mn);
    m = mn;
    l = l * a + p;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] * a + p * v[e];
  };
  if (sees) {
    for (int j = 0; j < C; ++j) {
      const long long blk = table[b * table_ld + j / TA_PAGE];
      const long long at = ((blk * Hkv + kvh) * TA_PAGE + j % TA_PAGE) * TA_DH;
      key(kc + at, vc + at, blk >= 0 && blk < num_blocks);
    }
    for (int j = 0; j < T; ++j)
      if ((sees >> j) & 1ull) {
        const __nv_bfloat16* row = qkv + (n0 + j) * ld;
        key(row + static_cast<long long>(Hq + kvh) * TA_DH, row + static_cast<long long>(Hq + Hkv + kvh) * TA_DH, true);
      }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint2 r;
  r.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  r.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<uint2*>(out + (static_cast<long long>(n0 + t) * Hq + h) * TA_DH + lane * 4) = r;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_tree_attn(const void* qkv, long long ld, const void* k_cache, const void* v_cache, int num_blocks, const int* table,
                              long long table_ld, int max_blocks, const int* ctx, const int* cu, const int* parents, int B, int N,
                              int max_nodes, int Hq, int Hkv, int Dh, float scale, void* out, void* stream) {
  if (B <= 0 || N <= 0) return 0;
  if (Dh != TA_DH || Hkv <= 0 || Hq % Hkv || max_nodes < 1 || max_nodes > TA_MAX_NODES) return -1;
  tree_attn_kernel<<<dim3(B, (Hq + 3) / 4, max_nodes), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const __nv_bfloat16*>(qkv), ld, reinterpret_cast<const __nv_bfloat16*>(k_cache),
      reinterpret_cast<const __nv_bfloat16*>(v_cache), table, table_ld, max_blocks, num_blocks, ctx, cu, parents, B, N, max_nodes, Hq, Hkv,
      scale, reinterpret_cast<__nv_bfloat16*>(out));
  return static_cast<int>(cudaGetLastError());
}
