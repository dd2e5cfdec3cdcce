// Attention of drafted token trees over the paged KV cache (speculative decoding), GQA, head_dim 128, on tcgen05.
//
// Sequence b owns the nodes cu[b] .. cu[b + 1] - 1 of the batch (rows of the fused qkv, RoPE applied).  Node n attends to the
// ctx[b] tokens of the sequence that are in the cache, to its ancestors in the tree and to itself:
//     o[n, h] = sum_j softmax_j(scale * q[n, h] . k[j]) v[j],   j in {0 .. ctx[b] - 1} and {n, parent(n), parent(parent(n)), ...}.
// Keys and values of the nodes come from their qkv rows, so nothing of a draft is in the cache before it is accepted.
// parents[n] is the parent's position inside the sequence (smaller than the node's own), -1 for a root, -2 for padding (a
// padding row gives zeros).
//
// Work.  All nodes of a sequence and all G query heads of a KV head read the same keys, so they are the rows of one matrix
// product: a row tile holds floor(128 / G) nodes x G heads, a UNIT is up to two row tiles of one (sequence, KV head), its keys
// come in tiles of 128 (two cache pages), the tree's own keys are one last tile of 64.  Per tile of keys the cache delivers
// 64 KB; the tensor cores need about 1000 cycles for the two products of a row tile and HBM about 2700 cycles of one SM's share for
// the 64 KB, so up to 256 rows are bound by the cache's bytes.
//
// Split.  The key tiles of all units, laid end to end, are shared out evenly over the CTAs (one per SM), whatever the
// sequences' lengths; a unit that crosses a border is finished in parts (unnormalised output, maximum and sum in fp32), which
// a second kernel joins in the order of the keys.  The shares are computed from ctx and cu on the device, so one captured graph
// serves every step.
//
// One CTA: warp 0 streams pages with TMA through a ring of five 32 KB buffers, warp 1 issues S = Q K^T and O += P V, two groups
// of four warps own the softmax (warps 4 to 7 and 8 to 11).  A unit of two row tiles gives each group one of them (the keys are loaded once for both); a
// unit of one row tile gives the groups alternate key tiles, merged at the end, so that one group's exponentials always run
// beside the other group's products.  P replaces S in tensor memory (bf16), O stays there for the whole unit and is rescaled
// only when the row maximum has grown by more than 2^8.
#include "common.cuh"

namespace b200 {

constexpr int TA_DH = 128;
constexpr int TA_PAGE = 64;
constexpr int TA_MAX_NODES = 64;
constexpr int TA_THREADS = 384;          // four warps for TMA and products (two of them idle), two groups of four for the softmax
// Registers: 12 warps at launch have 168 a thread.  The softmax holds a row of 128 scores and spills at that; the first group
// gives back what the other two take (72 + 2 * 216 = 3 * 168, checked against the launch).
constexpr int TA_REGS = 168, TA_REGS_ISSUE = 72, TA_REGS_SOFTMAX = 216;
static_assert(TA_REGS_ISSUE + 2 * TA_REGS_SOFTMAX <= 3 * TA_REGS, "the groups' shares exceed what the block is launched with");
constexpr int TA_SUB = 128 * 64 * 2;     // bytes of one [128 x 64] swizzled sub-tile
constexpr int TA_TILE = 2 * TA_SUB;      // a [128 keys or rows x 128] bf16 tile
constexpr int TA_RING = 5;
constexpr int TA_MIN_TILES = 2;          // key tiles a CTA takes at least: below that joining the parts costs more than it saves
constexpr float TA_LOG2E = 1.4426950408889634f;

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

struct TreeArgs {
  const int* table;
  long long table_ld;
  int max_blocks, num_blocks;
  const int* ctx;
  const int* cu;
  const int* parents;
  int B, N, max_nodes, Hq, Hkv;
  int G, npt;           // query heads per KV head, nodes per row tile
  int part_rows;        // rows of a part in the workspace
  float scale;
  __nv_bfloat16* out;
  float* part_o;        // [CTA][2][part_rows][128]
  float2* part_ml;      // [CTA][2][part_rows]: (maximum in the base-2 scale, sum)
  int4* joins;          // [CTA]: a unit that begins in this CTA and goes on in the next ones
  int* status;
};

// The CTA's share of the key tiles, unit by unit.  Every role of the CTA walks the same sequence on its own.
struct TreeWalk {
  int b, n0, T, C, nt, nru, unit, t0, t1;
  long long left;

  __device__ __forceinline__ void load(const TreeArgs& a) {
    n0 = min(max(a.cu[b], 0), a.N);
    T = min(min(max(a.cu[b + 1] - n0, 0), a.max_nodes), a.N - n0);
    C = min(max(a.ctx[b], 0), a.max_blocks * TA_PAGE);
    nt = (C + 127) / 128 + 1;
    nru = (T + 2 * a.npt - 1) / (2 * a.npt);
  }
  __device__ __forceinline__ long long tiles(const TreeArgs& a) const { return static_cast<long long>(a.Hkv) * nru * nt; }
  __device__ __forceinline__ void begin(const TreeArgs& a, int seq, long long offset, long long count) {
    b = seq;
    left = count;
    load(a);
    unit = static_cast<int>(offset / nt);
    t0 = static_cast<int>(offset % nt);
    t1 = static_cast<int>(min(static_cast<long long>(nt), t0 + left));
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next(const TreeArgs& a) {
    left -= t1 - t0;
    t0 = 0;
    if (left <= 0) return;
    if (++unit == a.Hkv * nru) {
      unit = 0;
      do {
        ++b;
        load(a);
      } while (T == 0);
    }
    t1 = static_cast<int>(min(static_cast<long long>(nt), left));
  }
  __device__ __forceinline__ int kvh() const { return unit / nru; }
  __device__ __forceinline__ int first_node(const TreeArgs& a) const { return unit % nru * 2 * a.npt; }
  __device__ __forceinline__ int row_tiles(const TreeArgs& a) const { return T - first_node(a) > a.npt ? 2 : 1; }
};

// Order of a segment's loads in the ring: K0 K1 V0 K2 V1 ... V(n-1), the order in which they are used.
__device__ __forceinline__ int ring_k(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int ring_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }

struct TreeSmem {
  uint8_t q[2][TA_TILE];
  uint8_t ring[TA_RING][TA_TILE];
  float2 ml[2][128];
  uint64_t q_full[2], q_empty[2], r_full[TA_RING], r_empty[TA_RING], s_full[2], p_full[2], o_full[2], ml_full[2], epi_done;
  long long scan[TA_THREADS / 32];
  long long at_off;
  int at_seq;
  uint32_t tmem_ptr;
  int abort_flag;
};

__device__ __forceinline__ uint64_t ta_desc_k(uint32_t tile, int k) { return umma_desc_sw128(tile + (k >> 2) * TA_SUB + (k & 3) * 32, 16, 1024); }
__device__ __forceinline__ uint64_t ta_desc_mn(uint32_t tile, int k) { return umma_desc_sw128(tile + k * 2048, TA_SUB, 1024); }
__device__ __forceinline__ bool ta_warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// the matching store of tmem_ld32 for 16 columns
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__global__ void __launch_bounds__(TA_THREADS, 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_node, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TreeArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  TreeSmem& sm = *reinterpret_cast<TreeSmem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &sm.abort_flag;
  griddep_launch_dependents();
  griddep_wait();

  // ---- this CTA's share: total number of key tiles, then the sequence in which the share begins
  auto block_scan = [&](long long v, long long& total) {  // inclusive prefix over the block's threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    __syncthreads();
    if (lane == 31) sm.scan[warp] = v;
    __syncthreads();
    long long before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < TA_THREADS / 32; ++w) {
      if (w < warp) before += sm.scan[w];
      total += sm.scan[w];
    }
    return v + before;
  };
  auto tiles_of = [&](int b) {
    if (b >= a.B) return 0ll;
    TreeWalk s;
    s.b = b;
    s.load(a);
    return s.tiles(a);
  };
  long long total = 0, chunk, mine = 0, incl = 0;
  for (int b0 = 0; b0 < a.B; b0 += TA_THREADS) {
    mine = tiles_of(b0 + tid);
    incl = block_scan(mine, chunk);
    total += chunk;
  }
  const long long want = total / TA_MIN_TILES;
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), max(want, 1ll)));
  const int cta = blockIdx.x;
  const long long begin = total * cta / ctas, end = total * (cta + 1) / ctas;
  if (cta >= ctas || begin >= end || (smem_u32(smem_raw) & 1023u)) {
    if (tid == 0) {
      a.joins[cta] = make_int4(0, 0, 0, 0);
      if (smem_u32(smem_raw) & 1023u) atomicCAS(a.status, 0, ST_BAD_ARG);
    }
    return;
  }
  {
    long long base = 0;
    for (int b0 = 0; b0 < a.B; b0 += TA_THREADS) {
      if (a.B > TA_THREADS) {  // more than one chunk: the values of this one again
        mine = tiles_of(b0 + tid);
        incl = block_scan(mine, chunk);
      }
      const long long lo = base + incl - mine;
      if (mine > 0 && begin >= lo && begin < lo + mine) {
        sm.at_seq = b0 + tid;
        sm.at_off = begin - lo;
      }
      base += chunk;
    }
  }

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 1);
      mbar_init(&sm.q_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_full[i], 1);
      mbar_init(&sm.ml_full[i], 4);
    }
    for (int i = 0; i < TA_RING; ++i) {
      mbar_init(&sm.r_full[i], 1);
      mbar_init(&sm.r_empty[i], 1);
    }
    mbar_init(&sm.epi_done, 8);
    sm.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_ptr, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_ptr;  // S (then P) of group w at column 128 w, O of group w at 256 + 128 w

  TreeWalk w;
  w.begin(a, sm.at_seq, sm.at_off, end - begin);

  if (warp < 4) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TA_REGS_ISSUE));
   if (warp == 0) {
    if (elect_one()) {
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
      uint32_t rc = 0, qc = 0;  // loads issued into the ring, row tiles issued
      bool ok = true;
      auto ring_slot = [&](uint32_t bytes) -> int {
        const int s = rc % TA_RING;
        if (!mbar_wait(&sm.r_empty[s], ((rc / TA_RING) & 1) ^ 1, abort_flag)) {
          atomicCAS(a.status, 0, ST_TIMEOUT_EMPTY);
          return -1;
        }
        mbar_expect_tx(&sm.r_full[s], bytes);
        ++rc;
        return s;
      };
      for (; w.more() && ok; w.next(a)) {
        const int kvh = w.kvh(), first = w.first_node(a), nrt = w.row_tiles(a), nq = w.nt - 1;
        for (int rt = 0; rt < nrt && ok; ++rt, ++qc) {
          const int s = qc & 1;
          if (!mbar_wait(&sm.q_empty[s], ((qc >> 1) & 1) ^ 1, abort_flag)) {
            atomicCAS(a.status, 0, ST_TIMEOUT_EMPTY);
            ok = false;
            break;
          }
          mbar_expect_tx(&sm.q_full[s], a.G * a.npt * 256);
          tma_load_3d(sm.q[s], &tm_q, &sm.q_full[s], 0, kvh * a.G, w.n0 + first + rt * a.npt);
          tma_load_3d(sm.q[s] + TA_SUB, &tm_q, &sm.q_full[s], 64, kvh * a.G, w.n0 + first + rt * a.npt);
        }
        const int* row = a.table + w.b * a.table_ld;
        int yk0 = 0, yk1 = 0, yv0 = 0, yv1 = 0;  // page rows of the tile whose K / V is next
        auto pages = [&](int t, int& y0, int& y1) {
          y0 = y1 = -1;
          if (t < nq) {
            auto at = [&](int p) {
              const int blk = row[p];
              return (min(static_cast<unsigned>(blk), static_cast<unsigned>(a.num_blocks)) * a.Hkv + kvh) * TA_PAGE;  // outside: past the end, reads as zeros
            };
            y0 = at(2 * t);
            if ((2 * t + 1) * TA_PAGE < w.C) y1 = at(2 * t + 1);
          }
        };
        auto load_tile = [&](const CUtensorMap* cache, int head, int t, int y0, int y1) -> bool {
          const bool tree = t == nq;
          const int s = ring_slot(tree || y1 < 0 ? TA_TILE / 2 : TA_TILE);
          if (s < 0) return false;
          uint8_t* dst = sm.ring[s];
          if (tree) {
            tma_load_3d(dst, &tm_node, &sm.r_full[s], 0, head, w.n0);
            tma_load_3d(dst + TA_SUB, &tm_node, &sm.r_full[s], 64, head, w.n0);
            return true;
          }
          tma_load_2d(dst, cache, &sm.r_full[s], 0, y0);
          tma_load_2d(dst + TA_SUB, cache, &sm.r_full[s], 64, y0);
          if (y1 >= 0) {
            tma_load_2d(dst + TA_SUB / 2, cache, &sm.r_full[s], 0, y1);
            tma_load_2d(dst + TA_SUB + TA_SUB / 2, cache, &sm.r_full[s], 64, y1);
          }
          return true;
        };
        if (ok) {
          pages(w.t0, yk0, yk1);
          ok = load_tile(&tm_k, a.Hq + kvh, w.t0, yk0, yk1);
        }
        for (int t = w.t0; t < w.t1 && ok; ++t) {
          yv0 = yk0;
          yv1 = yk1;
          if (t + 1 < w.t1) {
            pages(t + 1, yk0, yk1);
            ok = load_tile(&tm_k, a.Hq + kvh, t + 1, yk0, yk1);
          }
          if (ok) ok = load_tile(&tm_v, a.Hq + a.Hkv + kvh, t, yv0, yv1);
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128, false, false), idesc_s64 = umma_idesc_bf16(128, 64, false, false);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, 128, false, true);
      struct Job {
        int grp, vslot;
        uint32_t vpar;
        bool tree, wait_v, free_v, first, last, new_seg;
      };
      uint32_t jc = 0, rbase = 0, qc = 0, pc = 0, seg = 0;  // pc: bit g is the parity of group g's next P
      bool ok = true;
      auto give_up = [&](int code) {
        atomicCAS(a.status, 0, code);
        return false;
      };
      auto issue_pv = [&](const Job& j, uint32_t seg_of) -> bool {
        if (!mbar_wait(&sm.p_full[j.grp], (pc >> j.grp) & 1, abort_flag)) return give_up(ST_TIMEOUT_TMEM_EMPTY);
        pc ^= 1u << j.grp;
        if (j.wait_v && !mbar_wait(&sm.r_full[j.vslot], j.vpar, abort_flag)) return give_up(ST_TIMEOUT_FULL);
        // the first product of a unit overwrites O: both groups must have read the last unit's
        if (j.new_seg && seg_of > 0 && !mbar_wait(&sm.epi_done, (seg_of - 1) & 1, abort_flag)) return give_up(ST_TIMEOUT_TMEM_EMPTY);
        tc_fence_after();
        const uint32_t v = smem_u32(sm.ring[j.vslot]), p = tmem + j.grp * 128, o = tmem + 256 + j.grp * 128;
        const int steps = j.tree ? 4 : 8;
        for (int k = 0; k < steps; ++k) umma_ts(o, p + k * 8, ta_desc_mn(v, k), idesc_o, !(j.first && k == 0));
        if (j.free_v) umma_commit(&sm.r_empty[j.vslot]);
        if (j.last) umma_commit(&sm.o_full[j.grp]);
        return true;
      };
      Job prev;
      bool have = false;
      uint32_t prev_seg = 0;
      for (; w.more() && ok; w.next(a), ++seg) {
        const int n = w.t1 - w.t0, nrt = w.row_tiles(a), jobs = n * nrt;
        for (int x = 0; x < jobs && ok; ++x, ++jc) {
          const int i = nrt == 2 ? x >> 1 : x, rt = nrt == 2 ? x & 1 : 0;
          const bool tree = w.t0 + i == w.nt - 1;
          Job j;
          j.grp = jc & 1;
          const uint32_t kn = rbase + ring_k(i), vn = rbase + ring_v(i, n);
          const int ks = kn % TA_RING, qs = (qc + rt) & 1;
          j.vslot = vn % TA_RING;
          j.vpar = (vn / TA_RING) & 1;
          j.tree = tree;
          j.wait_v = rt == 0;
          j.free_v = rt == nrt - 1;
          j.first = x < 2;
          j.last = x >= jobs - 2;
          j.new_seg = x == 0;
          if (i == 0 && !mbar_wait(&sm.q_full[qs], ((qc + rt) >> 1) & 1, abort_flag)) {
            ok = give_up(ST_TIMEOUT_FULL);
            break;
          }
          if (rt == 0 && !mbar_wait(&sm.r_full[ks], (kn / TA_RING) & 1, abort_flag)) {
            ok = give_up(ST_TIMEOUT_FULL);
            break;
          }
          tc_fence_after();
          const uint32_t q = smem_u32(sm.q[qs]), kt = smem_u32(sm.ring[ks]);
#pragma unroll
          for (int k = 0; k < 8; ++k) umma_ss(tmem + j.grp * 128, ta_desc_k(q, k), ta_desc_k(kt, k), tree ? idesc_s64 : idesc_s, k != 0);
          if (rt == nrt - 1) umma_commit(&sm.r_empty[ks]);
          if (i == n - 1) umma_commit(&sm.q_empty[qs]);
          umma_commit(&sm.s_full[j.grp]);
          if (have) ok = issue_pv(prev, prev_seg);
          prev = j;
          prev_seg = seg;
          have = true;
        }
        rbase += 2 * n;
        qc += nrt;
      }
      if (ok && have) issue_pv(prev, prev_seg);
    }
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TA_REGS_SOFTMAX));
    const int grp = (warp - 4) >> 2, lg = warp & 3, r = lg * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(lg * 32) << 16;
    const uint32_t t_s = tmem + grp * 128 + lane_off, t_o = tmem + 256 + lane_off;
    const float c = a.scale * TA_LOG2E;
    uint32_t jc = 0, rbase = 0, sc = 0, oc0 = 0, oc1 = 0, mc_seg = 0, seg = 0;
    const int rn = r / a.G, rg = r - rn * a.G;  // node of the row tile and head of the group
    bool ok = true;
    for (; w.more() && ok; w.next(a), ++seg) {
      const int n = w.t1 - w.t0, nrt = w.row_tiles(a), kvh = w.kvh(), first = w.first_node(a), jobs = n * nrt;
      const int x0 = (grp ^ jc) & 1;           // my first job of this segment; then every second one
      const int rt = nrt == 2 ? x0 : 0;
      const int node = first + rt * a.npt + rn;
      const bool valid = rn < a.npt && node < w.T;
      const bool busy = __any_sync(0xffffffffu, valid);
      unsigned long long sees = 0;
      if (valid) sees = tree_ancestors(a.parents + w.n0, node);
      float m = -INFINITY, l = 0.f;
      for (int x = x0; x < jobs && ok; x += 2) {
        const int i = nrt == 2 ? x >> 1 : x, t = w.t0 + i;
        const bool tree = t == w.nt - 1;
        const int nkeys = tree ? w.T : min(128, w.C - t * 128);
        ok = ta_warp_wait(&sm.s_full[grp], sc & 1, abort_flag);
        ++sc;
        if (!ok) break;
        tc_fence_after();
        if (nkeys < (tree ? 64 : 128) && (nrt == 1 || rt == 0)) {
          // rows of V behind the last key hold whatever was there: 0 * NaN must not reach the output
          const uint32_t vn = rbase + ring_v(i, n);
          ok = ta_warp_wait(&sm.r_full[vn % TA_RING], (vn / TA_RING) & 1, abort_flag);
          if (!ok) break;
          if (r >= nkeys && r < (tree ? 64 : 128)) {
            uint4* row = reinterpret_cast<uint4*>(sm.ring[vn % TA_RING] + r * 128);
#pragma unroll
            for (int q = 0; q < 8; ++q) row[q] = row[q + TA_SUB / 16] = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async();
        }
        if (busy) {
          const int cols = tree ? 2 : 4;
          uint32_t sv[4][32];
#pragma unroll
          for (int cc = 0; cc < 4; ++cc)
            if (cc < cols) tmem_ld32(t_s + cc * 32, sv[cc]);
          tmem_ld_wait();
          if (tree) {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((sees >> (cc * 32 + e)) & 1ull)) sv[cc][e] = 0xff800000u;
#pragma unroll
            for (int cc = 2; cc < 4; ++cc)
#pragma unroll
              for (int e = 0; e < 32; ++e) sv[cc][e] = 0xff800000u;
          } else if (nkeys < 128) {
#pragma unroll
            for (int cc = 0; cc < 4; ++cc)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (cc * 32 + e >= nkeys) sv[cc][e] = 0xff800000u;
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int e = 0; e < 32; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(sv[cc][e]));
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          float alpha = 1.f;
          const bool grow = (mx - m) * c > 8.f;
          if (grow) {
            alpha = ex2_approx((m - mx) * c);
            m = mx;
            l *= alpha;
          }
          const float mc = m * c;
          float rs4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            if (cc < cols) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float p0 = ex2_approx(fmaf(__uint_as_float(sv[cc][e]), c, -mc));
                const float p1 = ex2_approx(fmaf(__uint_as_float(sv[cc][e + 1]), c, -mc));
                rs4[(e >> 1) & 3] += p0 + p1;
                pk[e >> 1] = pack_bf16x2(p0, p1);
              }
              tmem_st16(t_s + cc * 16, pk);
            }
          }
          l += (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]);
          // S of this job was issued after every earlier P V of this group, so O is at rest here
          if (x >= 2 && __any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
              uint32_t o[32];
              tmem_ld32(t_o + grp * 128 + cc * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st32(t_o + grp * 128 + cc * 32, o);
            }
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[grp]);
      }
      if (!ok) break;

      // ---- end of the segment: join the two groups (one row tile), write the result or a part of it
      const bool whole = w.t0 == 0 && w.t1 == w.nt;
      const long long part = (static_cast<long long>(cta) * 2 + (w.t0 == 0 ? 1 : 0)) * a.part_rows;
      const long long token = w.n0 + node;
      __nv_bfloat16* dst = a.out + (token * a.Hq + kvh * a.G + rg) * TA_DH;
      if (!sees) {
        m = -INFINITY;
        l = 0.f;
      }
      float a0 = 1.f, a1 = 0.f;
      int c0 = 0, c1 = 4;  // my columns, in steps of 32
      bool had0 = true, had1 = true;
      if (nrt == 2) {
        ok = ta_warp_wait(&sm.o_full[grp], (grp ? oc1 : oc0) & 1, abort_flag);
        ++oc0;
        ++oc1;
        if (!ok) break;
      } else {
        const int jobs0 = (jobs + 1 - (jc & 1)) / 2, jobs1 = jobs - jobs0;  // job 0 belongs to group jc & 1
        had0 = jobs0 > 0;
        had1 = jobs1 > 0;
        if (seg > 0) ok = ta_warp_wait(&sm.epi_done, (seg - 1) & 1, abort_flag);  // the other group has read the last pair
        if (!ok) break;
        sm.ml[grp][r] = make_float2(m * c, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.ml_full[grp]);
        ok = ta_warp_wait(&sm.ml_full[grp ^ 1], mc_seg & 1, abort_flag);
        ++mc_seg;
        if (!ok) break;
        const float2 other = sm.ml[grp ^ 1][r];
        const float2 m0 = grp == 0 ? make_float2(m * c, l) : other, m1 = grp == 0 ? other : make_float2(m * c, l);
        const float top = fmaxf(m0.x, m1.x);
        a0 = m0.y != 0.f ? ex2_approx(m0.x - top) : 0.f;
        a1 = m1.y != 0.f ? ex2_approx(m1.x - top) : 0.f;
        l = a0 * m0.y + a1 * m1.y;
        m = top;  // from here on in the base-2 scale
        c0 = grp * 2;
        c1 = c0 + 2;
        if (had0) {
          ok = ta_warp_wait(&sm.o_full[0], oc0 & 1, abort_flag);
          ++oc0;
        }
        if (ok && had1) {
          ok = ta_warp_wait(&sm.o_full[1], oc1 & 1, abort_flag);
          ++oc1;
        }
        if (!ok) break;
      }
      tc_fence_after();
      const float inv = l != 0.f ? 1.f / l : 0.f;  // an empty row gives zeros, a NaN stays one
      if (busy) {
        for (int cc = c0; cc < c1; ++cc) {
          uint32_t o[32], o1[32];
          if (nrt == 2) {
            tmem_ld32(t_o + grp * 128 + cc * 32, o);
            tmem_ld_wait();
          } else {
            if (had0) tmem_ld32(t_o + cc * 32, o);
            if (had1) tmem_ld32(t_o + 128 + cc * 32, o1);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x0v = a0 != 0.f ? a0 * __uint_as_float(o[e]) : 0.f, x1v = a1 != 0.f ? a1 * __uint_as_float(o1[e]) : 0.f;
              o[e] = __float_as_uint(x0v + x1v);
            }
          }
          if (!valid) continue;
          if (whole) {
#pragma unroll
            for (int g8 = 0; g8 < 4; ++g8) {
              uint4 v4;
              uint32_t* p4 = &v4.x;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float lo = __uint_as_float(o[g8 * 8 + 2 * e]) * inv, hi = __uint_as_float(o[g8 * 8 + 2 * e + 1]) * inv;
                p4[e] = sees ? pack_bf16x2(lo, hi) : 0u;
              }
              reinterpret_cast<uint4*>(dst + cc * 32)[g8] = v4;
            }
          } else {
            float4* to = reinterpret_cast<float4*>(a.part_o + (part + rt * 128 + r) * TA_DH + cc * 32);
#pragma unroll
            for (int g4 = 0; g4 < 8; ++g4)
              to[g4] = make_float4(__uint_as_float(o[4 * g4]), __uint_as_float(o[4 * g4 + 1]), __uint_as_float(o[4 * g4 + 2]),
                                   __uint_as_float(o[4 * g4 + 3]));
          }
        }
        if (!whole && valid && (nrt == 2 || grp == 0)) a.part_ml[part + rt * 128 + r] = make_float2(nrt == 2 ? m * c : m, l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.epi_done);
      jc += jobs;
      rbase += 2 * n;
      // a unit that begins here and goes on elsewhere: leave word for the kernel that joins the parts
      if (warp == 4 && lane == 0 && w.left == w.t1 - w.t0) {
        int4 join = make_int4(0, 0, 0, 0);
        if (w.t0 == 0 && !whole) {
          const long long last_tile = end - w.t1 + w.nt - 1;  // of the unit, in the order of all tiles
          int lastc = static_cast<int>(last_tile * ctas / total);
          while (total * (lastc + 1) / ctas <= last_tile) ++lastc;
          while (total * lastc / ctas > last_tile) --lastc;
          join = make_int4(lastc - cta + 1, w.n0 + first, min(2 * a.npt, w.T - first), kvh);
        }
        a.joins[cta] = join;
      }
    }
    if (!ok && lane == 0) atomicCAS(a.status, 0, ST_TIMEOUT_TMEM_FULL);
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // let copies in flight land before the shared memory goes
    if (tid == 0) a.joins[cta] = make_int4(0, 0, 0, 0);
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the units that cross a border between CTAs: block (x, y) rows 32 y .. of the unit that begins in CTA x.
// A warp takes a row, parts in the order of the keys.
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int cta = blockIdx.x;
  const int4 join = a.joins[cta];
  const int parts = join.x;
  if (parts == 0) return;
  const int lane = threadIdx.x & 31;
  for (int i = 0; i < 4; ++i) {
    const int row = blockIdx.y * 32 + i * 8 + (threadIdx.x >> 5), rt = row >> 7, r = row & 127;
    const int rn = r / a.G, node = rt * a.npt + rn;
    if (row >= a.part_rows || rn >= a.npt || node >= join.z) continue;
    auto at = [&](int p) { return (static_cast<long long>(cta + p) * 2 + (p == 0 ? 1 : 0)) * a.part_rows + row; };
    float top = -INFINITY;
    for (int p = lane; p < parts; p += 32) {
      const float2 ml = a.part_ml[at(p)];
      if (ml.y != 0.f) top = fmaxf(top, ml.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < parts; ++p) {
      const float2 ml = a.part_ml[at(p)];
      if (ml.y == 0.f) continue;
      const float w = ex2_approx(ml.x - top);
      const float4 v = reinterpret_cast<const float4*>(a.part_o + at(p) * TA_DH)[lane];
      l += w * ml.y;
      acc.x += w * v.x;
      acc.y += w * v.y;
      acc.z += w * v.z;
      acc.w += w * v.w;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;  // an empty row gives zeros, a NaN stays one
    uint2 res;
    res.x = pack_bf16x2(acc.x * inv, acc.y * inv);
    res.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    __nv_bfloat16* dst = a.out + ((static_cast<long long>(join.y) + node) * a.Hq + join.w * a.G + r % a.G) * TA_DH;
    reinterpret_cast<uint2*>(dst)[lane] = res;
  }
}

static int ta_sms() {
  static const int n = [] {
    int dev = 0, v = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    return v;
  }();
  return n;
}

static int ta_part_rows(int max_nodes, int G) {
  const int npt = 128 / G;
  return max_nodes <= npt ? max_nodes * G : 128 + (max_nodes <= 2 * npt ? (max_nodes - npt) * G : npt * G);
}

}  // namespace b200

using namespace b200;

// bytes of workspace that b200_tree_attn needs for trees of up to max_nodes nodes
extern "C" int b200_tree_attn_scratch(int max_nodes, int Hq, int Hkv) {
  if (Hkv <= 0 || Hq % Hkv || Hq / Hkv > 128 || Hq <= 0 || max_nodes < 1 || max_nodes > TA_MAX_NODES) return -1;
  return ta_sms() * (2 * ta_part_rows(max_nodes, Hq / Hkv) * (TA_DH * 4 + 8) + 16);
}

static int ta_map_3d(CUtensorMap* map, const void* qkv, long long ld, int heads, int N, int box_heads, int box_rows) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return -1;
  cuuint64_t dim[3] = {TA_DH, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(N)};
  cuuint64_t stride[2] = {TA_DH * 2, static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)}, step[3] = {1, 1, 1};
  return static_cast<int>(enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(qkv), dim, stride, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
}

extern "C" int b200_tree_attn(const void* qkv, long long ld, const void* k_cache, const void* v_cache, int num_blocks, const int* table,
                              long long table_ld, int max_blocks, const int* ctx, const int* cu, const int* parents, int B, int N,
                              int max_nodes, int Hq, int Hkv, int Dh, float scale, void* out, void* scratch, int* status, void* stream) {
  if (B <= 0 || N <= 0) return 0;
  const int need = b200_tree_attn_scratch(max_nodes, Hq, Hkv);
  if (Dh != TA_DH || need < 0 || num_blocks < 1 || max_blocks > (1 << 24)) return -1;
  if ((static_cast<long long>(num_blocks) + 1) * Hkv * TA_PAGE >= (1ll << 31)) return -3;  // rows of the cache are 32-bit TMA coordinates
  TreeArgs a;
  a.G = Hq / Hkv;
  a.npt = 128 / a.G;
  CUtensorMap tq, tn, tk, tv;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * Hkv * TA_PAGE;
  int r = ta_map_3d(&tq, qkv, ld, Hq + 2 * Hkv, N, a.G, a.npt);
  if (!r) r = ta_map_3d(&tn, qkv, ld, Hq + 2 * Hkv, N, 1, TA_MAX_NODES);
  if (!r) r = make_tmap_2d(&tk, k_cache, rows, TA_DH, TA_DH, TA_PAGE, 64, 2, true);
  if (!r) r = make_tmap_2d(&tv, v_cache, rows, TA_DH, TA_DH, TA_PAGE, 64, 2, true);
  if (r) return 10000 + r;
  const int sms = ta_sms();
  a.table = table;
  a.table_ld = table_ld;
  a.max_blocks = max_blocks;
  a.num_blocks = num_blocks;
  a.ctx = ctx;
  a.cu = cu;
  a.parents = parents;
  a.B = B;
  a.N = N;
  a.max_nodes = max_nodes;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.part_rows = ta_part_rows(max_nodes, a.G);
  a.scale = scale;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.joins = reinterpret_cast<int4*>(scratch);
  a.part_o = reinterpret_cast<float*>(a.joins + sms);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + static_cast<long long>(sms) * 2 * a.part_rows * TA_DH);
  a.status = status;
  const int smem = sizeof(TreeSmem);
  static std::atomic<unsigned long long> cfg{0};
  cudaError_t e = opt_in_shared_memory(tree_attn_kernel, smem, cfg);
  if (e != cudaSuccess) return static_cast<int>(e);
  static const int regs = [] {
    cudaFuncAttributes f = {};
    return cudaFuncGetAttributes(&f, tree_attn_kernel) == cudaSuccess ? f.numRegs : 0;
  }();
  if (regs != TA_REGS) return -4;  // the register split of the groups would wait for registers that the launch did not bring
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  e = launch_pdl(tree_attn_kernel, dim3(sms), dim3(TA_THREADS), smem, st, tq, tn, tk, tv, a);
  if (e != cudaSuccess) return static_cast<int>(e);
  e = launch_pdl(tree_join_kernel, dim3(sms, (a.part_rows + 31) / 32), dim3(256), 0, st, a);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
