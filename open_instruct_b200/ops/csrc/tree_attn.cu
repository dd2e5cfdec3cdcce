// Attention of drafted token trees over the paged KV cache (speculative decoding), GQA, head_dim 128, on tcgen05.
//
// Sequence b owns the nodes cu[b] .. cu[b + 1] - 1 of the batch (rows of the fused qkv, RoPE applied).  Node n attends to the
// ctx[b] tokens of the sequence that are in the cache, to its ancestors in the tree and to itself:
//     o[n, h] = sum_j softmax_j(scale * q[n, h] . k[j]) v[j],   j in {0 .. ctx[b] - 1} and {n, parent(n), parent(parent(n)), ...}.
// Keys and values of the nodes come from their qkv rows, so nothing of a draft is in the cache before it is accepted.
// parents[n] is the parent's position inside the sequence (smaller than the node's own), -1 for a root, -2 for padding (a
// padding row gives zeros, and may hold anything: its scores are replaced, its row of V is cleared in shared memory, since a
// product takes every row of V and 0 * NaN is NaN).
//
// Work.  All nodes of a sequence and all G query heads of a KV head read the same keys, so they are the rows of one matrix
// product: a row tile holds floor(128 / G) nodes x G heads, a UNIT is up to two row tiles of one (sequence, KV head), its keys
// come in tiles of 128 (two cache pages), the tree's own keys are the last 64 (beside an odd last page, or a half tile of their
// own).  HBM gives one SM's share of the 64 KB of a key tile in about 2700 cycles.  A row tile's products take the tensor cores
// 1300 cycles a key tile and its exponentials the special-function units 1024; what the softmax warps really need for them,
// with loads, maxima and packing, is 2560.  So units of one row tile run at the cache's bytes, two row tiles at the softmax.
//
// Split.  The work of all units - key tiles times row tiles, laid end to end - is shared out evenly over the CTAs (one per SM),
// whatever the sequences' lengths; a unit that crosses a border is finished in parts (unnormalised output, maximum and sum in
// fp32), which a second kernel joins in the order of the keys.  The shares are computed from ctx and cu on the device, so one
// captured graph serves every step.
//
// One CTA: warp 0 streams pages with TMA through a ring of 32 KB buffers, warp 2 plans the segments ahead, warps 1 and 3 issue
// S = Q K^T and O += P V, two groups of four warps own the softmax (warps 4 to 7 and 8 to 11).
//
// Wide kernel (more than 32 rows a unit): 128 rows by 64 keys a step.  A unit of two row tiles gives each group one of them (the
// keys are loaded once for both); a unit of one row tile gives each group its half of every key tile, merged at the end.  Each
// group has its own product thread and two buffers for S, so the next scores are there when a step's softmax is through.  P
// replaces S in tensor memory (bf16), O stays there for the whole unit and is rescaled only when the row maximum has grown by
// more than 2^8.  Measured: 16 trees of 64 nodes, 8 heads a KV head, contexts of 8192 to 32768: 697 GFLOP in 815 to 910 us = 765
// to 855 TFLOP/s, 0.6 of what a plain GEMM gets from the same power (the GPU is at its 1000 W limit, the SM clock at 1.5 GHz): the
// softmax bounds it, two warps a scheduler that wait for tensor memory in 900 of 2560 cycles a step.  Steps of 128 keys with one
// product thread (4 % behind), a later start of the second group, and scores fetched a step ahead (12 % behind) made no gain.
// 32 trees of 1 to 27 nodes, 7 heads a KV head: 88 to 97 us, 102 with shares in key tiles alone.
//
// Narrow kernel (at most 32 rows a unit: single tokens and short drafts).  As rows of a 128-row tile they would leave three
// quarters of the tensor work and most of the softmax warps to padding - and the padding is paid for in power: at 8 rows a unit
// the GPU ran at its 1000 W limit with the clock down to 1.5 GHz.  So the products are turned round, S^T = K Q^T and O^T = V^T P^T,
// with the 128 keys (the 128 dimensions) as the tile's rows and 32 columns: a quarter of the tensor work, every thread of a
// group has one key and 32 rows, and the result's rows are written by all of its warps.  The groups take alternate key tiles and
// have two O each, so that a unit is written while the next one runs (298 -> 289 us at one head a group).  Measured: 32 sequences
// of 4 nodes at 16384 tokens, 8 KV heads: 326 us, 6.6 TB/s; 128 trees of 8 nodes, 32 KV heads, contexts of 256 to 1024: 297 to 302 us,
// 4.7 TB/s (6 key tiles a unit: a sixth of the tiles are the trees' own, and a unit's end costs about 4000 cycles).
#include "common.cuh"

namespace b200 {

constexpr int TA_DH = 128;
constexpr int TA_PAGE = 64;
constexpr int TA_MAX_NODES = 64;
constexpr int TA_THREADS = 384;          // four warps for TMA, products and planning, two groups of four for the softmax
// Registers: 12 warps at launch have 168 a thread.  The softmax wants more, the issuing warps less: the first group gives back what
// the other two take.  No kernel spills with these splits (a few spilled words in the softmax loop had cost 10 %).
constexpr int TA_REGS = 168;
template <bool narrow>
struct TaRegs {
  static constexpr int issue = narrow ? 56 : 72, softmax = narrow ? 224 : 216;
  static_assert(issue + 2 * softmax <= 3 * TA_REGS, "the groups' shares exceed what the block is launched with");
};
constexpr int TA_SUB = 128 * 64 * 2;     // bytes of one [128 x 64] swizzled sub-tile
constexpr int TA_TILE = 2 * TA_SUB;      // a [128 keys or rows x 128] bf16 tile
constexpr int TA_RING = 4;               // two tiles of keys and values in flight; the narrow kernel has room for a fifth (no difference measured)
constexpr int TA_QSUB = 32 * 64 * 2;     // a narrow unit's queries: two [32 x 64] swizzled sub-tiles
constexpr int TA_MIN_WORK = 2;           // products of a key and a row tile that a CTA takes at least: below that joining the parts costs more than it saves
constexpr float TA_LOG2E = 1.4426950408889634f;

struct TreeArgs {
  const int* table;
  long long table_ld;
  int max_blocks, num_blocks;
  const int* ctx;
  const int* cu;
  const int* parents;
  int B, N, max_nodes, Hq, Hkv;
  int G, npt;           // query heads per KV head, nodes per row tile (narrow kernel: of 32 rows)
  int part_rows;        // rows of a part in the workspace
  float scale;
  __nv_bfloat16* out;
  float* part_o;        // [CTA][2][part_rows][128]
  float2* part_ml;      // [CTA][2][part_rows]: (maximum in the base-2 scale, sum)
  int4* joins;          // [CTA]: a unit that begins in this CTA and goes on in the next ones
  int* status;
};

// A sequence as the kernel sees it.  Tiles of 128 cached keys, then one tile with the tree's own keys; an odd last page shares
// that tile with the tree (page in rows 0 .. 63, tree in rows 64 .. 127; without such a page the tree is in rows 0 .. 63).
struct TreeSeq {
  int n0, T, C, nt, rts;  // first row, nodes, cached keys, key tiles, row tiles
  __device__ __forceinline__ void load(const TreeArgs& a, int b) {
    n0 = min(max(a.cu[b], 0), a.N);
    T = min(min(max(a.cu[b + 1] - n0, 0), a.max_nodes), a.N - n0);
    C = min(max(a.ctx[b], 0), a.max_blocks * TA_PAGE);
    nt = (C + TA_PAGE - 1) / TA_PAGE / 2 + 1;
    rts = (T + a.npt - 1) / a.npt;
  }
  // Work in products of a key tile with a row tile: what a unit of the wide kernel costs goes with its row tiles.  Shares in key
  // tiles alone left the busiest SM of an uneven batch with 1.33 times the mean (1.20 now), 102 us against 91.
  __device__ __forceinline__ int work(const TreeArgs& a) const { return a.Hkv * rts * nt; }
  __device__ __forceinline__ int pairs() const { return (rts + 1) >> 1; }  // of row tiles: units of a KV head
};

// Even shares of `total` products: the first `more` CTAs take one more than the others.  Inside a unit of two row tiles a boundary
// is rounded down to a whole key tile.
struct TreeShares {
  int each, more;
  __device__ __forceinline__ TreeShares(int total, int ctas) : each(total / ctas), more(total % ctas) {}
  __device__ __forceinline__ int begin(int cta) const { return each * cta + min(cta, more); }
  __device__ __forceinline__ int owner(int at) const {
    const int low = more * (each + 1);
    return at < low ? at / (each + 1) : more + (at - low) / each;
  }
};

// The part of one unit that a CTA works on, as the planning warp hands it to the others.
struct TreeSegment {
  int n0, T, C, nt;      // first row of the sequence in the batch, its nodes, its cached keys, tiles of the unit
  int t0, t1;            // tiles of this segment (none: the CTA is done)
  int kvh, first, nrt;   // KV head, first node of the unit, row tiles
  int y0, y1;            // cache rows of the first tile's pages (-1: none)
  int b;
  unsigned long long sees[TA_MAX_NODES];
};

// Order of a segment's loads in the ring: K0 K1 V0 K2 V1 ... V(n-1), the order in which they are used.
__device__ __forceinline__ int ring_k(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int ring_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }

template <bool NARROW>
struct TreeSmem {
  static constexpr int RING = NARROW ? TA_RING + 1 : TA_RING;
  uint8_t q[2][NARROW ? 2 * TA_QSUB : TA_TILE];
  uint8_t p[NARROW ? 2 : 1][NARROW ? 128 * 32 * 2 : 1024];  // narrow units: the groups' P^T, [128 keys x 32 rows]
  uint8_t ring[RING][TA_TILE];
  float ml[256];         // maxima and sums on their way to the group that writes a unit's result
  float ls[2][4][32], lm[2][32];  // narrow units: the same, by group, warp and row
  float mx[2][4][32];    // narrow units: row maxima by group and warp
  float wt[8][2][32];    // narrow units: a warp's weights of the rows, on their way from one lane to all
  uint32_t flags[2];     // narrow units: a byte for each warp of a group
  TreeSegment seg[2];
  uint64_t q_full[2], q_empty[2], r_full[RING], r_empty[RING], s_full[2][2], p_full[2][2], o_full[2][2], o_free[2][2],
      seg_full[2], seg_empty[2], ml_full[2], lx_full[2], flag_full[2], mx_full[2];
  int scan[TA_THREADS / 32];
  TreeSeq at;            // the sequence in which the CTA's share begins
  int at_seq, at_off;
  uint32_t tmem_ptr;
  int abort_flag;
};
static_assert(sizeof(TreeSmem<false>) <= 232448 && sizeof(TreeSmem<true>) <= 232448, "shared memory of a CTA");

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
__device__ __forceinline__ float max3(float x, float y, float z) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
  return d;
}
__device__ __forceinline__ float warp_max(float x) {
  float d;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(x));
  return d;
}
// MN-major operand of 32 bf16 (64 bytes) a row, 64-byte swizzle: rows indexed by K, groups of 8 rows 512 bytes apart
__device__ __forceinline__ uint64_t ta_desc_p(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(8192 >> 4) << 16;
  d |= static_cast<uint64_t>(512 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(4) << 61;  // SWIZZLE_64B
  return d;
}
// the low n bits, n in 0 .. 64
__device__ __forceinline__ unsigned long long low_bits(int n) { return n >= 64 ? ~0ull : (1ull << n) - 1ull; }

template <bool narrow>
__global__ void __launch_bounds__(TA_THREADS, 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_node, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ TreeArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  typedef TreeSmem<narrow> Smem;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  constexpr int RING = Smem::RING;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &sm.abort_flag;
  if (tid == 32) {
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_node);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 1);
      mbar_init(&sm.q_empty[i], narrow ? 1 : 2);  // the threads that issue products: one, or one a group
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sm.s_full[i][j], 1);
        mbar_init(&sm.p_full[i][j], 4);
        mbar_init(&sm.o_full[i][j], 1);
        mbar_init(&sm.o_free[i][j], 8);
      }
      mbar_init(&sm.ml_full[i], 4);
      mbar_init(&sm.lx_full[i], 4);
      mbar_init(&sm.flag_full[i], 4);
      mbar_init(&sm.mx_full[i], 4);
      mbar_init(&sm.seg_full[i], 1);
      mbar_init(&sm.seg_empty[i], narrow ? 10 : 11);  // the TMA and the product threads, eight softmax warps
    }
    for (int i = 0; i < RING; ++i) {
      mbar_init(&sm.r_full[i], 1);
      mbar_init(&sm.r_empty[i], narrow ? 1 : 2);
    }
    sm.abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (narrow) {  // rows that no query fills: finite whatever the memory held
    for (int i = tid; i < static_cast<int>(sizeof(sm.q) / 16); i += TA_THREADS) reinterpret_cast<uint4*>(sm.q)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();
  }
  griddep_launch_dependents();
  griddep_wait();

  // ---- this CTA's share: the batch's work, then the sequence in which the share begins
  auto block_scan = [&](int v, int& total) {  // inclusive prefix over the block's threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    __syncthreads();
    if (lane == 31) sm.scan[warp] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < TA_THREADS / 32; ++w) {
      if (w < warp) before += sm.scan[w];
      total += sm.scan[w];
    }
    return v + before;
  };
  TreeSeq seq;
  auto work_of = [&](int b) {
    if (b >= a.B) return 0;
    seq.load(a, b);
    return seq.work(a);
  };
  int total = 0, chunk, mine = 0, incl = 0;
  for (int b0 = 0; b0 < a.B; b0 += TA_THREADS) {
    mine = work_of(b0 + tid);
    incl = block_scan(mine, chunk);
    total += chunk;
  }
  const int ctas = min(static_cast<int>(gridDim.x), max(total / TA_MIN_WORK, 1)), cta = blockIdx.x;
  const TreeShares share(total, ctas);
  const int begin = share.begin(cta), end = share.begin(cta + 1);
  if (cta >= ctas || begin >= end || (smem_u32(smem_raw) & 1023u)) {
    if (tid == 0) {
      a.joins[cta] = make_int4(0, 0, 0, 0);
      if (smem_u32(smem_raw) & 1023u) atomicCAS(a.status, 0, ST_BAD_ARG);
    }
    return;
  }
  for (int b0 = 0, base = 0; b0 < a.B; b0 += TA_THREADS, base += chunk) {
    if (a.B > TA_THREADS) {  // more than one chunk: the values of this one again
      mine = work_of(b0 + tid);
      incl = block_scan(mine, chunk);
    }
    const int lo = base + incl - mine;
    if (begin >= lo && begin < lo + mine) {
      sm.at = seq;
      sm.at_seq = b0 + tid;
      sm.at_off = begin - lo;
    }
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_ptr, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_ptr;  // S (then P) of group g at column 128 g, O of group g at 256 + 128 g

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TaRegs<narrow>::issue));
    if (warp == 2) {
      // ---- planning: the CTA's segments one or two ahead of the others, so that their loads wait for no index
      TreeSeq q = sm.at;
      const int head = q.rts * q.nt, in_head = sm.at_off % head;  // work of a KV head
      int b = sm.at_seq, left = end - begin, kvh = sm.at_off / head, pair = in_head / (2 * q.nt), p0 = in_head % (2 * q.nt), have = -1;
      unsigned long long s0 = 0, s1 = 0;  // what nodes `lane` and `lane + 32` see
      bool ok = true;
      if (lane == 0) a.joins[cta] = make_int4(0, 0, 0, 0);
      for (uint32_t n = 0; ok; ++n) {
        TreeSegment& g = sm.seg[n & 1];
        if (n >= 2) ok = ta_warp_wait(&sm.seg_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag);
        if (!ok) break;
        const int nrt = min(2, q.rts - 2 * pair), p1 = min(q.nt * nrt, p0 + left), t0 = p0 / nrt, t1 = p1 / nrt;
        if (t0 < t1) {  // none: the share is done, or its last product is half a tile, which the next CTA has
          const int first = pair * 2 * a.npt;
          int blk = -1;
          if (lane < 2 && (2 * t0 + lane) * TA_PAGE < q.C) blk = a.table[b * a.table_ld + 2 * t0 + lane];
          if (have != b) {
            have = b;
            int u0 = lane < q.T ? a.parents[q.n0 + lane] : -2, u1 = lane + 32 < q.T ? a.parents[q.n0 + lane + 32] : -2;
            // Ancestors as bit sets, the paths' lengths doubling in every round: what a node sees, and where that path goes on.
            // Parents come before their children; anything else ends a path, so six rounds cover 64 nodes.
            s0 = u0 < -1 ? 0ull : 1ull << lane;
            s1 = u1 < -1 ? 0ull : 1ull << (lane + 32);
            if (u0 >= lane) u0 = -1;
            if (u1 >= lane + 32) u1 = -1;
            while (__any_sync(0xffffffffu, u0 >= 0 || u1 >= 0)) {
              // node u < 64 lives in lane u & 31, in its second word from 32 on; u0 is always in the first
              const unsigned long long f0 = __shfl_sync(0xffffffffu, s0, u0 & 31), f1 = __shfl_sync(0xffffffffu, s0, u1 & 31),
                                       g1 = __shfl_sync(0xffffffffu, s1, u1 & 31);
              const int v0 = __shfl_sync(0xffffffffu, u0, u0 & 31), v1 = __shfl_sync(0xffffffffu, u0, u1 & 31),
                        w1 = __shfl_sync(0xffffffffu, u1, u1 & 31);
              if (u0 >= 0) {
                s0 |= f0;
                u0 = v0;
              }
              if (u1 >= 0) {
                s1 |= u1 < 32 ? f1 : g1;
                u1 = u1 < 32 ? v1 : w1;
              }
            }
          }
          g.sees[lane] = s0;
          g.sees[lane + 32] = s1;
          if (lane < 2)
            (lane ? g.y1 : g.y0) = (2 * t0 + lane) * TA_PAGE < q.C
                                       ? static_cast<int>((min(static_cast<unsigned>(blk), static_cast<unsigned>(a.num_blocks)) * a.Hkv + kvh) * TA_PAGE)
                                       : -1;
          if (lane == 0) {
            g.n0 = q.n0;
            g.T = q.T;
            g.C = q.C;
            g.nt = q.nt;
            g.kvh = kvh;
            g.first = first;
            g.nrt = nrt;
            g.b = b;
            if (t0 == 0 && t1 < q.nt) {  // a unit that begins here and goes on in the next CTAs is joined from its parts
              const int c = share.owner(end - p1 + q.nt * nrt - 1);  // who has the unit's last product
              a.joins[cta] = make_int4(c - cta + 1, q.n0 + first, min(2 * a.npt, q.T - first), kvh);
            }
          }
        }
        if (lane == 0) {
          g.t0 = t0;
          g.t1 = t1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.seg_full[n & 1]);
        if (t1 == t0) break;
        left -= p1 - p0;
        p0 = 0;
        if (left > 0 && ++pair == q.pairs()) {
          pair = 0;
          if (++kvh == a.Hkv) {
            kvh = 0;
            do q.load(a, ++b);
            while (q.T == 0);
          }
        }
      }
      if (!ok && lane == 0) atomicCAS(a.status, 0, ST_TIMEOUT_EMPTY);
    } else if (warp == 0) {
      if (elect_one()) {
        uint32_t rc = 0, qc = 0;  // loads issued into the ring, row tiles issued
        bool ok = true;
        auto ring_slot = [&](uint32_t bytes) -> int {
          const int s = rc % RING;
          if (!mbar_wait(&sm.r_empty[s], ((rc / RING) & 1) ^ 1, abort_flag)) return -1;
          mbar_expect_tx(&sm.r_full[s], bytes);
          ++rc;
          return s;
        };
        for (uint32_t n = 0; ok; ++n) {
          const TreeSegment& g = sm.seg[n & 1];
          ok = mbar_wait(&sm.seg_full[n & 1], (n >> 1) & 1, abort_flag);
          if (!ok || g.t0 == g.t1) break;
          const int t0 = g.t0, t1 = g.t1, tree = g.nt - 1, kvh = g.kvh, C = g.C, n0 = g.n0;
          const int nrt = g.nrt;
          int yk0 = g.y0, yk1 = g.y1;  // page rows of the next tile of K
          const int q0 = n0 + g.first;
          const int* row = a.table + g.b * a.table_ld;
          mbar_arrive(&sm.seg_empty[n & 1]);
          for (int rt = 0; rt < nrt && ok; ++rt, ++qc) {
            const int s = qc & 1;
            ok = mbar_wait(&sm.q_empty[s], ((qc >> 1) & 1) ^ 1, abort_flag);
            if (!ok) break;
            mbar_expect_tx(&sm.q_full[s], a.G * a.npt * 256);
            constexpr int right = narrow ? TA_QSUB : TA_SUB;  // where the dimensions from 64 on start
            tma_load_3d(sm.q[s], &tm_q, &sm.q_full[s], 0, kvh * a.G, q0 + rt * a.npt);
            tma_load_3d(sm.q[s] + right, &tm_q, &sm.q_full[s], 64, kvh * a.G, q0 + rt * a.npt);
          }
          auto page = [&](int p) {  // a page outside the cache: rows past its end, which read as zeros
            if (p * TA_PAGE >= C) return -1;
            return static_cast<int>((min(static_cast<unsigned>(row[p]), static_cast<unsigned>(a.num_blocks)) * a.Hkv + kvh) * TA_PAGE);
          };
          auto load_tile = [&](const CUtensorMap* cache, int head, int t, int y0, int y1) -> bool {
            const int s = ring_slot((y0 >= 0 ? TA_TILE / 2 : 0) + (t == tree ? a.max_nodes * TA_DH * 2 : y1 >= 0 ? TA_TILE / 2 : 0));
            if (s < 0) return false;
            uint8_t* dst = sm.ring[s];
            if (y0 >= 0) {
              tma_load_2d(dst, cache, &sm.r_full[s], 0, y0);
              tma_load_2d(dst + TA_SUB, cache, &sm.r_full[s], 64, y0);
            }
            uint8_t* second = y0 >= 0 ? dst + TA_SUB / 2 : dst;
            if (t == tree) {
              tma_load_3d(second, &tm_node, &sm.r_full[s], 0, head, n0);
              tma_load_3d(second + TA_SUB, &tm_node, &sm.r_full[s], 64, head, n0);
            } else if (y1 >= 0) {
              tma_load_2d(second, cache, &sm.r_full[s], 0, y1);
              tma_load_2d(second + TA_SUB, cache, &sm.r_full[s], 64, y1);
            }
            return true;
          };
          int yn0 = -1, yn1 = -1;      // of the tile after that
          if (t0 + 1 < t1) yn0 = page(2 * t0 + 2), yn1 = page(2 * t0 + 3);
          if (ok) ok = load_tile(&tm_k, a.Hq + kvh, t0, yk0, yk1);
          for (int t = t0; t < t1 && ok; ++t) {
            const int yv0 = yk0, yv1 = yk1;
            yk0 = yn0;
            yk1 = yn1;
            if (t + 1 < t1) {
              if (t + 2 < t1) yn0 = page(2 * t + 4), yn1 = page(2 * t + 5);
              ok = load_tile(&tm_k, a.Hq + kvh, t + 1, yk0, yk1);
            }
            if (ok) ok = load_tile(&tm_v, a.Hq + a.Hkv + kvh, t, yv0, yv1);
          }
        }
        if (!ok) atomicCAS(a.status, 0, ST_TIMEOUT_EMPTY);
      }
    } else if (warp == 1 || (!narrow && warp == 3)) {
      if (elect_one()) {
        auto give_up = [&](int code) {
          atomicCAS(a.status, 0, code);
          return false;
        };
        if constexpr (narrow) {
          // Jobs (key tiles) alternate between the groups; S of a job is issued before P V of the one before.
          constexpr uint32_t idesc_s = umma_idesc_bf16(128, 32, false, false), idesc_o = umma_idesc_bf16(128, 32, true, true);
          struct Job {
            int grp, vslot;
            uint32_t vpar;
            bool half, first, last, alone;
          };
          uint32_t jc = 0, rbase = 0, qc = 0, pc = 0;  // pc: bit g is the parity of group g's next P
          bool ok = true;
          auto issue_pv = [&](const Job& j, uint32_t seg) -> bool {
            if (!mbar_wait(&sm.p_full[j.grp][0], (pc >> j.grp) & 1, abort_flag)) return give_up(ST_TIMEOUT_TMEM_EMPTY);
            pc ^= 1u << j.grp;
            if (!mbar_wait(&sm.r_full[j.vslot], j.vpar, abort_flag)) return give_up(ST_TIMEOUT_FULL);
            // A group's first product of a segment overwrites its O of the segment before the last, which must have been read: two O
            // for each group, so that a unit's result is written while the next unit's products go on.
            // (Each barrier is waited for once in two segments, so that a parity always means the phase before.)
            const int ob = seg & 1;
            if (j.first && seg > 1 &&
                !(mbar_wait(&sm.o_free[j.grp][ob], ((seg >> 1) - 1) & 1, abort_flag) &&
                  (!j.alone || mbar_wait(&sm.o_free[j.grp ^ 1][ob], ((seg >> 1) - 1) & 1, abort_flag))))
              return give_up(ST_TIMEOUT_TMEM_EMPTY);
            tc_fence_after();
            const uint32_t v = smem_u32(sm.ring[j.vslot]), p = smem_u32(sm.p[j.grp]), o = tmem + 256 + j.grp * 128 + ob * 32;
            const int steps = j.half ? 4 : 8;
            for (int k = 0; k < steps; ++k) umma_ss(o, ta_desc_mn(v, k), ta_desc_p(p + k * 1024), idesc_o, !(j.first && k == 0));
            umma_commit(&sm.r_empty[j.vslot]);
            if (j.last) umma_commit(&sm.o_full[j.grp][ob]);
            return true;
          };
          Job prev;
          bool have = false;
          uint32_t prev_seg = 0;
          for (uint32_t n = 0; ok; ++n) {
            const TreeSegment& g = sm.seg[n & 1];
            if (!mbar_wait(&sm.seg_full[n & 1], (n >> 1) & 1, abort_flag)) {
              ok = give_up(ST_TIMEOUT_FULL);
              break;
            }
            if (g.t0 == g.t1) break;
            const int count = g.t1 - g.t0;
            const int half_at = g.C <= (g.nt - 1) * 128 ? g.nt - 1 - g.t0 : -1;  // the tree's tile without a page: 64 keys
            mbar_arrive(&sm.seg_empty[n & 1]);
            const int qs = qc & 1;
            for (int x = 0; x < count && ok; ++x, ++jc) {
              Job j;
              j.grp = jc & 1;
              const uint32_t kn = rbase + ring_k(x), vn = rbase + ring_v(x, count);
              const int ks = kn % RING;
              j.vslot = vn % RING;
              j.vpar = (vn / RING) & 1;
              j.half = x == half_at;
              j.first = x < 2;
              j.alone = count == 1;
              j.last = x >= count - 2;
              if ((x == 0 && !mbar_wait(&sm.q_full[qs], (qc >> 1) & 1, abort_flag)) || !mbar_wait(&sm.r_full[ks], (kn / RING) & 1, abort_flag)) {
                ok = give_up(ST_TIMEOUT_FULL);
                break;
              }
              tc_fence_after();
              const uint32_t q = smem_u32(sm.q[qs]), kt = smem_u32(sm.ring[ks]);
              for (int k = 0; k < 8; ++k)
                umma_ss(tmem + j.grp * 128, ta_desc_k(kt, k), umma_desc_sw128(q + (k >> 2) * TA_QSUB + (k & 3) * 32, 16, 1024), idesc_s, k != 0);
              umma_commit(&sm.r_empty[ks]);
              if (x == count - 1) umma_commit(&sm.q_empty[qs]);
              umma_commit(&sm.s_full[j.grp][0]);
              if (have) ok = issue_pv(prev, prev_seg);
              prev = j;
              prev_seg = n;
              have = true;
            }
            rbase += 2 * count;
            ++qc;
          }
          if (ok && have) issue_pv(prev, prev_seg);
        } else {
          // Each group has a thread of its own here and steps of 64 keys: with two row tiles the halves of all key tiles in turn, with
          // one row tile its half of each.  S has two buffers of 64 columns, so S of a step is issued while the softmax still works
          // on the step before, and the groups do not wait for one another.  Both threads give back every load, used or not.
          constexpr uint32_t idesc_s = umma_idesc_bf16(128, 64, false, false), idesc_o = umma_idesc_bf16(128, 128, false, true);
          const int grp = warp >> 1;
          const uint32_t t_s = tmem + grp * 128, t_o = tmem + 256 + grp * 128;
          uint32_t rbase = 0, qc = 0, steps_s = 0, steps_o = 0;  // loads and row tiles so far; S and P V issued
          struct Step {
            uint32_t v;  // load
            int h;
            bool first, last;  // of the segment; of this V
          } prev{0u, 0, false, false};
          bool have = false, ok = true;
          uint32_t prev_seg = 0;
          auto loaded = [&](uint32_t load) { return mbar_wait(&sm.r_full[load % RING], (load / RING) & 1, abort_flag) || give_up(ST_TIMEOUT_FULL); };
          auto issue_pv = [&]() -> bool {
            const int b = steps_o & 1;
            if (!mbar_wait(&sm.p_full[grp][b], (steps_o >> 1) & 1, abort_flag)) return give_up(ST_TIMEOUT_TMEM_EMPTY);
            if (!loaded(prev.v)) return false;
            // the first product of a unit overwrites O: the last unit's must have been read
            if (prev.first && prev_seg > 0 && !mbar_wait(&sm.o_free[grp][0], (prev_seg - 1) & 1, abort_flag)) return give_up(ST_TIMEOUT_TMEM_EMPTY);
            tc_fence_after();
            const uint32_t v = smem_u32(sm.ring[prev.v % RING]) + prev.h * (TA_SUB / 2), p = t_s + b * 64;
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_ts(t_o, p + k * 8, ta_desc_mn(v, k), idesc_o, !(prev.first && k == 0));
            if (prev.last) umma_commit(&sm.r_empty[prev.v % RING]);
            umma_commit(&sm.o_full[grp][0]);  // of every step: the softmax rescales O between them
            ++steps_o;
            have = false;
            return true;
          };
          for (uint32_t n = 0; ok; ++n) {
            const TreeSegment& g = sm.seg[n & 1];
            if (!mbar_wait(&sm.seg_full[n & 1], (n >> 1) & 1, abort_flag)) {
              ok = give_up(ST_TIMEOUT_FULL);
              break;
            }
            if (g.t0 == g.t1) break;
            const int count = g.t1 - g.t0, tail = (g.C >> 7) - g.t0;  // from tile `tail` on the softmax may clear rows of V
            const bool two = g.nrt == 2, half_last = g.t1 == g.nt && g.C <= (g.nt - 1) * 128;
            mbar_arrive(&sm.seg_empty[n & 1]);
            const bool skips = !two && grp == 1 && half_last;  // the last tile has no half for this group
            const int steps = two ? 2 * count - half_last : count - skips;
            for (int rt = 0; rt <= two && ok; ++rt)
              if (!mbar_wait(&sm.q_full[(qc + rt) & 1], ((qc + rt) >> 1) & 1, abort_flag)) ok = give_up(ST_TIMEOUT_FULL);
            const int qs = (qc + (two ? grp : 0)) & 1;
            const uint32_t q = smem_u32(sm.q[qs]);
            for (int u = 0; u < steps && ok; ++u) {
              const int i = two ? u >> 1 : u, h = two ? u & 1 : grp;
              const uint32_t kn = rbase + ring_k(i), vn = rbase + ring_v(i, count);
              ok = loaded(kn) && (i < tail || loaded(vn));  // the softmax's own wait for V then cannot mean an older load
              if (!ok) break;
              const bool last = !two || h == 1 || (half_last && i == count - 1);
              tc_fence_after();
              const uint32_t kt = smem_u32(sm.ring[kn % RING]) + h * (TA_SUB / 2);
              const int b = steps_s++ & 1;
#pragma unroll
              for (int k = 0; k < 8; ++k) umma_ss(t_s + b * 64, ta_desc_k(q, k), ta_desc_k(kt, k), idesc_s, k != 0);
              umma_commit(&sm.s_full[grp][b]);
              if (last) umma_commit(&sm.r_empty[kn % RING]);
              if (u == steps - 1) umma_commit(&sm.q_empty[qs]);
              if (have) ok = issue_pv();
              prev = Step{vn, h, u == 0, last};
              prev_seg = n;
              have = true;
            }
            if (!ok) break;
            if (two) mbar_arrive(&sm.q_empty[qs ^ 1]);  // filled, and not used here
            if (skips) {
              if (have) ok = issue_pv();
              if (steps == 0) mbar_arrive(&sm.q_empty[qs]);
              const uint32_t kn = rbase + ring_k(count - 1), vn = rbase + ring_v(count - 1, count);
              ok = ok && loaded(kn);
              if (ok) mbar_arrive(&sm.r_empty[kn % RING]);
              ok = ok && loaded(vn);
              if (ok) mbar_arrive(&sm.r_empty[vn % RING]);
            }
            rbase += 2 * count;
            qc += two ? 2 : 1;
          }
          if (ok && have) issue_pv();
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TaRegs<narrow>::softmax));
    const int grp = (warp - 4) >> 2, lg = warp & 3, r = lg * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(lg * 32) << 16;
    const uint32_t t_s = tmem + grp * 128 + lane_off, t_o = tmem + 256 + lane_off;
    const float c = a.scale * TA_LOG2E;
    uint32_t rbase = 0;
    bool ok = true;
    // the last segment's end is over on both sides, what it left behind has been read.  Every warp waits for that in every
    // segment and says when it is through with this one, so no barrier is more than one phase away from a parity that is waited for.
    auto last_end = [&](uint32_t n) {
      const int ob = narrow ? (n - 1) & 1 : 0, par = (narrow ? (n - 1) >> 1 : n - 1) & 1;
      return n == 0 || (ta_warp_wait(&sm.o_free[0][ob], par, abort_flag) && ta_warp_wait(&sm.o_free[1][ob], par, abort_flag));
    };
    auto through = [&](uint32_t n) {
      const int ob = narrow ? n & 1 : 0;
      if (lane == 0) {
        mbar_arrive(&sm.o_free[0][ob]);
        mbar_arrive(&sm.o_free[1][ob]);
      }
    };
    if constexpr (narrow) {
      uint32_t jc = 0;
      uint32_t par_s = 0, par_o = 0, par_ml = 0, par_flag = 0, par_mx = 0, par_lx = 0;  // parities of the next S, of either group's O (bit: group, and 2 more in odd segments), of exchanges
      const int rn = lane / a.G, rg = lane - rn * a.G;  // node and head of row `lane`
      for (uint32_t n = 0; ok; ++n) {
        const TreeSegment& g = sm.seg[n & 1];
        ok = ta_warp_wait(&sm.seg_full[n & 1], (n >> 1) & 1, abort_flag);
        if (!ok || g.t0 == g.t1) break;
        const int t0 = g.t0, count = g.t1 - t0, nt = g.nt, T = g.T, C = g.C, jobs = count, ob = n & 1;
        const uint32_t t_on = t_o + ob * 32;
        const int x0 = (grp ^ jc) & 1;           // my first job of this segment; then every second one
        const bool valid = rn < T;
        const unsigned long long sees = valid ? g.sees[rn] : 0ull;
        const int own = r - (C > (nt - 1) * 128 ? 64 : 0);  // the node whose key is in this thread's row of the tree's tile
        const bool gap = own >= 0 && own < 64 && g.sees[own] == 0ull;  // there is none, or it is padding
        // Rows that see cached keys: a padding node's do not, so that its products are zeros.  (Zeros put in when the result is written
        // cost 4 to 8 us of 295 at one head a group.)
        const uint32_t alive = ~__ballot_sync(0xffffffffu, valid && !sees);
        const long long seg_at = (static_cast<long long>(g.n0) * a.Hq + g.kvh * a.G) * TA_DH;  // the sequence's first row in the result
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.seg_empty[n & 1]);
        float m = 0.f, l = 0.f;
        // The scores of tile x are there: its keys (as many as 128, fewer in the last tiles) and whether it is the tree's without a
        // page.  Rows of V that hold no key, or a padding node's, are cleared: 0 * NaN must not reach the output.
        auto begin_job = [&](int x, int& keys, bool& half) -> bool {
          if (!ta_warp_wait(&sm.s_full[grp][0], par_s, abort_flag)) return false;
          par_s ^= 1;
          tc_fence_after();
          const int t = t0 + x;
          keys = min(128, C - t * 128);
          half = t == nt - 1 && keys <= 0;
          if (t < nt - 1 && keys == 128) return true;
          const bool empty = t < nt - 1 ? r >= keys : gap || (r >= keys && r < 64 && !half);
          const uint32_t vn = rbase + ring_v(x, count);
          if (!ta_warp_wait(&sm.r_full[vn % RING], (vn / RING) & 1, abort_flag)) return false;
          if (empty) {
            uint4* row = reinterpret_cast<uint4*>(sm.ring[vn % RING] + r * 128);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int at = (q + lane) & 7;  // neighbouring rows start in different banks
              row[at] = row[at + TA_SUB / 16] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async();
          return true;
        };
        uint64_t nm[16], ln[16];  // reference points (negated) and sums of the 32 rows, this thread's keys
#pragma unroll
        for (int e = 0; e < 16; ++e) nm[e] = ln[e] = 0ull;
        for (int x = x0; x < jobs; x += 2) {
          const int t = t0 + x;
          int keys;
          bool half;
          ok = begin_job(x, keys, half);
          if (!ok) break;
          // ---- a thread has one key and all 32 rows.  The exponentials are taken against a reference point that starts at 0 and moves
          // to the rows' maxima only if a score exceeds it by 2^40, or if none of a unit's first scores comes up to 2^-40 of it:
          // fp32 and bf16 hold 2^+-126, so in between only the sums' exponents differ.
          uint32_t word = alive;  // the rows that see this key
          if (t == nt - 1) {
            const int node0 = (half ? lg : lg - 2) * 32;  // keys of the tree in this warp
            word = r < keys ? alive : 0u;
            if (node0 == 0) {
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const uint32_t rows = __ballot_sync(0xffffffffu, (sees >> e) & 1ull);
                if (lane == e) word = rows;
              }
            }
          } else if (r >= keys) {
            word = 0u;
          }
          uint32_t sv[32];
          tmem_ld32(t_s, sv);
          tmem_ld_wait();
          if (__any_sync(0xffffffffu, word != ~0u)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((word >> e) & 1u)) sv[e] = 0xff800000u;
          }
          const uint64_t c2 = pair2(c, c);
          float xs[32];
#pragma unroll
          for (int e = 0; e < 16; ++e) unpair2(fma2(pair2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), c2, nm[e]), xs[2 * e], xs[2 * e + 1]);
          float hi2[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; e += 2) hi2[e / 2 & 1] = max3(hi2[e / 2 & 1], xs[e], xs[e + 1]);
          uint32_t flag = __any_sync(0xffffffffu, fmaxf(hi2[0], hi2[1]) > 40.f) ? 1u : 0u;
          if (x < 2) {
            float low = INFINITY;
            const int rows = T * a.G;
#pragma unroll
            for (int e = 0; e < 32; ++e) low = e < rows ? fminf(low, xs[e]) : low;
            flag |= __any_sync(0xffffffffu, low > -40.f) ? 2u : 0u;  // one key that is not far below the reference for any row
          } else {
            flag |= 2u;
          }
          if (lane == 0) {
            reinterpret_cast<volatile uint8_t*>(&sm.flags[grp])[lg] = static_cast<uint8_t>(flag);
            mbar_arrive(&sm.flag_full[grp]);
          }
          ok = ta_warp_wait(&sm.flag_full[grp], par_flag, abort_flag);
          par_flag ^= 1;
          if (!ok) break;
          const uint32_t flags = *reinterpret_cast<volatile uint32_t*>(&sm.flags[grp]);
          if ((flags & 0x01010101u) || !(flags & 0x02020202u)) {
            // move the rows' reference points to their maxima (after the first scores: only upwards)
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float v = warp_max(xs[e]);
              if (lane == e) top = v;
            }
            sm.mx[grp][lg][lane] = top;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.mx_full[grp]);
            ok = ta_warp_wait(&sm.mx_full[grp], par_mx, abort_flag);
            par_mx ^= 1;
            if (!ok) break;
            top = fmaxf(fmaxf(sm.mx[grp][0][lane], sm.mx[grp][1][lane]), fmaxf(sm.mx[grp][2][lane], sm.mx[grp][3][lane]));
            if (top == -INFINITY || (x >= 2 && top < 0.f)) top = 0.f;  // a row without a key so far stays where it is
            m += top;
            sm.wt[warp - 4][0][lane] = -top;
            sm.wt[warp - 4][1][lane] = x < 2 ? 1.f : ex2_approx(-top);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 v = *reinterpret_cast<const float4*>(&sm.wt[warp - 4][0][e]), w = *reinterpret_cast<const float4*>(&sm.wt[warp - 4][1][e]);
              nm[e / 2] = add2(nm[e / 2], pair2(v.x, v.y));
              nm[e / 2 + 1] = add2(nm[e / 2 + 1], pair2(v.z, v.w));
              ln[e / 2] = mul2(ln[e / 2], pair2(w.x, w.y));
              ln[e / 2 + 1] = mul2(ln[e / 2 + 1], pair2(w.z, w.w));
              xs[e] += v.x;
              xs[e + 1] += v.y;
              xs[e + 2] += v.z;
              xs[e + 3] += v.w;
            }
            if (x >= 2) {
              uint32_t o[32];
              tmem_ld32(t_on + grp * 128, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float4 w = *reinterpret_cast<const float4*>(&sm.wt[warp - 4][1][e]);
                o[e] = __float_as_uint(__uint_as_float(o[e]) * w.x);
                o[e + 1] = __float_as_uint(__uint_as_float(o[e + 1]) * w.y);
                o[e + 2] = __float_as_uint(__uint_as_float(o[e + 2]) * w.z);
                o[e + 3] = __float_as_uint(__uint_as_float(o[e + 3]) * w.w);
              }
              tmem_st32(t_on + grp * 128, o);
              tmem_st_wait();
            }
            __syncwarp();
          }
          uint8_t* prow = sm.p[grp] + r * 64;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i2 = q * 4 + e;
              const float p0 = ex2_approx(xs[2 * i2]), p1 = ex2_approx(xs[2 * i2 + 1]);
              ln[i2] = add2(ln[i2], pair2(p0, p1));
              pk[e] = pack_bf16x2(p0, p1);
            }
            *reinterpret_cast<uint4*>(prow + ((q ^ (r >> 1 & 3)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
          fence_proxy_async();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[grp][0]);
        }
        if (!ok) break;
        // 32 sums over the warp's keys: halve the rows and the lanes that share them, until lane i has row i
        float v[32];
#pragma unroll
        for (int e = 0; e < 16; ++e) unpair2(ln[e], v[2 * e], v[2 * e + 1]);
#pragma unroll
        for (int h = 16; h > 0; h >>= 1) {
          const bool upper = lane & h;
#pragma unroll
          for (int e = 0; e < h; ++e) {
            const float send = upper ? v[e] : v[e + h], keep = upper ? v[e + h] : v[e];
            v[e] = keep + __shfl_xor_sync(0xffffffffu, send, h);
          }
        }
        l = sees ? v[0] : 0.f;

        // ---- end of the segment: the group of the last job joins both and writes, the other hands over its maxima and sums and goes on
        const int last = (jc + jobs - 1) & 1;
        const bool both = jobs > 1;
        jc += jobs;
        rbase += 2 * count;
        ok = last_end(n);
        if (!ok) break;
        if (grp != last) {
          if (both) {
            sm.ls[grp][lg][lane] = l;
            sm.lm[grp][lane] = m;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.ml_full[grp]);
          }
          through(n);
          par_o ^= (both ? 3 : 1 << last) << 2 * ob;
          continue;
        }
        float a0 = 1.f, a1 = 0.f;  // weights of my own O and of the other group's
        sm.ls[grp][lg][lane] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.lx_full[grp]);
        ok = ta_warp_wait(&sm.lx_full[grp], par_lx, abort_flag);
        par_lx ^= 1;
        if (!ok) break;
        l = (sm.ls[grp][0][lane] + sm.ls[grp][1][lane]) + (sm.ls[grp][2][lane] + sm.ls[grp][3][lane]);
        if (both) {
          ok = ta_warp_wait(&sm.ml_full[grp ^ 1], par_ml, abort_flag);
          par_ml ^= 1;
          if (ok) ok = ta_warp_wait(&sm.o_full[grp ^ 1][ob], par_o >> (2 * ob + (grp ^ 1)) & 1, abort_flag);
          if (!ok) break;
          const float* o = &sm.ls[grp ^ 1][0][lane];
          const float l_other = (o[0] + o[32]) + (o[64] + o[96]), m_other = sm.lm[grp ^ 1][lane], top = fmaxf(m, m_other);
          a0 = l != 0.f ? ex2_approx(m - top) : 0.f;
          a1 = l_other != 0.f ? ex2_approx(m_other - top) : 0.f;
          l = a0 * l + a1 * l_other;
          m = top;
        }
        ok = ta_warp_wait(&sm.o_full[grp][ob], par_o >> (2 * ob + grp) & 1, abort_flag);
        par_o ^= (both ? 3 : 1 << grp) << 2 * ob;
        if (!ok) break;
        tc_fence_after();
        const bool whole = t0 == 0 && count == nt;
        const long long part = (static_cast<long long>(cta) * 2 + (t0 == 0 ? 1 : 0)) * a.part_rows + lane;
        // O^T: a thread has one dimension (r) of all 32 rows; the rows' weights come from the lanes that hold them
        const float inv = whole ? (l != 0.f ? 1.f / l : 0.f) : 1.f;  // an empty row gives zeros, a NaN stays one
        sm.wt[warp - 4][0][lane] = a0 * inv;
        sm.wt[warp - 4][1][lane] = a1 * inv;
        if (!whole && valid && lg == 0) a.part_ml[part] = make_float2(m, l);
        const int to = valid ? (rn * a.Hq + rg) * TA_DH : -1;
        uint32_t o0[32], o1[32];
        tmem_ld32(t_on + grp * 128, o0);
        if (both) tmem_ld32(t_on + (grp ^ 1) * 128, o1);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 w = *reinterpret_cast<const float4*>(&sm.wt[warp - 4][0][e]), z = *reinterpret_cast<const float4*>(&sm.wt[warp - 4][1][e]);
          f[e] = w.x * __uint_as_float(o0[e]);
          f[e + 1] = w.y * __uint_as_float(o0[e + 1]);
          f[e + 2] = w.z * __uint_as_float(o0[e + 2]);
          f[e + 3] = w.w * __uint_as_float(o0[e + 3]);
          if (both) {
            f[e] = fmaf(z.x, __uint_as_float(o1[e]), f[e]);
            f[e + 1] = fmaf(z.y, __uint_as_float(o1[e + 1]), f[e + 1]);
            f[e + 2] = fmaf(z.z, __uint_as_float(o1[e + 2]), f[e + 2]);
            f[e + 3] = fmaf(z.w, __uint_as_float(o1[e + 3]), f[e + 3]);
          }
        }
        __syncwarp();
        through(n);
        const int rows = T * a.G;
        if (whole) {
          __nv_bfloat16* dst = a.out + seg_at + (r & ~1);  // two neighbouring dimensions of every second row
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            if (e >= rows) break;
            const bool odd = lane & 1;
            const float got = __shfl_xor_sync(0xffffffffu, odd ? f[e] : f[e + 1], 1);
            const int row = __shfl_sync(0xffffffffu, to, e + (lane & 1));
            if (row >= 0) *reinterpret_cast<uint32_t*>(dst + row) = odd ? pack_bf16x2(got, f[e + 1]) : pack_bf16x2(f[e], got);
          }
        } else {
          float* dst = a.part_o + (part - lane) * TA_DH + r;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (e < rows) dst[e * TA_DH] = f[e];
        }
      }
    } else {
      uint32_t mine = 0, other = 0, par_ml = 0;  // steps of this group and of the other one before this segment
      const int rn = r / a.G, rg = r - rn * a.G;  // node of the row tile and head of the group
      for (uint32_t n = 0; ok; ++n) {
        const TreeSegment& g = sm.seg[n & 1];
        ok = ta_warp_wait(&sm.seg_full[n & 1], (n >> 1) & 1, abort_flag);
        if (!ok || g.t0 == g.t1) break;
        const int t0 = g.t0, count = g.t1 - t0, nt = g.nt, T = g.T, C = g.C;
        const bool two = g.nrt == 2, half_last = t0 + count == nt && C <= (nt - 1) * 128;
        const int all = two ? 2 * count - half_last : count;                  // steps of group 0 in this segment
        const int steps = two || grp == 0 ? all : all - half_last, others = two || grp == 1 ? all : all - half_last;
        const int rt = two ? grp : 0, node = g.first + rt * a.npt + rn;
        const bool valid = rn < a.npt && node < T;
        const unsigned long long sees = valid ? g.sees[node] : 0ull;
        const bool empty = g.sees[r & 63] == 0ull;  // the tree has no node, or padding, at this thread's key
        const bool empties = __any_sync(0xffffffffu, empty);
        const long long out_at = ((static_cast<long long>(g.n0) + node) * a.Hq + g.kvh * a.G + rg) * TA_DH;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.seg_empty[n & 1]);
        const bool busy = __any_sync(0xffffffffu, valid);
        float m = -INFINITY, l = 0.f;
        for (int u = 0; u < steps; ++u) {
          const uint32_t U = mine + u;
          const int b = U & 1, i = two ? u >> 1 : u, h = two ? u & 1 : grp, t = t0 + i;
          ok = ta_warp_wait(&sm.s_full[grp][b], (U >> 1) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          // the keys of this half: as many as 64 cached ones, or the tree's
          const int keys = min(64, C - t * 128 - h * 64);
          const bool tree = t == nt - 1 && (h == 1 || keys <= 0);
          const unsigned long long live = tree ? sees : low_bits(max(keys, 0));
          if (tree ? empties : keys < 64) {  // rows of V that hold no key are cleared (by either group: the same zeros): 0 * NaN must not reach the output
            const uint32_t vn = rbase + ring_v(i, count);
            ok = ta_warp_wait(&sm.r_full[vn % RING], (vn / RING) & 1, abort_flag);
            if (!ok) break;
            if (tree ? empty : (r & 63) >= keys) {
              uint4* row = reinterpret_cast<uint4*>(sm.ring[vn % RING] + (r >> 6) * TA_SUB + (h * 64 + (r & 63)) * 128);
#pragma unroll
              for (int q = 0; q < 8; ++q) row[(q + lane) & 7] = make_uint4(0u, 0u, 0u, 0u);  // neighbouring rows start in different banks
            }
            fence_proxy_async();
          }
          float alpha = 1.f;
          bool grow = false;
          if (busy) {
            const uint32_t ts = t_s + b * 64;
            uint32_t sv[2][32];
            tmem_ld32(ts, sv[0]);
            tmem_ld32(ts + 32, sv[1]);
            tmem_ld_wait();
            if (__any_sync(0xffffffffu, live != ~0ull)) {
              const uint32_t words[2] = {static_cast<uint32_t>(live), static_cast<uint32_t>(live >> 32)};
#pragma unroll
              for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (!((words[cc] >> e) & 1u)) sv[cc][e] = 0xff800000u;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
              for (int e = 0; e < 32; e += 2) mx4[e / 2 & 3] = max3(mx4[e / 2 & 3], __uint_as_float(sv[cc][e]), __uint_as_float(sv[cc][e + 1]));
            const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]);
            grow = (mx - m) * c > 8.f;
            if (grow) {
              alpha = ex2_approx((m - mx) * c);
              m = mx;
              l *= alpha;
            }
            const float at0 = m == -INFINITY ? 0.f : -m * c;  // no score above -inf yet: weights of zero, not -inf + inf
            const uint64_t c2 = pair2(c, c), mc2 = pair2(at0, at0);
            uint64_t sum[2] = {0ull, 0ull};  // two pairs of zeros
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                float p0, p1;
                unpair2(fma2(pair2(__uint_as_float(sv[cc][e]), __uint_as_float(sv[cc][e + 1])), c2, mc2), p0, p1);
                p0 = ex2_approx(p0);
                p1 = ex2_approx(p1);
                sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pair2(p0, p1));
                pk[e >> 1] = pack_bf16x2(p0, p1);
              }
              tmem_st16(ts + cc * 16, pk);
            }
            float s0, s1;
            unpair2(add2(sum[0], sum[1]), s0, s1);
            l += s0 + s1;
          }
          // The product of the step before is waited for where O is to be rescaled, and in the last step: from there on the parity of
          // the last product's phase can only mean that one.
          const bool rescale = u > 0 && __any_sync(0xffffffffu, grow);
          if (U > 0 && (rescale || u == steps - 1)) {
            ok = ta_warp_wait(&sm.o_full[grp][0], (U - 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
          }
          if (rescale) {
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
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[grp][b]);
        }
        if (!ok) break;
        if (!sees) {
          m = -INFINITY;
          l = 0.f;
        }
        m *= c;  // base-2 scale from here on

        // ---- end of the segment: the result or a part of it.  Two row tiles: each group writes its own.  One: the group of the last
        // step joins both, the other hands over its maxima and sums and goes on with the next unit.
        const uint32_t my_last = mine + steps - 1, their_last = other + others - 1;
        const bool both = !two && steps > 0 && others > 0;
        const int last = both ? !half_last : 0;
        mine += steps;
        other += others;
        rbase += 2 * count;
        ok = last_end(n);
        if (!ok) break;
        float a0 = 1.f, a1 = 0.f;  // weights of my own O and of the other group's
        if (two) {
          if (lane == 0) mbar_arrive(&sm.o_free[grp ^ 1][0]);
        } else if (grp != last) {
          if (both) {
            sm.ml[r] = l;
            sm.ml[128 + r] = m;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.ml_full[grp]);
          }
          through(n);
          continue;
        } else if (both) {
          ok = ta_warp_wait(&sm.ml_full[grp ^ 1], par_ml >> (grp ^ 1) & 1, abort_flag) && ta_warp_wait(&sm.o_full[grp ^ 1][0], their_last & 1, abort_flag);
          par_ml ^= 1u << (grp ^ 1);
          if (!ok) break;
          const float l_other = sm.ml[r], m_other = sm.ml[128 + r], top = fmaxf(m, m_other);
          a0 = l != 0.f ? ex2_approx(m - top) : 0.f;
          a1 = l_other != 0.f ? ex2_approx(m_other - top) : 0.f;
          l = a0 * l + a1 * l_other;
          m = top;
        }
        ok = steps == 0 || ta_warp_wait(&sm.o_full[grp][0], my_last & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const bool whole = t0 == 0 && count == nt;
        const long long part = (static_cast<long long>(cta) * 2 + (t0 == 0 ? 1 : 0)) * a.part_rows + rt * 128 + r;
        if (whole) {  // a row that sees nothing gives zeros (below), a NaN stays one
          a0 *= 1.f / l;
          a1 *= 1.f / l;
        }
        const uint64_t w0 = pair2(a0, a0), w1 = pair2(a1, a1);
        if (busy) {
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t v[32], u[32];
            tmem_ld32(t_o + grp * 128 + cc * 32, v);
            if (both) tmem_ld32(t_o + (grp ^ 1) * 128 + cc * 32, u);
            tmem_ld_wait();
            float f[32];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              uint64_t y = mul2(pair2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), w0);
              if (both) y = fma2(pair2(__uint_as_float(u[e]), __uint_as_float(u[e + 1])), w1, y);
              unpair2(y, f[e], f[e + 1]);
            }
            if (whole) {
              if (valid) {
                uint4* dst = reinterpret_cast<uint4*>(a.out + out_at + cc * 32);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint4 y = make_uint4(pack_bf16x2(f[8 * e], f[8 * e + 1]), pack_bf16x2(f[8 * e + 2], f[8 * e + 3]),
                                             pack_bf16x2(f[8 * e + 4], f[8 * e + 5]), pack_bf16x2(f[8 * e + 6], f[8 * e + 7]));
                  dst[e] = sees ? y : make_uint4(0u, 0u, 0u, 0u);
                }
              }
            } else if (valid) {
              float4* dst = reinterpret_cast<float4*>(a.part_o + part * TA_DH + cc * 32);
#pragma unroll
              for (int e = 0; e < 8; ++e) dst[e] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.o_free[grp][0]);
          if (!two) mbar_arrive(&sm.o_free[grp ^ 1][0]);
        }
        if (valid && !whole) a.part_ml[part] = make_float2(m, l);
        __syncwarp();
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
// Parts in the order of the keys.
//
// Nothing is launched early behind this kernel, so whatever follows the attention starts when all of its CTAs have left and their
// tensor memory is free.  Launched early, the pairs of a decode GEMM two kernels further took over SMs the moment the attention's
// last CTAs left them, and their allocation of tensor memory for a pair, right behind the release by a single CTA, never returned
// (5 rows at 8B, within 60 decode steps; the bounded waits cannot end that one).
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeArgs a) {
  griddep_wait();
  const int cta = blockIdx.x;
  const int4 join = a.joins[cta];
  const int parts = join.x;
  if (parts == 0) return;
  // A warp joins four rows at a time, all their loads in flight together: one row after the other took 15.5 us for parts of 256
  // rows (75 MB of parts), this 9.6; with four rows in all it is 0.5 us slower (12.7 against 12.2 us for the whole call).
  constexpr int ROWS = 4;
  const int lane = threadIdx.x & 31, row0 = blockIdx.y * 32 + (threadIdx.x >> 5);  // and every eighth row from there
  int node[ROWS];  // -1: no row
  float top[ROWS], l[ROWS];
  float4 acc[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = row0 + 8 * i, rn = (row & 127) / a.G;
    node[i] = (row >> 7) * a.npt + rn;
    if (row >= a.part_rows || rn >= a.npt || node[i] >= join.z) node[i] = -1;
    top[i] = -INFINITY;
    l[i] = 0.f;
    acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  auto at = [&](int p, int i) { return (static_cast<long long>(cta + p) * 2 + (p == 0 ? 1 : 0)) * a.part_rows + row0 + 8 * i; };
  for (int p = lane; p < parts; p += 32) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (node[i] < 0) continue;
      const float2 ml = a.part_ml[at(p, i)];
      if (ml.y != 0.f) top[i] = fmaxf(top[i], ml.x);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < ROWS; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
  for (int p = 0; p < parts; ++p) {
    float2 ml[ROWS];
    float4 v[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      ml[i] = make_float2(0.f, 0.f);
      if (node[i] < 0) continue;
      ml[i] = a.part_ml[at(p, i)];
      v[i] = reinterpret_cast<const float4*>(a.part_o + at(p, i) * TA_DH)[lane];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (ml[i].y == 0.f) continue;
      const float w = ex2_approx(ml[i].x - top[i]);
      l[i] += w * ml[i].y;
      acc[i].x += w * v[i].x;
      acc[i].y += w * v[i].y;
      acc[i].z += w * v[i].z;
      acc[i].w += w * v[i].w;
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (node[i] < 0) continue;
    const float inv = l[i] != 0.f ? 1.f / l[i] : 0.f;  // an empty row gives zeros, a NaN stays one
    uint2 res;
    res.x = pack_bf16x2(acc[i].x * inv, acc[i].y * inv);
    res.y = pack_bf16x2(acc[i].z * inv, acc[i].w * inv);
    __nv_bfloat16* dst = a.out + ((static_cast<long long>(join.y) + node[i]) * a.Hq + join.w * a.G + ((row0 + 8 * i) & 127) % a.G) * TA_DH;
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

template <bool narrow>
static int ta_launch(const CUtensorMap& tq, const CUtensorMap& tn, const CUtensorMap& tk, const CUtensorMap& tv, const TreeArgs& a, int sms,
                     cudaStream_t st) {
  const auto kern = tree_attn_kernel<narrow>;
  const int smem = sizeof(TreeSmem<narrow>);
  static std::atomic<unsigned long long> cfg{0};
  const cudaError_t e = opt_in_shared_memory(kern, smem, cfg);
  if (e != cudaSuccess) return static_cast<int>(e);
  static const int regs = [&] {
    cudaFuncAttributes f = {};
    return cudaFuncGetAttributes(&f, kern) == cudaSuccess ? f.numRegs : 0;
  }();
  if (regs != TA_REGS) return -4;  // the register split of the groups would wait for registers that the launch did not bring
  return static_cast<int>(launch_pdl(kern, dim3(sms), dim3(TA_THREADS), smem, st, tq, tn, tk, tv, a));
}

extern "C" int b200_tree_attn(const void* qkv, long long ld, const void* k_cache, const void* v_cache, int num_blocks, const int* table,
                              long long table_ld, int max_blocks, const int* ctx, const int* cu, const int* parents, int B, int N,
                              int max_nodes, int Hq, int Hkv, int Dh, float scale, void* out, void* scratch, int* status, void* stream) {
  if (B <= 0 || N <= 0) return 0;
  const int need = b200_tree_attn_scratch(max_nodes, Hq, Hkv);
  if (Dh != TA_DH || need < 0 || num_blocks < 1 || max_blocks > (1 << 24)) return -1;
  // rows of the cache are 32-bit TMA coordinates, work is counted in 32 bits
  if ((static_cast<long long>(num_blocks) + 1) * Hkv * TA_PAGE >= (1ll << 31)) return -3;
  if (static_cast<double>(B) * Hkv * ((max_nodes + 128 / (Hq / Hkv) - 1) / (128 / (Hq / Hkv))) * (max_blocks / 2 + 2) >= 2147483648.0) return -3;
  TreeArgs a;
  a.G = Hq / Hkv;
  // The narrow kernel where every tree fits into 32 rows.  Narrow against wide: 32 rows at contexts of 16384, 345 against 368 us, of
  // 1024, 68 against 75; 20 rows, 69 against 81; 8 rows, 290 against 350; single tokens, 12.0 against 15.0.
  const bool narrow = max_nodes * a.G <= 32;
  a.npt = (narrow ? 32 : 128) / a.G;
  CUtensorMap tq, tn, tk, tv;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * Hkv * TA_PAGE;
  int r = ta_map_3d(&tq, qkv, ld, Hq + 2 * Hkv, N, a.G, a.npt);
  if (!r) r = ta_map_3d(&tn, qkv, ld, Hq + 2 * Hkv, N, 1, max_nodes);
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  r = narrow ? ta_launch<true>(tq, tn, tk, tv, a, sms, st) : ta_launch<false>(tq, tn, tk, tv, a, sms, st);
  if (r) return r;
  const cudaError_t e = launch_pdl(tree_join_kernel, dim3(sms, (a.part_rows + 31) / 32), dim3(256), 0, st, a);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
