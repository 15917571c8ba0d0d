// Gradient of the weights of the contiguous BF16 grouped GEMM:
//
//   dW[g][n][k] = sum over rows i with m_indices[i] = g of dY[i][n] * X[i][k]
//
// written in the packed layout of the weight itself, [g][k / 64][n][k % 64], so that an optimiser
// steps over weight and gradient element by element.  The contraction runs along the rows of both
// operands, i.e. both are stored along M / N: a TMA box of 64 columns x 64 rows (128-byte swizzle)
// is exactly the tensor cores' operand for 64 steps of the contraction, and neither operand is
// transposed anywhere.
//
// Tiles and roles.  kSplit: below.  CL = 2: a cluster of two blocks computes 256 (n) x 256 (k) with
// tcgen05.mma.cta_group::2, block r owning rows [128 r, 128 r + 128) of the tile (its part of dY, its
// accumulator, its epilogue) and holding 128 of the 256 columns of X.  CL = 1: one block, 128 x 128,
// for problems with few tiles.  Either way a ring stage holds 64 rows of 128 columns of each
// operand (32 KB); six stages, five where eight epilogue warps (below) need the room, and one fewer
// where the table of very many rows does.  A work item is (group, tile); its contraction walks the 128-row
// blocks of the group in ascending order, 64 rows (a chunk) at a time.
//   warp 0      TMA producer (each block its own copies)
//   warp 1      UMMA issuer (leader)
//   warps 2..5  epilogue (fp32: 8..11 too): accumulator -> bf16 or fp32 -> 32-row strip in shared memory -> TMA store
//               (or TMA reduce-add, when the gradient is added to what is there)
//   warp 6      ragged steps.  The products run in steps of 16 rows.  Rows that stand for nothing
//               (padding, rows behind the last group) must not reach a sum, whatever they hold (NaN,
//               infinities): a step that has some beside rows that count is copied by this warp,
//               with zeros in their place in both operands, into a buffer of its own, ahead of its
//               use (a group usually ends in one).  Steps whose 16 rows all count, nearly every one,
//               come from the ring.
//   warp 7      watcher (leader): waits on the barriers in the UMMA issuer's place and posts counts in
//               plain shared-memory words (store-release, load-acquire).  The issuer has 512 cycles for a chunk (four instructions
//               of 256 x 256 x 16); a first look at a barrier alone takes 200 of them.
// Which rows count is known beforehand: every block of the grid reads all of m_indices once (from
// L2) and keeps a byte for each 128 rows.  Two earlier forms cleared the rows in the ring, in
// front of the tensor cores: for every chunk that cost 1.0 us a chunk (a remote arrival with
// cluster-wide release and an acquire to match, on the path of every stage), for ragged chunks
// alone still 0.5 us a work item (32 groups of 300 to 3000 rows, 4096 x 7168: 1.65 ms instead of 1.55).
// kSplit (CL = 1): few tiles and many rows.  A cluster of 2, 4 or 8 blocks takes one tile, each block
// its share of the group's row blocks; the fp32 partial tiles stay in shared memory (in the ring,
// which is idle by then) and each block adds its share of the tile's rows over the cluster, in the
// order of the blocks, so no result depends on timing (1 group of 8000 rows, 512 x 768: 40.6 -> 19.4
// us; 2 of 4000 rows, 256 x 256: 24.2 -> 12.7).
// Precision.  The tensor cores' fp32 accumulation rounds towards zero: the sum of R rows comes out
// smaller by about 0.65e-9 R of itself (measured: relative error 1.0e-6 at 1024 rows, 9.1e-6 at 8192;
// plain fp32 sums 2.5e-7).  Beside a bf16 result that is nothing.  An fp32 result is made of segments
// of at most kWgSegment row blocks, each accumulated by itself and added to the ones before it with
// correct rounding, in order, in the epilogue's registers: eight epilogue warps (kWide), each with
// half of a tile's columns, hold a lane's 128 sums.  32 groups of 1024 rows, 4096 x 7168, i.e. two segments
// each, fp32: 1.79 ms, added to what is there 2.05 to 2.31 (cards differ): about as if
// what a bf16 result does not move (1.9 GB, added 5.6) came on top of its 1.44 ms at the copy rate.  The
// 256-wide form has 168 registers for its sums and all else (384 threads leave no more) and spills 80
// bytes.  With four warps and the segments added in memory by the
// TMA's reduce-add 2.2 and 2.7; 8 groups of 4096 rows 1.71 instead of 2.07.  Groups of one segment are on
// average where they were (768 rows 1.58 and 1.60 ms, 896 rows 1.72 and 1.51, 512 rows, 4096 x 4096, 361 and
// 404 us); bf16 results (1.44 ms) need no segments and keep four warps and the sixth ring stage.
// Groups without rows give zeros (or, added, nothing) and cost no products.
//
// Every mbarrier wait is bounded, as in the other kernels.
#pragma once

#include "deepgemm_b200.h"
#include "dg_ptx.cuh"
#include <cuda_bf16.h>

namespace dg {

constexpr int kWgStages = 6;                       // less one with eight epilogue warps, less one for a large table
constexpr int kWgThreads = 256;
constexpr int kWgWideThreads = 384;                // kWide: warps 8..11 are a second set of epilogue warps
constexpr uint32_t kWgBoxBytes = 64 * 128;         // 64 columns x 64 rows
constexpr uint32_t kWgOperand = 2 * kWgBoxBytes;   // 128 columns x 64 rows
constexpr uint32_t kWgStageBytes = 2 * kWgOperand;
constexpr uint32_t kWgTailBox = 64 * 2 * 16;       // 64 columns x 16 rows
constexpr uint32_t kWgTailBytes = 4 * kWgTailBox;  // 128 columns of both operands

constexpr int kWgSegment = 7;       // row blocks: 896 rows, 0.9e-6
constexpr int kWgIrregular = 255;  // rows that count lie between others: looked up where they are used

enum : int { WG_SITE_EMPTY = 21, WG_SITE_TAIL_EMPTY = 22, WG_SITE_READY = 23, WG_SITE_ACC_EMPTY = 24, WG_SITE_ACC_FULL = 25,
             WG_SITE_TAIL_READY = 26 };

struct WgradParams {
  int G, M, N, K;
  int n_tiles, k_tiles;      // tiles of a group
  int m_blocks;              // ceil(M / 128)
  const int32_t* m_indices;
  const __nv_bfloat16* dy;
  const __nv_bfloat16* x;
  int32_t* status;
  int f32;                   // output type: fp32 (else bf16)
  int add;                   // fp32 only: add to what the output holds
  int segment;               // most row blocks that are accumulated at once
  int split;                 // kSplit: blocks of a cluster
  void* dw;                  // kSplit: the output
  int whole_blocks;          // every row with an entry >= 0 counts for its block's group (else those of that group)
  int dy_blocks;             // N % 64 == 0: dy's map counts 64-column blocks, as x's always does
};

// EPI: epilogue warps, 4 KB each.
template <int S, int EPI>
struct WgradSmem {
  static constexpr int off_stage = 0;
  static constexpr int off_tail = off_stage + S * kWgStageBytes;
  static constexpr int off_strip = off_tail + kWgTailBytes;
  // ready[S], empty[S], tail_ready, tail_empty, acc_full[2], acc_empty[2], drain
  static constexpr int kNumBars = 2 * S + 7;
  static constexpr int off_bar = off_strip + EPI * 4096;
  static constexpr int off_misc = off_bar + kNumBars * 8;  // tmem slot, abort, stages ready, items ready, tails ready
  static constexpr int off_table = off_misc + 24;
  // table: first[G + 1] (int32), the groups' 128-row blocks in order (uint16), rows that count (uint8)
  __host__ __device__ static constexpr int total(int groups, int blocks) {
    return off_table + (groups + 1) * 4 + blocks * 3 + 16 + 1024;
  }
  // The table is built from m_indices[128 b] of every block b, held as int16 in the (still empty) ring.
  static_assert(S * static_cast<int>(kWgStageBytes) >= DG_MAX_CONTIG_ROWS / 128 * 2, "");
  static_assert(off_table % 4 == 0 && off_strip % 1024 == 0 && off_tail % 1024 == 0, "");
};
static_assert(WgradSmem<kWgStages - 1, 4>::total(DG_MAX_GROUPS, DG_MAX_CONTIG_ROWS / 128) <= 232448, "");
static_assert(WgradSmem<kWgStages - 2, 8>::total(DG_MAX_GROUPS, DG_MAX_CONTIG_ROWS / 128) <= 232448, "");

// An arrival on another block's mbarrier that orders nothing (the copies it announces are ordered by
// the barrier's byte count).
__device__ __forceinline__ void wg_arrive_remote_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void wg_fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }

__device__ __forceinline__ void wg_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src),
               "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void wg_add_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
               "r"(src), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void wg_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wg_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void wg_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ float4 wg_load_cluster(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

// kSegments: items may be more than one segment.
// Such items without kSplit take eight epilogue warps (kWide).
__host__ __device__ constexpr bool wg_wide(bool segments, bool split) { return segments && !split; }
__host__ __device__ constexpr int wg_threads(bool segments, bool split) {
  return wg_wide(segments, split) ? kWgWideThreads : kWgThreads;
}
template <int CL, int S, bool kSegments, bool kSplit = false>
__global__ void __launch_bounds__(wg_threads(kSegments, kSplit), 1)
grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_d, const WgradParams p) {
  constexpr bool kWide = wg_wide(kSegments, kSplit);
  constexpr int kThreads = wg_threads(kSegments, kSplit), kEpi = kWide ? 8 : 4;
  using L = WgradSmem<S, kEpi>;
  constexpr int BT = 128 * CL;  // tile edge
  constexpr uint32_t kIdesc = umma_idesc(1u, 1u, BT, BT) | kIdescAMn | kIdescBMn;
  constexpr int kTmemCols = 2 * BT;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  static_assert(!kSplit || CL == 1, "a split tile is computed by single blocks");
  const uint32_t rank = CL == 2 ? cluster_ctarank() : 0u;
  const int part = kSplit ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = kSplit ? blockIdx.x / p.split : blockIdx.x / CL, units = kSplit ? gridDim.x / p.split : gridDim.x / CL;

  auto bar_ready = [&](int s) { return base + L::off_bar + 8u * s; };
  auto bar_empty = [&](int s) { return base + L::off_bar + 8u * (S + s); };
  const uint32_t bar_tail_ready = base + L::off_bar + 8u * (2 * S);
  const uint32_t bar_tail_empty = base + L::off_bar + 8u * (2 * S + 1);
  auto bar_acc_full = [&](int b) { return base + L::off_bar + 8u * (2 * S + 2 + b); };
  auto bar_acc_empty = [&](int b) { return base + L::off_bar + 8u * (2 * S + 4 + b); };
  const uint32_t bar_drain = base + L::off_bar + 8u * (2 * S + 6);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::off_misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 4);
  const uint32_t stages_addr = base + L::off_misc + 8;  // stages whose operands are ready
  const uint32_t items_addr = base + L::off_misc + 12;  // work items whose accumulator is free
  const uint32_t tails_addr = base + L::off_misc + 16;  // ragged steps whose operands are ready
  int32_t* first = reinterpret_cast<int32_t*>(smem + L::off_table);
  uint16_t* blocks = reinterpret_cast<uint16_t*>(first + p.G + 1);
  uint8_t* valid = reinterpret_cast<uint8_t*>(blocks + p.m_blocks);  // of each 128-row block

  if (tid == 0) {
    *abort_flag = 0;
    *reinterpret_cast<volatile uint32_t*>(smem + L::off_misc + 8) = 0;
    *reinterpret_cast<volatile uint32_t*>(smem + L::off_misc + 12) = 0;
    *reinterpret_cast<volatile uint32_t*>(smem + L::off_misc + 16) = 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_ready(s), CL);  // the producer of each block
      mbar_init(bar_empty(s), 1);
    }
    mbar_init(bar_tail_ready, CL);  // warp 6 of each block
    mbar_init(bar_tail_empty, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), kEpi * CL);
    }
    mbar_init(bar_drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tm_dy);
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_d);
  }

  // Table: the 128-row blocks of every group in ascending order (counting sort, stable).
  {
    int16_t* of_block = reinterpret_cast<int16_t*>(smem + L::off_stage);
    for (int g = tid; g <= p.G; g += kThreads) first[g] = 0;
    __syncthreads();
    bool bad = false;
#pragma unroll 4
    for (int b = warp; b < p.m_blocks; b += kThreads / 32) {
      int m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = b * 128 + 32 * i + lane;
        m[i] = row < p.M ? __ldg(p.m_indices + row) : -1;
      }
      const int e = __shfl_sync(0xffffffffu, m[0], 0);
      uint32_t in_group[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) in_group[i] = __ballot_sync(0xffffffffu, p.whole_blocks ? m[i] >= 0 : m[i] == e);
      if (lane == 0) {
        const bool in = e >= 0 && e < p.G;
        bad |= e >= p.G;
        // rows 0 .. n - 1 and no others?
        const int n = __popc(in_group[0]) + __popc(in_group[1]) + __popc(in_group[2]) + __popc(in_group[3]);
        bool prefix = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int here = max(0, min(32, n - 32 * i));
          prefix &= in_group[i] == (here == 32 ? 0xffffffffu : (1u << here) - 1u);
        }
        of_block[b] = static_cast<int16_t>(in ? e : -1);
        valid[b] = static_cast<uint8_t>(prefix ? n : kWgIrregular);
        if (in) atomicAdd(&first[e], 1);
      }
    }
    if (bad && blockIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, DG_DEV_OK, DG_DEV_BAD_GROUP_INDEX);
    __syncthreads();
    if (warp == 0) {
      int running = 0;
      for (int g0 = 0; g0 < p.G; g0 += 32) {
        const int g = g0 + lane;
        const int v = g < p.G ? first[g] : 0;
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (g < p.G) first[g] = running + x - v;
        running += __shfl_sync(0xffffffffu, x, 31);
      }
      __syncwarp();
      // place the blocks; first[g] walks to the group's end and is the next group's beginning after
      for (int b0 = 0; b0 < p.m_blocks; b0 += 32) {
        const int b = b0 + lane;
        const int e = b < p.m_blocks ? of_block[b] : -1;
        const unsigned same = __match_any_sync(0xffffffffu, e);
        const int r = __popc(same & ((1u << lane) - 1u));
        int at = 0;
        if (e >= 0) at = first[e] + r;
        __syncwarp();
        if (e >= 0) {
          blocks[at] = static_cast<uint16_t>(b);
          if (r == 0) first[e] += __popc(same);
        }
        __syncwarp();
      }
    }
  }
  if (warp == 1) {
    if constexpr (CL == 2) {
      tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish();
    }
  }
  // the ring held the table's source: those reads are done before any copy lands there
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CL == 2) cluster_sync_all();
  tc_fence_after_sync();

  const uint32_t tmem_base = *tmem_slot;
  const int tiles = p.n_tiles * p.k_tiles;
  const int n_items = p.G * tiles;
  struct Item {
    int g, n0, k0, b0, blocks;  // blocks[b0 .. b0 + blocks) are the group's
  };
  auto item_of = [&](int item) {
    Item it;
    it.g = item / tiles;
    const int t = item - it.g * tiles;
    const int nt = t / p.k_tiles;
    it.n0 = nt * BT;
    it.k0 = (t - nt * p.k_tiles) * BT;
    it.b0 = it.g > 0 ? first[it.g - 1] : 0;
    it.blocks = first[it.g] - it.b0;
    if constexpr (kSplit) {  // this block's share of them
      const int lo = it.blocks * part / p.split, hi = it.blocks * (part + 1) / p.split;
      it.b0 += lo;
      it.blocks = hi - lo;
    }
    return it;
  };

  // An item's blocks in segments (a group without rows is one empty segment).
  auto segments = [&](const Item& w) { return kSegments && w.blocks > p.segment ? (w.blocks + p.segment - 1) / p.segment : 1; };
  auto segment = [&](const Item& whole, int i, int of) {
    if (!kSegments || of == 1) return whole;
    Item w = whole;
    const int lo = whole.blocks * i / of;
    w.b0 += lo;
    w.blocks = whole.blocks * (i + 1) / of - lo;
    return w;
  };

  // A block whose table entry is n: steps of 16 rows of its first and second 64 rows that come from
  // the ring, and ragged steps behind them (all eight steps of an irregular block).
  auto ring_steps = [&](int n, int half) { return n == kWgIrregular ? 0 : max(0, min(4, n / 16 - 4 * half)); };
  auto ragged_steps = [&](int n) { return n == kWgIrregular ? 8 : (n % 16 != 0 ? 1 : 0); };

  if (warp == 0) {
    if (lane == 0) {
      // ---- TMA producer
      const uint64_t pol = l2_policy_evict_last();  // the rows of a group are read by all of its tiles
      uint32_t it = 0;
      bool ok = true;
      for (int item = unit; ok && item < n_items; item += units) {
        const Item w = item_of(item);  // (segments follow one another: nothing to do for them here)
        const int n = w.n0 + static_cast<int>(rank) * 128, k = w.k0 + static_cast<int>(rank) * 128;
        for (int i = 0; ok && i < w.blocks; ++i) {
          const int b = blocks[w.b0 + i];
          const int count = valid[b];
          for (int half = 0; half < 2; ++half) {
            if (ring_steps(count, half) == 0) break;
            const int s = it % S;
            if (!mbar_wait_bounded(bar_empty(s), ((it / S) & 1u) ^ 1u, abort_flag, WG_SITE_EMPTY)) {
              ok = false;
              break;
            }
            ++it;
            const int row = b * 128 + half * 64;
            const uint32_t dst = base + L::off_stage + s * kWgStageBytes;
            // 64 rows x 128 columns of an operand are one box (two blocks of 64 columns): with a box
            // for each block the copies alone took 1.27 ms instead of 1.06 (32 groups of 1024 rows,
            // 4096 x 7168), the whole kernel 1.50 instead of 1.42.
            if constexpr (CL == 2) {
              // the copies of both blocks complete on the leader's barrier
              const uint32_t bar = mapa_shared(bar_ready(s), 0);
              if (rank == 0) mbar_arrive_expect_tx(bar_ready(s), 2 * kWgStageBytes); else wg_arrive_remote_relaxed(bar);
              if (p.dy_blocks) {
                tma_load_3d_pair(dst, &tm_dy, bar, 0, row, n / 64, pol);
              } else {
                tma_load_2d_pair(dst, &tm_dy, bar, n, row, pol);
                tma_load_2d_pair(dst + kWgBoxBytes, &tm_dy, bar, n + 64, row, pol);
              }
              tma_load_3d_pair(dst + kWgOperand, &tm_x, bar, 0, row, k / 64, pol);
            } else {
              mbar_arrive_expect_tx(bar_ready(s), kWgStageBytes);
              if (p.dy_blocks) {
                tma_load_3d(dst, &tm_dy, bar_ready(s), 0, row, n / 64, pol);
              } else {
                tma_load_2d(dst, &tm_dy, bar_ready(s), n, row, pol);
                tma_load_2d(dst + kWgBoxBytes, &tm_dy, bar_ready(s), n + 64, row, pol);
              }
              tma_load_3d(dst + kWgOperand, &tm_x, bar_ready(s), 0, row, k / 64, pol);
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ---- UMMA issuer.  It touches no barrier and looks a block of rows ahead in the table.
      uint32_t it = 0, tile = 0, tail = 0, stages_known = 0, items_known = 0, tails_known = 0;
      bool ok = true;
      for (int item = unit; ok && item < n_items; item += units) {
        const Item whole = item_of(item);
        if (whole.blocks == 0) continue;
        const int segs = segments(whole);
        for (int sg = 0; ok && sg < segs; ++sg) {
          const Item w = segment(whole, sg, segs);
          const uint32_t buf = tile & 1u;
          int n_next = valid[blocks[w.b0]];
          if (items_known <= tile && (items_known = poll_above(items_addr, tile, abort_flag, WG_SITE_ACC_EMPTY)) == 0) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + buf * BT;
          uint32_t acc = 0;  // the first product of a segment overwrites
          auto step = [&](uint64_t a_desc, uint64_t b_desc) {
            if constexpr (CL == 2)
              umma_ss_pair<UMMA_F16>(d_tmem, a_desc, b_desc, kIdesc, acc);
            else
              umma_ss<UMMA_F16>(d_tmem, a_desc, b_desc, kIdesc, acc);
            acc = 1;
          };
          auto commit = [&](uint32_t bar) {
            if constexpr (CL == 2) umma_commit_pair(bar, 3); else umma_commit(bar);
          };
          for (int i = 0; ok && i < w.blocks; ++i) {
            const int n = n_next;
            if (i + 1 < w.blocks) n_next = valid[blocks[w.b0 + i + 1]];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int steps = ring_steps(n, half);
              if (steps == 0) break;
              const int s = it % S;
              if (stages_known <= it) {
                if ((stages_known = poll_above(stages_addr, it, abort_flag, WG_SITE_READY)) == 0) {
                  ok = false;
                  break;
                }
                tc_fence_after_sync();
              }
              ++it;
              const uint32_t at = base + L::off_stage + s * kWgStageBytes;
              const uint64_t a_desc = umma_desc_mn_sw128(at, kWgBoxBytes);
              const uint64_t b_desc = umma_desc_mn_sw128(at + kWgOperand, kWgBoxBytes);
              if (steps == 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) step(a_desc + 128u * k, b_desc + 128u * k);  // 2048 bytes on in every box
              } else {
                for (int k = 0; k < steps; ++k) step(a_desc + 128u * k, b_desc + 128u * k);
              }
              commit(bar_empty(s));
            }
            for (int r = ragged_steps(n); ok && r > 0; --r) {
              if (tails_known <= tail) {
                if ((tails_known = poll_above(tails_addr, tail, abort_flag, WG_SITE_TAIL_READY)) == 0) {
                  ok = false;
                  break;
                }
                tc_fence_after_sync();
              }
              ++tail;
              const uint32_t at = base + L::off_tail;
              step(umma_desc_mn_sw128(at, kWgTailBox), umma_desc_mn_sw128(at + 2 * kWgTailBox, kWgTailBox));
              commit(bar_tail_empty);
            }
          }
          if (ok) commit(bar_acc_full(buf));
          ++tile;
        }
      }
      if (*abort_flag) {
        int local_abort = 0;
        if constexpr (CL == 2) umma_commit_pair(bar_drain, 1); else umma_commit(bar_drain);
        mbar_wait_bounded(bar_drain, 0, &local_abort, 0);
      }
    }
  } else if (warp == 7) {
    if (lane == 0 && rank == 0) {
      // ---- watcher
      uint32_t it = 0, tile = 0, tail = 0;
      bool ok = true;
      for (int item = unit; ok && item < n_items; item += units) {
        const Item whole = item_of(item);
        if (whole.blocks == 0) continue;
        const int segs = segments(whole);
        for (int sg = 0; ok && sg < segs; ++sg) {
          const Item w = segment(whole, sg, segs);
          if (!mbar_wait_bounded(bar_acc_empty(tile & 1u), ((tile >> 1) & 1u) ^ 1u, abort_flag, WG_SITE_ACC_EMPTY)) {
            ok = false;
            break;
          }
          post_count(items_addr, ++tile);
          for (int i = 0; ok && i < w.blocks; ++i) {
            const int n = valid[blocks[w.b0 + i]];
            for (int half = 0; half < 2; ++half) {
              if (ring_steps(n, half) == 0) break;
              if (!mbar_wait_bounded(bar_ready(it % S), (it / S) & 1u, abort_flag, WG_SITE_READY)) {
                ok = false;
                break;
              }
              post_count(stages_addr, ++it);
            }
            for (int r = ragged_steps(n); ok && r > 0; --r) {
              if (!mbar_wait_bounded(bar_tail_ready, tail & 1u, abort_flag, WG_SITE_TAIL_READY)) {
                ok = false;
                break;
              }
              if constexpr (CL == 2) wg_fence_cluster();  // the other block's stores
              post_count(tails_addr, ++tail);
            }
          }
        }
      }
    }
  } else if (warp == 6) {
    // ---- ragged steps: 16 rows x 128 columns of both operands through registers, fetched before the
    // buffer is free.  Lane l takes the 16-byte piece l % 16 (64-column block (l % 16) / 8) of rows
    // l / 16, l / 16 + 2, ...
    const int piece = lane & 15, rsub = lane >> 4;
    uint32_t tail = 0;
    bool ok = true;
    for (int item = unit; ok && item < n_items; item += units) {
      const Item w = item_of(item);
      const int cn = w.n0 + static_cast<int>(rank) * 128 + piece * 8;
      const int ck = w.k0 + static_cast<int>(rank) * 128 + piece * 8;
      for (int i = 0; ok && i < w.blocks; ++i) {
        const int b = blocks[w.b0 + i];
        const int n = valid[b];
        const int count = ragged_steps(n);
        for (int r = 0; ok && r < count; ++r, ++tail) {
          const int row0 = b * 128 + 16 * (n == kWgIrregular ? r : n / 16);
          uint32_t rows = (1u << (n & 15)) - 1u;  // rows of the step that count
          if (n == kWgIrregular) {
            const int row = row0 + lane;
            const int e = lane < 16 && row < p.M ? __ldg(p.m_indices + row) : -1;
            rows = __ballot_sync(0xffffffffu, p.whole_blocks ? e >= 0 : e == w.g);
          }
          uint4 dy[8], x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int rr = rsub + 2 * j;
            const size_t row = static_cast<size_t>(row0 + rr);
            const bool in = (rows >> rr) & 1u;
            dy[j] = x[j] = make_uint4(0u, 0u, 0u, 0u);
            if (in && cn < p.N) dy[j] = __ldg(reinterpret_cast<const uint4*>(p.dy + row * p.N + cn));
            if (in && ck < p.K) x[j] = __ldg(reinterpret_cast<const uint4*>(p.x + row * p.K + ck));
          }
          if (!mbar_wait_warp(bar_tail_empty, (tail & 1u) ^ 1u, abort_flag, WG_SITE_TAIL_EMPTY)) {
            ok = false;
            break;
          }
          uint8_t* at = smem + L::off_tail + (piece >> 3) * kWgTailBox;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int rr = rsub + 2 * j;
            const int off = rr * 128 + (((piece & 7) ^ (rr & 7)) << 4);
            *reinterpret_cast<uint4*>(at + off) = dy[j];
            *reinterpret_cast<uint4*>(at + 2 * kWgTailBox + off) = x[j];
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CL == 2) mbar_arrive_remote(mapa_shared(bar_tail_ready, 0)); else mbar_arrive(bar_tail_ready);
          }
        }
      }
    }
  } else {
    // ---- epilogue: rows n0 + 128 rank + 32 q .. + 31 of the tile; kWide: warps 2..5 the first half of its
    // columns, 8..11 the second
    constexpr int kCols = kWide ? BT / 2 : BT;
    const int q = warp & 3, half = kWide ? warp >> 3 : 0;
    const uint32_t strip = base + L::off_strip + (half * 4 + q) * 4096;
    uint8_t* strip_p = smem + L::off_strip + (half * 4 + q) * 4096;
    const uint32_t acc_empty[2] = {CL == 2 ? mapa_shared(bar_acc_empty(0), 0) : bar_acc_empty(0),
                                   CL == 2 ? mapa_shared(bar_acc_empty(1), 0) : bar_acc_empty(1)};
    const int kb_all = p.K / 64;
    uint32_t tile = 0;
    // 128 bytes of this lane's row, 16 at a time, where the 128-byte swizzle puts them
    auto put = [&](int piece, uint4 v) {
      *reinterpret_cast<uint4*>(strip_p + lane * 128 + ((piece ^ (lane & 7)) << 4)) = v;
    };
    auto before = [&]() {  // the strip's last store has read it
      if (lane == 0) wg_store_wait_read();
      __syncwarp();
    };
    auto after = [&](int x, int n, int z) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (p.add) wg_add_3d(&tm_d, strip, x, n, z); else wg_store_3d(&tm_d, strip, x, n, z);
        wg_store_commit();
      }
    };
    auto release = [&](uint32_t buf) {  // the accumulator's columns are in registers
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CL == 2) mbar_arrive_remote(acc_empty[buf]); else mbar_arrive(acc_empty[buf]);
      }
    };
    for (int item = unit; item < n_items; item += units) {
      const Item w = item_of(item);
      const int n = w.n0 + static_cast<int>(rank) * 128 + q * 32;
      const int kb0 = w.k0 / 64 + half * (kCols / 64);
      const int kbs = n < p.N ? max(0, min(kCols / 64, kb_all - kb0)) : 0;  // 64-column blocks to store
      if constexpr (kSplit) {
        // this block's partial tile: a lane's row of it in registers over the segments, then in shared
        // memory, row r at 512 r, 16-byte pieces swizzled with the row
        float sum[128];
#pragma unroll
        for (int i = 0; i < 128; ++i) sum[i] = 0.0f;
        const int segs = w.blocks > 0 ? segments(w) : 0;
        bool ok = true;
        for (int sg = 0; sg < segs; ++sg, ++tile) {
          const uint32_t buf = tile & 1u;
          if (!mbar_wait_warp(bar_acc_full(buf), (tile >> 1) & 1u, abort_flag, WG_SITE_ACC_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            uint32_t v[32];
            tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BT + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[c + i] += __uint_as_float(v[i]);
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty[buf]);
        }
        if (ok) {  // every copy and product is done: the ring is free
          const int r = q * 32 + lane;
          float* row = reinterpret_cast<float*>(smem + L::off_stage + r * 512);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            *reinterpret_cast<float4*>(row + 4 * (i ^ (r & 7))) = make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
        }
        break;  // one tile for a cluster
      }
      if (w.blocks == 0) {
        if (!p.add && kbs > 0) {
          before();
#pragma unroll
          for (int i = 0; i < 8; ++i) put(i, make_uint4(0u, 0u, 0u, 0u));
          for (int b = 0; b < kbs; ++b)
            for (int x = 0; x < 64; x += p.f32 ? 32 : 64) after(x, n, w.g * kb_all + kb0 + b);
        }
        continue;
      }
      if constexpr (kWide) {
        // this lane's row of the half tile, summed over the segments in registers
        float sum[kCols];
        const int segs = segments(w);
        bool ok = true;
        for (int sg = 0; sg < segs; ++sg, ++tile) {
          const uint32_t buf = tile & 1u;
          if (!mbar_wait_warp(bar_acc_full(buf), (tile >> 1) & 1u, abort_flag, WG_SITE_ACC_FULL)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BT + half * kCols;
#pragma unroll
          for (int c = 0; c < kCols; c += 16) {
            uint32_t v[16];
            tmem_ld_32x16(t_row + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[c + i] = sg == 0 ? __uint_as_float(v[i]) : sum[c + i] + __uint_as_float(v[i]);
          }
          release(buf);
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          if (c / 64 >= kbs) continue;
          before();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            put(i, make_uint4(__float_as_uint(sum[c + 4 * i]), __float_as_uint(sum[c + 4 * i + 1]), __float_as_uint(sum[c + 4 * i + 2]),
                              __float_as_uint(sum[c + 4 * i + 3])));
          after(c % 64, n, w.g * kb_all + kb0 + c / 64);
        }
      } else if constexpr (!kSplit) {
        const uint32_t buf = tile & 1u;
        if (!mbar_wait_warp(bar_acc_full(buf), (tile >> 1) & 1u, abort_flag, WG_SITE_ACC_FULL)) break;
        tc_fence_after_sync();
        const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BT;
        for (int b = 0; b < kbs; ++b) {
          uint32_t r0[32], r1[32];
          tmem_ld_32x32(t_row + b * 64, r0);
          tmem_ld_32x32(t_row + b * 64 + 32, r1);
          tmem_ld_wait();
          auto two = [](uint32_t a, uint32_t b2) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(a), __uint_as_float(b2));
            return *reinterpret_cast<const uint32_t*>(&h);
          };
          before();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            put(i, make_uint4(two(r0[8 * i], r0[8 * i + 1]), two(r0[8 * i + 2], r0[8 * i + 3]),
                              two(r0[8 * i + 4], r0[8 * i + 5]), two(r0[8 * i + 6], r0[8 * i + 7])));
            put(4 + i, make_uint4(two(r1[8 * i], r1[8 * i + 1]), two(r1[8 * i + 2], r1[8 * i + 3]),
                                  two(r1[8 * i + 4], r1[8 * i + 5]), two(r1[8 * i + 6], r1[8 * i + 7])));
          }
          after(0, n, w.g * kb_all + kb0 + b);
        }
        release(buf);
        ++tile;
      }
    }
    if (lane == 0) wg_store_wait();  // the strip lives until its last store is done
  }

  if constexpr (kSplit) {
    // ---- the cluster's partial tiles added up: rows [128 / split * part, ...) of the tile here
    __syncthreads();
    cluster_sync_all();
    if (unit < n_items) {
      const Item w = item_of(unit);
      const int rows = 128 / p.split, r0 = part * rows;
      const int kb_all = p.K / 64;
      for (int i = tid; i < rows * 32; i += kThreads) {
        const int r = r0 + (i >> 5), piece = i & 31;
        const int n = w.n0 + r, k = w.k0 + 4 * piece;
        if (n >= p.N || k >= p.K) continue;
        const uint32_t at = base + L::off_stage + r * 512 + ((piece ^ (r & 7)) << 4);
        float4 s = wg_load_cluster(mapa_shared(at, 0));
        for (int b = 1; b < p.split; ++b) {
          const float4 v = wg_load_cluster(mapa_shared(at, b));
          s.x += v.x;
          s.y += v.y;
          s.z += v.z;
          s.w += v.w;
        }
        const size_t o = ((static_cast<size_t>(w.g) * kb_all + k / 64) * p.N + n) * 64 + k % 64;
        if (p.f32) {
          float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.dw) + o);
          if (p.add) {
            const float4 v = *d;
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
          }
          *d = s;
        } else {
          const __nv_bfloat162 h0 = __floats2bfloat162_rn(s.x, s.y), h1 = __floats2bfloat162_rn(s.z, s.w);
          *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.dw) + o) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
        }
      }
    }
    cluster_sync_all();  // nobody leaves while another block reads its partial tile
  }

  // ---- tear-down
  if (*abort_flag != 0 && tid == 0) {
    const uint64_t t0 = global_timer_ns();  // abnormal exit: copies still in flight get time to land
    while (global_timer_ns() - t0 < 200000ull) {
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CL == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (CL == 2) tmem_dealloc_pair(tmem_base, kTmemCols); else tmem_dealloc(tmem_base, kTmemCols);
  }
  if (tid == 0 && *abort_flag != 0 && p.status != nullptr) {
    if (atomicCAS(p.status, DG_DEV_OK, DG_DEV_WAIT_EXPIRED) == DG_DEV_OK) {
      p.status[1] = blockIdx.x;
      p.status[2] = *abort_flag;
      p.status[3] = n_items;
    }
  }
}

}  // namespace dg
