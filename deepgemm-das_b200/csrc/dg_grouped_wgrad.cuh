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
// Tiles and roles.  CL = 2: a cluster of two blocks computes 256 (n) x 256 (k) with
// tcgen05.mma.cta_group::2, block r owning rows [128 r, 128 r + 128) of the tile (its part of dY, its
// accumulator, its epilogue) and holding 128 of the 256 columns of X.  CL = 1: one block, 128 x 128,
// for problems with few tiles.  Either way a ring stage holds 64 rows of 128 columns of each
// operand (32 KB), six stages.  A work item is (group, tile); its contraction walks the 128-row
// blocks of the group in ascending order, 64 rows (a chunk) at a time.
//   warp 0      TMA producer (each block its own copies)
//   warp 1      UMMA issuer (leader)
//   warps 2..5  epilogue: accumulator -> bf16 or fp32 -> 32-row strip in shared memory -> TMA store
//               (or TMA reduce-add, when the gradient is added to what is there)
//   warp 6      row filter.  Rows that stand for nothing (padding, rows behind the last group) are
//               set to zero in shared memory, in both operands, so that whatever they held (NaN,
//               infinities) does not reach a sum; of a chunk's four 16-row steps only those up to
//               its last row are issued, and a block's second chunk is left out when it is empty.
//   warp 7      watcher (leader): waits on the barriers in the UMMA issuer's place and posts counts in
//               plain shared-memory words.  The issuer has 512 cycles for a chunk (four instructions
//               of 256 x 256 x 16); a first look at a barrier alone takes 200 of them.
// A chunk whose 64 rows all count, i.e. nearly every one, goes straight to the tensor cores: the
// copies of both blocks complete on the leader's `ready` barrier.  Only the others complete on their
// own block's `full` barrier, for the filter, which then arrives on `ready` in the producers' place.
// (With the filter between every chunk and its products, each stage paid a remote arrival with
// cluster-wide release and an acquire to match: 1.0 us a chunk, whatever the tensor cores did.)
// Which rows count is known beforehand: every block of the grid reads all of m_indices once (from
// L2) and keeps a byte for each 128 rows.
// Groups without rows give zeros (or, added, nothing) and cost no products.
//
// Every mbarrier wait is bounded, as in the other kernels.
#pragma once

#include "deepgemm_b200.h"
#include "dg_ptx.cuh"
#include <cuda_bf16.h>

namespace dg {

constexpr int kWgStages = 6;
constexpr int kWgThreads = 256;
constexpr uint32_t kWgBoxBytes = 64 * 128;         // 64 columns x 64 rows
constexpr uint32_t kWgOperand = 2 * kWgBoxBytes;   // 128 columns x 64 rows
constexpr uint32_t kWgStageBytes = 2 * kWgOperand;

constexpr int kWgIrregular = 255;  // rows that count lie between others: looked up where they are used

enum : int { WG_SITE_EMPTY = 21, WG_SITE_FILTER = 22, WG_SITE_READY = 23, WG_SITE_ACC_EMPTY = 24, WG_SITE_ACC_FULL = 25 };

struct WgradParams {
  int G, M, N, K;
  int n_tiles, k_tiles;      // tiles of a group
  int m_blocks;              // ceil(M / 128)
  const int32_t* m_indices;
  int32_t* status;
  int f32;                   // output type: fp32 (else bf16)
  int add;                   // fp32 only: add to what the output holds
  int dy_blocks;             // N % 64 == 0: dy's map counts 64-column blocks, as x's always does
};

struct WgradSmem {
  static constexpr int off_stage = 0;
  static constexpr int off_strip = off_stage + kWgStages * kWgStageBytes;  // 4 KB for each epilogue warp
  // full[S], ready[S], empty[S], acc_full[2], acc_empty[2], drain
  static constexpr int kNumBars = 3 * kWgStages + 5;
  static constexpr int off_bar = off_strip + 4 * 4096;
  static constexpr int off_misc = off_bar + kNumBars * 8;  // tmem slot, abort, stages ready, items ready
  static constexpr int off_steps = off_misc + 16;          // per stage: 16-row steps to issue
  static constexpr int off_table = off_steps + kWgStages * 4;
  // table: first[G + 1] (int32), the groups' 128-row blocks in order (uint16), rows that count (uint8)
  __host__ __device__ static constexpr int total(int groups, int blocks) {
    return off_table + (groups + 1) * 4 + blocks * 3 + 16 + 1024;
  }
  // The table is built from m_indices[128 b] of every block b, held as int16 in the (still empty) ring.
  static_assert(kWgStages * static_cast<int>(kWgStageBytes) >= DG_MAX_CONTIG_ROWS / 128 * 2, "");
};

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

template <int CL>
__global__ void __launch_bounds__(kWgThreads, 1)
grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_x,
                     const __grid_constant__ CUtensorMap tm_d, const WgradParams p) {
  using L = WgradSmem;
  constexpr int S = kWgStages;
  constexpr int BT = 128 * CL;  // tile edge
  constexpr uint32_t kIdesc = umma_idesc(1u, 1u, BT, BT) | kIdescAMn | kIdescBMn;
  constexpr int kTmemCols = 2 * BT;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = CL == 2 ? cluster_ctarank() : 0u;
  const int unit = blockIdx.x / CL, units = gridDim.x / CL;

  auto bar_full = [&](int s) { return base + L::off_bar + 8u * s; };
  auto bar_ready = [&](int s) { return base + L::off_bar + 8u * (S + s); };
  auto bar_empty = [&](int s) { return base + L::off_bar + 8u * (2 * S + s); };
  auto bar_acc_full = [&](int b) { return base + L::off_bar + 8u * (3 * S + b); };
  auto bar_acc_empty = [&](int b) { return base + L::off_bar + 8u * (3 * S + 2 + b); };
  const uint32_t bar_drain = base + L::off_bar + 8u * (3 * S + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::off_misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::off_misc + 4);
  const uint32_t stages_addr = base + L::off_misc + 8;  // stages whose operands are ready
  const uint32_t items_addr = base + L::off_misc + 12;  // work items whose accumulator is free
  volatile int* steps_s = reinterpret_cast<volatile int*>(smem + L::off_steps);
  int32_t* first = reinterpret_cast<int32_t*>(smem + L::off_table);
  uint16_t* blocks = reinterpret_cast<uint16_t*>(first + p.G + 1);
  uint8_t* valid = reinterpret_cast<uint8_t*>(blocks + p.m_blocks);  // of each 128-row block

  if (tid == 0) {
    *abort_flag = 0;
    *reinterpret_cast<volatile uint32_t*>(smem + L::off_misc + 8) = 0;
    *reinterpret_cast<volatile uint32_t*>(smem + L::off_misc + 12) = 0;
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_ready(s), CL);  // the producer of each block, or its filter
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), 4 * CL);
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
    for (int g = tid; g <= p.G; g += kWgThreads) first[g] = 0;
    __syncthreads();
    bool bad = false;
#pragma unroll 4
    for (int b = warp; b < p.m_blocks; b += kWgThreads / 32) {
      int m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = b * 128 + 32 * i + lane;
        m[i] = row < p.M ? __ldg(p.m_indices + row) : -1;
      }
      const int e = __shfl_sync(0xffffffffu, m[0], 0);
      uint32_t in_group[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) in_group[i] = __ballot_sync(0xffffffffu, m[i] == e);
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
    int g, n0, k0, b0, chunks;
  };
  auto item_of = [&](int item) {
    Item it;
    it.g = item / tiles;
    const int t = item - it.g * tiles;
    const int nt = t / p.k_tiles;
    it.n0 = nt * BT;
    it.k0 = (t - nt * p.k_tiles) * BT;
    it.b0 = it.g > 0 ? first[it.g - 1] : 0;
    it.chunks = 2 * (first[it.g] - it.b0);
    return it;
  };

  // Rows that count in half c & 1 of a block with the table's entry n: 0 (left out), 1..63, 64, or
  // kWgIrregular.
  auto rows_of = [&](int n, int c) { return n == kWgIrregular ? n : max(0, min(64, n - 64 * (c & 1))); };

  if (warp == 0) {
    if (lane == 0) {
      // ---- TMA producer
      const uint64_t pol = l2_policy_evict_last();  // the rows of a group are read by all of its tiles
      uint32_t it = 0;
      bool ok = true;
      for (int item = unit; ok && item < n_items; item += units) {
        const Item w = item_of(item);
        for (int c = 0; c < w.chunks; ++c) {
          const int b = blocks[w.b0 + (c >> 1)];
          const int rows = rows_of(valid[b], c);
          if (rows == 0) continue;
          const int s = it % S;
          if (!mbar_wait_bounded(bar_empty(s), ((it / S) & 1u) ^ 1u, abort_flag, WG_SITE_EMPTY)) {
            ok = false;
            break;
          }
          ++it;
          const int row = b * 128 + (c & 1) * 64;
          const uint32_t dst = base + L::off_stage + s * kWgStageBytes;
          const int n = w.n0 + static_cast<int>(rank) * 128, k = w.k0 + static_cast<int>(rank) * 128;
          // 64 rows x 128 columns of an operand are one box (two blocks of 64 columns): with a box for
          // each block the copies alone took 1.27 ms instead of 1.06 (32 groups of 1024 rows, 4096 x
          // 7168), the whole kernel 1.50 instead of 1.42.
          if (CL == 2 && rows == 64) {
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
            const uint32_t bar = rows == 64 ? bar_ready(s) : bar_full(s);
            mbar_arrive_expect_tx(bar, kWgStageBytes);
            if (p.dy_blocks) {
              tma_load_3d(dst, &tm_dy, bar, 0, row, n / 64, pol);
            } else {
              tma_load_2d(dst, &tm_dy, bar, n, row, pol);
              tma_load_2d(dst + kWgBoxBytes, &tm_dy, bar, n + 64, row, pol);
            }
            tma_load_3d(dst + kWgOperand, &tm_x, bar, 0, row, k / 64, pol);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ---- UMMA issuer.  It touches no barrier and looks a block of rows ahead in the table.
      auto poll_above = [&](uint32_t addr, uint32_t have, int site) -> uint32_t {
        uint32_t v;
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          asm volatile("ld.volatile.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
          if (v > have) return v;
        }
        const uint64_t t0 = global_timer_ns();
        uint32_t spins = 0;
        while (true) {
          asm volatile("ld.volatile.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
          if (v > have) return v;
          if ((++spins & 63u) == 0 && (*abort_flag || global_timer_ns() - t0 > 1500000000ull)) {
            if (!*abort_flag) *abort_flag = site;
            return 0;
          }
        }
      };
      uint32_t it = 0, tile = 0, stages_known = 0, items_known = 0;
      bool ok = true;
      for (int item = unit; ok && item < n_items; item += units) {
        const Item w = item_of(item);
        if (w.chunks == 0) continue;
        const uint32_t buf = tile & 1u;
        int n_next = valid[blocks[w.b0]];
        if (items_known <= tile && (items_known = poll_above(items_addr, tile, WG_SITE_ACC_EMPTY)) == 0) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + buf * BT;
        uint32_t acc = 0;
        for (int i = 0; ok && 2 * i < w.chunks; ++i) {
          const int n = n_next;
          if (2 * (i + 1) < w.chunks) n_next = valid[blocks[w.b0 + i + 1]];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int rows = rows_of(n, half);
            if (rows == 0) continue;
            const int s = it % S;
            if (stages_known <= it) {
              if ((stages_known = poll_above(stages_addr, it, WG_SITE_READY)) == 0) {
                ok = false;
                break;
              }
              tc_fence_after_sync();
            }
            ++it;
            const uint32_t at = base + L::off_stage + s * kWgStageBytes;
            const uint64_t a_desc = umma_desc_mn_sw128(at, kWgBoxBytes);
            const uint64_t b_desc = umma_desc_mn_sw128(at + kWgOperand, kWgBoxBytes);
            auto step = [&](int k) {  // 16 rows: 2048 bytes on in every box
              if constexpr (CL == 2)
                umma_ss_pair<UMMA_F16>(d_tmem, a_desc + 128u * k, b_desc + 128u * k, kIdesc, acc);
              else
                umma_ss<UMMA_F16>(d_tmem, a_desc + 128u * k, b_desc + 128u * k, kIdesc, acc);
              acc = 1;
            };
            if (rows == 64) {
#pragma unroll
              for (int k = 0; k < 4; ++k) step(k);
            } else {
              const int steps = rows == kWgIrregular ? steps_s[s] : (rows + 15) / 16;
              for (int k = 0; k < steps; ++k) step(k);
            }
            if constexpr (CL == 2) umma_commit_pair(bar_empty(s), 3); else umma_commit(bar_empty(s));
          }
        }
        if (ok) {
          if constexpr (CL == 2) umma_commit_pair(bar_acc_full(buf), 3); else umma_commit(bar_acc_full(buf));
        }
        ++tile;
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
      uint32_t it = 0, tile = 0;
      bool ok = true;
      for (int item = unit; ok && item < n_items; item += units) {
        const Item w = item_of(item);
        if (w.chunks == 0) continue;
        if (!mbar_wait_bounded(bar_acc_empty(tile & 1u), ((tile >> 1) & 1u) ^ 1u, abort_flag, WG_SITE_ACC_EMPTY)) break;
        ++tile;
        asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(items_addr), "r"(tile) : "memory");
        for (int c = 0; c < w.chunks; ++c) {
          const int rows = rows_of(valid[blocks[w.b0 + (c >> 1)]], c);
          if (rows == 0) continue;
          if (!mbar_wait_bounded(bar_ready(it % S), (it / S) & 1u, abort_flag, WG_SITE_READY)) {
            ok = false;
            break;
          }
          ++it;
          if (rows != 64) wg_fence_cluster();  // both filters' writes
          asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(stages_addr), "r"(it) : "memory");
        }
      }
    }
  } else if (warp == 6) {
    // ---- row filter
    uint32_t it = 0, phase = 0;  // bit s: parity of the next use of stage s's full barrier
    bool ok = true;
    for (int item = unit; ok && item < n_items; item += units) {
      const Item w = item_of(item);
      for (int c = 0; c < w.chunks; ++c) {
        const int b = blocks[w.b0 + (c >> 1)];
        int rows = rows_of(valid[b], c);
        if (rows == 0) continue;
        const int s = it % S;
        ++it;
        if (rows == 64) continue;
        uint32_t lo, hi;  // rows of the chunk that count
        if (rows == kWgIrregular) {
          const int row = b * 128 + (c & 1) * 64 + lane;
          lo = __ballot_sync(0xffffffffu, (row < p.M ? __ldg(p.m_indices + row) : -1) == w.g);
          hi = __ballot_sync(0xffffffffu, (row + 32 < p.M ? __ldg(p.m_indices + row + 32) : -1) == w.g);
          rows = hi ? 64 - __clz(hi) : 32 - __clz(lo);
        } else {
          lo = rows >= 32 ? 0xffffffffu : (1u << rows) - 1u;
          hi = rows > 32 ? (1u << (rows - 32)) - 1u : 0u;
        }
        // steps of 16 rows; at least one, so that every stage has an instruction for its commit to follow
        const int steps = max(1, (rows + 15) / 16);
        if (!mbar_wait_warp(bar_full(s), (phase >> s) & 1u, abort_flag, WG_SITE_FILTER)) {
          ok = false;
          break;
        }
        phase ^= 1u << s;
        uint32_t zlo = ~lo, zhi = ~hi;  // rows to clear, of those that are issued
        if (steps < 2) zlo &= 0xffffu;
        if (steps < 3) zhi = 0;
        else if (steps < 4) zhi &= 0xffffu;
        {
          // a row is 128 bytes in each of the four boxes: one 16-byte store of every lane
          uint8_t* at = smem + L::off_stage + s * kWgStageBytes + (lane >> 3) * kWgBoxBytes + (lane & 7) * 16;
          while (zlo) {
            const int r = __ffs(zlo) - 1;
            zlo &= zlo - 1;
            *reinterpret_cast<uint4*>(at + r * 128) = make_uint4(0u, 0u, 0u, 0u);
          }
          while (zhi) {
            const int r = __ffs(zhi) - 1;
            zhi &= zhi - 1;
            *reinterpret_cast<uint4*>(at + (32 + r) * 128) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) {
          if (rank == 0) steps_s[s] = steps;
          if constexpr (CL == 2)
            mbar_arrive_remote(mapa_shared(bar_ready(s), 0));
          else
            mbar_arrive(bar_ready(s));
        }
      }
    }
  } else {
    // ---- epilogue: rows n0 + 128 rank + 32 q .. + 31 of the tile
    const int q = warp & 3;
    const uint32_t strip = base + L::off_strip + q * 4096;
    uint8_t* strip_p = smem + L::off_strip + q * 4096;
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
    for (int item = unit; item < n_items; item += units) {
      const Item w = item_of(item);
      const int n = w.n0 + static_cast<int>(rank) * 128 + q * 32;
      const int kb0 = w.k0 / 64;
      const int kbs = n < p.N ? min(BT / 64, kb_all - kb0) : 0;  // 64-column blocks to store
      if (w.chunks == 0) {
        if (!p.add && kbs > 0) {
          before();
#pragma unroll
          for (int i = 0; i < 8; ++i) put(i, make_uint4(0u, 0u, 0u, 0u));
          for (int b = 0; b < kbs; ++b)
            for (int x = 0; x < 64; x += p.f32 ? 32 : 64) after(x, n, w.g * kb_all + kb0 + b);
        }
        continue;
      }
      const uint32_t buf = tile & 1u;
      if (!mbar_wait_warp(bar_acc_full(buf), (tile >> 1) & 1u, abort_flag, WG_SITE_ACC_FULL)) break;
      tc_fence_after_sync();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * BT;
      for (int b = 0; b < kbs; ++b) {
        uint32_t r0[32], r1[32];
        tmem_ld_32x32(t_row + b * 64, r0);
        tmem_ld_32x32(t_row + b * 64 + 32, r1);
        tmem_ld_wait();
        const int z = w.g * kb_all + kb0 + b;
        if (p.f32) {
          before();
#pragma unroll
          for (int i = 0; i < 8; ++i) put(i, make_uint4(r0[4 * i], r0[4 * i + 1], r0[4 * i + 2], r0[4 * i + 3]));
          after(0, n, z);
          before();
#pragma unroll
          for (int i = 0; i < 8; ++i) put(i, make_uint4(r1[4 * i], r1[4 * i + 1], r1[4 * i + 2], r1[4 * i + 3]));
          after(32, n, z);
        } else {
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
          after(0, n, z);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CL == 2) mbar_arrive_remote(acc_empty[buf]); else mbar_arrive(acc_empty[buf]);
      }
      ++tile;
    }
    if (lane == 0) wg_store_wait();  // the strip lives until its last store is done
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
