// Tokens sorted by expert and back.
//
// A router names top_k experts for each of T tokens; pair p = t * top_k + j.  With
//   count[e]  = #{p : id[p] = e},        offset[e] = sum_{e' < e} roundup(count[e'], align),
//   dest[p]   = offset[id[p]] + #{p' < p : id[p'] = id[p]}
// the sorted layout holds row dest[p] = x[t], m_indices[dest[p]] = id[p], and m_indices = -1 in
// rows that stand for no pair (an expert's padding, everything behind the last expert).  The way
// back and the gradients:
//   out[t]     = sum_j w[t][j] * y[dest[t][j]]
//   dy[dest]   = w[t][j] * dout[t]           dw[t][j] = <dout[t], y[dest[t][j]]>
//   dx[t]      = sum_j drows[dest[t][j]]     (the way back without weights)
// A pair whose id is negative (an expert that lives elsewhere) has dest = -1 and contributes
// nothing; an id >= G is treated the same and reported in the status words.
//
// All of it moves rows and is bound by HBM; sums are held in fp32 in the order j = 0, 1, ..., so
// no result depends on the launch shape, and nothing uses an atomic on a floating-point value.
#pragma once

#include "dg_rows.cuh"

namespace dg {

struct TokenSortParams {
  const void* x;
  const void* ids;      // int32 or int64 [T][top_k]
  int ids64;
  int T, top_k, G, align, cap;
  int row_bytes;        // bytes of a row
  long long x_stride;   // bytes between rows of x
  void* rows;           // [cap] rows
  int32_t* dest;        // [T][top_k]
  int32_t* m_indices;   // [cap]
  int32_t* counts;      // [G]
  int32_t* offsets;     // [G]
  int32_t* m_total;     // [1]
  int32_t* status;
  const int32_t* hist;  // NULL, or [chunks + 1][G]: pairs of each expert before each block's chunk, then totals
  int tokens_per_block;
  int clear;            // write zeros into rows that stand for no pair
  int rep;              // copies of the shared-memory histogram (fewer lanes meet at one address)
};

constexpr int kSortThreads = 1024;
constexpr int kSortMaxChunk = 2048;  // pairs of one block

__device__ __forceinline__ int sort_id(const TokenSortParams& p, long long i) {
  if (p.ids64) {
    const long long v = static_cast<const long long*>(p.ids)[i];
    return v < 0 ? -1 : (v >= p.G ? p.G : static_cast<int>(v));
  }
  const int v = static_cast<const int32_t*>(p.ids)[i];
  return v < 0 ? -1 : (v >= p.G ? p.G : v);
}

// Pairs of each expert in each block's chunk (more pairs than one block should count by itself).
__global__ void __launch_bounds__(kSortThreads) sort_hist_kernel(const TokenSortParams p, int32_t* hist) {
  extern __shared__ int32_t cnt[];
  for (int e = threadIdx.x; e < p.G; e += kSortThreads) cnt[e] = 0;
  __syncthreads();
  const long long p0 = (long long)blockIdx.x * p.tokens_per_block * p.top_k;
  const long long p1 = min(p0 + (long long)p.tokens_per_block * p.top_k, (long long)p.T * p.top_k);
  for (long long i = p0 + threadIdx.x; i < p1; i += kSortThreads) {
    const int e = sort_id(p, i);
    if (e >= 0 && e < p.G) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.G; e += kSortThreads) hist[(size_t)blockIdx.x * p.G + e] = cnt[e];
}

// Running sums over the chunks, one warp per expert; entry [chunks] is the total.
__global__ void __launch_bounds__(256) sort_scan_kernel(int32_t* hist, int chunks, int G) {
  const int e = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (e >= G) return;
  int running = 0;
  for (int c0 = 0; c0 < chunks; c0 += 32) {
    const int c = c0 + lane;
    const int v = c < chunks ? hist[(size_t)c * G + e] : 0;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (c < chunks) hist[(size_t)c * G + e] = running + x - v;
    running += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) hist[(size_t)chunks * G + e] = running;
}

// Values of VB bytes that a lane moves at once, and those of a warp.
__host__ __device__ constexpr int sort_each(int vb) { return vb == 16 ? 4 : (vb == 4 ? 8 : 16); }
__host__ __device__ constexpr int sort_seg(int vb) { return 32 * sort_each(vb); }

template <int VB>
struct BytesOf;
template <>
struct BytesOf<16> { using type = uint4; };
template <>
struct BytesOf<4> { using type = uint32_t; };
template <>
struct BytesOf<2> { using type = uint16_t; };

// Plan and copy in one launch.  Every block counts all pairs itself (their ids stay in L2; where they
// are many, the two kernels above have counted), so no block waits for another; it then places the
// pairs of its own tokens and copies their rows, each read once and written top_k times.  blockIdx.y
// splits the columns of a row when there are few tokens.  Nine tenths of the bytes are written: 4096
// tokens x top-8 x 7168 bf16 in 32 experts padded to 128 rows, 586 MB: 122 us = 4.8 TB/s, 110 us without
// padding.  HBM takes more (a plain fp32 fill of as many bytes writes 7.1 TB/s) and issue slots are 20 %
// busy; with one block of 32 warps on an SM, each reading a piece before it writes it, latency is the
// likely rest, but it was not isolated.  (Streaming stores: 1024 tokens 32 -> 28 us, 4096 x top-4
// 67 -> 63.)
template <int VB>
__global__ void __launch_bounds__(kSortThreads) token_sort_kernel(const TokenSortParams p) {
  using V = typename BytesOf<VB>::type;
  extern __shared__ int32_t sm[];
  int32_t* before = sm;               // [G] pairs of e before this block's (then: placed so far)
  int32_t* count = before + p.G;      // [G]
  int32_t* offset = count + p.G;      // [G + 1]
  int32_t* dest_s = offset + p.G + 1; // [tokens_per_block * top_k]
  int32_t* hist = dest_s + p.tokens_per_block * p.top_k;  // [2][G][rep]
  __shared__ int bad_s, list_n;
  __shared__ int list[kSortThreads];
  __shared__ int warp_sum[32];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long R = (long long)p.T * p.top_k;
  const int t0 = blockIdx.x * p.tokens_per_block;
  const int nt = min(p.tokens_per_block, p.T - t0);
  const long long p0 = (long long)t0 * p.top_k;
  const int np = nt * p.top_k;
  const bool first = blockIdx.y == 0;

  if (tid == 0) bad_s = 0;
  for (int i = tid; i < np; i += kSortThreads) dest_s[i] = sort_id(p, p0 + i);
  if (p.hist == nullptr) {
    for (int i = tid; i < 2 * p.G * p.rep; i += kSortThreads) hist[i] = 0;
    __syncthreads();
    const int mine = lane & (p.rep - 1);
    auto note = [&](int e, long long i) {
      if (e < 0) return;
      if (e >= p.G) {
        bad_s = 1;
        return;
      }
      atomicAdd(&hist[((i < p0 ? 0 : p.G) + e) * p.rep + mine], 1);
    };
    if (!p.ids64 && (reinterpret_cast<uintptr_t>(p.ids) & 15u) == 0) {
      const int4* v = static_cast<const int4*>(p.ids);
      const long long nv = R / 4;
#pragma unroll 4
      for (long long i = tid; i < nv; i += kSortThreads) {
        const int4 q = __ldg(v + i);
        note(min(q.x, p.G), 4 * i);
        note(min(q.y, p.G), 4 * i + 1);
        note(min(q.z, p.G), 4 * i + 2);
        note(min(q.w, p.G), 4 * i + 3);
      }
      for (long long i = 4 * nv + tid; i < R; i += kSortThreads) note(sort_id(p, i), i);
    } else {
#pragma unroll 4
      for (long long i = tid; i < R; i += kSortThreads) note(sort_id(p, i), i);
    }
    __syncthreads();
    for (int e = tid; e < p.G; e += kSortThreads) {
      int b = 0, r = 0;
      for (int c = 0; c < p.rep; ++c) {
        b += hist[e * p.rep + c];
        r += hist[(p.G + e) * p.rep + c];
      }
      before[e] = b;
      count[e] = b + r;
    }
  } else {
    for (int e = tid; e < p.G; e += kSortThreads) {
      before[e] = p.hist[(size_t)blockIdx.x * p.G + e];
      count[e] = p.hist[(size_t)gridDim.x * p.G + e];
    }
    __syncthreads();  // bad_s is zero before the ids below are looked at
    for (int i = tid; i < np; i += kSortThreads)
      if (dest_s[i] >= p.G) bad_s = 1;
  }
  __syncthreads();
  // where the experts begin: a thread for each (G <= 1024 = kSortThreads)
  {
    static_assert(DG_MAX_GROUPS <= kSortThreads, "");
    // (unsigned: pairs + align - 1 may pass 2^31 where no place does)
    const unsigned align = p.align;
    const int v = tid < p.G ? static_cast<int>((static_cast<unsigned>(count[tid]) + align - 1u) / align * align) : 0;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int before_warp = 0;
    if (warp * 32 < p.G)
      for (int w = 0; w < warp; ++w) before_warp += warp_sum[w];
    if (tid < p.G) offset[tid] = before_warp + x - v;
    if (tid == p.G - 1) offset[p.G] = before_warp + x;
    __syncthreads();
  }
  if (warp == 0) {
    // stable places of this block's pairs, 32 at a time
    for (int i0 = 0; i0 < np; i0 += 32) {
      const int i = i0 + lane;
      const int e = i < np ? dest_s[i] : -1;
      const bool in = e >= 0 && e < p.G;
      const unsigned same = __match_any_sync(0xffffffffu, in ? e : -1);
      const int rank = __popc(same & ((1u << lane) - 1u));
      int d = -1;
      if (in) d = offset[e] + before[e] + rank;
      __syncwarp();
      if (in && rank == 0) before[e] += __popc(same);
      __syncwarp();
      if (i < np) {
        dest_s[i] = d;
        if (first) p.dest[p0 + i] = d;
      }
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && first) {
    for (int e = tid; e < p.G; e += kSortThreads) {
      p.counts[e] = count[e];
      p.offsets[e] = offset[e];
    }
    if (tid == 0) *p.m_total = offset[p.G];
  }
  if (tid == 0 && first && bad_s && p.status != nullptr) atomicCAS(p.status, DG_DEV_OK, DG_DEV_BAD_GROUP_INDEX);

  // rows: a warp takes kEach x 32 values of one token at a time
  const int nv = p.row_bytes / VB;
  constexpr int kEach = sort_each(VB), kSeg = sort_seg(VB);
  const int segs_all = (nv + kSeg - 1) / kSeg;
  const int segs_per = (segs_all + gridDim.y - 1) / gridDim.y;
  const int seg0 = blockIdx.y * segs_per, seg1 = min(seg0 + segs_per, segs_all);
  const int segs = max(seg1 - seg0, 0);
  char* rows = static_cast<char*>(p.rows);
  for (int u = warp; u < nt * segs; u += kSortThreads / 32) {
    const int t = u / segs, v0 = (seg0 + u - t * segs) * kSeg + lane;
    const V* src = reinterpret_cast<const V*>(static_cast<const char*>(p.x) + (long long)(t0 + t) * p.x_stride);
    V v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (v0 + 32 * i < nv) v[i] = __ldg(src + v0 + 32 * i);
    for (int j = 0; j < p.top_k; ++j) {
      const int d = dest_s[t * p.top_k + j];
      if (d < 0) continue;
      V* dst = reinterpret_cast<V*>(rows + (size_t)d * p.row_bytes);
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (v0 + 32 * i < nv) __stcs(dst + v0 + 32 * i, v[i]);
    }
  }

  // m_indices: a stretch of rows for each block
  auto expert_of = [&](long long r) {  // -1: the row stands for no pair
    int lo = 0, hi = p.G;  // the last expert that begins at or before r (empty ones begin where the next does)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (offset[mid] <= r) lo = mid; else hi = mid;
    }
    return r < (long long)offset[lo] + count[lo] ? lo : -1;
  };
  if (first) {
    const int per = (p.cap + gridDim.x - 1) / gridDim.x;
    const long long r1 = min((long long)(blockIdx.x + 1) * per, (long long)p.cap);
    for (long long r = (long long)blockIdx.x * per + tid; r < r1; r += kSortThreads) p.m_indices[r] = expert_of(r);
  }
  // zeros in the rows that stand for no pair; most of them lie together, so the blocks take every
  // gridDim.x-th row
  if (p.clear) {
    for (long long rb = 0; rb < p.cap; rb += (long long)gridDim.x * kSortThreads) {
      if (tid == 0) list_n = 0;
      __syncthreads();
      const long long r = rb + (long long)tid * gridDim.x + blockIdx.x;
      if (r < p.cap && expert_of(r) < 0) list[atomicAdd(&list_n, 1)] = static_cast<int>(r);
      __syncthreads();
      const int n = list_n;
      for (int u = warp; u < n * segs; u += kSortThreads / 32) {
        const int i = u / segs, v0 = (seg0 + u - i * segs) * kSeg + lane;
        V* dst = reinterpret_cast<V*>(rows + (size_t)list[i] * p.row_bytes);
#pragma unroll
        for (int k = 0; k < kEach; ++k)
          if (v0 + 32 * k < nv) dst[v0 + 32 * k] = V{};
      }
      __syncthreads();
    }
  }
}

struct TokenUnsortParams {
  const void* y;         // [rows] rows of H values
  const int32_t* dest;   // [T][top_k]
  const float* weights;  // [T][top_k] or NULL
  void* out;             // [T][H]
  int T, top_k, H, rows;
  long long y_stride;    // values between rows of y
};

// out[t] = sum_j w * y[dest]: a warp takes kPairs pairs of one token at once and kPieces pieces of 256
// columns of their rows, all of them on their way before the first is used, and adds the pairs in
// order.  What a lane holds (kPairs x kPieces pieces on their way, kPieces sums) is kept to 64
// registers, so that 32 warps share an SM: with eight pieces whatever type and top_k are, and 128
// registers or more, 4096 tokens x top-4 x 7168 bf16 took 49.3 us instead of 40.6 (7.2 TB/s), 16384 x top-1
// 77 instead of 73, in fp32 171 instead of 141, with rows of 2043 bf16 47 instead of 35; only 16384 x
// top-2 x 4096 was better off, 62 and 64.
constexpr int kUnsortThreads = 256;
__host__ __device__ constexpr int unsort_pairs(bool vec, int bytes, int pairs) {  // at most
  const int most = vec && bytes == 2 ? 8 : 4;
  return pairs < most ? pairs : most;
}
__host__ __device__ constexpr int unsort_pieces(bool vec, int bytes, int pairs) {
  if (!vec) return pairs == 1 ? 2 : 1;
  if (bytes == 4) return pairs <= 2 ? 2 : 1;
  return pairs == 1 ? 4 : (pairs == 8 ? 1 : 2);
}
template <class T, bool VEC, int kPairs>
__global__ void __launch_bounds__(kUnsortThreads, 4) token_unsort_kernel(const TokenUnsortParams p) {
  static_assert(unsort_pairs(VEC, sizeof(T), kPairs) == kPairs, "");
  constexpr int kPieces = unsort_pieces(VEC, sizeof(T), kPairs);
  const int lane = threadIdx.x & 31;
  const unsigned segs = (p.H + 256u * kPieces - 1u) / (256u * kPieces);
  const unsigned u = blockIdx.x * (kUnsortThreads / 32u) + (threadIdx.x >> 5);  // the host keeps units below 2^32
  const unsigned t = u / segs;
  if (t >= static_cast<unsigned>(p.T)) return;
  const int c0 = static_cast<int>(u - t * segs) * 256 * kPieces;
  float acc[kPieces][8] = {};
  for (int j0 = 0; j0 < p.top_k; j0 += kPairs) {
    int d = -1;
    float w = 1.0f;
    if (lane < kPairs && j0 + lane < p.top_k) {
      const size_t i = (size_t)t * p.top_k + j0 + lane;
      d = p.dest[i];
      if (d >= p.rows) d = -1;
      if (p.weights) w = p.weights[i];
    }
    Eight<T, VEC, 32> v[kPairs][kPieces];
    int dj[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      dj[j] = __shfl_sync(0xffffffffu, d, j);
      const T* row = static_cast<const T*>(p.y) + (size_t)max(dj[j], 0) * p.y_stride;
#pragma unroll
      for (int s = 0; s < kPieces; ++s) v[j][s].load(row, c0 + 256 * s, lane, p.H, dj[j] >= 0);
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      if (dj[j] >= 0) {  // a pair without a row adds nothing, whatever its weight is
#pragma unroll
        for (int s = 0; s < kPieces; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[s][i] = fmaf(wj, v[j][s].get(i), acc[s][i]);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < kPieces; ++s) {
    Eight<T, VEC, 32> o;
#pragma unroll
    for (int i = 0; i < 8; i += 2) o.set2(i, acc[s][i], acc[s][i + 1]);
    o.template store<true>(static_cast<T*>(p.out) + (size_t)t * p.H, c0 + 256 * s, lane, p.H);
  }
}

struct TokenUnsortGradParams {
  const void* dout;          // [T] rows
  const void* y;             // [rows] rows
  const int32_t* dest;       // [T][top_k]
  const float* weights;      // or NULL (weights of one; dw is not written)
  const int32_t* m_indices;  // [rows]; with clear: rows with m_indices < 0 are set to zero
  void* dy;                  // [rows][H]
  float* dw;                 // [T][top_k] or NULL
  int T, top_k, H, rows;
  long long y_stride, dout_stride;
  int per;                   // pairs of a token that one block takes
  int clear_blocks;          // blocks behind those of the tokens that clear rows
};

// Sets rows with m_indices < 0 to zero (groups > 0: and those of a 128-row block whose first entry is not
// in [0, groups)): block `b` of `nb`.  Most of them lie together, so the warps take every so-many-th
// row; lane l looks at the warp's l-th.
template <class T, bool VEC>
__device__ __forceinline__ void clear_rows_block(T* out, const int32_t* m_indices, int rows, int H, int b, int nb, int groups = 0) {
  const int lane = threadIdx.x & 31;
  const int warps = nb * (blockDim.x >> 5);
  const int first = b * (blockDim.x >> 5) + (threadIdx.x >> 5);
  for (long long rb = 0; rb < rows; rb += 32LL * warps) {
    const long long mine = rb + (long long)lane * warps + first;
    const bool stands_for_none =
        mine < rows && (m_indices[mine] < 0 || (groups > 0 && static_cast<unsigned>(m_indices[mine & ~127LL]) >= static_cast<unsigned>(groups)));
    unsigned mask = __ballot_sync(0xffffffffu, stands_for_none);
    while (mask) {
      const int i = __ffs(mask) - 1;
      mask &= mask - 1;
      T* row = out + (size_t)(rb + (long long)i * warps + first) * H;
      const Eight<T, VEC, 32> zero;
      for (int c0 = 0; c0 < H; c0 += 256) zero.store(row, c0, lane, H);
    }
  }
}

// One block takes `per` pairs of one token, a warp kPairs of them and kPieces pieces of 256 columns at
// a time: its pieces of dout[t] stay in registers while those of the pairs' rows go by, all of them on
// their way before the first is used.  A pair's product is summed over a lane's columns, the lanes
// and the warps in that fixed order.
// Value by value (not VEC) a piece is eight loads instead of one, and one or two pieces are enough.  As
// above, what a lane holds is kept to 64 registers (VEC; 48 if not): blocks of eight warps with up to 128
// took 129 us instead of 105 for 16384 tokens x top-1 x 7168 bf16 (6.7 TB/s), 289 instead of 206 for fp32,
// 425 instead of 337 for 4096 x top-8 x 7168 fp32, 55 instead of 46 for 4096 x top-4 x 1002 fp32.  Streaming
// stores are 3 to 5 % of that.  Six of the forms spill for it: 16-bit with eight pairs 28 bytes stored and 36
// loaded, with four 8 and 8; fp32 with four pairs 16 and 28, with two 8 and 16.
constexpr int kUnsortGradWarps = 4;
__host__ __device__ constexpr int grad_pairs(bool vec, int bytes, int pairs) {  // at most
  const int most = !vec ? 2 : (bytes == 4 ? 4 : 8);
  return pairs < most ? pairs : most;
}
__host__ __device__ constexpr int grad_pieces(bool vec, int bytes, int pairs) {
  return !vec ? (pairs == 1 ? 2 : 1) : (bytes == 4 ? 4 : 8) / pairs;
}
__host__ __device__ constexpr int grad_blocks(bool vec) { return vec ? 8 : 10; }  // resident on an SM
template <class T, bool VEC, int kPairs>
__global__ void __launch_bounds__(32 * kUnsortGradWarps, grad_blocks(VEC)) token_unsort_grad_kernel(const TokenUnsortGradParams p) {
  static_assert(grad_pairs(VEC, sizeof(T), kPairs) == kPairs, "");
  constexpr int kPieces = grad_pieces(VEC, sizeof(T), kPairs);
  __shared__ float part[kUnsortGradWarps][kPairs];
  const int warps = blockDim.x >> 5;
  const unsigned splits = (p.top_k + p.per - 1) / p.per;
  const unsigned token_blocks = static_cast<unsigned>(p.T) * splits;
  if (blockIdx.x >= token_blocks) {
    clear_rows_block<T, VEC>(static_cast<T*>(p.dy), p.m_indices, p.rows, p.H, static_cast<int>(blockIdx.x - token_blocks), p.clear_blocks);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned t = blockIdx.x / splits;
  const int j_begin = static_cast<int>(blockIdx.x - t * splits) * p.per;
  const int j_end = min(j_begin + p.per, p.top_k);
  const T* dout = static_cast<const T*>(p.dout) + (size_t)t * p.dout_stride;
  for (int j0 = j_begin; j0 < j_end; j0 += kPairs) {
    int d_lane = -1;
    float w_lane = 1.0f;
    if (lane < kPairs && j0 + lane < j_end) {
      const size_t i = (size_t)t * p.top_k + j0 + lane;
      d_lane = p.dest[i];
      if (d_lane >= p.rows) d_lane = -1;
      if (p.weights) w_lane = p.weights[i];
    }
    float dot[kPairs] = {};
    for (int c0 = warp * 256 * kPieces; c0 < p.H; c0 += warps * 256 * kPieces) {
      Eight<T, VEC, 32> g[kPieces];
#pragma unroll
      for (int s = 0; s < kPieces; ++s) g[s].load(dout, c0 + 256 * s, lane, p.H);
      if (p.dw != nullptr) {
        Eight<T, VEC, 32> v[kPairs][kPieces];
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const int d = __shfl_sync(0xffffffffu, d_lane, j);
          const T* row = static_cast<const T*>(p.y) + (size_t)max(d, 0) * p.y_stride;
#pragma unroll
          for (int s = 0; s < kPieces; ++s) v[j][s].load(row, c0 + 256 * s, lane, p.H, d >= 0);
        }
#pragma unroll
        for (int j = 0; j < kPairs; ++j)  // columns behind the row's end and rows of no pair hold zeros
#pragma unroll
          for (int s = 0; s < kPieces; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) dot[j] = fmaf(g[s].get(i), v[j][s].get(i), dot[j]);
      }
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int d = __shfl_sync(0xffffffffu, d_lane, j);
        const float w = __shfl_sync(0xffffffffu, w_lane, j);
        if (d < 0) continue;
#pragma unroll
        for (int s = 0; s < kPieces; ++s) {
          Eight<T, VEC, 32> o;
#pragma unroll
          for (int i = 0; i < 8; i += 2) o.set2(i, w * g[s].get(i), w * g[s].get(i + 1));
          o.template store<true>(static_cast<T*>(p.dy) + (size_t)d * p.H, c0 + 256 * s, lane, p.H);
        }
      }
    }
    if (p.dw != nullptr) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int d = __shfl_sync(0xffffffffu, d_lane, j);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
        if (lane == 0) part[warp][j] = d < 0 ? 0.0f : dot[j];  // (0 * dout is NaN where dout is infinite)
      }
      __syncthreads();
      if (threadIdx.x < kPairs && j0 + static_cast<int>(threadIdx.x) < j_end) {
        float s = part[0][threadIdx.x];
        for (int w = 1; w < warps; ++w) s += part[w][threadIdx.x];
        p.dw[(size_t)t * p.top_k + j0 + threadIdx.x] = s;
      }
      __syncthreads();
    }
  }
}

constexpr int kClearThreads = 128;
template <class T, bool VEC>
__global__ void __launch_bounds__(kClearThreads) clear_rows_kernel(T* out, const int32_t* m_indices, int rows, int H, int groups) {
  clear_rows_block<T, VEC>(out, m_indices, rows, H, blockIdx.x, gridDim.x, groups);
}

}  // namespace dg
