// C ABI of the operators of a training step that move rows: tokens sorted by expert and back with
// their gradients, activation checkpoints in 8 bits.  Argument checks and launches; no torch
// types, no allocation, no stream synchronisation.
#include "dg_host.h"
#include "dg_checkpoint.cuh"
#include "dg_token_sort.cuh"

namespace {

using namespace dg;
using namespace dg::host;

bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

size_t elem_size(int elem) { return elem == DG_OUT_F32 ? 4 : 2; }
bool bad_elem(int elem) { return elem < DG_OUT_BF16 || elem > DG_OUT_F32; }

// Rows of `h` values every 8 of which can be moved at once.
bool vec_rows(const void* p, long long stride, int h, int elem) {
  return h % 8 == 0 && stride % 8 == 0 && aligned16(p);
}

// f(type, vec): calls a generic lambda with a value of the element type and a bool constant.
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
template <class F>
void by_type(int elem, bool vec, F f) {
  if (elem == DG_OUT_BF16) {
    if (vec) f(__nv_bfloat16(), Yes{}); else f(__nv_bfloat16(), No{});
  } else if (elem == DG_OUT_F16) {
    if (vec) f(__half(), Yes{}); else f(__half(), No{});
  } else {
    if (vec) f(float(), Yes{}); else f(float(), No{});
  }
}

// f(n): n = 1, 2, 4 or 8 pairs of a token that a warp handles at once.
template <int N>
struct Num { static constexpr int value = N; };
template <class F>
void by_pairs(int pairs, F f) {
  if (pairs <= 1) f(Num<1>{});
  else if (pairs <= 2) f(Num<2>{});
  else if (pairs <= 4) f(Num<4>{});
  else f(Num<8>{});
}

int launched(int n) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e);
  count_launches(n);
  return DG_OK;
}

// Blocks that leave the device full with `per_sm` resident on each SM, but no more than there is
// work for.
int blocks_for(long long units, int per_block, const DeviceInfo& dev, int per_sm) {
  const long long want = (units + per_block - 1) / per_block;
  const long long most = (long long)dev.sm_count * per_sm;
  return static_cast<int>(want < 1 ? 1 : (want < most ? want : most));
}

// The pairs above which a block does not count all of them itself, but two launches before the sort do
// (us without and with them, 32 experts x 1024 bf16: 4800 pairs 10.3 / 12.0, 16384 14.5 / 15.4, 32768 21.8 /
// 21.5, 65536 43.8 / 40.4).
constexpr long long kSortSelfCount = 16384;

int sort_tokens_per_block(int tokens, int top_k, int sms) {
  long long per = ((long long)tokens + sms - 1) / sms;
  const long long most = kSortMaxChunk / top_k;
  if (per > most) per = most;
  return static_cast<int>(per < 1 ? 1 : per);
}

}  // namespace

extern "C" {

int64_t dg_token_sort_capacity(int64_t pairs, int32_t num_groups, int32_t align) {
  if (pairs < 0 || num_groups < 1 || align < 1) return -1;
  const int64_t used = pairs < num_groups ? pairs : num_groups;
  return (pairs + used * (align - 1)) / align * align;
}

size_t dg_token_sort_scratch_bytes(int32_t num_tokens, int32_t top_k, int32_t num_groups) {
  if (num_tokens < 0 || top_k < 1 || num_groups < 1) return 0;
  if ((long long)num_tokens * top_k <= kSortSelfCount) return 0;
  // the smallest block takes one token, the largest kSortMaxChunk pairs; sized for any device
  const int per = sort_tokens_per_block(num_tokens, top_k, 1024);
  const long long chunks = ((long long)num_tokens + per - 1) / per;
  return static_cast<size_t>((chunks + 1) * num_groups) * sizeof(int32_t);
}

int dg_token_sort(const dg_token_sort_args* a, void* stream) {
  if (a == nullptr) return DG_ERR_NULL_POINTER;
  if (a->elem_bytes != 2 && a->elem_bytes != 4) return DG_ERR_BAD_ARGUMENT;
  if (a->num_tokens < 0 || a->top_k < 1 || a->num_groups < 1 || a->hidden < 1 || a->align < 1 || a->cap < 0)
    return DG_ERR_BAD_SHAPE;
  if (a->num_groups > DG_MAX_GROUPS || a->top_k > DG_MAX_TOP_K) return DG_ERR_TOO_LARGE;
  const long long pairs = (long long)a->num_tokens * a->top_k;
  if (pairs > 0x7fffffffLL || (long long)a->hidden * a->elem_bytes > 0x7fffffffLL) return DG_ERR_TOO_LARGE;
  // every place that a pair can be given lies below this
  if (a->cap < dg_token_sort_capacity(pairs, a->num_groups, a->align)) return DG_ERR_BAD_SHAPE;
  if (!a->counts || !a->offsets || !a->m_total) return DG_ERR_NULL_POINTER;
  if (pairs > 0 && (!a->x || !a->ids || !a->dest)) return DG_ERR_NULL_POINTER;
  if (a->cap > 0 && (!a->rows || !a->m_indices)) return DG_ERR_NULL_POINTER;
  if (a->num_tokens > 1 && a->x_stride < a->hidden) return DG_ERR_BAD_SHAPE;
  const size_t need = dg_token_sort_scratch_bytes(a->num_tokens, a->top_k, a->num_groups);
  if (need > 0 && (!a->scratch || a->scratch_bytes < need)) return DG_ERR_BAD_ARGUMENT;
  if (!aligned_to(a->x, a->elem_bytes) || !aligned_to(a->rows, a->elem_bytes) || !aligned_to(a->ids, a->ids64 ? 8 : 4))
    return DG_ERR_BAD_ALIGNMENT;
  const long long rows_bytes = (long long)a->cap * a->hidden * a->elem_bytes;
  if (overlap(a->rows, rows_bytes, a->x, row_span(a->num_tokens, a->x_stride, a->hidden, a->elem_bytes)) ||
      overlap(a->rows, rows_bytes, a->ids, pairs * (a->ids64 ? 8 : 4)))
    return DG_ERR_BAD_ARGUMENT;
  const DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != DG_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  TokenSortParams p{};
  p.x = a->x;
  p.ids = a->ids;
  p.ids64 = a->ids64 != 0;
  p.T = a->num_tokens;
  p.top_k = a->top_k;
  p.G = a->num_groups;
  p.align = a->align;
  p.cap = a->cap;
  p.row_bytes = a->hidden * a->elem_bytes;
  p.x_stride = a->x_stride * a->elem_bytes;
  p.rows = a->rows;
  p.dest = a->dest;
  p.m_indices = a->m_indices;
  p.counts = a->counts;
  p.offsets = a->offsets;
  p.m_total = a->m_total;
  p.status = a->status;
  p.clear = a->clear != 0;
  p.tokens_per_block = sort_tokens_per_block(p.T, p.top_k, dev->sm_count);
  p.rep = 1;
  while (p.rep < 32 && p.rep * 2 * p.G <= 1024) p.rep *= 2;
  const int chunks = p.T > 0 ? (p.T + p.tokens_per_block - 1) / p.tokens_per_block : 1;
  int launches = 1;
  if (need > 0) {
    int32_t* hist = static_cast<int32_t*>(a->scratch);
    sort_hist_kernel<<<chunks, kSortThreads, p.G * 4, st>>>(p, hist);
    sort_scan_kernel<<<(p.G + 7) / 8, 256, 0, st>>>(hist, chunks, p.G);
    p.hist = hist;
    launches = 3;
  }
  const unsigned long long all = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.rows) |
                                 static_cast<unsigned long long>(p.row_bytes) | static_cast<unsigned long long>(p.x_stride);
  const int vb = (all & 15u) == 0 ? 16 : ((all & 3u) == 0 ? 4 : 2);
  // few tokens: the columns are split as well, so that more SMs take part (one block on each: a second
  // round would pay for the counting again)
  const int segs = (p.row_bytes / vb + sort_seg(vb) - 1) / sort_seg(vb);
  int split = chunks < dev->sm_count ? dev->sm_count / chunks : 1;
  if (split > segs) split = segs;
  const dim3 grid(chunks, split, 1);
  const int smem = (3 * p.G + 1 + p.tokens_per_block * p.top_k + (p.hist ? 0 : 2 * p.G * p.rep)) * 4;
  if (vb == 16)
    token_sort_kernel<16><<<grid, kSortThreads, smem, st>>>(p);
  else if (vb == 4)
    token_sort_kernel<4><<<grid, kSortThreads, smem, st>>>(p);
  else
    token_sort_kernel<2><<<grid, kSortThreads, smem, st>>>(p);
  return launched(launches);
}

int dg_token_unsort(const dg_token_unsort_args* a, void* stream) {
  if (a == nullptr) return DG_ERR_NULL_POINTER;
  if (bad_elem(a->elem)) return DG_ERR_BAD_KIND;
  if (a->num_tokens < 0 || a->top_k < 1 || a->hidden < 1 || a->num_rows < 0) return DG_ERR_BAD_SHAPE;
  if (a->num_rows > 1 && a->y_stride < a->hidden) return DG_ERR_BAD_SHAPE;
  if ((long long)a->num_tokens * a->top_k > 0x7fffffffLL) return DG_ERR_TOO_LARGE;
  if (a->num_tokens == 0) return DG_OK;
  if (!a->dest || !a->out || (a->num_rows > 0 && !a->y)) return DG_ERR_NULL_POINTER;
  const size_t es = elem_size(a->elem);
  if (!aligned_to(a->y, es) || !aligned_to(a->out, es)) return DG_ERR_BAD_ALIGNMENT;
  const long long out_bytes = (long long)es * a->num_tokens * a->hidden, pair_bytes = 4LL * a->num_tokens * a->top_k;
  if (overlap(a->out, out_bytes, a->y, row_span(a->num_rows, a->y_stride, a->hidden, es)) ||
      overlap(a->out, out_bytes, a->dest, pair_bytes) || overlap(a->out, out_bytes, a->weights, pair_bytes))
    return DG_ERR_BAD_ARGUMENT;
  const DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != DG_OK) return rc;
  TokenUnsortParams p{};
  p.y = a->y;
  p.dest = a->dest;
  p.weights = a->weights;
  p.out = a->out;
  p.T = a->num_tokens;
  p.top_k = a->top_k;
  p.H = a->hidden;
  p.rows = a->num_rows;
  p.y_stride = a->y_stride;
  const bool vec = vec_rows(p.y, p.y_stride, p.H, a->elem) && aligned16(p.out);
  int rc2 = DG_OK;
  by_type(a->elem, vec, [&](auto t, auto v) {
    by_pairs(p.top_k, [&](auto pairs) {
      constexpr int kBytes = static_cast<int>(sizeof(decltype(t)));
      constexpr bool V = decltype(v)::value;
      constexpr int kPairs = unsort_pairs(V, kBytes, decltype(pairs)::value);
      constexpr int kCols = 256 * unsort_pieces(V, kBytes, kPairs);
      const long long units = (long long)p.T * ((p.H + kCols - 1) / kCols);  // < 2^31 tokens x pairs, rows < 2^31 values
      const long long grid = (units + kUnsortThreads / 32 - 1) / (kUnsortThreads / 32);
      if (grid > 0x1fffffffLL) {
        rc2 = DG_ERR_TOO_LARGE;
        return;
      }
      token_unsort_kernel<decltype(t), V, kPairs>
          <<<static_cast<unsigned>(grid), kUnsortThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    });
  });
  if (rc2 != DG_OK) return rc2;
  return launched(1);
}

int dg_token_unsort_grad(const dg_token_unsort_grad_args* a, void* stream) {
  if (a == nullptr) return DG_ERR_NULL_POINTER;
  if (bad_elem(a->elem)) return DG_ERR_BAD_KIND;
  if (a->num_tokens < 0 || a->top_k < 1 || a->hidden < 1 || a->num_rows < 0) return DG_ERR_BAD_SHAPE;
  if (a->num_rows > 1 && a->y_stride < a->hidden) return DG_ERR_BAD_SHAPE;
  if (a->num_tokens > 1 && a->dout_stride < a->hidden) return DG_ERR_BAD_SHAPE;
  if ((long long)a->num_tokens * a->top_k > 0x7fff0000LL) return DG_ERR_TOO_LARGE;
  if (a->num_tokens == 0 && (!a->clear || a->num_rows == 0)) return DG_OK;
  if (a->num_tokens > 0 && (!a->dout || !a->dest)) return DG_ERR_NULL_POINTER;
  if (a->num_rows > 0 && (!a->dy || (a->dw && !a->y) || (a->clear && !a->m_indices))) return DG_ERR_NULL_POINTER;
  const size_t es = elem_size(a->elem);
  if (!aligned_to(a->y, es) || !aligned_to(a->dy, es) || !aligned_to(a->dout, es)) return DG_ERR_BAD_ALIGNMENT;
  const long long dy_bytes = (long long)es * a->num_rows * a->hidden;
  if (overlap(a->dy, dy_bytes, a->dout, row_span(a->num_tokens, a->dout_stride, a->hidden, es)) ||
      (a->dw && overlap(a->dy, dy_bytes, a->y, row_span(a->num_rows, a->y_stride, a->hidden, es))))
    return DG_ERR_BAD_ARGUMENT;
  const DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != DG_OK) return rc;
  TokenUnsortGradParams p{};
  p.dout = a->dout;
  p.y = a->y;
  p.dest = a->dest;
  p.weights = a->weights;
  p.m_indices = a->m_indices;
  p.dy = a->dy;
  p.dw = a->dw;
  p.T = a->num_tokens;
  p.top_k = a->top_k;
  p.H = a->hidden;
  p.rows = a->num_rows;
  p.y_stride = a->y_stride;
  p.dout_stride = a->dout_stride;
  // few tokens: a block for every pair, so that more SMs take part (top-8 x 7168 bf16, us with and without:
  // 148 tokens 7.5 / 8.0, 296 14.7 / 14.9, 600 34.1 / 32.6, 2400 128 / 108)
  p.per = (long long)p.T >= 4LL * dev->sm_count ? p.top_k : 1;
  p.clear_blocks = a->clear && p.rows > 0 ? blocks_for(p.rows, 16, *dev, 2) : 0;
  const long long grid = (long long)p.T * ((p.top_k + p.per - 1) / p.per) + p.clear_blocks;
  if (grid == 0) return DG_OK;
  const bool vec = vec_rows(p.dout, p.dout_stride, p.H, a->elem) && aligned16(p.dy) &&
                   (!p.dw || vec_rows(p.y, p.y_stride, p.H, a->elem));
  by_type(a->elem, vec, [&](auto t, auto v) {
    constexpr bool V = decltype(v)::value;
    by_pairs(p.per, [&](auto pairs) {
      constexpr int kBytes = static_cast<int>(sizeof(decltype(t)));
      constexpr int kPairs = grad_pairs(V, kBytes, decltype(pairs)::value);
      constexpr int kCols = 256 * grad_pieces(V, kBytes, kPairs);
      // as many warps as divide the row's pieces evenly
      const int pieces = (p.H + kCols - 1) / kCols;
      const int turns = (pieces + kUnsortGradWarps - 1) / kUnsortGradWarps, warps = (pieces + turns - 1) / turns;
      token_unsort_grad_kernel<decltype(t), V, kPairs>
          <<<static_cast<unsigned>(grid), 32 * warps, 0, static_cast<cudaStream_t>(stream)>>>(p);
    });
  });
  return launched(1);
}

int dg_clear_padding_rows(const dg_clear_rows_args* a, void* stream) {
  if (a == nullptr) return DG_ERR_NULL_POINTER;
  if (bad_elem(a->elem)) return DG_ERR_BAD_KIND;
  if (a->num_rows < 0 || a->hidden < 1 || a->num_groups < 0) return DG_ERR_BAD_SHAPE;
  if (a->num_rows == 0) return DG_OK;
  if (!a->rows || !a->m_indices) return DG_ERR_NULL_POINTER;
  if (!aligned_to(a->rows, elem_size(a->elem))) return DG_ERR_BAD_ALIGNMENT;
  const DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != DG_OK) return rc;
  const int grid = blocks_for(a->num_rows, 16, *dev, 8);
  by_type(a->elem, vec_rows(a->rows, a->hidden, a->hidden, a->elem), [&](auto t, auto v) {
    using T = decltype(t);
    clear_rows_kernel<T, decltype(v)::value><<<grid, kClearThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<T*>(a->rows), a->m_indices, a->num_rows, a->hidden, a->num_groups);
  });
  return launched(1);
}

static int checkpoint_common(bool restore, const dg_checkpoint_args* a, void* stream) {
  if (a == nullptr) return DG_ERR_NULL_POINTER;
  if (bad_elem(a->elem) || (a->kind != DG_KIND_E4M3 && a->kind != DG_KIND_I8)) return DG_ERR_BAD_KIND;
  if (a->num_rows < 0 || a->hidden < 1 || (a->num_rows > 1 && a->x_stride < a->hidden)) return DG_ERR_BAD_SHAPE;
  if (a->num_rows == 0) return DG_OK;
  if (!a->x || !a->q || !a->scale) return DG_ERR_NULL_POINTER;
  if (!aligned_to(a->x, elem_size(a->elem)) || !aligned_to(a->scale, 4)) return DG_ERR_BAD_ALIGNMENT;
  const DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != DG_OK) return rc;
  CheckpointParams p{};
  p.x = a->x;
  p.out = a->x;
  p.q = static_cast<uint8_t*>(a->q);
  p.scale = a->scale;
  p.rows = a->num_rows;
  p.H = a->hidden;
  p.x_stride = a->x_stride;
  const bool vec = vec_rows(p.x, p.x_stride, p.H, a->elem) && aligned_to(p.q, 8);
  const long long units = (long long)p.rows * ((p.H + kCkBlock - 1) / kCkBlock);
  const int per_block = vec ? kCkUnits<true> * kCkThreads / 8 : kCkUnits<false> * kCkThreads / 32;
  const long long want = (units + per_block - 1) / per_block;
  if (want > 0x7fffffffLL) return DG_ERR_TOO_LARGE;
  const unsigned grid = static_cast<unsigned>(want);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  by_type(a->elem, vec, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr bool V = decltype(v)::value;
    if (restore) {
      if (a->kind == DG_KIND_E4M3)
        restore_rows_kernel<T, V, DG_KIND_E4M3><<<grid, kCkThreads, 0, st>>>(p);
      else
        restore_rows_kernel<T, V, DG_KIND_I8><<<grid, kCkThreads, 0, st>>>(p);
    } else {
      if (a->kind == DG_KIND_E4M3)
        checkpoint_rows_kernel<T, V, DG_KIND_E4M3><<<grid, kCkThreads, 0, st>>>(p);
      else
        checkpoint_rows_kernel<T, V, DG_KIND_I8><<<grid, kCkThreads, 0, st>>>(p);
    }
  });
  return launched(1);
}

int dg_checkpoint_rows(const dg_checkpoint_args* a, void* stream) { return checkpoint_common(false, a, stream); }

int dg_restore_rows(const dg_checkpoint_args* a, void* stream) {
  if (a != nullptr && a->num_rows > 1 && a->x_stride != a->hidden) return DG_ERR_BAD_SHAPE;  // written row after row
  return checkpoint_common(true, a, stream);
}

static int act_checkpoint_common(bool grad, const dg_act_checkpoint_args* a, void* stream) {
  if (a == nullptr) return DG_ERR_NULL_POINTER;
  if (bad_elem(a->elem) || (a->kind != DG_KIND_E4M3 && a->kind != DG_KIND_I8)) return DG_ERR_BAD_KIND;
  if (a->num_rows < 0 || a->hidden < 1 || a->hidden > 0x3fffffff) return DG_ERR_BAD_SHAPE;
  if (a->num_rows > 1 && (grad ? a->dact_stride < a->hidden : a->x_stride < 2LL * a->hidden)) return DG_ERR_BAD_SHAPE;
  if (a->num_rows == 0) return DG_OK;
  if (!a->q || !a->scale || (grad ? (!a->dact || !a->dx) : (!a->x || !a->act))) return DG_ERR_NULL_POINTER;
  const size_t es = elem_size(a->elem);
  if (!aligned_to(a->x, es) || !aligned_to(a->dact, es) || !aligned_to(a->dx, es) || !aligned_to(a->act, es) ||
      !aligned_to(a->scale, 4))
    return DG_ERR_BAD_ALIGNMENT;
  const DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != DG_OK) return rc;
  ActCheckpointParams p{};
  p.x = a->x;
  p.dact = a->dact;
  p.q = static_cast<uint8_t*>(a->q);
  p.scale = a->scale;
  p.act = a->act;
  p.dx = a->dx;
  p.m_indices = a->m_indices;
  p.rows = a->num_rows;
  p.H = a->hidden;
  p.clear = a->clear != 0;
  p.x_stride = a->x_stride;
  p.dact_stride = a->dact_stride;
  const bool vec = p.H % 8 == 0 && aligned_to(p.q, 8) && aligned16(p.act) &&
                   (grad ? aligned16(p.dx) && vec_rows(p.dact, p.dact_stride, p.H, a->elem)
                         : vec_rows(p.x, p.x_stride, p.H, a->elem));
  const long long units = (long long)p.rows * ((p.H + kCkBlock - 1) / kCkBlock);
  const int per_block = kCkActUnits * kCkThreads / (vec ? 8 : 32);
  const long long want = (units + per_block - 1) / per_block;
  if (want > 0x7fffffffLL) return DG_ERR_TOO_LARGE;
  const unsigned grid = static_cast<unsigned>(want);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  by_type(a->elem, vec, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr bool V = decltype(v)::value;
    if (grad) {
      if (a->kind == DG_KIND_E4M3)
        act_checkpoint_grad_kernel<T, V, DG_KIND_E4M3><<<grid, kCkThreads, 0, st>>>(p);
      else
        act_checkpoint_grad_kernel<T, V, DG_KIND_I8><<<grid, kCkThreads, 0, st>>>(p);
    } else {
      if (a->kind == DG_KIND_E4M3)
        act_checkpoint_kernel<T, V, DG_KIND_E4M3><<<grid, kCkThreads, 0, st>>>(p);
      else
        act_checkpoint_kernel<T, V, DG_KIND_I8><<<grid, kCkThreads, 0, st>>>(p);
    }
  });
  return launched(1);
}

int dg_act_checkpoint(const dg_act_checkpoint_args* a, void* stream) { return act_checkpoint_common(false, a, stream); }
int dg_act_checkpoint_grad(const dg_act_checkpoint_args* a, void* stream) { return act_checkpoint_common(true, a, stream); }

}  // extern "C"
