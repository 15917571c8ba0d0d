// Host fast path between torch tensors and the C ABI of libdeepgemm_b200.so.
//
// The reference binds its launchers to Python from C++ (csrc/common/deepgemm_ops.cpp:127-144), so
// a call costs a pybind argument conversion and the TORCH_CHECKs.  The Python marshalling in
// deepgemm/_core.py does the same checks with tensor attribute reads, about 7 us a call; for a
// sparse decode step that is half of what the kernel takes.  This module does them natively.
//
// It is deliberately only the accepting half: each function returns true (or its results) when the
// arguments passed every check and the launch was enqueued, false (or None) when anything at all is unusual (a
// check failed, a layout this file does not know, a device that is not current, a launch error).
// On false nothing was enqueued and the caller runs the Python marshalling, which either raises
// the error with its full message or handles the unusual case.  No message text lives here.
//
// It is not part of the C ABI boundary (include/deepgemm_b200.h has no torch types); it is a
// client of it, like the ctypes marshalling.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <array>

#include "deepgemm_b200.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

constexpr int kMaxDevices = 64;
std::array<Tensor, kMaxDevices> g_status;  // int32[DG_STATUS_WORDS] per device, registered from Python
int64_t g_accepted = 0, g_declined = 0;     // calls enqueued here / handed back (under the GIL)

inline bool on(const Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev && t.is_contiguous(); }

// activation / weight / output element types per kind (deepgemm/_core.py: _A_DTYPES, _B_DTYPES)
inline bool a_dtype_ok(int kind, at::ScalarType t) {
  switch (kind) {
    case DG_KIND_I8: case DG_KIND_W4A8: return t == at::kChar;
    case DG_KIND_E4M3: return t == at::kFloat8_e4m3fn;
    case DG_KIND_BF16: return t == at::kBFloat16;
  }
  return false;
}
inline bool b_dtype_ok(int kind, at::ScalarType t) {
  switch (kind) {
    case DG_KIND_I8: case DG_KIND_W4A8: return t == at::kChar || t == at::kByte;
    case DG_KIND_E4M3: return t == at::kFloat8_e4m3fn || t == at::kChar || t == at::kByte;
    case DG_KIND_BF16: return t == at::kBFloat16;
  }
  return false;
}
// the packed weight of an INT8 / FP8 problem with K % 128 == 64 carries one zero-padded block more
inline bool k_matches(int kind, int64_t packed_k, int64_t k) {
  return packed_k == k || ((kind == DG_KIND_I8 || kind == DG_KIND_E4M3) && k % 128 == 64 && packed_k == k + 64);
}
inline bool d_dtype_ok(int kind, at::ScalarType t) {
  return t == at::kBFloat16 || (kind == DG_KIND_W4A8 && t == at::kHalf);
}

// 4-D packed weight [G, K / block, N, row]; the 3-D W4A8 form needs the Python side's registry
inline bool weight_dims(const Tensor& b, int kind, int64_t* g, int64_t* n, int64_t* k) {
  if (b.dim() != 4) return false;
  const int64_t row = (kind == DG_KIND_BF16) ? 64 : 128;
  const int64_t k_per_block = (kind == DG_KIND_BF16) ? 64 : (kind == DG_KIND_W4A8 ? 256 : 128);
  if (b.size(3) != row) return false;
  *g = b.size(0);
  *n = b.size(2);
  *k = b.size(1) * k_per_block;
  return true;
}

// fp32, contiguous, 16-byte aligned, shape (s0[, s1]) optionally followed by a 1
inline const float* scale_ptr(const OptTensor& t, int dev, int64_t s0, int64_t s1) {
  if (!t.has_value()) return nullptr;
  const Tensor& x = *t;
  if (!on(x, dev) || x.scalar_type() != at::kFloat) return nullptr;
  const int64_t want = s1 < 0 ? 1 : 2;
  const int64_t nd = x.dim();
  if (!(nd == want || (nd == want + 1 && x.size(nd - 1) == 1))) return nullptr;
  if (x.size(0) != s0 || (s1 >= 0 && x.size(1) != s1)) return nullptr;
  const float* p = x.data_ptr<float>();
  return (reinterpret_cast<uintptr_t>(p) % 16 == 0) ? p : nullptr;
}

inline int32_t* status_ptr(const OptTensor& status, int dev) {
  const Tensor& s = status.has_value() ? *status : g_status[dev];
  if (!s.defined() || !on(s, dev) || s.scalar_type() != at::kInt || s.numel() < DG_STATUS_WORDS) return nullptr;
  return s.data_ptr<int32_t>();
}

bool masked_impl(int64_t kind, int64_t scale_mode, const Tensor& a, const Tensor& b, const Tensor& d,
            const OptTensor& a_scale, const OptTensor& b_scale, const Tensor& masked_m, int64_t expected_m,
            int64_t block_n, const OptTensor& status, const OptTensor& signal) {
  if (!a.is_cuda()) return false;
  const int dev = static_cast<int>(a.get_device());
  if (dev < 0 || dev >= kMaxDevices || dev != c10::cuda::current_device()) return false;
  if (a.dim() != 3 || d.dim() != 3) return false;
  if (!on(a, dev) || !on(b, dev) || !on(d, dev) || !on(masked_m, dev)) return false;
  const int ki = static_cast<int>(kind);
  if (!a_dtype_ok(ki, a.scalar_type()) || !b_dtype_ok(ki, b.scalar_type()) || !d_dtype_ok(ki, d.scalar_type()))
    return false;
  if (masked_m.scalar_type() != at::kInt) return false;
  int64_t bg, n, bk;
  if (!weight_dims(b, ki, &bg, &n, &bk)) return false;
  const int64_t g = a.size(0), max_m = a.size(1), k = a.size(2);
  if (bg != g || !k_matches(ki, bk, k) || d.size(0) != g || d.size(1) != max_m || d.size(2) != n || masked_m.numel() != g)
    return false;
  if (g > INT32_MAX || max_m > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return false;

  dg_masked_args args{};
  args.kind = ki;
  args.scale_mode = static_cast<int32_t>(scale_mode);
  if (scale_mode != DG_SCALE_NONE) {
    args.a_scale = scale_ptr(a_scale, dev, g, max_m);
    args.b_scale = scale_ptr(b_scale, dev, g, scale_mode == DG_SCALE_PER_CHANNEL ? n : -1);
    if (args.a_scale == nullptr || args.b_scale == nullptr) return false;
  }
  args.status = status_ptr(status, dev);
  if (args.status == nullptr) return false;
  if (signal.has_value()) {
    const Tensor& s = *signal;
    if (!on(s, dev) || s.scalar_type() != at::kInt || s.numel() != g * ((max_m + 127) / 128)) return false;
    if (ki == DG_KIND_W4A8 || n % 32 != 0) return false;
    args.signal = s.data_ptr<int32_t>();
  }
  args.a = a.data_ptr();
  args.b_packed = b.data_ptr();
  args.d = d.data_ptr();
  args.masked_m = masked_m.data_ptr<int32_t>();
  args.num_groups = static_cast<int32_t>(g);
  args.max_m = static_cast<int32_t>(max_m);
  args.n = static_cast<int32_t>(n);
  args.k = static_cast<int32_t>(k);
  args.expected_m = static_cast<int32_t>(expected_m);
  args.block_n = static_cast<int32_t>(block_n);
  args.out_kind = d.scalar_type() == at::kHalf ? DG_OUT_F16 : DG_OUT_BF16;
  return dg_masked_gemm(&args, c10::cuda::getCurrentCUDAStream(dev).stream()) == DG_OK;
}

bool contiguous_impl(int64_t kind, int64_t scale_mode, const Tensor& a, const Tensor& b, const Tensor& d,
                const OptTensor& a_scale, const OptTensor& b_scale, const Tensor& m_indices, int64_t block_n,
                const OptTensor& status) {
  if (!a.is_cuda()) return false;
  const int dev = static_cast<int>(a.get_device());
  if (dev < 0 || dev >= kMaxDevices || dev != c10::cuda::current_device()) return false;
  if (a.dim() != 2 || d.dim() != 2) return false;
  if (!on(a, dev) || !on(b, dev) || !on(d, dev) || !on(m_indices, dev)) return false;
  const int ki = static_cast<int>(kind);
  if (!a_dtype_ok(ki, a.scalar_type()) || !b_dtype_ok(ki, b.scalar_type()) || !d_dtype_ok(ki, d.scalar_type()))
    return false;
  if (m_indices.scalar_type() != at::kInt) return false;
  int64_t g, n, bk;
  if (!weight_dims(b, ki, &g, &n, &bk)) return false;
  const int64_t m_total = a.size(0), k = a.size(1);
  if (!k_matches(ki, bk, k) || d.size(0) != m_total || d.size(1) != n || m_indices.numel() != m_total) return false;
  if (g > INT32_MAX || m_total > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return false;

  dg_contig_args args{};
  args.kind = ki;
  args.scale_mode = static_cast<int32_t>(scale_mode);
  if (scale_mode != DG_SCALE_NONE) {
    args.a_scale = scale_ptr(a_scale, dev, m_total, -1);
    args.b_scale = scale_ptr(b_scale, dev, g, scale_mode == DG_SCALE_PER_CHANNEL ? n : -1);
    if (args.a_scale == nullptr || args.b_scale == nullptr) return false;
  }
  args.status = status_ptr(status, dev);
  if (args.status == nullptr) return false;
  args.a = a.data_ptr();
  args.b_packed = b.data_ptr();
  args.d = d.data_ptr();
  args.m_indices = m_indices.data_ptr<int32_t>();
  args.num_groups = static_cast<int32_t>(g);
  args.m_total = static_cast<int32_t>(m_total);
  args.n = static_cast<int32_t>(n);
  args.k = static_cast<int32_t>(k);
  args.block_n = static_cast<int32_t>(block_n);
  args.out_kind = d.scalar_type() == at::kHalf ? DG_OUT_F16 : DG_OUT_BF16;
  return dg_contig_gemm(&args, c10::cuda::getCurrentCUDAStream(dev).stream()) == DG_OK;
}

inline bool count(bool ok) {
  ++(ok ? g_accepted : g_declined);
  return ok;
}

bool masked(int64_t kind, int64_t scale_mode, const Tensor& a, const Tensor& b, const Tensor& d,
            const OptTensor& a_scale, const OptTensor& b_scale, const Tensor& masked_m, int64_t expected_m,
            int64_t block_n, const OptTensor& status, const OptTensor& signal) {
  return count(masked_impl(kind, scale_mode, a, b, d, a_scale, b_scale, masked_m, expected_m, block_n, status, signal));
}

bool contiguous(int64_t kind, int64_t scale_mode, const Tensor& a, const Tensor& b, const Tensor& d,
                const OptTensor& a_scale, const OptTensor& b_scale, const Tensor& m_indices, int64_t block_n,
                const OptTensor& status) {
  return count(contiguous_impl(kind, scale_mode, a, b, d, a_scale, b_scale, m_indices, block_n, status));
}

// ------------------------------------------------------------------ operators of a training step
// These allocate their results as the Python functions do (deepgemm/token_sort.py,
// activation_checkpoint.py, grouped_grad.py) and return them, or None with nothing enqueued.
namespace py = pybind11;

inline int elem_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return DG_OUT_BF16;
    case at::kHalf: return DG_OUT_F16;
    case at::kFloat: return DG_OUT_F32;
    default: return -1;
  }
}
inline int code_kind(at::ScalarType t) {
  return t == at::kFloat8_e4m3fn ? DG_KIND_E4M3 : (t == at::kChar ? DG_KIND_I8 : -1);
}
inline int current(const Tensor& t) {  // the tensor's device if it is the current one, else -1
  if (!t.is_cuda()) return -1;
  const int dev = static_cast<int>(t.get_device());
  return dev >= 0 && dev < kMaxDevices && dev == c10::cuda::current_device() ? dev : -1;
}
// [rows, H] of a known type on `dev`, rows whole and apart
inline bool rows_ok(const Tensor& t, int dev) {
  return t.is_cuda() && t.get_device() == dev && t.dim() == 2 && elem_of(t) >= 0 && t.size(1) >= 1 && t.size(0) <= INT32_MAX &&
         t.size(1) <= INT32_MAX / 8 && (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) < 2 || t.stride(0) >= t.size(1));
}
inline int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
inline bool ints_ok(const Tensor& t, int dev, int64_t n) { return on(t, dev) && t.scalar_type() == at::kInt && t.numel() == n; }
inline void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
inline Tensor make(at::IntArrayRef size, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), c10::nullopt);  // at::empty without the dispatcher
}
// `size` values of an int32 buffer from `first` on, as a tensor of its own (no dispatcher, no allocation)
inline Tensor part(const Tensor& whole, int64_t first, at::IntArrayRef size) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(whole.storage_offset() + first);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
  return t;
}
inline py::object count_obj(py::object o) {
  count(!o.is_none());
  return o;
}

py::object sort_impl(const Tensor& x, const Tensor& ids, int64_t experts, int64_t align, const OptTensor& out) {
  const int dev = current(x);
  if (dev < 0 || !rows_ok(x, dev) || !on(ids, dev) || ids.dim() != 2 || ids.size(0) != x.size(0)) return py::none();
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) return py::none();
  const int64_t t = ids.size(0), k = ids.size(1), h = x.size(1);
  if (k < 1 || k > DG_MAX_TOP_K || experts < 1 || experts > DG_MAX_GROUPS || align < 1 || align > INT32_MAX) return py::none();
  int32_t* status = status_ptr(c10::nullopt, dev);
  const int64_t cap = dg_token_sort_capacity(t * k, static_cast<int32_t>(experts), static_cast<int32_t>(align));
  if (status == nullptr || cap < 0 || cap > INT32_MAX) return py::none();
  if (out.has_value() && (!on(*out, dev) || out->scalar_type() != x.scalar_type() || out->dim() != 2 || out->size(0) != cap || out->size(1) != h))
    return py::none();
  Tensor rows = out.has_value() ? *out : make({cap, h}, x.scalar_type(), x);
  // the plan's five arrays in one buffer, each on a 16-byte boundary
  const int64_t at_m = (t * k + 3) / 4 * 4, at_c = at_m + (cap + 3) / 4 * 4, at_o = at_c + (experts + 3) / 4 * 4,
                at_t = at_o + (experts + 3) / 4 * 4;
  Tensor ints = make({at_t + 1}, at::kInt, x), scratch;
  Tensor dest = part(ints, 0, {t, k}), m_indices = part(ints, at_m, {cap}), counts = part(ints, at_c, {experts}),
         offsets = part(ints, at_o, {experts}), m_total = part(ints, at_t, {1});
  dg_token_sort_args a{};
  a.elem_bytes = static_cast<int32_t>(x.element_size());
  a.ids64 = ids.scalar_type() == at::kLong;
  a.num_tokens = static_cast<int32_t>(t);
  a.top_k = static_cast<int32_t>(k);
  a.num_groups = static_cast<int32_t>(experts);
  a.hidden = static_cast<int32_t>(h);
  a.align = static_cast<int32_t>(align);
  a.cap = static_cast<int32_t>(cap);
  a.x_stride = row_stride(x);
  a.x = x.data_ptr();
  a.ids = ids.data_ptr();
  a.rows = rows.data_ptr();
  a.dest = dest.data_ptr<int32_t>();
  a.m_indices = m_indices.data_ptr<int32_t>();
  a.counts = counts.data_ptr<int32_t>();
  a.offsets = offsets.data_ptr<int32_t>();
  a.m_total = m_total.data_ptr<int32_t>();
  a.scratch_bytes = dg_token_sort_scratch_bytes(a.num_tokens, a.top_k, a.num_groups);
  if (a.scratch_bytes > 0) {
    scratch = make({static_cast<int64_t>(a.scratch_bytes)}, at::kByte, x);
    a.scratch = scratch.data_ptr();
  }
  a.status = status;
  a.clear = !out.has_value();
  if (dg_token_sort(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::make_tuple(rows, dest, m_indices, counts, offsets, m_total);
}

py::object unsort_impl(const Tensor& y, const Tensor& dest, const Tensor& m_indices, const OptTensor& weights, const OptTensor& out) {
  const int dev = current(y);
  if (dev < 0 || !rows_ok(y, dev) || !on(dest, dev) || dest.scalar_type() != at::kInt || dest.dim() != 2 ||
      !ints_ok(m_indices, dev, y.size(0)))
    return py::none();
  const int64_t t = dest.size(0), k = dest.size(1), h = y.size(1);
  if (weights.has_value() && (!on(*weights, dev) || weights->scalar_type() != at::kFloat || weights->sizes() != dest.sizes())) return py::none();
  if (out.has_value() && (!on(*out, dev) || out->scalar_type() != y.scalar_type() || out->dim() != 2 || out->size(0) != t || out->size(1) != h))
    return py::none();
  Tensor o = out.has_value() ? *out : make({t, h}, y.scalar_type(), y);
  dg_token_unsort_args a{};
  a.elem = elem_of(y);
  a.num_tokens = static_cast<int32_t>(t);
  a.top_k = static_cast<int32_t>(k);
  a.hidden = static_cast<int32_t>(h);
  a.num_rows = static_cast<int32_t>(y.size(0));
  a.y_stride = row_stride(y);
  a.y = y.data_ptr();
  a.dest = dest.data_ptr<int32_t>();
  a.weights = weights.has_value() ? weights->data_ptr<float>() : nullptr;
  a.out = o.data_ptr();
  if (dg_token_unsort(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::cast(o);
}

// without y: the gradient of the rows alone
py::object unsort_grad_impl(const Tensor& dout, const OptTensor& y, const Tensor& dest, const Tensor& m_indices, const OptTensor& weights,
                            bool need_dweights) {
  const int dev = current(dout);
  if (dev < 0 || !rows_ok(dout, dev) || !on(dest, dev) || dest.scalar_type() != at::kInt || dest.dim() != 2)
    return py::none();
  const int64_t t = dest.size(0), k = dest.size(1), h = dout.size(1), rows = m_indices.numel();
  if (dout.size(0) != t || rows > INT32_MAX || !ints_ok(m_indices, dev, rows)) return py::none();
  if (y.has_value() ? (!rows_ok(*y, dev) || y->scalar_type() != dout.scalar_type() || y->size(0) != rows || y->size(1) != h)
                    : (weights.has_value() && need_dweights))
    return py::none();
  if (weights.has_value() && (!on(*weights, dev) || weights->scalar_type() != at::kFloat || weights->sizes() != dest.sizes())) return py::none();
  Tensor dy = make({rows, h}, dout.scalar_type(), dout), dw;
  if (weights.has_value() && need_dweights) dw = make({t, k}, at::kFloat, dout);
  dg_token_unsort_grad_args a{};
  a.elem = elem_of(dout);
  a.num_tokens = static_cast<int32_t>(t);
  a.top_k = static_cast<int32_t>(k);
  a.hidden = static_cast<int32_t>(h);
  a.num_rows = static_cast<int32_t>(rows);
  a.clear = 1;
  a.y_stride = y.has_value() ? row_stride(*y) : h;
  a.dout_stride = row_stride(dout);
  a.dout = dout.data_ptr();
  a.y = y.has_value() ? y->data_ptr() : nullptr;
  a.dest = dest.data_ptr<int32_t>();
  a.weights = weights.has_value() ? weights->data_ptr<float>() : nullptr;
  a.m_indices = m_indices.data_ptr<int32_t>();
  a.dy = dy.data_ptr();
  a.dw = dw.defined() ? dw.data_ptr<float>() : nullptr;
  if (dg_token_unsort_grad(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::make_tuple(dy, dw.defined() ? py::cast(dw) : py::none());
}

inline int64_t scale_blocks(int64_t h) { return (h + 127) / 128; }

py::object checkpoint_impl(const Tensor& x, int64_t kind) {
  const int dev = current(x);
  if (dev < 0 || !rows_ok(x, dev)) return py::none();
  Tensor q = make(x.sizes(), kind == DG_KIND_E4M3 ? at::kFloat8_e4m3fn : at::kChar, x);
  Tensor scale = make({x.size(0), scale_blocks(x.size(1))}, at::kFloat, x);
  dg_checkpoint_args a{};
  a.elem = elem_of(x);
  a.kind = static_cast<int32_t>(kind);
  a.num_rows = static_cast<int32_t>(x.size(0));
  a.hidden = static_cast<int32_t>(x.size(1));
  a.x_stride = row_stride(x);
  a.x = x.data_ptr();
  a.q = q.data_ptr();
  a.scale = scale.data_ptr<float>();
  if (dg_checkpoint_rows(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::make_tuple(q, scale);
}

// the checkpoint of rows that consist of `halves` parts with blocks of their own
inline bool kept_ok(const Tensor& q, const Tensor& scale, int dev, int64_t halves) {
  return on(q, dev) && on(scale, dev) && q.dim() == 2 && code_kind(q.scalar_type()) >= 0 && q.size(1) >= halves && q.size(1) % halves == 0 &&
         q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX / 8 && scale.scalar_type() == at::kFloat && scale.dim() == 2 &&
         scale.size(0) == q.size(0) && scale.size(1) == halves * scale_blocks(q.size(1) / halves);
}

py::object restore_impl(const Tensor& q, const Tensor& scale, int64_t elem) {
  const int dev = current(q);
  const at::ScalarType type = elem == DG_OUT_F32 ? at::kFloat : (elem == DG_OUT_F16 ? at::kHalf : at::kBFloat16);
  if (dev < 0 || !kept_ok(q, scale, dev, 1)) return py::none();
  Tensor x = make(q.sizes(), type, q);
  dg_checkpoint_args a{};
  a.elem = elem_of(x);
  a.kind = code_kind(q.scalar_type());
  a.num_rows = static_cast<int32_t>(q.size(0));
  a.hidden = static_cast<int32_t>(q.size(1));
  a.x_stride = q.size(1);
  a.x = x.data_ptr();
  a.q = q.data_ptr();
  a.scale = scale.data_ptr<float>();
  if (dg_restore_rows(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::cast(x);
}

py::object act_impl(const Tensor& x, int64_t kind, const OptTensor& m_indices) {
  const int dev = current(x);
  if (dev < 0 || !rows_ok(x, dev) || x.size(1) % 2 != 0 || (m_indices.has_value() && !ints_ok(*m_indices, dev, x.size(0)))) return py::none();
  const int64_t m = x.size(0), h = x.size(1) / 2;
  Tensor act = make({m, h}, x.scalar_type(), x), q = make(x.sizes(), kind == DG_KIND_E4M3 ? at::kFloat8_e4m3fn : at::kChar, x),
         scale = make({m, 2 * scale_blocks(h)}, at::kFloat, x);
  dg_act_checkpoint_args a{};
  a.elem = elem_of(x);
  a.kind = static_cast<int32_t>(kind);
  a.num_rows = static_cast<int32_t>(m);
  a.hidden = static_cast<int32_t>(h);
  a.clear = 1;
  a.x_stride = row_stride(x);
  a.x = x.data_ptr();
  a.q = q.data_ptr();
  a.scale = scale.data_ptr<float>();
  a.act = act.data_ptr();
  a.m_indices = m_indices.has_value() ? m_indices->data_ptr<int32_t>() : nullptr;
  if (dg_act_checkpoint(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::make_tuple(act, q, scale);
}

py::object act_grad_impl(const Tensor& q, const Tensor& scale, const Tensor& dact, const OptTensor& m_indices, bool need_act) {
  const int dev = current(q);
  if (dev < 0 || !kept_ok(q, scale, dev, 2) || !rows_ok(dact, dev) || dact.size(0) != q.size(0) || 2 * dact.size(1) != q.size(1) ||
      (m_indices.has_value() && !ints_ok(*m_indices, dev, q.size(0))))
    return py::none();
  const int64_t m = dact.size(0), h = dact.size(1);
  Tensor dx = make({m, 2 * h}, dact.scalar_type(), q), act;
  if (need_act) act = make({m, h}, dact.scalar_type(), q);
  dg_act_checkpoint_args a{};
  a.elem = elem_of(dact);
  a.kind = code_kind(q.scalar_type());
  a.num_rows = static_cast<int32_t>(m);
  a.hidden = static_cast<int32_t>(h);
  a.clear = 1;
  a.dact_stride = row_stride(dact);
  a.dact = dact.data_ptr();
  a.q = q.data_ptr();
  a.scale = scale.data_ptr<float>();
  a.act = act.defined() ? act.data_ptr() : nullptr;
  a.dx = dx.data_ptr();
  a.m_indices = m_indices.has_value() ? m_indices->data_ptr<int32_t>() : nullptr;
  if (dg_act_checkpoint_grad(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::make_tuple(dx, act.defined() ? py::cast(act) : py::none());
}

// a contiguous bf16 [rows, columns] operand of the grouped products
inline bool operand_ok(const Tensor& t, int dev) {
  return on(t, dev) && t.dim() == 2 && t.scalar_type() == at::kBFloat16 && t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX;
}

py::object input_grad_impl(const Tensor& dy, const Tensor& w, const Tensor& m_indices, const OptTensor& out, int64_t block_n) {
  const int dev = current(dy);
  int64_t g, n, k;
  if (dev < 0 || !operand_ok(dy, dev) || !on(w, dev) || w.scalar_type() != at::kBFloat16 || !weight_dims(w, DG_KIND_BF16, &g, &n, &k) ||
      dy.size(1) != n || g > INT32_MAX || k > INT32_MAX || m_indices.dim() != 1 || !ints_ok(m_indices, dev, dy.size(0)))
    return py::none();
  if (out.has_value() && (!operand_ok(*out, dev) || out->size(0) != dy.size(0) || out->size(1) != k)) return py::none();
  int32_t* status = status_ptr(c10::nullopt, dev);
  if (status == nullptr) return py::none();
  Tensor dx = out.has_value() ? *out : make({dy.size(0), k}, at::kBFloat16, dy);
  dg_input_grad_args a{};
  a.dy = dy.data_ptr();
  a.w_packed = w.data_ptr();
  a.dx = dx.data_ptr();
  a.m_indices = m_indices.data_ptr<int32_t>();
  a.num_groups = static_cast<int32_t>(g);
  a.m_total = static_cast<int32_t>(dy.size(0));
  a.n = static_cast<int32_t>(n);
  a.k = static_cast<int32_t>(k);
  a.block_n = static_cast<int32_t>(block_n);
  a.clear = !out.has_value();
  a.status = status;
  if (dg_grouped_input_grad(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::cast(dx);
}

py::object weight_grad_impl(const Tensor& dy, const Tensor& x, const Tensor& m_indices, int64_t groups, const OptTensor& out, bool f32,
                            bool accumulate, int64_t tile, bool whole_blocks) {
  const int dev = current(dy);
  if (dev < 0 || !operand_ok(dy, dev) || !operand_ok(x, dev) || x.size(0) != dy.size(0) || m_indices.dim() != 1 ||
      !ints_ok(m_indices, dev, dy.size(0)) || groups < 1 || groups > DG_MAX_GROUPS)
    return py::none();
  const int64_t n = dy.size(1), k = x.size(1);
  if (n < 16 || n % 16 != 0 || k < 64 || k % 64 != 0 || (accumulate && !out.has_value())) return py::none();
  if (out.has_value()) {
    const Tensor& o = *out;
    if (!on(o, dev) || o.dim() != 4 || o.size(0) != groups || o.size(1) != k / 64 || o.size(2) != n || o.size(3) != 64 ||
        (o.scalar_type() != at::kBFloat16 && o.scalar_type() != at::kFloat) || (accumulate && o.scalar_type() != at::kFloat))
      return py::none();
  }
  int32_t* status = status_ptr(c10::nullopt, dev);
  if (status == nullptr) return py::none();
  Tensor dw = out.has_value() ? *out : make({groups, k / 64, n, 64}, f32 ? at::kFloat : at::kBFloat16, dy);
  dg_weight_grad_args a{};
  a.dy = dy.data_ptr();
  a.x = x.data_ptr();
  a.dw = dw.data_ptr();
  a.m_indices = m_indices.data_ptr<int32_t>();
  a.num_groups = static_cast<int32_t>(groups);
  a.m_total = static_cast<int32_t>(dy.size(0));
  a.n = static_cast<int32_t>(n);
  a.k = static_cast<int32_t>(k);
  a.out_kind = dw.scalar_type() == at::kFloat ? DG_OUT_F32 : DG_OUT_BF16;
  a.accumulate = accumulate;
  a.tile = static_cast<int32_t>(tile);
  a.whole_blocks = whole_blocks;
  a.status = status;
  if (dg_grouped_weight_grad(&a, stream_of(dev)) != DG_OK) return py::none();
  return py::cast(dw);
}

void set_status_words(int64_t device, const Tensor& words) {
  TORCH_CHECK(device >= 0 && device < kMaxDevices, "device index out of range");
  TORCH_CHECK(words.is_cuda() && words.get_device() == device && words.scalar_type() == at::kInt &&
                  words.is_contiguous() && words.numel() >= DG_STATUS_WORDS,
              "status words must be a contiguous int32 CUDA tensor on that device");
  g_status[device] = words;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "native argument checks and launch for the grouped GEMM entry points (accepting half only)";
  m.def("masked", &masked, "enqueue dg_masked_gemm if every check passes; False otherwise");
  m.def("contiguous", &contiguous, "enqueue dg_contig_gemm if every check passes; False otherwise");
  // results, or None with nothing enqueued
  m.def("sort_tokens", [](const Tensor& x, const Tensor& ids, int64_t e, int64_t align, const OptTensor& out) {
    return count_obj(sort_impl(x, ids, e, align, out));
  });
  m.def("unsort_tokens", [](const Tensor& y, const Tensor& dest, const Tensor& mi, const OptTensor& w, const OptTensor& out) {
    return count_obj(unsort_impl(y, dest, mi, w, out));
  });
  m.def("unsort_tokens_grad", [](const Tensor& dout, const OptTensor& y, const Tensor& dest, const Tensor& mi, const OptTensor& w, bool need) {
    return count_obj(unsort_grad_impl(dout, y, dest, mi, w, need));
  });
  m.def("checkpoint_rows", [](const Tensor& x, int64_t kind) { return count_obj(checkpoint_impl(x, kind)); });
  m.def("restore_rows", [](const Tensor& q, const Tensor& s, int64_t elem) { return count_obj(restore_impl(q, s, elem)); });
  m.def("silu_mul_checkpoint", [](const Tensor& x, int64_t kind, const OptTensor& mi) { return count_obj(act_impl(x, kind, mi)); });
  m.def("silu_mul_checkpoint_grad", [](const Tensor& q, const Tensor& s, const Tensor& d, const OptTensor& mi, bool need) {
    return count_obj(act_grad_impl(q, s, d, mi, need));
  });
  m.def("input_grad", [](const Tensor& dy, const Tensor& w, const Tensor& mi, const OptTensor& out, int64_t bn) {
    return count_obj(input_grad_impl(dy, w, mi, out, bn));
  });
  m.def("weight_grad", [](const Tensor& dy, const Tensor& x, const Tensor& mi, int64_t g, const OptTensor& out, bool f32, bool acc, int64_t tile,
                          bool whole) {
    return count_obj(weight_grad_impl(dy, x, mi, g, out, f32, acc, tile, whole));
  });
  m.def("set_status_words", &set_status_words);
  m.def("stats", []() { return std::make_pair(g_accepted, g_declined); }, "(calls enqueued here, calls handed back)");
  // the header this file was compiled against; the caller compares it with the library's own
  m.def("abi_version", []() { return static_cast<int64_t>(DG_ABI_VERSION); });
}
