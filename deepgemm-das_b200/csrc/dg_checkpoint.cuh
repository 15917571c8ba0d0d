// Activation checkpoints in 8 bits, and the experts' activation that is taken back from one.
//
// Every 128 columns of a row share one fp32 scale s; the stored code q stands for q * s.
//   e4m3:  s = the smallest power of two with max|x| / s <= 448.  A power of two costs a
//          floating-point format no precision (only its range ends a factor of up to two earlier),
//          x / s is exact, and q * s is exact in bf16: taking the rows out again adds no rounding.
//   int8:  s = max|x| / 127, q = rint(x * (1 / s)) (within 1.6e-5 steps of the nearest: two
//          roundings of 2^-24 on at most 127 steps).
// s = 1 for a block of zeros and never less than 2^-126; a block that holds a NaN or an infinity
// gets s = NaN, so that it comes back as NaN and an overflow is not lost in the checkpoint.  Values
// come back at most as large as the largest finite one of their type.
//
//   act   = g * sig(g) * u                                  (g = gate, u = up, sig(g) = 1 / (1 + exp(-g)))
//   dg    = d * u * sig(g) * (1 + g * (1 - sig(g)))         du = d * g * sig(g)
// all in fp32, rounded once.  The backward kernel also hands out act again, which the gradient
// of the weights behind it needs, so that the forward pass need not keep it.
//
// Bound by HBM: 8 bytes per activation forward (4 read, 2 + 2 written), 10 backward (2 + 2 read,
// 4 + 2 written).  16 lanes hold the 128 columns of one scale, eight each.
#pragma once

#include <cuda_fp8.h>

#include "dg_rows.cuh"

namespace dg {

constexpr int kCkBlock = 128;    // columns of one scale
constexpr int kCkThreads = 256;
constexpr int kCkLanes = 16;     // lanes of one block of columns

// Bits of the largest magnitude (NaN and infinities order above everything finite), over the 16
// lanes of a block of columns.
__device__ __forceinline__ uint32_t ck_max_bits(uint32_t m) {
#pragma unroll
  for (int o = kCkLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// Scale and its reciprocal for a block whose largest magnitude has the bits `top`.
template <int KIND>
__device__ __forceinline__ void ck_scale(uint32_t top, float& s, float& inv) {
  if (top >= 0x7f800000u) {
    s = inv = __uint_as_float(0x7fc00000u);
    return;
  }
  if (top == 0) {
    s = inv = 1.0f;
    return;
  }
  if constexpr (KIND == DG_KIND_E4M3) {
    // top = m * 2^e, 1 <= m < 2: 448 = 1.75 * 2^8, so s = 2^(e - 8) if m <= 1.75, else 2^(e - 7)
    int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, 1);  // 2^-126
    s = __uint_as_float(static_cast<uint32_t>(e) << 23);
    inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
  } else {
    s = fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), __uint_as_float(1u << 23));
    inv = __frcp_rn(s);
  }
}

template <int KIND>
__device__ __forceinline__ uint8_t ck_code(float x, float inv) {
  const float v = x * inv;
  if constexpr (KIND == DG_KIND_E4M3)
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  else
    return static_cast<uint8_t>(max(-127, min(127, __float2int_rn(v))));
}
// The value that a code stands for, at most `most` in magnitude (NaN stays NaN): a value just below
// the largest of its type may have been rounded up to a code beyond it (255 to 256 of 2^120, say)
// and still comes back finite.
template <int KIND>
__device__ __forceinline__ float ck_value(uint8_t q, float s, float most) {
  float v;
  if constexpr (KIND == DG_KIND_E4M3)
    v = __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3))) * s;
  else
    v = static_cast<float>(static_cast<int8_t>(q)) * s;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(most));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(v), "f"(-most));
  return v;
}
constexpr float kCkMaxF32 = 3.402823466e+38f;
template <class T>
__device__ __forceinline__ float ck_most();
template <>
__device__ __forceinline__ float ck_most<float>() { return kCkMaxF32; }
template <>
__device__ __forceinline__ float ck_most<__half>() { return 65504.0f; }
template <>
__device__ __forceinline__ float ck_most<__nv_bfloat16>() { return 3.3895313892515355e+38f; }

template <class T, bool VEC>
__device__ __forceinline__ uint32_t ck_lane_max(const Eight<T, VEC, kCkLanes>& v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v.get(i)) & 0x7fffffffu);
  return m;
}

// 1 / (1 + exp(-g)).  16-bit results take the hardware's exp and reciprocal (relative error below
// 2^-21 where the sigmoid is not negligible), 32-bit ones the exact forms.
template <class T>
__device__ __forceinline__ float ck_sigmoid(float g) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
  return __fdividef(1.0f, 1.0f + __expf(-g));
}
template <class T>
__device__ __forceinline__ float ck_silu(float g) {
  if constexpr (sizeof(T) == 4) return g / (1.0f + expf(-g));
  return __fdividef(g, 1.0f + __expf(-g));
}

struct CheckpointParams {
  const void* x;    // [rows] rows of H values (restore: written)
  uint8_t* q;       // [rows][H]
  float* scale;     // [rows][blocks]
  void* out;        // restore: [rows][H]
  int rows, H;
  long long x_stride;
};

// Rows into a checkpoint.  A unit is 128 columns of one row.
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) checkpoint_rows_kernel(const CheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  const long long units = (long long)p.rows * blocks;
  const long long step = (long long)gridDim.x * (kCkThreads / kCkLanes);
  const long long first = (long long)blockIdx.x * (kCkThreads / kCkLanes) + threadIdx.x / kCkLanes;
  for (long long base = first; base - first < units; base += step) {  // the same number of rounds for a whole warp
    const long long u = min(base, units - 1);
    const long long r = u / blocks;
    const int b = static_cast<int>(u - r * blocks);
    Eight<T, VEC, kCkLanes> v;
    v.load(static_cast<const T*>(p.x) + (size_t)r * p.x_stride, b * kCkBlock, lane, p.H);
    float s, inv;
    ck_scale<KIND>(ck_max_bits(ck_lane_max(v)), s, inv);
    if (base >= units) continue;
    EightBytes<VEC, kCkLanes> q;
#pragma unroll
    for (int i = 0; i < 8; ++i) q.val[i] = ck_code<KIND>(v.get(i), inv);
    q.store(p.q + (size_t)r * p.H, b * kCkBlock, lane, p.H);
    if (lane == 0) p.scale[u] = s;
  }
}

// And out of it.
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) restore_rows_kernel(const CheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  const long long units = (long long)p.rows * blocks;
  const long long step = (long long)gridDim.x * (kCkThreads / kCkLanes);
  for (long long u = (long long)blockIdx.x * (kCkThreads / kCkLanes) + threadIdx.x / kCkLanes; u < units; u += step) {
    const long long r = u / blocks;
    const int b = static_cast<int>(u - r * blocks);
    const float s = p.scale[u];
    EightBytes<VEC, kCkLanes> q;
    q.load(p.q + (size_t)r * p.H, b * kCkBlock, lane, p.H);
    Eight<T, VEC, kCkLanes> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.set(i, ck_value<KIND>(q.val[i], s, ck_most<T>()));
    v.store(static_cast<T*>(p.out) + (size_t)r * p.H, b * kCkBlock, lane, p.H);
  }
}

struct ActCheckpointParams {
  const void* x;             // [rows] rows of 2 H values: gate, up
  const void* dact;          // backward: [rows] rows of H
  uint8_t* q;                // [rows][2 H]
  float* scale;              // [rows][2 * blocks]: gate's, then up's
  void* act;                 // [rows][H]
  void* dx;                  // backward: [rows][2 H]
  const int32_t* m_indices;  // NULL, or rows with m_indices < 0 are skipped
  int rows, H, clear;        // clear: skipped rows of the outputs are set to zero
  long long x_stride, dact_stride;
};

template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) act_checkpoint_kernel(const ActCheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  const long long units = (long long)p.rows * blocks;
  const long long step = (long long)gridDim.x * (kCkThreads / kCkLanes);
  const long long first = (long long)blockIdx.x * (kCkThreads / kCkLanes) + threadIdx.x / kCkLanes;
  for (long long base = first; base - first < units; base += step) {
    const long long u = min(base, units - 1);
    const long long r = u / blocks;
    const int b = static_cast<int>(u - r * blocks), c0 = b * kCkBlock;
    const bool skip = p.m_indices != nullptr && p.m_indices[r] < 0;
    Eight<T, VEC, kCkLanes> g, up;
    if (!skip) {
      const T* x = static_cast<const T*>(p.x) + (size_t)r * p.x_stride;
      g.load(x, c0, lane, p.H);
      up.load(x + p.H, c0, lane, p.H);
    }
    float sg, ig, su, iu;
    ck_scale<KIND>(ck_max_bits(ck_lane_max(g)), sg, ig);
    ck_scale<KIND>(ck_max_bits(ck_lane_max(up)), su, iu);
    if (base >= units || (skip && !p.clear)) continue;
    EightBytes<VEC, kCkLanes> qg, qu;
    Eight<T, VEC, kCkLanes> a;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float gv = g.get(i), uv = up.get(i);
      qg.val[i] = ck_code<KIND>(gv, ig);
      qu.val[i] = ck_code<KIND>(uv, iu);
      a.set(i, ck_silu<T>(gv) * uv);
    }
    a.store(static_cast<T*>(p.act) + (size_t)r * p.H, c0, lane, p.H);
    uint8_t* q = p.q + (size_t)r * 2 * p.H;
    qg.store(q, c0, lane, p.H);
    qu.store(q + p.H, c0, lane, p.H);
    if (lane == 0) {
      float* s = p.scale + (size_t)r * 2 * blocks;
      s[b] = sg;
      s[blocks + b] = su;
    }
  }
}

template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) act_checkpoint_grad_kernel(const ActCheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  const long long units = (long long)p.rows * blocks;
  const long long step = (long long)gridDim.x * (kCkThreads / kCkLanes);
  for (long long u = (long long)blockIdx.x * (kCkThreads / kCkLanes) + threadIdx.x / kCkLanes; u < units; u += step) {
    const long long r = u / blocks;
    const int b = static_cast<int>(u - r * blocks), c0 = b * kCkBlock;
    const bool skip = p.m_indices != nullptr && p.m_indices[r] < 0;
    if (skip && !p.clear) continue;
    Eight<T, VEC, kCkLanes> dg, du, a;
    if (!skip) {
      const float* s = p.scale + (size_t)r * 2 * blocks;
      const float sg = s[b], su = s[blocks + b];
      const uint8_t* q = p.q + (size_t)r * 2 * p.H;
      EightBytes<VEC, kCkLanes> qg, qu;
      Eight<T, VEC, kCkLanes> d;
      qg.load(q, c0, lane, p.H);
      qu.load(q + p.H, c0, lane, p.H);
      d.load(static_cast<const T*>(p.dact) + (size_t)r * p.dact_stride, c0, lane, p.H);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float gv = ck_value<KIND>(qg.val[i], sg, kCkMaxF32), uv = ck_value<KIND>(qu.val[i], su, kCkMaxF32), dv = d.get(i);
        const float sig = ck_sigmoid<T>(gv);
        const float silu = gv * sig;
        dg.set(i, dv * uv * sig * fmaf(gv, 1.0f - sig, 1.0f));
        du.set(i, dv * silu);
        a.set(i, silu * uv);
      }
    }
    T* dx = static_cast<T*>(p.dx) + (size_t)r * 2 * p.H;
    dg.store(dx, c0, lane, p.H);
    du.store(dx + p.H, c0, lane, p.H);
    if (p.act != nullptr) a.store(static_cast<T*>(p.act) + (size_t)r * p.H, c0, lane, p.H);
  }
}

}  // namespace dg
