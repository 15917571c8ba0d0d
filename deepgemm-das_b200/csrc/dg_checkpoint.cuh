// Activation checkpoints in 8 bits, and the experts' activation that is taken back from one.
//
// Every 128 columns of a row share one fp32 scale s; the stored code q stands for q * s.
//   e4m3:  s = the smallest power of two with max|x| / s <= 448.  A power of two costs a
//          floating-point format no precision (only its range ends a factor of up to two earlier),
//          x / s is exact, and q * s is exact in bf16: taking the rows out again adds no rounding.
//   int8:  s = max|x| / 127, q = rint(x / s).
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

#include <type_traits>

#include "dg_rows.cuh"

namespace dg {

constexpr int kCkBlock = 128;    // columns of one scale
constexpr int kCkThreads = 256;
constexpr int kCkLanes = 16;     // lanes of one block of columns

// The largest magnitude of 128 columns, over the 16 lanes that hold them, as the bits of an fp32
// value.  Magnitudes order like their bits, NaN and infinities above everything finite.  16-bit
// types compare two at a time, and two blocks of columns (gate and up) share the exchanges between
// the lanes.
__device__ __forceinline__ uint32_t ck_max2(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
template <class T>
__device__ __forceinline__ uint32_t ck_bits16(uint32_t b) {  // bits of a 16-bit value -> bits of it in fp32
  if constexpr (sizeof(T) == 4) return b;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return b << 16;
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(b))));
}
template <class T, bool VEC>
__device__ __forceinline__ uint32_t ck_lane_max16(const Eight<T, VEC, kCkLanes>& v) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(v.raw);
  const uint32_t m = ck_max2(ck_max2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), ck_max2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
  return max(m >> 16, m & 0xffffu);
}
template <class T, bool VEC>
__device__ __forceinline__ uint32_t ck_lane_max32(const Eight<T, VEC, kCkLanes>& v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v.get(i)) & 0x7fffffffu);
  return m;
}
template <class T, bool VEC>
__device__ __forceinline__ uint32_t ck_top(const Eight<T, VEC, kCkLanes>& v) {
  uint32_t m = sizeof(T) == 2 ? ck_lane_max16(v) : ck_lane_max32(v);
#pragma unroll
  for (int o = kCkLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return ck_bits16<T>(m);
}
template <class T, bool VEC>
__device__ __forceinline__ void ck_top_of_two(const Eight<T, VEC, kCkLanes>& v0, const Eight<T, VEC, kCkLanes>& v1, uint32_t& t0,
                                              uint32_t& t1) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = (ck_lane_max16(v0) << 16) | ck_lane_max16(v1);
#pragma unroll
    for (int o = kCkLanes / 2; o > 0; o >>= 1) m = ck_max2(m, __shfl_xor_sync(0xffffffffu, m, o));
    t0 = ck_bits16<T>(m >> 16);
    t1 = ck_bits16<T>(m & 0xffffu);
  } else {
    t0 = ck_top(v0);
    t1 = ck_top(v1);
  }
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

// x / s, correctly rounded, from inv = 1 / s correctly rounded (Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990: q + (x - q s) inv with fused operations).
// Near a tie of rint the product x * inv alone picks the further of two steps.
__device__ __forceinline__ float ck_quotient(float x, float s, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, s, x), inv, q);
}

// Codes of eight values.
template <int KIND, bool VEC, class Values>
__device__ __forceinline__ EightBytes<VEC, kCkLanes> ck_codes(const Values& x, float s, float inv) {
  EightBytes<VEC, kCkLanes> q;
  if constexpr (KIND == DG_KIND_E4M3) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q.half[i] = __nv_cvt_float2_to_fp8x2(make_float2(x.get(2 * i) * inv, x.get(2 * i + 1) * inv), __NV_SATFINITE, __NV_E4M3);
  } else {
    // Adding 1.5 * 2^23 rounds to a whole number (nearest, ties to even) and leaves it in the low bits;
    // |x| <= 127 s up to a rounding, so nothing lies beyond 127.
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = __float_as_uint(ck_quotient(x.get(i), s, inv) + 12582912.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      q.word[i] = __byte_perm(__byte_perm(n[4 * i], n[4 * i + 1], 0x0040), __byte_perm(n[4 * i + 2], n[4 * i + 3], 0x0040), 0x5410);
  }
  return q;
}

// The values that eight codes stand for, at most `most` in magnitude (NaN stays NaN): a value just
// below the largest of its type may have been rounded up to a code beyond it (255 to 256 of 2^120,
// say) and still comes back finite.
template <int KIND, bool VEC>
__device__ __forceinline__ void ck_values(const EightBytes<VEC, kCkLanes>& q, float s, float most, float (&v)[8]) {
  if constexpr (KIND == DG_KIND_E4M3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(q.half[i], __NV_E4M3)));
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
  } else {
    // byte + 128 under the exponent of 2^23: 8388608 + byte + 128
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = (__uint_as_float(__byte_perm(q.word[i / 4] ^ 0x80808080u, 0x4b000000u, 0x7440 + i % 4)) - 8388736.0f) * s;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(v[i]) : "f"(v[i]), "f"(most));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v[i]) : "f"(v[i]), "f"(-most));
  }
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

// A unit is 128 columns of one row, the work of 16 lanes; a block takes kCkUnits of them for each
// group of 16 lanes, all of whose loads are under way before the first is used.
constexpr int kCkUnits = 4;
constexpr int kCkGroups = kCkThreads / kCkLanes;
struct CkUnit {
  long long u, r;  // u: the unit; r: its row, -1 behind the last unit
  int b;           // its block of columns
};
template <int UNITS = kCkUnits>
__device__ __forceinline__ CkUnit ck_unit(int k, int rows, int blocks) {
  CkUnit w;
  w.u = ((long long)blockIdx.x * UNITS + k) * kCkGroups + threadIdx.x / kCkLanes;
  const long long all = (long long)rows * blocks;
  if (all <= 0xffffffffLL) {
    const uint32_t r = static_cast<uint32_t>(w.u) / static_cast<uint32_t>(blocks);
    w.r = r;
    w.b = static_cast<int>(static_cast<uint32_t>(w.u) - r * static_cast<uint32_t>(blocks));
  } else {
    w.r = w.u / blocks;
    w.b = static_cast<int>(w.u - w.r * blocks);
  }
  if (w.u >= all) w.r = -1;
  return w;
}

// Rows into a checkpoint.
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) checkpoint_rows_kernel(const CheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[kCkUnits];
  Eight<T, VEC, kCkLanes> v[kCkUnits];
#pragma unroll
  for (int k = 0; k < kCkUnits; ++k) {
    w[k] = ck_unit(k, p.rows, blocks);
    v[k].load(static_cast<const T*>(p.x) + (size_t)max(w[k].r, 0LL) * p.x_stride, w[k].b * kCkBlock, lane, p.H, w[k].r >= 0);
  }
#pragma unroll
  for (int k = 0; k < kCkUnits; ++k) {
    float s, inv;
    ck_scale<KIND>(ck_top(v[k]), s, inv);  // every lane takes part
    if (w[k].r < 0) continue;
    ck_codes<KIND, VEC>(v[k], s, inv).store(p.q + (size_t)w[k].r * p.H, w[k].b * kCkBlock, lane, p.H);
    if (lane == 0) p.scale[w[k].u] = s;
  }
}

// And out of it.
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) restore_rows_kernel(const CheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[kCkUnits];
  EightBytes<VEC, kCkLanes> q[kCkUnits];
  float s[kCkUnits];
#pragma unroll
  for (int k = 0; k < kCkUnits; ++k) {
    w[k] = ck_unit(k, p.rows, blocks);
    q[k].load(p.q + (size_t)max(w[k].r, 0LL) * p.H, w[k].b * kCkBlock, lane, p.H, w[k].r >= 0);
    s[k] = w[k].r >= 0 ? p.scale[w[k].u] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kCkUnits; ++k) {
    if (w[k].r < 0) continue;
    float f[8];
    ck_values<KIND, VEC>(q[k], s[k], ck_most<T>(), f);
    Eight<T, VEC, kCkLanes> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.set(i, f[i]);
    v.store(static_cast<T*>(p.out) + (size_t)w[k].r * p.H, w[k].b * kCkBlock, lane, p.H);
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

constexpr int kCkActUnits = 2;

template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) act_checkpoint_kernel(const ActCheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[kCkActUnits];
  bool skip[kCkActUnits];
  Eight<T, VEC, kCkLanes> g[kCkActUnits], up[kCkActUnits];
#pragma unroll
  for (int k = 0; k < kCkActUnits; ++k) {
    w[k] = ck_unit<kCkActUnits>(k, p.rows, blocks);
    skip[k] = w[k].r < 0 || (p.m_indices != nullptr && p.m_indices[w[k].r] < 0);
  }
#pragma unroll
  for (int k = 0; k < kCkActUnits; ++k) {
    const T* x = static_cast<const T*>(p.x) + (size_t)max(w[k].r, 0LL) * p.x_stride;
    g[k].load(x, w[k].b * kCkBlock, lane, p.H, !skip[k]);
    up[k].load(x + p.H, w[k].b * kCkBlock, lane, p.H, !skip[k]);
  }
#pragma unroll
  for (int k = 0; k < kCkActUnits; ++k) {
    float sg, ig, su, iu;
    uint32_t tg, tu;
    ck_top_of_two(g[k], up[k], tg, tu);  // every lane takes part
    ck_scale<KIND>(tg, sg, ig);
    ck_scale<KIND>(tu, su, iu);
    if (w[k].r < 0 || (skip[k] && !p.clear)) continue;
    const int c0 = w[k].b * kCkBlock;
    Eight<T, VEC, kCkLanes> a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a.set(i, ck_silu<T>(g[k].get(i)) * up[k].get(i));
    a.store(static_cast<T*>(p.act) + (size_t)w[k].r * p.H, c0, lane, p.H);
    uint8_t* q = p.q + (size_t)w[k].r * 2 * p.H;
    ck_codes<KIND, VEC>(g[k], sg, ig).store(q, c0, lane, p.H);
    ck_codes<KIND, VEC>(up[k], su, iu).store(q + p.H, c0, lane, p.H);
    if (lane == 0) {
      float* s = p.scale + (size_t)w[k].r * 2 * blocks;
      s[w[k].b] = sg;
      s[blocks + w[k].b] = su;
    }
  }
}

template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) act_checkpoint_grad_kernel(const ActCheckpointParams p) {
  const int lane = threadIdx.x & (kCkLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[kCkActUnits];
  bool skip[kCkActUnits];
  EightBytes<VEC, kCkLanes> qg[kCkActUnits], qu[kCkActUnits];
  Eight<T, VEC, kCkLanes> d[kCkActUnits];
  float sg[kCkActUnits], su[kCkActUnits];
#pragma unroll
  for (int k = 0; k < kCkActUnits; ++k) {
    w[k] = ck_unit<kCkActUnits>(k, p.rows, blocks);
    skip[k] = w[k].r < 0 || (p.m_indices != nullptr && p.m_indices[w[k].r] < 0);
  }
#pragma unroll
  for (int k = 0; k < kCkActUnits; ++k) {
    const size_t r = static_cast<size_t>(max(w[k].r, 0LL));
    const float* s = p.scale + r * 2 * blocks;
    const uint8_t* q = p.q + r * 2 * p.H;
    const int c0 = w[k].b * kCkBlock;
    qg[k].load(q, c0, lane, p.H, !skip[k]);
    qu[k].load(q + p.H, c0, lane, p.H, !skip[k]);
    d[k].load(static_cast<const T*>(p.dact) + r * p.dact_stride, c0, lane, p.H, !skip[k]);
    sg[k] = skip[k] ? 0.0f : s[w[k].b];
    su[k] = skip[k] ? 0.0f : s[blocks + w[k].b];
  }
#pragma unroll
  for (int k = 0; k < kCkActUnits; ++k) {
    if (w[k].r < 0 || (skip[k] && !p.clear)) continue;
    Eight<T, VEC, kCkLanes> dg, du, a;
    if (!skip[k]) {
      float gv[8], uv[8];
      ck_values<KIND, VEC>(qg[k], sg[k], kCkMaxF32, gv);
      ck_values<KIND, VEC>(qu[k], su[k], kCkMaxF32, uv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float dv = d[k].get(i);
        const float sig = ck_sigmoid<T>(gv[i]);
        const float silu = gv[i] * sig;
        dg.set(i, dv * uv[i] * sig * fmaf(gv[i], 1.0f - sig, 1.0f));
        du.set(i, dv * silu);
        a.set(i, silu * uv[i]);
      }
    }
    const int c0 = w[k].b * kCkBlock;
    T* dx = static_cast<T*>(p.dx) + (size_t)w[k].r * 2 * p.H;
    dg.store(dx, c0, lane, p.H);
    du.store(dx + p.H, c0, lane, p.H);
    if (p.act != nullptr) a.store(static_cast<T*>(p.act) + (size_t)w[k].r * p.H, c0, lane, p.H);
  }
}

}  // namespace dg
