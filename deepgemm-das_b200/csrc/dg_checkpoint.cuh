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
// HBM moves 8 bytes per activation forward (4 read, 2 + 2 written) and 10 backward (2 + 2 read, 4 + 2
// written); with that little work per byte the instructions count as much as the bytes.  So 8 lanes
// hold the 128 columns of one scale, sixteen each (what a block of columns costs once, its
// address, exchanges between lanes and scale, is spread over twice the columns that 16 lanes give:
// forward 117 -> 99 us, backward 128 -> 113, rows to int8 89 -> 68), 16-bit magnitudes are compared two at a time and codes are made
// and read two (e4m3) or four (int8) at a time.
#pragma once

#include <cuda_fp8.h>

#include <string.h>

#include <type_traits>

#include "dg_rows.cuh"

namespace dg {

constexpr int kCkBlock = 128;    // columns of one scale
constexpr int kCkThreads = 256;

// What a lane holds of a block's 128 columns.  VEC: 8 lanes, each eight of the first 64 columns and
// eight of the others.  Otherwise (rows that begin anywhere) 32 lanes, columns lane, lane + 32, ...,
// so that a warp's accesses of single values lie side by side.
template <class T, bool VEC>
struct CkValues {
  static constexpr int kLanes = 8, N = 16;
  Eight<T, true, 8> h[2];
  __device__ __forceinline__ void load(const T* row, int c0, int lane, int cols, bool on) {
    h[0].load(row, c0, lane, cols, on);
    h[1].load(row, c0 + 64, lane, cols, on);
  }
  __device__ __forceinline__ void store(T* row, int c0, int lane, int cols) const {
    h[0].template store<true>(row, c0, lane, cols);
    h[1].template store<true>(row, c0 + 64, lane, cols);
  }
  __device__ __forceinline__ float get(int i) const { return h[i / 8].get(i % 8); }
  __device__ __forceinline__ void set2(int i, float a, float b) { h[i / 8].set2(i % 8, a, b); }
  __device__ __forceinline__ uint32_t pair(int i) const { return reinterpret_cast<const uint32_t*>(h[i / 4].raw)[i % 4]; }
};
template <class T>
struct CkValues<T, false> {
  static constexpr int kLanes = 32, N = 4;
  T val[4] = {T(), T(), T(), T()};
  __device__ __forceinline__ void load(const T* row, int c0, int lane, int cols, bool on) {
#pragma unroll
    for (int i = 0; i < 4; ++i) val[i] = load_value(row + c0 + lane + 32 * i, on && c0 + lane + 32 * i < cols);
  }
  __device__ __forceinline__ void store(T* row, int c0, int lane, int cols) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c0 + lane + 32 * i < cols) row[c0 + lane + 32 * i] = val[i];
  }
  __device__ __forceinline__ float get(int i) const { return to_f32(val[i]); }
  __device__ __forceinline__ void set2(int i, float a, float b) {
    val[i] = from_f32<T>(a);
    val[i + 1] = from_f32<T>(b);
  }
  __device__ __forceinline__ uint32_t pair(int i) const {
    const T two[2] = {val[2 * i], val[2 * i + 1]};
    uint32_t v;
    memcpy(&v, two, 4);
    return v;
  }
};
template <bool VEC>
struct CkCodes {
  EightBytes h[2];
  __device__ __forceinline__ void load(const uint8_t* row, int c0, int lane, int cols, bool on) {
    h[0].load(row, c0, lane, cols, on);
    h[1].load(row, c0 + 64, lane, cols, on);
  }
  __device__ __forceinline__ void store(uint8_t* row, int c0, int lane, int cols) const {
    h[0].store(row, c0, lane, cols);
    h[1].store(row, c0 + 64, lane, cols);
  }
  __device__ __forceinline__ uint16_t& two(int i) { return h[i / 4].half[i % 4]; }
  __device__ __forceinline__ uint16_t two(int i) const { return h[i / 4].half[i % 4]; }
  __device__ __forceinline__ uint32_t& four(int i) { return h[i / 2].word[i % 2]; }
  __device__ __forceinline__ uint32_t four(int i) const { return h[i / 2].word[i % 2]; }
};
template <>
struct CkCodes<false> {
  uint32_t word = 0;
  __device__ __forceinline__ void load(const uint8_t* row, int c0, int lane, int cols, bool on) {
    word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (on && c0 + lane + 32 * i < cols) word |= static_cast<uint32_t>(row[c0 + lane + 32 * i]) << (8 * i);
  }
  __device__ __forceinline__ void store(uint8_t* row, int c0, int lane, int cols) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c0 + lane + 32 * i < cols) row[c0 + lane + 32 * i] = static_cast<uint8_t>(word >> (8 * i));
  }
  __device__ __forceinline__ uint16_t& two(int i) { return reinterpret_cast<uint16_t*>(&word)[i]; }
  __device__ __forceinline__ uint16_t two(int i) const { return static_cast<uint16_t>(word >> (16 * i)); }
  __device__ __forceinline__ uint32_t& four(int) { return word; }
  __device__ __forceinline__ uint32_t four(int) const { return word; }
};

// The largest magnitude of 128 columns, over the lanes that hold them, as the bits of an fp32
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
__device__ __forceinline__ uint32_t ck_lane_max(const CkValues<T, VEC>& v) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < v.N / 2; ++i) m = ck_max2(m, v.pair(i) & 0x7fff7fffu);
    return max(m >> 16, m & 0xffffu);
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < v.N; ++i) m = max(m, __float_as_uint(v.get(i)) & 0x7fffffffu);
    return m;
  }
}
template <class T, bool VEC>
__device__ __forceinline__ uint32_t ck_top(const CkValues<T, VEC>& v) {
  uint32_t m = ck_lane_max(v);
#pragma unroll
  for (int o = v.kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return ck_bits16<T>(m);
}
template <class T, bool VEC>
__device__ __forceinline__ void ck_top_of_two(const CkValues<T, VEC>& v0, const CkValues<T, VEC>& v1, uint32_t& t0, uint32_t& t1) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = (ck_lane_max(v0) << 16) | ck_lane_max(v1);
#pragma unroll
    for (int o = v0.kLanes / 2; o > 0; o >>= 1) m = ck_max2(m, __shfl_xor_sync(0xffffffffu, m, o));
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

// Codes of a lane's values.
template <int KIND, class T, bool VEC>
__device__ __forceinline__ CkCodes<VEC> ck_codes(const CkValues<T, VEC>& x, float s, float inv) {
  CkCodes<VEC> q;
  if constexpr (KIND == DG_KIND_E4M3) {
#pragma unroll
    for (int i = 0; i < x.N / 2; ++i)
      q.two(i) = __nv_cvt_float2_to_fp8x2(make_float2(x.get(2 * i) * inv, x.get(2 * i + 1) * inv), __NV_SATFINITE, __NV_E4M3);
  } else {
    // Adding 1.5 * 2^23 rounds to a whole number (nearest, ties to even) and leaves it in the low bits;
    // |x| <= 127 s up to a rounding, so nothing lies beyond 127.
#pragma unroll
    for (int i = 0; i < x.N / 4; ++i) {
      uint32_t n[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] = __float_as_uint(ck_quotient(x.get(4 * i + k), s, inv) + 12582912.0f);
      q.four(i) = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    }
  }
  return q;
}

// The values that a lane's codes stand for, at most `most` in magnitude (NaN stays NaN): a value just
// below the largest of its type may have been rounded up to a code beyond it (255 to 256 of 2^120,
// say) and still comes back finite.
template <int KIND, bool VEC, int N>
__device__ __forceinline__ void ck_values(const CkCodes<VEC>& q, float s, float most, float (&v)[N]) {
  if constexpr (KIND == DG_KIND_E4M3) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(q.two(i), __NV_E4M3)));
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
  } else {
    // byte + 128 under the exponent of 2^23: 8388608 + byte + 128
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = (__uint_as_float(__byte_perm(q.four(i / 4) ^ 0x80808080u, 0x4b000000u, 0x7440 + i % 4)) - 8388736.0f) * s;
  }
  if (448.0f * s > most) {  // (no code stands for more than 448 s; not so for NaN, which stays)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fminf(fmaxf(v[i], -most), most);
  }
}
template <class T>
__device__ __forceinline__ float ck_most();
template <>
__device__ __forceinline__ float ck_most<float>() { return 3.402823466e+38f; }
template <>
__device__ __forceinline__ float ck_most<__half>() { return 65504.0f; }
template <>
__device__ __forceinline__ float ck_most<__nv_bfloat16>() { return 3.3895313892515355e+38f; }

// 1 / (1 + exp(-g)).  16-bit results take the hardware's 2^x and reciprocal without their handling
// of subnormal numbers (exp(-g) below 2^-126 disappears beside the 1, a sigmoid below 2^-126 is 0),
// 32-bit ones the exact forms.
template <class T>
__device__ __forceinline__ float ck_sigmoid(float g) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
template <class T>
__device__ __forceinline__ float ck_silu(float g) {
  if constexpr (sizeof(T) == 4) return g / (1.0f + expf(-g));
  return g * ck_sigmoid<T>(g);
}

struct CheckpointParams {
  const void* x;    // [rows] rows of H values (restore: written)
  uint8_t* q;       // [rows][H]
  float* scale;     // [rows][blocks]
  void* out;        // restore: [rows][H]
  int rows, H;
  long long x_stride;
};

// A unit is 128 columns of one row, the work of 8 lanes; a block takes kCkUnits of them for each
// group of 8 lanes, all of whose loads are under way before the first is used.
template <bool VEC>
constexpr int kCkUnits = VEC ? 1 : 2;
struct CkUnit {
  long long u, r;  // u: the unit; r: its row, -1 behind the last unit
  int b;           // its block of columns
};
template <int LANES, int UNITS>
__device__ __forceinline__ CkUnit ck_unit(int k, int rows, int blocks) {
  CkUnit w;
  w.u = ((long long)blockIdx.x * UNITS + k) * (kCkThreads / LANES) + threadIdx.x / LANES;
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

// Rows into a checkpoint.  16383 x 7168 bf16: e4m3 59.7 us (5.9 TB/s), int8 66.6 (5.3; its quotients
// keep the schedulers busy 84 % of the time).
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) checkpoint_rows_kernel(const CheckpointParams p) {
  constexpr int kLanes = CkValues<T, VEC>::kLanes, U = kCkUnits<VEC>;
  const int lane = threadIdx.x & (kLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[U];
  CkValues<T, VEC> v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    w[k] = ck_unit<kLanes, U>(k, p.rows, blocks);
    v[k].load(static_cast<const T*>(p.x) + (size_t)max(w[k].r, 0LL) * p.x_stride, w[k].b * kCkBlock, lane, p.H, w[k].r >= 0);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    float s, inv;
    ck_scale<KIND>(ck_top(v[k]), s, inv);  // every lane takes part
    if (w[k].r < 0) continue;
    ck_codes<KIND>(v[k], s, inv).store(p.q + (size_t)w[k].r * p.H, w[k].b * kCkBlock, lane, p.H);
    if (lane == 0) p.scale[w[k].u] = s;
  }
}

// And out of it: 55.5 us (6.3 TB/s) from int8, 55.6 from e4m3.
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) restore_rows_kernel(const CheckpointParams p) {
  constexpr int kLanes = CkValues<T, VEC>::kLanes, N = CkValues<T, VEC>::N, U = kCkUnits<VEC>;
  const int lane = threadIdx.x & (kLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[U];
  CkCodes<VEC> q[U];
  float s[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    w[k] = ck_unit<kLanes, U>(k, p.rows, blocks);
    q[k].load(p.q + (size_t)max(w[k].r, 0LL) * p.H, w[k].b * kCkBlock, lane, p.H, w[k].r >= 0);
    s[k] = w[k].r >= 0 ? p.scale[w[k].u] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    if (w[k].r < 0) continue;
    float f[N];
    ck_values<KIND, VEC>(q[k], s[k], ck_most<T>(), f);
    CkValues<T, VEC> v;
#pragma unroll
    for (int i = 0; i < N; i += 2) v.set2(i, f[i], f[i + 1]);
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

// Activation and checkpoint.  32768 rows of 2 x 2048 bf16 (and as much padding as 32 experts have) to
// e4m3: 92.5 us = 6.2 TB/s; int8 102.8; rows of 2 x 2043, value by value, 215.
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) act_checkpoint_kernel(const ActCheckpointParams p) {
  constexpr int kLanes = CkValues<T, VEC>::kLanes, N = CkValues<T, VEC>::N, U = kCkActUnits;
  const int lane = threadIdx.x & (kLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[U];
  bool skip[U];
  CkValues<T, VEC> g[U], up[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    w[k] = ck_unit<kLanes, U>(k, p.rows, blocks);
    skip[k] = w[k].r < 0 || (p.m_indices != nullptr && p.m_indices[w[k].r] < 0);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const T* x = static_cast<const T*>(p.x) + (size_t)max(w[k].r, 0LL) * p.x_stride;
    g[k].load(x, w[k].b * kCkBlock, lane, p.H, !skip[k]);
    up[k].load(x + p.H, w[k].b * kCkBlock, lane, p.H, !skip[k]);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    float sg, ig, su, iu;
    uint32_t tg, tu;
    ck_top_of_two(g[k], up[k], tg, tu);  // every lane takes part
    ck_scale<KIND>(tg, sg, ig);
    ck_scale<KIND>(tu, su, iu);
    if (w[k].r < 0 || (skip[k] && !p.clear)) continue;
    const int c0 = w[k].b * kCkBlock;
    CkValues<T, VEC> a;
#pragma unroll
    for (int i = 0; i < N; i += 2)
      a.set2(i, ck_silu<T>(g[k].get(i)) * up[k].get(i), ck_silu<T>(g[k].get(i + 1)) * up[k].get(i + 1));
    a.store(static_cast<T*>(p.act) + (size_t)w[k].r * p.H, c0, lane, p.H);
    uint8_t* q = p.q + (size_t)w[k].r * 2 * p.H;
    ck_codes<KIND>(g[k], sg, ig).store(q, c0, lane, p.H);
    ck_codes<KIND>(up[k], su, iu).store(q + p.H, c0, lane, p.H);
    if (lane == 0) {
      float* s = p.scale + (size_t)w[k].r * 2 * blocks;
      s[w[k].b] = sg;
      s[blocks + w[k].b] = su;
    }
  }
}

// Backward from the checkpoint: 108.9 us = 6.6 TB/s for the same rows.  Gate and up are at most
// the largest finite value of their type, as in restore_rows_kernel: an fp16 65504 that is held as
// 65536 does not overflow the activation it is multiplied into.
template <class T, bool VEC, int KIND>
__global__ void __launch_bounds__(kCkThreads) act_checkpoint_grad_kernel(const ActCheckpointParams p) {
  constexpr int kLanes = CkValues<T, VEC>::kLanes, N = CkValues<T, VEC>::N, U = kCkActUnits;
  const int lane = threadIdx.x & (kLanes - 1);
  const int blocks = (p.H + kCkBlock - 1) / kCkBlock;
  CkUnit w[U];
  bool skip[U];
  CkCodes<VEC> qg[U], qu[U];
  CkValues<T, VEC> d[U];
  float sg[U], su[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    w[k] = ck_unit<kLanes, U>(k, p.rows, blocks);
    skip[k] = w[k].r < 0 || (p.m_indices != nullptr && p.m_indices[w[k].r] < 0);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
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
  for (int k = 0; k < U; ++k) {
    if (w[k].r < 0 || (skip[k] && !p.clear)) continue;
    CkValues<T, VEC> dg, du, a;
    if (!skip[k]) {
      float gv[N], uv[N];
      ck_values<KIND, VEC>(qg[k], sg[k], ck_most<T>(), gv);
      ck_values<KIND, VEC>(qu[k], su[k], ck_most<T>(), uv);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        float fg[2], fu[2], fa[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float dv = d[k].get(i + j), gj = gv[i + j], uj = uv[i + j];
          const float sig = ck_sigmoid<T>(gj);
          const float silu = gj * sig;
          fg[j] = dv * uj * sig * fmaf(gj, 1.0f - sig, 1.0f);
          fu[j] = dv * silu;
          fa[j] = silu * uj;
        }
        dg.set2(i, fg[0], fg[1]);
        du.set2(i, fu[0], fu[1]);
        a.set2(i, fa[0], fa[1]);
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
