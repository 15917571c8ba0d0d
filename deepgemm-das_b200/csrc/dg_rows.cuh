// Rows of bf16 / fp16 / fp32 values as the memory-bound kernels of a training step handle them:
// eight values of a row per thread, through 16-byte accesses where every row starts on a 16-byte
// boundary and ends on one, value by value where not.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "deepgemm_b200.h"

namespace dg {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// 16 (8) bytes that are read once, or zeros where `on` is false (nothing is read).  One predicated
// instruction and volatile: several of these in a row stay together in front of their first use.
// Written as a branch around a plain load, the compiler moved each load and what uses it into the
// branch, which put eight memory latencies behind one another in the gradient of the way back
// (380 us instead of 180).
__device__ __forceinline__ uint4 load_once(const void* p, bool on) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred on;\n\tsetp.ne.u32 on, %5, 0;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
      "@on ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"(static_cast<uint32_t>(on)));
  return v;
}
__device__ __forceinline__ uint2 load_once8(const void* p, bool on) {
  uint2 v;
  asm volatile(
      "{\n\t.reg .pred on;\n\tsetp.ne.u32 on, %3, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t"
      "@on ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];\n\t}"
      : "=&r"(v.x), "=&r"(v.y)
      : "l"(p), "r"(static_cast<uint32_t>(on)));
  return v;
}

// One value of two or four bytes, likewise.
template <class T>
__device__ __forceinline__ T load_value(const T* p, bool on) {
  T v;
  if constexpr (sizeof(T) == 4) {
    uint32_t b;
    asm volatile(
        "{\n\t.reg .pred on;\n\tsetp.ne.u32 on, %2, 0;\n\tmov.u32 %0, 0;\n\t@on ld.global.nc.u32 %0, [%1];\n\t}"
        : "=&r"(b)
        : "l"(p), "r"(static_cast<uint32_t>(on)));
    v = *reinterpret_cast<const T*>(&b);
  } else {
    uint16_t b;
    asm volatile(
        "{\n\t.reg .pred on;\n\tsetp.ne.u32 on, %2, 0;\n\tmov.u16 %0, 0;\n\t@on ld.global.nc.u16 %0, [%1];\n\t}"
        : "=&h"(b)
        : "l"(p), "r"(static_cast<uint32_t>(on)));
    v = *reinterpret_cast<const T*>(&b);
  }
  return v;
}

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight values of the 8 * LANES columns that begin at column c0, held by lane `lane` of LANES:
// VEC: columns c0 + 8 * lane + i (c0, the row length and the row's address are multiples of 16
// bytes); otherwise columns c0 + lane + LANES * i, so that a warp's accesses stay side by side.
template <class T, bool VEC, int LANES>
struct Eight {
  union {
    uint4 raw[sizeof(T) / 2];
    T val[8];
  };
  __device__ __forceinline__ Eight() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  static __device__ __forceinline__ int col(int c0, int lane, int i) {
    return VEC ? c0 + 8 * lane + i : c0 + lane + LANES * i;
  }
  // columns at or beyond `cols` are zero, and all of them where `on` is false
  __device__ __forceinline__ void load(const T* row, int c0, int lane, int cols, bool on = true) {
    if constexpr (VEC) {
      const int c = c0 + 8 * lane;
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        raw[i] = load_once(reinterpret_cast<const uint4*>(row + c) + i, on && c < cols);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + lane + LANES * i;
        val[i] = load_value(row + c, on && c < cols);
      }
    }
  }
  // kStream: the lines leave L2 before others when room is needed (a result that does not fit there
  // anyway costs 3 to 6 % less time; a small one stays all the same).
  template <bool kStream = false>
  __device__ __forceinline__ void store(T* row, int c0, int lane, int cols) const {
    if constexpr (VEC) {
      const int c = c0 + 8 * lane;
      if (c < cols) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
          if constexpr (kStream) __stcs(reinterpret_cast<uint4*>(row + c) + i, raw[i]);
          else *(reinterpret_cast<uint4*>(row + c) + i) = raw[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + lane + LANES * i;
        if (c < cols) row[c] = val[i];
      }
    }
  }
  __device__ __forceinline__ float get(int i) const { return to_f32(val[i]); }
  __device__ __forceinline__ void set(int i, float v) { val[i] = from_f32<T>(v); }  // round to nearest even
  __device__ __forceinline__ void set2(int i, float a, float b) {                   // i and i + 1 (i even)
    if constexpr (sizeof(T) == 4) {
      set(i, a);
      set(i + 1, b);
    } else {
      reinterpret_cast<uint32_t*>(raw)[i / 2] = pack2(a, b, T());
    }
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Eight 8-bit codes, columns c0 + 8 * lane + i, in one 8-byte access.
struct EightBytes {
  union {
    uint2 raw;
    uint32_t word[2];
    uint16_t half[4];
  };
  __device__ __forceinline__ EightBytes() { raw = make_uint2(0u, 0u); }
  __device__ __forceinline__ void load(const uint8_t* row, int c0, int lane, int cols, bool on) {
    const int c = c0 + 8 * lane;
    raw = load_once8(row + c, on && c < cols);
  }
  __device__ __forceinline__ void store(uint8_t* row, int c0, int lane, int cols) const {
    const int c = c0 + 8 * lane;
    if (c < cols) __stcs(reinterpret_cast<uint2*>(row + c), raw);  // not read again soon
  }
};

}  // namespace dg
