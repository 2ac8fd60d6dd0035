// Device-side building blocks shared by the gfx950 kernels: element types, 16-byte
// vector loads/stores, wave64 cross-lane exchanges and fp32 helpers.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <stdint.h>

#include "../../include/tinyserve_amd.h"

namespace ts {

using f16 = _Float16;
using bf16 = __bf16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWave = 64;

// 16 bytes moved as one global_load_dwordx4 / global_store_dwordx4.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Pack16 {
  static constexpr int N = 16 / sizeof(T);
  union {
    u32x4 raw;
    T v[16 / sizeof(T)];
  };
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  return static_cast<float>(x);
}

template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  return static_cast<T>(x);  // round to nearest even for f16 and bf16
}

// from_f32 of a product or sum that is rounded to float32 first. Without the empty asm the compiler
// makes the operation and the conversion to f16 one v_fma_mixlo_f16, which rounds once, in some
// places and not in others, and the same values would come out differently by where they stand.
template <typename T>
__device__ __forceinline__ T round_f32(float x) {
  asm("" : "+v"(x));
  return from_f32<T>(x);
}

template <typename T>
__device__ __forceinline__ Pack16<T> load16(const T* p) {
  Pack16<T> r;
  r.raw = *reinterpret_cast<const u32x4*>(p);
  return r;
}

template <typename T>
__device__ __forceinline__ void store16(T* p, const Pack16<T>& x) {
  *reinterpret_cast<u32x4*>(p) = x.raw;
}

// 16 bytes at any address: the same global_load / store_dwordx4 (gfx950 takes unaligned ones).
typedef u32x4 u32x4_loose __attribute__((aligned(1), may_alias));

template <typename T>
__device__ __forceinline__ Pack16<T> load16_loose(const T* p) {
  Pack16<T> r;
  r.raw = *reinterpret_cast<const u32x4_loose*>(p);
  return r;
}

template <typename T>
__device__ __forceinline__ void store16_loose(T* p, const Pack16<T>& x) {
  *reinterpret_cast<u32x4_loose*>(p) = x.raw;
}

// x from the lane whose id is (this lane's id) XOR OFF. OFF < 32 stays inside a
// 32-lane half and uses ds_swizzle's xor mode (no address computation); OFF == 32
// crosses the halves through ds_bpermute.
template <int OFF>
__device__ __forceinline__ float xor_lane(float x) {
  static_assert(OFF > 0 && OFF <= 32 && (OFF & (OFF - 1)) == 0, "power-of-2 offset");
  if constexpr (OFF == 32) {
    return __shfl_xor(x, 32);
  } else {
    constexpr int pattern = (OFF << 10) | 0x1f;  // and_mask 31, or_mask 0, xor_mask OFF
    return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(x), pattern));
  }
}

#define TS_LDS __attribute__((address_space(3)))

// One direct-to-LDS load of 16 bytes per lane with a scalar base address and a 32-bit
// per-lane byte offset (global_load_lds_dwordx4 voffset, saddr): lane l's bytes land at
// dst + 16 l. Inline asm, since the compiler's wait-count pass would guard every later LDS
// read with a wait for all such loads in flight; the kernel orders them itself with counted
// waits before its barriers.
// M0 is bound through the asm operand, so the compiler sets it (one instruction) and
// knows it is taken.
__device__ __forceinline__ void lds_load16_s(const void* base, uint32_t voff, TS_LDS void* dst) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(dst));
  asm volatile("global_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(base), "{m0}"(lds) : "memory");
#endif
}

// Wait until at most N of this wave's vector-memory operations are in flight and all its
// LDS operations are done, then meet the other waves at s_barrier. __syncthreads() would
// also fence workgroup memory, which waits for every load in flight (vmcnt(0)) and so
// drains the ring; the tiles' visibility needs only each wave's own counted wait. The
// signal fences (no instructions) keep the compiler from moving memory accesses across.
template <int N>
__device__ __forceinline__ void ring_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  // vmcnt N (bits 3:0 and 15:14), expcnt 7 (no wait), lgkmcnt 0
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Sum / max over groups of N consecutive lanes (N a power of 2 <= 64); every lane of a
// group ends with the group's total.
template <int N>
__device__ __forceinline__ float group_sum(float x) {
  if constexpr (N >= 2) x += xor_lane<1>(x);
  if constexpr (N >= 4) x += xor_lane<2>(x);
  if constexpr (N >= 8) x += xor_lane<4>(x);
  if constexpr (N >= 16) x += xor_lane<8>(x);
  if constexpr (N >= 32) x += xor_lane<16>(x);
  if constexpr (N >= 64) x += xor_lane<32>(x);
  return x;
}

// Max / sum of x over lanes l and l ^ 32 (the two 32-lane halves), via gfx950's
// v_permlane32_swap: with both operands x, one result holds x of this lane and the other
// x of the partner lane (in either order per half), so max/sum of the pair is the answer.
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// RMSNorm's output element: y = (T)(x * r) * w, the multiply by w in T's precision (exact
// product, one rounding), as layers.py:14-38 computes it in the model dtype.
template <typename T>
__device__ __forceinline__ T norm_scale(T x, float r, T w) {
  const T xn = from_f32<T>(to_f32(x) * r);
  return from_f32<T>(to_f32(xn) * to_f32(w));
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

inline int ilog2(int x) {
  int r = 0;
  while ((1 << r) < x) ++r;
  return r;
}

inline bool is_pow2(int x) { return x > 0 && (x & (x - 1)) == 0; }

inline int elem_size(int dtype) { return dtype == TS_F32 ? 4 : 2; }

// Compute units of the current device (cached per device; 256 on MI355X).
inline int compute_units() {
  static std::atomic<int> cache[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 256;
  if (dev < 64) {
    const int hit = cache[dev].load(std::memory_order_relaxed);
    if (hit > 0) return hit;
  }
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    n = 256;
  if (dev < 64) cache[dev].store(n, std::memory_order_relaxed);
  return n;
}

inline int launch_status() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : static_cast<int>(e);
}

}  // namespace ts
