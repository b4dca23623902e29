// What the row and page kernels (embedding.hip, pages.hip) share: accesses of 16 bytes at any alignment, element
// types widened to 32-bit floats and rounded back once, and the hooks of the host build that runs them with one
// thread per GPU thread.
#pragma once

#include <hip/hip_runtime.h>

#include "reduce_ops.h"

// the workgroup's one LDS object (a host build that emulates workgroups with threads supplies its own definition)
#ifndef DFCCL_WG_SHARED
#define DFCCL_WG_SHARED(T, name) __shared__ T name
#endif
// between the lanes of one wave that hand values to each other through LDS: see daemon.hip
#ifndef DFCCL_WAVE_LDS_SYNC
#define DFCCL_WAVE_LDS_SYNC()                              \
  do {                                                     \
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront"); \
    __builtin_amdgcn_wave_barrier();                       \
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront"); \
  } while (0)
#endif
// the value, loaded, is here from this place on: loads whose values several such statements in a row name are waited for
// together, where the compiler would move one behind a branch that only needs the other
#ifndef DFCCL_LOADED
#define DFCCL_LOADED(v) asm volatile("" : "+v"(v))
#endif
// a launch whose workgroups do not wait for each other (the host build runs a few of them at a time)
#ifndef DFCCL_LAUNCH_BLOCKS
#define DFCCL_LAUNCH_BLOCKS(kernel, grid, block, stream, ...) \
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(block), 0, stream, __VA_ARGS__)
#endif

namespace dfccl {

// 16 bytes at an address that is only aligned to A bytes. The hardware takes such addresses in one instruction
// (the compiler knows that and does not split the access), so rows whose length or stride is odd need no path of
// their own.
template <int A>
struct Pack16;
template <>
struct Pack16<1> {
  typedef u32x4 type __attribute__((aligned(1)));
};
template <>
struct Pack16<2> {
  typedef u32x4 type __attribute__((aligned(2)));
};
template <>
struct Pack16<4> {
  typedef u32x4 type __attribute__((aligned(4)));
};
// NT: what is not used again soon does not stay in the caches
template <int A, bool NT = false>
__device__ __forceinline__ u32x4 load16(const char* p) {
  if constexpr (NT) return __builtin_nontemporal_load((const DFCCL_GLOBAL typename Pack16<A>::type*)p);
  else return *(const DFCCL_GLOBAL typename Pack16<A>::type*)p;
}
template <int A, bool NT = false>
__device__ __forceinline__ void store16(char* p, u32x4 v) {
  if constexpr (NT) __builtin_nontemporal_store(v, (DFCCL_GLOBAL typename Pack16<A>::type*)p);
  else *(DFCCL_GLOBAL typename Pack16<A>::type*)p = v;
}

__device__ __forceinline__ int waveInBlock() {  // the same in every lane: say so
  return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
}

// a value that every lane of the wave holds alike: kept in scalar registers from there on
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)uniform((uint32_t)((uint64_t)v >> 32)) << 32) | uniform((uint32_t)v));
}

// ---- eight elements of a floating type, as 32-bit floats
constexpr int kVec = 8;

template <int DT>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (DT == kF32) return __uint_as_float(bits);
  else if constexpr (DT == kBF16) return __uint_as_float(bits << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
// round to nearest even
template <int DT>
__device__ __forceinline__ uint32_t narrow(float x) {
  if constexpr (DT == kF32) return __float_as_uint(x);
  else if constexpr (DT == kF16) return __builtin_bit_cast(uint16_t, (_Float16)x);
  else {
    f32x2 two;
    two.x = x;
    two.y = 0.0f;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2)) & 0xffffu;
  }
}
template <int DT>
__device__ __forceinline__ void widenWord(uint32_t w, float& lo, float& hi) {
  if constexpr (DT == kBF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const f16x2 two = __builtin_bit_cast(f16x2, w);
    lo = (float)two.x;
    hi = (float)two.y;
  }
}
template <int DT>
__device__ __forceinline__ uint32_t narrowWord(float lo, float hi) {
  f32x2 two;
  two.x = lo;
  two.y = hi;
  if constexpr (DT == kBF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(two, f16x2));
}

// the raw words of eight elements: four for the 16-bit types, eight for fp32
template <int DT>
struct Raw8 {
  u32x4 w[typeSize(DT) / 2];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> loadRaw8(const char* p) {
  Raw8<DT> r;
  r.w[0] = load16<typeSize(DT)>(p);
  if constexpr (DT == kF32) r.w[1] = load16<4>(p + 16);
  return r;
}
template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float (&f)[kVec]) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      f[i] = __uint_as_float(r.w[0][i]);
      f[4 + i] = __uint_as_float(r.w[1][i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) widenWord<DT>(r.w[0][i], f[2 * i], f[2 * i + 1]);
  }
}
template <int DT>
__device__ __forceinline__ Raw8<DT> narrow8(const float (&f)[kVec]) {  // to nearest even
  Raw8<DT> r;
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      r.w[0][i] = __float_as_uint(f[i]);
      r.w[1][i] = __float_as_uint(f[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) r.w[0][i] = narrowWord<DT>(f[2 * i], f[2 * i + 1]);
  }
  return r;
}
template <int DT, bool NT = false>
__device__ __forceinline__ void store8(char* p, const float (&f)[kVec]) {
  const Raw8<DT> r = narrow8<DT>(f);
  store16<typeSize(DT), NT>(p, r.w[0]);
  if constexpr (DT == kF32) store16<4, NT>(p + 16, r.w[1]);
}
// the last, shorter vector of a row: `left` elements (1..7)
template <int DT>
__device__ __forceinline__ void loadTail(const char* p, int left, float (&f)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; i++) f[i] = i < left ? widen<DT>((uint32_t)loadElem<typeSize(DT)>(p, i)) : 0.0f;
}
template <int DT>
__device__ __forceinline__ void storeTail(char* p, int left, const float (&f)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; i++)
    if (i < left) storeElem<typeSize(DT)>(p, i, narrow<DT>(f[i]));
}

}  // namespace dfccl
