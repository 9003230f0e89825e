// head_common.hpp -- what the detection head's operators share: element types, vector loads, rounding.
//
// These operators are held to their formulas in 64 bits, not to a bit pattern: unlike the proposal path they may use fused
// multiply-adds (written out, the library is built with -ffp-contract=off) and the hardware's exp2 / rcp.  Every sum and
// statistic is held in fp32; a value is rounded to its tensor's type once, at the store.
#pragma once

#include "common.hpp"

namespace frcnn {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

static const int kQuantBlock = 128;          // elements per scale along a row
static const float kE4M3Max = 448.0f;        // largest finite e4m3

static const long long kGridThreads = (1ll << 32) - 1;  // threads of one launch at most

static inline size_t type_bytes(int type) { return type == FRCNN_F32 ? 4 : 2; }
static inline bool type_known(int type) { return type == FRCNN_F32 || type == FRCNN_F16 || type == FRCNN_BF16; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }

// VEC elements of T as they lie in memory: 16 bytes (VEC = 16 / sizeof(T)) or one element (VEC = 1, for rows whose start
// or length is not a multiple of 16 bytes).
template <typename T, int VEC>
struct Pack {
  static_assert(VEC * sizeof(T) == 16, "a pack is 16 bytes or one element");
  u32x4 w;
  __device__ __forceinline__ static Pack load(const T *p) { return Pack{*reinterpret_cast<const u32x4 *>(p)}; }
  __device__ __forceinline__ static Pack zero() { return Pack{u32x4{0, 0, 0, 0}}; }
  __device__ __forceinline__ void unpack(float (&f)[VEC]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = u2f(w[i]);
    } else if constexpr (__is_same(T, __bf16)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = u2f(w[i] << 16);
        f[2 * i + 1] = u2f(w[i] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = w[i];  // a value of its own: the cast of a vector element reads element 0
        const f16x2 h = __builtin_bit_cast(f16x2, u);
        f[2 * i] = (float)h.x;
        f[2 * i + 1] = (float)h.y;
      }
    }
  }
  __device__ __forceinline__ static u32x4 packed(const float (&f)[VEC]) {
    u32x4 o;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = f2u(f[i]);
    } else if constexpr (__is_same(T, __bf16)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)f[2 * i], (__bf16)f[2 * i + 1]});
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
    }
    return o;
  }
  // PAST: past the caches, for results that fill whole lines
  template <bool PAST = false>
  __device__ __forceinline__ static void store(T *p, const float (&f)[VEC]) {
    if constexpr (PAST)
      __builtin_nontemporal_store(packed(f), reinterpret_cast<u32x4 *>(p));
    else
      *reinterpret_cast<u32x4 *>(p) = packed(f);
  }
};

template <typename T>
struct Pack<T, 1> {
  T w;
  __device__ __forceinline__ static Pack load(const T *p) { return Pack{*p}; }
  __device__ __forceinline__ static Pack zero() { return Pack{(T)0.0f}; }
  __device__ __forceinline__ void unpack(float (&f)[1]) const { f[0] = to_float(w); }
  template <bool PAST = false>
  __device__ __forceinline__ static void store(T *p, const float (&f)[1]) { *p = (T)f[0]; }
};

// Workgroups are dealt to the 8 XCDs in turn; this order gives each XCD a contiguous range of n places.
__device__ __forceinline__ int xcd_contiguous(int i, int n) {
  const int x = i & 7, base = n >> 3, more = n & 7;
  return x * base + min(x, more) + (i >> 3);
}

}  // namespace frcnn
