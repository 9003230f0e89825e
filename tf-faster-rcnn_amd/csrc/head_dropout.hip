// head_dropout.hip -- dropout whose mask is computed, never stored.
//
// Element i of the tensor (row-major order) keeps its value iff word i % 4 of block i / 4 of the generator is at least
// round(rate * 2^32); the kept ones are multiplied by 1 / (1 - rate).  The generator is Philox4x32 (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with 7 rounds, the fewest that the authors report passing all
// of BigCrush: key = the seed, counter = (block index, offset), both 64 bits.  The gradient is the same function of dy.
//
// Bound by memory: one read and one write of the tensor.  The rounds cost 14 full 32x32 products per four elements.
#include "head_common.hpp"

namespace frcnn {

struct PhiloxKeys {  // the seven round keys
  uint32_t k0[7], k1[7];
};

__device__ __forceinline__ PhiloxKeys philox_keys(uint64_t seed) {
  PhiloxKeys k;
  uint32_t a = (uint32_t)seed, b = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    k.k0[r] = a;
    k.k1[r] = b;
    a += 0x9E3779B9u;
    b += 0xBB67AE85u;
  }
  return k;
}

__device__ __forceinline__ u32x4 philox4x32_7(uint64_t block, uint64_t offset, const PhiloxKeys &k) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ k.k0[r];
    c1 = (uint32_t)q;
    c2 = (uint32_t)(p >> 32) ^ c3 ^ k.k1[r];
    c3 = (uint32_t)p;
  }
  return u32x4{c0, c1, c2, c3};
}

// One pack of VEC elements per thread and step (VEC = 4 with element loads where a pointer is not 16-byte aligned).
template <typename T, int VEC, bool ALIGNED>
__global__ __launch_bounds__(256) void dropout_kernel(const T *__restrict__ x, T *__restrict__ y, long long count,
                                                      uint32_t threshold, float scale, uint64_t seed, uint64_t offset,
                                                      const uint64_t *__restrict__ state) {
  if (state) {  // uniform: a device-held (seed, offset) pair, so that a captured graph can draw anew on each replay
    seed = state[0];
    offset = state[1];
  }
  const PhiloxKeys keys = philox_keys(seed);
  const long long packs = (count + VEC - 1) / VEC;
  const long long stride = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < packs; i += stride) {
    const long long at = i * VEC;
    const bool whole = ALIGNED && at + VEC <= count;
    float f[VEC];
    if constexpr (ALIGNED) {
      if (whole) Pack<T, VEC>::load(x + at).unpack(f);
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = at + e < count ? to_float(x[at + e]) : 0.0f;
    }
#pragma unroll
    for (int b = 0; b < VEC / 4; ++b) {
      const u32x4 r = philox4x32_7((uint64_t)(at / 4 + b), offset, keys);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * b + e] = r[e] >= threshold ? f[4 * b + e] * scale : 0.0f;
    }
    if constexpr (ALIGNED) {
      if (whole) Pack<T, VEC>::store(y + at, f);
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (at + e < count) y[at + e] = (T)f[e];
    }
  }
}

// Where rate * 2^32 rounds to 2^32 no word of 32 bits is large enough: nothing is kept.
template <typename T>
__global__ __launch_bounds__(256) void drop_all_kernel(T *__restrict__ y, long long count) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) y[i] = (T)0.0f;
}

template <typename T>
static int launch_dropout(const void *x, void *y, long long count, uint64_t least, float scale, uint64_t seed, uint64_t offset,
                          const uint64_t *state, hipStream_t stream) {
  const bool aligned = aligned_to(x, 16) && aligned_to(y, 16);
  const int vec = aligned ? (int)(16 / sizeof(T)) : 4;
  long long blocks = ((count + vec - 1) / vec + 255) / 256;
  if (blocks > 16384) blocks = 16384;
  const uint32_t threshold = (uint32_t)least;
  if (least >> 32)
    hipLaunchKernelGGL(drop_all_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (T *)y, count);
  else if (aligned)
    hipLaunchKernelGGL((dropout_kernel<T, 16 / sizeof(T), true>), dim3((unsigned)blocks), dim3(256), 0, stream, (const T *)x,
                       (T *)y, count, threshold, scale, seed, offset, state);
  else
    hipLaunchKernelGGL((dropout_kernel<T, 4, false>), dim3((unsigned)blocks), dim3(256), 0, stream, (const T *)x, (T *)y, count,
                       threshold, scale, seed, offset, state);
  return check_launch("dropout");
}

}  // namespace frcnn

using namespace frcnn;

extern "C" int frcnn_dropout(const void *x, void *y, int type, int64_t count, double rate, uint64_t seed, uint64_t offset,
                             const uint64_t *state, frcnn_stream_t stream) {
  FRCNN_REQUIRE(type_known(type), "dropout: unknown element type %d", type);
  FRCNN_REQUIRE(rate >= 0.0 && rate < 1.0, "dropout: rate %g is not in [0, 1)", rate);
  FRCNN_REQUIRE(count >= 0 && count < ((int64_t)1 << 62), "dropout: bad element count");
  if (count == 0) return FRCNN_OK;
  FRCNN_REQUIRE(x && y, "dropout: null pointer");
  FRCNN_REQUIRE(aligned_to(x, type_bytes(type)) && aligned_to(y, type_bytes(type)), "dropout: pointers must be element aligned");
  FRCNN_REQUIRE(!state || aligned_to(state, 8), "dropout: state must be 8-byte aligned");
  const uint64_t least = (uint64_t)__builtin_rint(rate * 4294967296.0);  // 0 .. 2^32
  const float scale = (float)(1.0 / (1.0 - rate));
  hipStream_t s = (hipStream_t)stream;
  if (type == FRCNN_F32) return launch_dropout<float>(x, y, count, least, scale, seed, offset, state, s);
  if (type == FRCNN_F16) return launch_dropout<_Float16>(x, y, count, least, scale, seed, offset, state, s);
  return launch_dropout<__bf16>(x, y, count, least, scale, seed, offset, state, s);
}
