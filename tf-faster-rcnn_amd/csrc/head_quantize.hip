// head_quantize.hip -- rows to e4m3 with one scale per block of 128 elements.
//
// scale = max(amax * (1 / 448), 2^-126) over the block's finite values (1 where they are all zero; 1 / 448 rounded to fp32, the
// product too), or the smallest power of two that is not below amax / 448; q = x / scale, the correctly rounded fp32 quotient,
// rounded to the nearest e4m3, ties to even.  NaN and infinities become e4m3's
// NaN and leave the scale to their finite neighbours.  Blocks are 1 x 128 (activations) or 128 x 128 (weights).
//
// Bound by memory: 2 or 4 bytes read and one written per element.  16 lanes hold a block's row, 8 elements each.
#include "head_common.hpp"

namespace frcnn {

// four e4m3 from four floats (round to nearest even; |v| <= 448 or NaN)
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}

__device__ __forceinline__ float block_scale(float amax, bool power_of_two) {
  if (amax == 0.0f) return 1.0f;
  if (!power_of_two) {
    const float s = amax * (1.0f / kE4M3Max);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;
  }
  // amax = 1.f * 2^e: amax / 448 = (1.f / 1.75) * 2^(e - 8)
  const uint32_t u = f2u(amax);
  int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  if (e < 1) e = 1;  // 2^-126 at least (also for a subnormal amax)
  return u2f((uint32_t)e << 23);
}

template <typename T, bool VECTOR>
__device__ __forceinline__ void load8(const T *__restrict__ row, int col, int K, float (&f)[8]) {
  if (VECTOR && col + 8 <= K) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / V; ++h) {
      float g[V];
      Pack<T, V>::load(row + col + h * V).unpack(g);
#pragma unroll
      for (int e = 0; e < V; ++e) f[h * V + e] = g[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = col + e < K ? to_float(row[col + e]) : 0.0f;
  }
}

__device__ __forceinline__ float finite_abs(float v) {
  const float a = __builtin_fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;  // false for NaN too
}

__device__ __forceinline__ float quotient(float v, float scale) {
  const float a = __builtin_fabsf(v);
  return a <= 3.402823466e38f ? v / scale : u2f(0x7FC00000u);
}

__device__ __forceinline__ void store_scale(void *scales, long long at, float s, bool power_of_two) {
  if (power_of_two)
    reinterpret_cast<uint8_t *>(scales)[at] = (uint8_t)(f2u(s) >> 23);
  else
    reinterpret_cast<float *>(scales)[at] = s;
}

// BR = 1: a workgroup takes 64 rows of one block column; BR = 128: one 128 x 128 block.
template <typename T, bool VECTOR, int BR>
__global__ __launch_bounds__(256) void quantize_kernel(const T *__restrict__ x, long long ldx, int rows, int K,
                                                       uint8_t *__restrict__ q, long long ldq, void *__restrict__ scales,
                                                       long long scale_row, long long scale_block, int power_of_two,
                                                       int across) {
  constexpr int PASSES = BR == 1 ? 4 : 8;
  const int kb = (int)(blockIdx.x % (unsigned)across);
  const int tile = (int)(blockIdx.x / (unsigned)across);
  const int sub = threadIdx.x & 15, lane_row = threadIdx.x >> 4;
  const int col = kb * kQuantBlock + sub * 8;
  float f[PASSES][8];
  float amax[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const long long r = (long long)tile * (16 * PASSES) + p * 16 + lane_row;
    if (r < rows)
      load8<T, VECTOR>(x + r * ldx, col, K, f[p]);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) f[p][e] = 0.0f;
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = __builtin_fmaxf(m, finite_abs(f[p][e]));
    amax[p] = m;
  }
  if (BR == 1) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) amax[p] = __builtin_fmaxf(amax[p], __shfl_xor(amax[p], d));
  } else {
    __shared__ float part[4];
    float m = amax[0];
#pragma unroll
    for (int p = 1; p < PASSES; ++p) m = __builtin_fmaxf(m, amax[p]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = __builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3]));
#pragma unroll
    for (int p = 0; p < PASSES; ++p) amax[p] = m;
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const long long r = (long long)tile * (16 * PASSES) + p * 16 + lane_row;
    if (r >= rows) continue;
    const float s = block_scale(amax[p], power_of_two != 0);
    float g[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = quotient(f[p][e], s);
    if (col < (K + 15) / 16 * 16)  // the bytes up to the next multiple of 16 are written too, as zeros
      *reinterpret_cast<u32x2 *>(q + r * ldq + col) = u32x2{to_e4m3x4(g[0], g[1], g[2], g[3]), to_e4m3x4(g[4], g[5], g[6], g[7])};
    if (BR == 1) {
      if (sub == 0) store_scale(scales, r * scale_row + kb * scale_block, s, power_of_two != 0);
    } else if (p == 0 && threadIdx.x == 0) {
      store_scale(scales, (long long)tile * scale_row + kb * scale_block, s, power_of_two != 0);
    }
  }
}

template <typename T, int BR>
static int launch_quantize(const void *x, long long ldx, int rows, int K, void *q, long long ldq, void *scales,
                           long long scale_row, long long scale_block, int power_of_two, hipStream_t stream) {
  const int across = (K + kQuantBlock - 1) / kQuantBlock;
  const int per = BR == 1 ? 64 : 128;
  if (((long long)rows + per - 1) / per * across >= (1ll << 31)) return set_error(FRCNN_EUNSUPPORTED, "quantize_blocks: too many blocks");
  const bool vector = aligned_to(x, 16) && (ldx * (long long)sizeof(T)) % 16 == 0;
  const long long most = kGridThreads / 256 / across * per;  // rows of one launch
  for (long long first = 0; first < rows; first += most) {
    const int count = (int)(rows - first < most ? rows - first : most);
    const dim3 grid((unsigned)(((long long)count + per - 1) / per * across));
    const T *from = (const T *)x + first * ldx;
    uint8_t *to = (uint8_t *)q + first * ldq;
    void *s = (uint8_t *)scales + first / BR * scale_row * (power_of_two ? 1 : 4);
    if (vector)
      hipLaunchKernelGGL((quantize_kernel<T, true, BR>), grid, dim3(256), 0, stream, from, ldx, count, K, to, ldq, s, scale_row, scale_block,
                         power_of_two, across);
    else
      hipLaunchKernelGGL((quantize_kernel<T, false, BR>), grid, dim3(256), 0, stream, from, ldx, count, K, to, ldq, s, scale_row, scale_block,
                         power_of_two, across);
    const int rc = check_launch("quantize_blocks");
    if (rc) return rc;
  }
  return FRCNN_OK;
}

}  // namespace frcnn

using namespace frcnn;

extern "C" int frcnn_quantize_blocks(const void *x, int type, int64_t ldx, int64_t rows, int64_t K, int block_rows, void *q,
                                     int64_t ldq, void *scales, int scale_type, int64_t scale_row_stride,
                                     int64_t scale_block_stride, frcnn_stream_t stream) {
  FRCNN_REQUIRE(type_known(type), "quantize_blocks: unknown element type %d", type);
  FRCNN_REQUIRE(scale_type == FRCNN_SCALE_F32 || scale_type == FRCNN_SCALE_E8M0, "quantize_blocks: unknown scale type %d", scale_type);
  FRCNN_REQUIRE(block_rows == 1 || block_rows == kQuantBlock, "quantize_blocks: block_rows must be 1 or 128, got %d", block_rows);
  FRCNN_REQUIRE(rows >= 0 && K >= 0, "quantize_blocks: negative shape");
  if (rows == 0 || K == 0) return FRCNN_OK;
  FRCNN_REQUIRE(x && q && scales, "quantize_blocks: null pointer");
  FRCNN_REQUIRE(ldx >= K && ldq >= K && ldq % 16 == 0, "quantize_blocks: row strides must cover the row, q's in multiples of 16");
  // q's rows are written up to the next multiple of 16: the stride leaves room for that
  FRCNN_REQUIRE(aligned_to(x, type_bytes(type)) && aligned_to(q, 16) && (scale_type == FRCNN_SCALE_E8M0 || aligned_to(scales, 4)),
                "quantize_blocks: misaligned pointer");
  FRCNN_REQUIRE(scale_row_stride >= 0 && scale_block_stride >= 0, "quantize_blocks: negative scale stride");
  if (rows >= (1ll << 31) || K > (1 << 30))
    return set_error(FRCNN_EUNSUPPORTED, "quantize_blocks: (%lld, %lld) is beyond what the kernels index", (long long)rows, (long long)K);
  const int p2 = scale_type == FRCNN_SCALE_E8M0;
  hipStream_t s = (hipStream_t)stream;
#define FRCNN_QUANT(T)                                                                                                        \
  (block_rows == 1 ? launch_quantize<T, 1>(x, ldx, (int)rows, (int)K, q, ldq, scales, scale_row_stride, scale_block_stride, p2, s)      \
                   : launch_quantize<T, 128>(x, ldx, (int)rows, (int)K, q, ldq, scales, scale_row_stride, scale_block_stride, p2, s))
  if (type == FRCNN_F32) return FRCNN_QUANT(float);
  if (type == FRCNN_F16) return FRCNN_QUANT(_Float16);
  return FRCNN_QUANT(__bf16);
#undef FRCNN_QUANT
}
