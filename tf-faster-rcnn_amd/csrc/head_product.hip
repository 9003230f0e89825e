// head_product.hip -- matrix product of two block-scaled e4m3 operands, for the dense layers behind RoIPooling.
//
//   y[m, n] = act( sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} a[m, k] b[n, k]  + bias[n] )
//
// a (M, K) activations with a scale per 1 x 128 block, b (N, K) weights with a scale per 128 x 128 block.  The inner sum of a
// block is one v_mfma_f32_16x16x128_f8f6f4; with fp32 scales its result is multiplied by sa sb and added to the fp32
// accumulator by four fused multiply-adds per lane, with power-of-two scales the instruction takes them and accumulates.
// The weights are the instruction's first operand, so that a lane holds four neighbouring columns of one row of y.
#include "head_common.hpp"

namespace frcnn {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct ProductArgs {
  const uint8_t *a;
  const uint8_t *b;
  long long lda, ldb;
  const void *sa;  // float or e8m0
  const void *sb;
  long long sa_row, sa_block, sb_row, sb_block;  // element strides
  const float *bias;                              // may be null
  void *y;
  long long ldy;
  int M, N, K, blocks;  // blocks = ceil(K / 128)
  int act, out;
};

// The 16 bytes at `col` of a row of K bytes; bytes at K and beyond are zero.
__device__ __forceinline__ u32x4 load_chunk(const uint8_t *row, int col, int K) {
  if (col + 16 <= K) return *reinterpret_cast<const u32x4 *>(row + col);
  u32x4 w = {0, 0, 0, 0};
  for (int i = 0; i < 16; ++i)
    if (col + i < K) w[i >> 2] |= (uint32_t)row[col + i] << (8 * (i & 3));
  return w;
}

// Lane l of an operand holds row l % 16 and, of the block's eight 16-byte chunks, number l / 16 and l / 16 + 4 (both operands
// alike, so the order of the 128 products does not matter).
__device__ __forceinline__ i32x8 load_operand(const uint8_t *row, int block, int K) {
  const int col = block * kQuantBlock + (lane_id() >> 4) * 16;
  const u32x4 lo = load_chunk(row, col, K), hi = load_chunk(row, col + 64, K);
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// How a block's 128 products are formed.  The e4m3 matrix instructions drop low bits while they line the products up: 1.1e-5
// of the result in the mean over random blocks (measured; 16x16x128, 32x32x64 and the K = 32 forms alike), a 150th of the
// rounding to bf16 and a 12th of fp16's.  For an fp32 result the operands are widened to fp16, which holds every e4m3 value, and
// the fp16 instructions (5e-9 on the same blocks) multiply them at half the rate.
enum { kNarrowF32, kNarrowE8M0, kWideF32, kWideE8M0 };

template <int MODE>
struct Scale {  // fp32 scales, or e8m0 ones widened to fp32
  using type = float;
  __device__ __forceinline__ static float load(const void *p, long long at) {
    if constexpr (MODE == kWideE8M0) {
      const uint32_t e = reinterpret_cast<const uint8_t *>(p)[at];
      return u2f(e == 255 ? 0x7FC00000u : e == 0 ? 0x00400000u : e << 23);
    } else {
      return reinterpret_cast<const float *>(p)[at];
    }
  }
};
template <>
struct Scale<kNarrowE8M0> {  // the byte that the matrix instruction takes
  using type = int;
  __device__ __forceinline__ static int load(const void *p, long long at) { return reinterpret_cast<const uint8_t *>(p)[at]; }
};

template <int MODE>
struct Operand {
  using type = i32x8;
  __device__ __forceinline__ static i32x8 of(i32x8 v) { return v; }
};
struct WideOperand {
  f16x8 h[4];
};
template <>
struct Operand<kWideF32> {
  using type = WideOperand;
  __device__ __forceinline__ static WideOperand of(i32x8 v) {
    WideOperand o;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int w = v[i];
      const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
      o.h[i >> 1][4 * (i & 1)] = lo.x;
      o.h[i >> 1][4 * (i & 1) + 1] = lo.y;
      o.h[i >> 1][4 * (i & 1) + 2] = hi.x;
      o.h[i >> 1][4 * (i & 1) + 3] = hi.y;
    }
    return o;
  }
};
template <>
struct Operand<kWideE8M0> : Operand<kWideF32> {};

template <int MODE>
__device__ __forceinline__ f32x4 multiply(const typename Operand<MODE>::type &w, const typename Operand<MODE>::type &a, f32x4 acc,
                                          typename Scale<MODE>::type sw, typename Scale<MODE>::type sa) {
  if constexpr (MODE == kNarrowE8M0) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 0, 0, 0, sw, 0, sa);
  } else {
    f32x4 d = {0, 0, 0, 0};
    if constexpr (MODE == kNarrowF32) {
      d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, d, 0, 0, 0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.h[i], a.h[i], d, 0, 0, 0);
    }
    const float s = sw * sa;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(d[i], s, acc[i]);
    return acc;
  }
}

// Bias, activation, rounding and store of four neighbouring columns n .. n + 3 of row m.
template <typename T>
__device__ __forceinline__ void store4(const ProductArgs &p, int m, int n, f32x4 v) {
  T *row = reinterpret_cast<T *>(p.y) + (long long)m * p.ldy + n;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.N) {
      float f = v[i] + (p.bias ? p.bias[n + i] : 0.0f);
      if (p.act == FRCNN_ACT_RELU) f = f > 0.0f ? f : (f != f ? f : 0.0f);
      row[i] = (T)f;
    }
}

__device__ __forceinline__ void finish4(const ProductArgs &p, int m, int n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  if (p.out == FRCNN_F32) store4<float>(p, m, n, v);
  else if (p.out == FRCNN_F16) store4<_Float16>(p, m, n, v);
  else store4<__bf16>(p, m, n, v);
}

// TM x TN tiles of 16 x 16 per workgroup; its W waves share the blocks of K and add their sums in LDS, in the waves' order.
template <int TM, int TN, int W, int MODE>
__global__ __launch_bounds__(64 * W) void product_split_kernel(ProductArgs p, int tiles_n) {
  using S = Scale<MODE>;
  using O = Operand<MODE>;
  const int tn = (int)(blockIdx.x % (unsigned)tiles_n), tm = (int)(blockIdx.x / (unsigned)tiles_n);
  const int wave = threadIdx.x >> 6, lane = lane_id();
  const int m0 = tm * TM * 16, n0 = tn * TN * 16;
  const uint8_t *arow[TM], *brow[TN];
  long long sa_at[TM], sb_at[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = min(m0 + i * 16 + (lane & 15), p.M - 1);  // rows beyond the end repeat the last one and are not stored
    arow[i] = p.a + m * p.lda;
    sa_at[i] = m * p.sa_row;
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = min(n0 + j * 16 + (lane & 15), p.N - 1);
    brow[j] = p.b + n * p.ldb;
    sb_at[j] = (long long)(min(n0 + j * 16, p.N - 1) / kQuantBlock) * p.sb_row;
  }
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  for (int kb = wave; kb < p.blocks; kb += W) {
    typename O::type a[TM], b[TN];
    typename S::type sa[TM], sb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      b[j] = O::of(load_operand(brow[j], kb, p.K));
      sb[j] = S::load(p.sb, sb_at[j] + kb * p.sb_block);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      a[i] = O::of(load_operand(arow[i], kb, p.K));
      sa[i] = S::load(p.sa, sa_at[i] + kb * p.sa_block);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = multiply<MODE>(b[j], a[i], acc[i][j], sb[j], sa[i]);
  }
  __shared__ f32x4 part[W][TM * TN][64];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) part[wave][i * TN + j][lane] = acc[i][j];
  __syncthreads();
  for (int t = wave; t < TM * TN; t += W) {
    f32x4 v = part[0][t][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += part[w][t][lane];
    finish4(p, m0 + (t / TN) * 16 + (lane & 15), n0 + (t % TN) * 16 + (lane >> 4) * 4, v);
  }
}

}  // namespace frcnn

using namespace frcnn;

extern "C" {

size_t frcnn_scaled_matmul_workspace_bytes(int M, int N, int K) {
  (void)M, (void)N, (void)K;
  return 0;
}

int frcnn_scaled_matmul(const void *a, int64_t lda, const void *a_scales, int64_t a_scale_row_stride, int64_t a_scale_block_stride,
                        const void *b, int64_t ldb, const void *b_scales, int64_t b_scale_row_stride, int64_t b_scale_block_stride,
                        int scale_type, const float *bias, int activation, int M, int N, int K, void *y, int y_type, int64_t ldy,
                        void *workspace, size_t workspace_bytes, frcnn_stream_t stream) {
  FRCNN_REQUIRE(scale_type == FRCNN_SCALE_F32 || scale_type == FRCNN_SCALE_E8M0, "scaled_matmul: unknown scale type %d", scale_type);
  FRCNN_REQUIRE(type_known(y_type), "scaled_matmul: unknown output type %d", y_type);
  FRCNN_REQUIRE(activation == FRCNN_ACT_NONE || activation == FRCNN_ACT_RELU, "scaled_matmul: unknown activation %d", activation);
  FRCNN_REQUIRE(M >= 0 && N >= 0 && K >= 0, "scaled_matmul: negative shape");
  if (M == 0 || N == 0) return FRCNN_OK;
  FRCNN_REQUIRE(y && ldy >= N && aligned_to(y, type_bytes(y_type)), "scaled_matmul: bad output");
  FRCNN_REQUIRE(aligned_to(bias, 4), "scaled_matmul: misaligned bias");
  if (K > 0) {
    FRCNN_REQUIRE(a && b && a_scales && b_scales, "scaled_matmul: null pointer");
    FRCNN_REQUIRE(lda >= K && ldb >= K && lda % 16 == 0 && ldb % 16 == 0 && aligned_to(a, 16) && aligned_to(b, 16),
                  "scaled_matmul: operand rows must start at multiples of 16 bytes");
    FRCNN_REQUIRE(scale_type == FRCNN_SCALE_E8M0 || (aligned_to(a_scales, 4) && aligned_to(b_scales, 4)), "scaled_matmul: misaligned scales");
    FRCNN_REQUIRE(a_scale_row_stride >= 0 && a_scale_block_stride >= 0 && b_scale_row_stride >= 0 && b_scale_block_stride >= 0,
                  "scaled_matmul: negative scale stride");
  }
  if (K > (1 << 22) || lda > (1 << 23) || ldb > (1 << 23) || N > (1 << 24))
    return set_error(FRCNN_EUNSUPPORTED, "scaled_matmul: K=%d (row strides %lld, %lld), N=%d is beyond what the kernels index", K,
                     (long long)lda, (long long)ldb, N);
  (void)workspace, (void)workspace_bytes;
  const ProductArgs p = {(const uint8_t *)a, (const uint8_t *)b, lda, ldb, a_scales, b_scales, a_scale_row_stride, a_scale_block_stride,
                         b_scale_row_stride, b_scale_block_stride, bias, y, ldy, M, N, K, (K + kQuantBlock - 1) / kQuantBlock,
                         activation, y_type};
  const int mode = (y_type == FRCNN_F32 ? kWideF32 : kNarrowF32) + (scale_type == FRCNN_SCALE_E8M0);
  hipStream_t s = (hipStream_t)stream;
#define FRCNN_SPLIT(TM, TN, W)                                                                                                 \
  {                                                                                                                            \
    const long long tm = (M + TM * 16 - 1) / (TM * 16), tn = (N + TN * 16 - 1) / (TN * 16);                                    \
    if (tm * tn >= (1ll << 31)) return set_error(FRCNN_EUNSUPPORTED, "scaled_matmul: too many tiles");                         \
    const dim3 grid((unsigned)(tm * tn)), block(64 * W);                                                                       \
    if (mode == kNarrowF32) hipLaunchKernelGGL((product_split_kernel<TM, TN, W, kNarrowF32>), grid, block, 0, s, p, (int)tn);  \
    else if (mode == kNarrowE8M0) hipLaunchKernelGGL((product_split_kernel<TM, TN, W, kNarrowE8M0>), grid, block, 0, s, p, (int)tn); \
    else if (mode == kWideF32) hipLaunchKernelGGL((product_split_kernel<TM, TN, W, kWideF32>), grid, block, 0, s, p, (int)tn); \
    else hipLaunchKernelGGL((product_split_kernel<TM, TN, W, kWideE8M0>), grid, block, 0, s, p, (int)tn);                      \
  }
  if (M <= 16) FRCNN_SPLIT(1, 1, 16) else FRCNN_SPLIT(4, 2, 4)
#undef FRCNN_SPLIT
  return check_launch("scaled_matmul");
}

}  // extern "C"
