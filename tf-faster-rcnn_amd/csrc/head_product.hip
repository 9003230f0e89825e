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
  int quads;  // N, ldy and the pointers allow four columns at a time
  int rows16;  // y's rows start at multiples of 16 bytes
};

// The 16 bytes at `col` of a row of K bytes; bytes at K and beyond are zero.
__device__ __forceinline__ u32x4 load_chunk(const uint8_t *row, int col, int K) {
  if (col + 16 <= K) return *reinterpret_cast<const u32x4 *>(row + col);
  uint64_t lo = 0, hi = 0;
#pragma unroll 1
  for (int i = K - col - 1; i >= 0; --i) {
    hi = hi << 8 | lo >> 56;
    lo = lo << 8 | row[col + i];
  }
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// Lane l of an operand holds row l % 16 and, of the block's eight 16-byte chunks, number l / 16 and l / 16 + 4 (both operands
// alike, so the order of the 128 products does not matter).
__device__ __forceinline__ i32x8 load_operand(const uint8_t *row, int block, int K) {
  const int col = block * kQuantBlock + (lane_id() >> 4) * 16;
  const u32x4 lo = load_chunk(row, col, K), hi = load_chunk(row, col + 64, K);
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// How a block's 128 products are formed.  The e4m3 matrix instructions line the products of 8 neighbouring columns up with the
// largest of them and cut each below 2^-13 of it (measured: 16x16x128, 32x32x64 and the K = 32 forms alike); the sums of the
// eights, of the blocks and, with e8m0 scales, the instruction's own accumulator are fp32.  That is 1.1e-5 of the result in the
// median for operands of random signs, a 150th of the rounding to bf16 and a 12th of fp16's, and 2.5e-6 for positive ones, but a
// large pair that cancels within an eight takes its small neighbours with it.  "Narrow" is for 16-bit results of the tile forms,
// whose time is the products: 4800 x 4096 x 28224 takes 467 us so and 1003 widened, 300 rows 63 and 101.  "Wide", for all
// others: the operands are widened to fp16, which holds every e4m3 value and every product's bits, and the fp16 instructions
// multiply them at half the rate (5e-9 on the same blocks).  The split-K form waits for memory either way: 1 row 23 us, 16 rows
// 34 us, narrow and wide.
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

// The 128 products of a block onto acc: with its scales only where the instruction takes them.
template <int MODE>
__device__ __forceinline__ f32x4 block_product(const typename Operand<MODE>::type &w, const typename Operand<MODE>::type &a, f32x4 acc,
                                               typename Scale<MODE>::type sw, typename Scale<MODE>::type sa) {
  if constexpr (MODE == kNarrowE8M0) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 0, 0, 0, sw, 0, sa);
  } else if constexpr (MODE == kNarrowF32) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 0, 0, 0, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.h[i], a.h[i], acc, 0, 0, 0);
    return acc;
  }
}

__device__ __forceinline__ void add_scaled(f32x4 &acc, f32x4 d, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(d[i], s, acc[i]);
}

// Is the product of two scales no normal number, other than for a zero among them?  Times a block's sum (2^-18 to 2^25) it may be one.
__device__ __forceinline__ bool far_scales(float sw, float sa) {
  const float f = sw * sa;
  return __builtin_amdgcn_classf(f, 0x297) || (f == 0.0f && sw != 0.0f && sa != 0.0f);  // NaN, infinity, subnormal; vanished
}

// acc + d sw sa for such scales: their powers of two are applied last.
__device__ __forceinline__ void add_far_scaled(f32x4 &acc, f32x4 d, float sw, float sa) {
  const float m = __builtin_amdgcn_frexp_mantf(sw) * __builtin_amdgcn_frexp_mantf(sa);
  const int e = __builtin_amdgcn_frexp_expf(sw) + __builtin_amdgcn_frexp_expf(sa);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] += __builtin_amdgcn_ldexpf(d[i] * m, e);
}

__device__ __forceinline__ float relu(float v) { return v > 0.0f ? v : (v != v ? v : 0.0f); }

// The bias of columns n .. n + 3; zeros without one or beyond the last column.
__device__ __forceinline__ f32x4 bias4(const ProductArgs &p, int n) {
  f32x4 v = {0, 0, 0, 0};
  if (!p.bias || n >= p.N) return v;
  if (p.quads) return *reinterpret_cast<const f32x4 *>(p.bias + n);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.N) v[i] = p.bias[n + i];
  return v;
}

// Activation, rounding and store of four neighbouring columns n .. n + 3 of row m.
template <typename T>
__device__ __forceinline__ void store4(const ProductArgs &p, int m, int n, f32x4 v) {
  T *row = reinterpret_cast<T *>(p.y) + (long long)m * p.ldy + n;
  if (p.act == FRCNN_ACT_RELU)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = relu(v[i]);
  if (p.quads) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4 *>(row) = v;
    } else {
      typedef T tx4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<tx4 *>(row) = __builtin_convertvector(v, tx4);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.N) row[i] = (T)v[i];
}

// 16 rows from m and 16 NT columns from n, all of them columns of y, by way of the wave's own piece of LDS: a store instruction
// then fills whole rows of the tile instead of 32 bytes of each.
template <typename T, int NT>
struct RowStore {
  static constexpr int ROW = NT * 16 * sizeof(T), STRIDE = ROW + 16, BYTES = 16 * STRIDE;
  static constexpr int LANES = ROW / 16, PER = 64 / LANES;  // lanes per row, rows per store
  __device__ __forceinline__ static void run(const ProductArgs &p, uint8_t *scratch, int m, int n, f32x4 (&v)[NT]) {
    typedef T tx4 __attribute__((ext_vector_type(4)));
    const int lane = lane_id();
    uint8_t *to = scratch + (lane & 15) * STRIDE + (lane >> 4) * 4 * sizeof(T);
#pragma unroll
    for (int j = 0; j < NT; ++j) *reinterpret_cast<tx4 *>(to + j * 16 * sizeof(T)) = __builtin_convertvector(v[j], tx4);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's lanes read what others of them wrote
    const int row = lane / LANES, chunk = lane % LANES;
    T *out = reinterpret_cast<T *>(p.y) + (long long)(m + row) * p.ldy + n + chunk * (16 / sizeof(T));
#pragma unroll
    for (int s = 0; s < 16 / PER; ++s) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(scratch + (s * PER + row) * STRIDE + chunk * 16);
      if (m + s * PER + row < p.M) *reinterpret_cast<u32x4 *>(out + (long long)s * PER * p.ldy) = w;
    }
    asm volatile("" ::: "memory");
  }
};

// f(T) for the output's type T: one uniform branch around all of a thread's stores.
template <typename F>
__device__ __forceinline__ void with_output_type(const ProductArgs &p, F f) {
  if (p.out == FRCNN_F32) f((float *)nullptr);
  else if (p.out == FRCNN_F16) f((_Float16 *)nullptr);
  else f((__bf16 *)nullptr);
}

// One 16 x 16 tile per workgroup; its 16 waves share the blocks of K and add their sums in LDS, in the waves' order.  For few
// rows, where the weights' way from memory is all there is: 116 MB for one row in 24 us, 4.8 TB/s.  More blocks in flight per wave
// (two, four) gave nothing.
static const int kSplitWaves = 16;

template <int MODE>
__global__ __launch_bounds__(64 * kSplitWaves) void product_split_kernel(ProductArgs p, int tiles_n) {
  using S = Scale<MODE>;
  using O = Operand<MODE>;
  const int tn = (int)(blockIdx.x % (unsigned)tiles_n), tm = (int)(blockIdx.x / (unsigned)tiles_n);
  const int wave = threadIdx.x >> 6, lane = lane_id();
  // rows beyond the end repeat the last one and are not stored
  const int row = min(tm * 16 + (lane & 15), p.M - 1), column = min(tn * 16 + (lane & 15), p.N - 1);
  const uint8_t *arow = p.a + row * p.lda, *brow = p.b + column * p.ldb;
  const long long sa_at = row * p.sa_row, sb_at = (long long)(tn * 16 / kQuantBlock) * p.sb_row;
  f32x4 acc = {0, 0, 0, 0};
  for (int kb = wave; kb < p.blocks; kb += kSplitWaves) {
    const typename O::type b = O::of(load_operand(brow, kb, p.K));
    const float sb = S::load(p.sb, sb_at + kb * p.sb_block);
    const typename O::type a = O::of(load_operand(arow, kb, p.K));
    const float sa = S::load(p.sa, sa_at + kb * p.sa_block);
    const f32x4 d = block_product<MODE>(b, a, f32x4{0, 0, 0, 0}, sb, sa);
    const float both = sb * sa;
    if (__builtin_expect(__any(__builtin_amdgcn_classf(both, 0x2F7)), 0) && far_scales(sb, sa))  // no normal number
      add_far_scaled(acc, d, sb, sa);
    else
      add_scaled(acc, d, both);
  }
  __shared__ f32x4 part[kSplitWaves][64];
  part[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
  f32x4 v = part[0][lane];
#pragma unroll
  for (int w = 1; w < kSplitWaves; ++w) v += part[w][lane];
  const int m = tm * 16 + (lane & 15), n = tn * 16 + (lane >> 4) * 4;
  v += bias4(p, n);
  if (m < p.M && n < p.N) with_output_type(p, [&](auto *type) { store4<__remove_pointer(decltype(type))>(p, m, n, v); });
}

// ---- large products: tiles through LDS ------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves computes a BM x BN tile, 16 MT x 16 NT per wave, one block of 128 columns at a time: the next
// blocks travel from memory straight to other parts of LDS while the matrix instructions work on this one.  In LDS a row of
// 128 bytes keeps its 16-byte chunk c at place c ^ (row % 8), so that the 16 rows of an operand read fall on all banks.
//
// The tiles fill the chip in rounds of one workgroup per CU; the tiles of a last, unfilled round are cut along K into `pieces`
// of whole blocks, whose sums go to the workspace and are added in their order by product_join_kernel.
static const int kProductCus = 256;

struct TilePlan {
  int tiles_m, tiles_n;
  int whole;   // tiles computed by one workgroup each: the first ones of the order
  int rest;    // the others
  int pieces;  // workgroups per tile of the rest
};

static const int kStripRows = 4;

// Each XCD takes a contiguous range of an order that runs down strips of kStripRows row tiles, so that the 32 tiles it works on
// share 4 rows' and 8 columns' operands in its L2.
__device__ __forceinline__ void tile_of(const TilePlan &t, int order, int &m, int &n) {
  const int strip = order / (kStripRows * t.tiles_n), at = order - strip * kStripRows * t.tiles_n;
  const int rows = min(kStripRows, t.tiles_m - strip * kStripRows);
  n = at / rows;
  m = strip * kStripRows + at - n * rows;
}

typedef __attribute__((address_space(3))) void *lds_ptr;

// The R rows of one operand's tile, a block at a time, into LDS.
template <int R, int THREADS>
struct TileLoader {
  static constexpr int N = (R * 8 + THREADS - 1) / THREADS;  // 16-byte chunks per thread
  static_assert(R % 8 == 0, "whole waves of chunks");
  // the first chunk of the thread's (wave's) i-th load; waves beyond the last chunk load others' again, so that every wave has
  // the same number of loads in flight
  __device__ __forceinline__ static int chunk(int i, int thread) {
    const int c = i * THREADS + thread;
    return (i + 1) * THREADS <= R * 8 || c < R * 8 ? c : c - (N * THREADS - R * 8);
  }
  const uint8_t *base;  // the tile's first row
  int offset[N];
  int first, rows, ld, bytes;
  __device__ __forceinline__ TileLoader(const uint8_t *operand, long long stride, int first_row, int total_rows, int K)
      : base(operand + first_row * stride), first(first_row), rows(total_rows), ld((int)stride) {
    bytes = (min(R, rows - first) - 1) * ld + K;  // under R * 2^23
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = chunk(i, (int)threadIdx.x), row = c >> 3;
      offset[i] = min(row, rows - 1 - first) * ld + (((c & 7) ^ (row & 7)) << 4);  // rows beyond the end: the last one
    }
  }
  // Buffer loads: the block's offset is a scalar operand, and unlike the flat forms they leave the order of the wave's other
  // loads known to the compiler, whose waits are then for what they have to be.
  __device__ __forceinline__ void start_one(int i, int block, uint8_t *lds) const {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass does not know the builtins' types
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, bytes, 0x00027000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_ptr)(lds + chunk(i, wave * 64) * 16), 16, offset[i], block * kQuantBlock, 0, 0);
#endif
  }
  __device__ __forceinline__ void start(int block, uint8_t *lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) start_one(i, block, lds);
  }
  // the last, partial block: zeros behind the row's end
  __device__ __forceinline__ void partial(int block, int K, uint8_t *lds) const {
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      const int c = chunk(i, (int)threadIdx.x), row = c >> 3;
      const uint8_t *r = base + (long long)min(row, rows - 1 - first) * ld;
      *reinterpret_cast<u32x4 *>(lds + c * 16) = load_chunk(r, block * kQuantBlock + ((c & 7) ^ (row & 7)) * 16, K);
    }
  }
};

// `at`: the first of the lane's two chunks in row lane % 16 of the operand's tile; rows further down are 2 KB per 16 apart.
__device__ __forceinline__ i32x8 read_operand(const uint8_t *lds, int at, int sixteens) {
  const u32x4 lo = *reinterpret_cast<const u32x4 *>(lds + at + sixteens * (16 * kQuantBlock));
  const u32x4 hi = *reinterpret_cast<const u32x4 *>(lds + (at ^ 64) + sixteens * (16 * kQuantBlock));
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// out[r] = v of lane 16 r + lane % 16: each of the wave's four rows of 16 lanes spread over all of them.
template <typename V>
__device__ __forceinline__ void rows_of_16_to_all(V v, V *out) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto halves = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // rows 0 1 0 1, rows 2 3 2 3
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned w = halves[h];
    const auto rows = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    const unsigned r0 = rows[0], r1 = rows[1];
    out[2 * h] = __builtin_bit_cast(V, r0);
    out[2 * h + 1] = __builtin_bit_cast(V, r1);
  }
}

// Waits until at most `left` of the wave's loads are in flight and all its LDS reads are back, then for the other waves.
template <int LEFT>
__device__ __forceinline__ void step_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int MT, int NT, int WM, int WN, int PER_CU, int DB, int MODE>
__global__ __launch_bounds__(64 * WM * WN, WM * WN * PER_CU / 4) void product_tile_kernel(ProductArgs p, TilePlan plan, f32x4 *__restrict__ partial) {
  constexpr int THREADS = 64 * WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
  constexpr int ROWS = 16 * MT, SCALES = (ROWS + 63) / 64;  // a wave's rows of a; registers that hold their scales
  using S = Scale<MODE>;
  using O = Operand<MODE>;
  extern __shared__ uint8_t smem[];  // three tiles of a, DB of b
  int tile, k0 = 0, k1 = p.blocks, piece = -1;
  if ((int)blockIdx.x < plan.whole) {
    tile = xcd_contiguous((int)blockIdx.x, plan.whole);
  } else {  // the same blocks of K of neighbouring tiles next to each other
    const int r = xcd_contiguous((int)blockIdx.x - plan.whole, plan.rest * plan.pieces);
    const int part = r / plan.rest, t = r - part * plan.rest;
    tile = plan.whole + t;
    k0 = __builtin_amdgcn_readfirstlane((int)((long long)p.blocks * part / plan.pieces));
    k1 = __builtin_amdgcn_readfirstlane((int)((long long)p.blocks * (part + 1) / plan.pieces));
    if (plan.pieces > 1) piece = t * plan.pieces + part;
  }
  int tm, tn;
  tile_of(plan, tile, tm, tn);
  const int m0 = __builtin_amdgcn_readfirstlane(tm) * BM, n0 = __builtin_amdgcn_readfirstlane(tn) * BN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id();
  const int wm = (wave % WM) * ROWS, wn = (wave / WM) * NT * 16;  // the wave's corner in the tile
  const TileLoader<BM, THREADS> load_a(p.a, p.lda, m0, p.M, p.K);
  const TileLoader<BN, THREADS> load_b(p.b, p.ldb, n0, p.N, p.K);
  const int last = min(k1, p.K / kQuantBlock);  // whole blocks end here

  // NT * 16 divides 128: one row of b's scales.  The lane's part of the address is zero, but keeps it a vector load: scalar
  // loads would make every wait for LDS one for all of them
  int zero = 0;
  asm("" : "+v"(zero));
  const long long sb_at = (long long)(min(n0 + wn, p.N - 1) / kQuantBlock) * p.sb_row + zero;
  long long sa_at[SCALES];
#pragma unroll
  for (int i = 0; i < SCALES; ++i) sa_at[i] = (long long)min(m0 + wm + min(i * 64 + lane, ROWS - 1), p.M - 1) * p.sa_row;

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  typename S::type sa_next[SCALES], sb_next;
  auto fetch_scales = [&](int block) {
#pragma unroll
    for (int i = 0; i < SCALES; ++i) sa_next[i] = S::load(p.sa, sa_at[i] + block * p.sa_block);
    sb_next = S::load(p.sb, sb_at + block * p.sb_block);
  };
  // For row i * 16 + lane % 16 and every i: what the instruction takes, a's scale, with b's beside it; otherwise the product of the two
  typename S::type sa[SCALES * 4], sb;
  uint64_t far = 0;  // not zero: rows whose scales are far from 1 were left out (times 0), and come last
  auto take_scales = [&]() {
    if constexpr (MODE == kNarrowE8M0) {
      sb = sb_next;
#pragma unroll
      for (int i = 0; i < SCALES; ++i) rows_of_16_to_all(sa_next[i], sa + 4 * i);
    } else {
      float both[SCALES];
      uint64_t odd = 0;
#pragma unroll
      for (int i = 0; i < SCALES; ++i) {
        both[i] = sb_next * sa_next[i];
        odd |= __builtin_amdgcn_ballot_w64(__builtin_amdgcn_classf(both[i], 0x2F7));  // no normal number
      }
      if (__builtin_expect(odd != 0, 0))
#pragma unroll
        for (int i = 0; i < SCALES; ++i) {
          const bool f = far_scales(sb_next, sa_next[i]);
          far |= __builtin_amdgcn_ballot_w64(f);
          both[i] = f ? 0.0f : both[i];
        }
#pragma unroll
      for (int i = 0; i < SCALES; ++i) rows_of_16_to_all(both[i], sa + 4 * i);
    }
  };
  const int lane_at = (lane & 15) * kQuantBlock + (((lane >> 4) ^ (lane & 7)) << 4);
  // a's next operand is read while this one is multiplied, and a group's scaled sums follow the next group's products
  auto compute = [&](const uint8_t *a_tile, const uint8_t *b_tile, auto &&between) {
    const uint8_t *a = a_tile + wm * kQuantBlock, *b = b_tile + wn * kQuantBlock;
    i32x8 x = read_operand(a, lane_at, 0);
    typename O::type w[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) w[j] = O::of(read_operand(b, lane_at, j));
    f32x4 before[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      i32x8 coming;
      if (i + 1 < MT) coming = read_operand(a, lane_at, i + 1);
      between(i);
      const typename O::type v = O::of(x);
      f32x4 now[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if constexpr (MODE == kNarrowE8M0)
          acc[i][j] = block_product<MODE>(w[j], v, acc[i][j], sb, sa[i]);
        else
          now[j] = block_product<MODE>(w[j], v, f32x4{0, 0, 0, 0}, sb, sa[i]);
      }
      if constexpr (MODE != kNarrowE8M0) {
        if (i > 0)
#pragma unroll
          for (int j = 0; j < NT; ++j) add_scaled(acc[i - 1][j], before[j], sa[i - 1]);
#pragma unroll
        for (int j = 0; j < NT; ++j) before[j] = now[j];
      }
      x = coming;
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MODE != kNarrowE8M0)
#pragma unroll
      for (int j = 0; j < NT; ++j) add_scaled(acc[MT - 1][j], before[j], sa[MT - 1]);
  };
  constexpr int A = BM * kQuantBlock, B = BN * kQuantBlock;
  uint8_t *const bs = smem + 3 * A;
  if (k0 < last) {
    // Block k of a lives in tile k % 3, of b in tile k % DB.  Step k computes block k while a's block k + 2 and b's block
    // k + DB - 1 are on their way: what has two steps' time keeps loads in flight all along.  Past the end the last block is
    // fetched again and not used.
    constexpr int NA = TileLoader<BM, THREADS>::N, NB = TileLoader<BN, THREADS>::N, PER = (NA + NB + MT - 1) / MT;
    load_a.start(k0, smem);
    load_b.start(k0, bs);
    fetch_scales(k0);
    __builtin_amdgcn_sched_barrier(0);  // the first barrier counts on this order
    if (DB == 3) load_b.start(min(k0 + 1, last - 1), bs + B);
    load_a.start(min(k0 + 1, last - 1), smem + A);
    int at = 0, bt = 0;  // offsets of this step's tiles
    for (int kb = k0; kb < last; ++kb) {
      step_barrier<DB == 3 ? NA + NB : NA>();
      take_scales();  // before this step's loads are issued: a wait for the scales is then none for them
      __builtin_amdgcn_sched_barrier(0);
      const int after = min(kb + 2, last - 1), b_next = DB == 3 ? after : min(kb + 1, last - 1);
      fetch_scales(min(kb + 1, last - 1));
      uint8_t *const to_a = smem + (at == 0 ? 2 * A : at - A), *const to_b = bs + (bt == 0 ? (DB - 1) * B : bt - B);
      // the loads are issued between the groups of products: all at once they would fill the memory pipe's queue and hold up
      // the first products
      compute(smem + at, bs + bt, [&](int i) {
#pragma unroll
        for (int l = i * PER; l < (i + 1) * PER; ++l) {
          if (l < NB) load_b.start_one(l, b_next, to_b);
          else if (l < NB + NA) load_a.start_one(l - NB, after, to_a);
        }
      });
      at = at == 2 * A ? 0 : at + A;
      bt = bt == (DB - 1) * B ? 0 : bt + B;
    }
    step_barrier<0>();
  }
  if (last < k1) {  // the partial block behind the whole ones
    load_a.partial(last, p.K, smem);
    load_b.partial(last, p.K, bs);
    fetch_scales(last);
    take_scales();
    step_barrier<0>();
    compute(smem, bs, [](int) {});
    step_barrier<0>();  // LDS is free for the results
  }
  if constexpr (MODE != kNarrowE8M0)
    if (far) {
#pragma unroll 1
      for (int kb = k0; kb < k1; ++kb) {
        const float sw = S::load(p.sb, sb_at + kb * p.sb_block);
        int row = lane & 15;  // seen as new in each block: addresses kept over the loop would take registers that the sums need
        asm volatile("" : "+v"(row));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int m = min(m0 + wm + i * 16 + row, p.M - 1);
          const float sv = S::load(p.sa, m * p.sa_row + kb * p.sa_block);
          const bool mine = far_scales(sw, sv);
          if (!__any(mine)) continue;
          const typename O::type v = O::of(load_operand(p.a + m * p.lda, kb, p.K));
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const int n = min(n0 + wn + j * 16 + row, p.N - 1);
            const f32x4 d = block_product<MODE>(O::of(load_operand(p.b + n * p.ldb, kb, p.K)), v, f32x4{0, 0, 0, 0}, sw, sv);
            if (mine) add_far_scaled(acc[i][j], d, sw, sv);
            __builtin_amdgcn_sched_barrier(0);  // few registers beside the sums
          }
        }
      }
    }
  if (piece >= 0) {
    f32x4 *out = partial + (long long)piece * (MT * NT * THREADS) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) out[(i * NT + j) * THREADS] = acc[i][j];
  } else {
    f32x4 bias[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) bias[j] = bias4(p, n0 + wn + j * 16 + (lane >> 4) * 4);
    const bool whole_rows = p.rows16 && n0 + wn + NT * 16 <= p.N;
    with_output_type(p, [&](auto *type) {
      using T = __remove_pointer(decltype(type));
      using R = RowStore<T, NT>;
      static_assert(R::BYTES * WM * WN <= 3 * A + DB * B, "the waves' pieces of LDS");
      if (whole_rows) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          f32x4 v[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            v[j] = acc[i][j] + bias[j];
            if (p.act == FRCNN_ACT_RELU)
#pragma unroll
              for (int e = 0; e < 4; ++e) v[j][e] = relu(v[j][e]);
          }
          R::run(p, smem + wave * R::BYTES, m0 + wm + i * 16, n0 + wn, v);
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + wm + i * 16 + (lane & 15);
        if (m < p.M)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
            if (n < p.N) store4<T>(p, m, n, acc[i][j] + bias[j]);
          }
      }
    });
  }
}

// One workgroup per 16 x 16 tile index of a cut tile's waves: the pieces' sums in their order, then what a whole tile does.
template <int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product_join_kernel(ProductArgs p, TilePlan plan, const f32x4 *__restrict__ partial) {
  constexpr int THREADS = 64 * WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
  const int t = (int)(blockIdx.x / (MT * NT)), f = (int)(blockIdx.x % (MT * NT));
  int tm, tn;
  tile_of(plan, plan.whole + t, tm, tn);
  const int wave = threadIdx.x >> 6, lane = lane_id();
  const int m = tm * BM + (wave % WM) * MT * 16 + (f / NT) * 16 + (lane & 15);
  const int n = tn * BN + (wave / WM) * NT * 16 + (f % NT) * 16 + (lane >> 4) * 4;
  const f32x4 *in = partial + ((long long)t * plan.pieces * (MT * NT) + f) * THREADS + threadIdx.x;
  f32x4 v = in[0];
#pragma unroll 8
  for (int i = 1; i < plan.pieces; ++i) v += in[(long long)i * (MT * NT * THREADS)];
  v += bias4(p, n);
  if (m < p.M && n < p.N) with_output_type(p, [&](auto *type) { store4<__remove_pointer(decltype(type))>(p, m, n, v); });
}

// The tile forms, and how long one takes for a block of 128 columns when the chip is full of them (measured between K = 8320 and
// 16640, fp32 scales; `wide`: for fp32 results).  Large tiles move the fewest bytes per product: per product the 160 x 256 tile
// takes 1.04 times as long as the 256 x 256 one, 128 x 128 1.28 and 64 x 128 1.95 times.  Small ones fill the chip when there are
// few rows, and waste less of a ragged edge.  `best_form` takes the form with the shortest time by these figures.
// They are too low for plans cut along K, whose weights come from memory on first touch: 300 rows of 4096 x 28224 are 47 us by them
// and 63 measured.  The choice was therefore compared with every form forced, 17 to 4800 rows, N = 4096, bf16 results, chosen /
// best other (us): K = 28224: 64 rows 35 / 39, 150 rows 48 / 52, 300 rows 63 / 69, 600 rows 97 / 104, 1200 rows 163 / 155 (the worst),
// 2400 rows 280 / 314, 4800 rows 465 / 521; K = 4096: 300 rows 21 / 24, 600 rows 30 / 26 and 1200 rows 39 / 36 (the worst), 2400 rows
// 43 / 55, 4800 rows 87 / 93.
struct TileForm {
  int bm, bn, per_cu;
  float block_us, wide_us;
};
static const TileForm kTileForms[] = {{256, 256, 1, 1.63f, 0.0f}, {160, 256, 1, 1.06f, 0.0f}, {128, 128, 2, 1.04f, 1.96f}, {64, 128, 2, 0.80f, 1.17f}};
static const int kTileFormCount = sizeof(kTileForms) / sizeof(kTileForms[0]);

static bool product_size_known(int64_t M, int64_t N, int64_t K) {
  return M <= (1 << 30) && N <= (1 << 24) && K <= (1 << 22) && (M + 63) / 64 * ((N + 63) / 64) < (1ll << 30);
}

// One launch holds the form's tiles, 512 threads each, and the pieces of a round of them.
static bool form_fits(const TileForm &f, int M, int N) {
  return (((long long)M + f.bm - 1) / f.bm) * (((long long)N + f.bn - 1) / f.bn) <= kGridThreads / 512 - kProductCus * f.per_cu;
}

static TilePlan tile_plan(const TileForm &f, int M, int N, int blocks) {
  TilePlan t;
  t.tiles_m = (M + f.bm - 1) / f.bm;
  t.tiles_n = (N + f.bn - 1) / f.bn;
  const long long tiles = (long long)t.tiles_m * t.tiles_n;
  const int slots = kProductCus * f.per_cu;
  t.whole = (int)(tiles / slots * slots);
  t.rest = (int)(tiles - t.whole);
  t.pieces = t.rest ? slots / t.rest : 1;
  if (t.pieces > blocks / 4) t.pieces = blocks / 4;  // at least four blocks each: the first one's latency is not hidden
  if (t.pieces < 1) t.pieces = 1;
  return t;
}

static size_t plan_bytes(const TileForm &f, const TilePlan &t) {
  return t.pieces > 1 ? (size_t)t.rest * t.pieces * f.bm * f.bn * sizeof(float) : 0;
}

static double plan_us(const TileForm &f, const TilePlan &t, int blocks, bool wide) {
  const double block = wide ? f.wide_us : f.block_us;
  const int slots = kProductCus * f.per_cu;
  double us = (double)(t.whole / slots) * (blocks * block + 5.0);
  if (t.rest) us += (blocks + t.pieces - 1) / t.pieces * block + 5.0;
  if (t.pieces > 1) us += 4.0 + (double)t.rest * t.pieces * f.bm * f.bn * 8 / 9.5e6;  // the sums' way through memory: 9.5 TB/s
  return us;
}

static int best_form(int M, int N, int blocks, bool wide) {
  const int forced = knob(kKnobProductForm, -1);
  if (forced >= 0 && forced < kTileFormCount && !(wide && kTileForms[forced].wide_us == 0.0f)) return forced;
  int best = 2;  // every result type has it
  double least = 1e30;
  for (int i = 0; i < kTileFormCount; ++i) {
    if (wide && kTileForms[i].wide_us == 0.0f) continue;
    const double us = plan_us(kTileForms[i], tile_plan(kTileForms[i], M, N, blocks), blocks, wide);
    if (us < least) best = i, least = us;
  }
  return best;
}

// A workgroup of product_split_kernel streams 4 KB per 16 x 16 tile and block through the chip at about 7.5 TB/s.
static bool use_tiles(int M, int N, int blocks, bool wide) {
  if (blocks == 0) return false;
  const TileForm &f = kTileForms[best_form(M, N, blocks, wide)];
  if (!form_fits(f, M, N)) return false;
  const int forced = knob(kKnobProductForm, -1);
  if (forced >= 0) return forced < kTileFormCount;
  if (M <= 16) return false;
  const double split_us = 4.0 + (double)((M + 15) / 16) * ((N + 15) / 16) * blocks * 5.5e-4;
  return plan_us(f, tile_plan(f, M, N, blocks), blocks, wide) < split_us;
}

template <int MT, int NT, int WM, int WN, int PER_CU, int DB, int MODE>
static int launch_tile(const ProductArgs &p, const TileForm &f, void *workspace, size_t workspace_bytes, hipStream_t s) {
  if (f.bm != 16 * MT * WM || f.bn != 16 * NT * WN) return set_error(FRCNN_EINVAL, "scaled_matmul: a %d x %d tile has no kernel", f.bm, f.bn);
  const TilePlan plan = tile_plan(f, p.M, p.N, p.blocks);
  const size_t need = plan_bytes(f, plan);
  if (need && !(workspace && workspace_bytes >= need))
    return set_error(FRCNN_EINVAL, "scaled_matmul: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
  constexpr int THREADS = 64 * WM * WN;
  constexpr size_t lds = (3 * 16 * MT * WM + DB * 16 * NT * WN) * kQuantBlock;
  static_assert(lds * PER_CU <= 160 * 1024, "LDS of a CU");
  int rc = ensure_dynamic_lds((const void *)product_tile_kernel<MT, NT, WM, WN, PER_CU, DB, MODE>, lds, "scaled_matmul");
  if (rc) return rc;
  hipLaunchKernelGGL((product_tile_kernel<MT, NT, WM, WN, PER_CU, DB, MODE>), dim3((unsigned)(plan.whole + plan.rest * plan.pieces)),
                     dim3(THREADS), lds, s, p, plan, (f32x4 *)workspace);
  rc = check_launch("scaled_matmul");
  if (rc || plan.pieces == 1) return rc;
  hipLaunchKernelGGL((product_join_kernel<MT, NT, WM, WN>), dim3((unsigned)(plan.rest * MT * NT)), dim3(THREADS), 0, s, p, plan,
                     (const f32x4 *)workspace);
  return check_launch("scaled_matmul");
}

template <int MODE>
static int launch_tiles(const ProductArgs &p, void *workspace, size_t workspace_bytes, hipStream_t s) {
  constexpr bool wide = MODE == kWideF32 || MODE == kWideE8M0;
  const int form = best_form(p.M, p.N, p.blocks, wide);
  const TileForm &f = kTileForms[form];
  if constexpr (!wide) {
    if (form == 0) return launch_tile<8, 4, 2, 4, 1, 2, MODE>(p, f, workspace, workspace_bytes, s);
    if (form == 1) return launch_tile<5, 4, 2, 4, 1, 3, MODE>(p, f, workspace, workspace_bytes, s);
  }
  if (form == 2) return launch_tile<4, 2, 2, 4, 2, 2, MODE>(p, f, workspace, workspace_bytes, s);
  return launch_tile<2, 2, 2, 4, 2, 3, MODE>(p, f, workspace, workspace_bytes, s);
}

template <int MODE>
static int launch_split(const ProductArgs &p, hipStream_t s) {
  const long long tn = ((long long)p.N + 15) / 16;
  const long long most = kGridThreads / (64 * kSplitWaves) / tn * 16;  // rows of one launch; N <= 2^24 leaves some
  for (long long first = 0; first < p.M; first += most) {
    ProductArgs part = p;
    part.M = (int)(p.M - first < most ? p.M - first : most);
    part.a += first * p.lda;
    part.sa = (const uint8_t *)p.sa + first * p.sa_row * (MODE == kWideE8M0 ? 1 : 4);
    part.y = (uint8_t *)p.y + first * p.ldy * (long long)type_bytes(p.out);
    const long long tm = ((long long)part.M + 15) / 16;
    hipLaunchKernelGGL((product_split_kernel<MODE>), dim3((unsigned)(tm * tn)), dim3(64 * kSplitWaves), 0, s, part, (int)tn);
    const int rc = check_launch("scaled_matmul");
    if (rc) return rc;
  }
  return FRCNN_OK;
}

template <int MODE>
static int launch_product(const ProductArgs &p, void *workspace, size_t workspace_bytes, hipStream_t s) {
  if (use_tiles(p.M, p.N, p.blocks, MODE == kWideF32 || MODE == kWideE8M0)) return launch_tiles<MODE>(p, workspace, workspace_bytes, s);
  return launch_split<MODE == kNarrowE8M0 || MODE == kWideE8M0 ? kWideE8M0 : kWideF32>(p, s);
}

}  // namespace frcnn

using namespace frcnn;

extern "C" {

size_t frcnn_scaled_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m < 1 || n < 1 || k < 1 || !product_size_known(m, n, k)) return 0;
  const int M = (int)m, N = (int)n, blocks = (int)((k + kQuantBlock - 1) / kQuantBlock);
  size_t most = 0;
  for (int wide = 0; wide < 2; ++wide) {  // the output's type decides
    if (!use_tiles(M, N, blocks, wide != 0)) continue;
    const TileForm &f = kTileForms[best_form(M, N, blocks, wide != 0)];
    const size_t bytes = plan_bytes(f, tile_plan(f, M, N, blocks));
    if (bytes > most) most = bytes;
  }
  return most;
}

int frcnn_scaled_matmul(const void *a, int64_t lda, const void *a_scales, int64_t a_scale_row_stride, int64_t a_scale_block_stride,
                        const void *b, int64_t ldb, const void *b_scales, int64_t b_scale_row_stride, int64_t b_scale_block_stride,
                        int scale_type, const float *bias, int activation, int64_t M, int64_t N, int64_t K, void *y, int y_type, int64_t ldy,
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
  if (!product_size_known(M, N, K) || lda > (1 << 23) || ldb > (1 << 23))
    return set_error(FRCNN_EUNSUPPORTED, "scaled_matmul: M=%lld, N=%lld, K=%lld (row strides %lld, %lld) is beyond what the kernels index",
                     (long long)M, (long long)N, (long long)K, (long long)lda, (long long)ldb);
  const size_t need = frcnn_scaled_matmul_workspace_bytes(M, N, K);
  FRCNN_REQUIRE(need == 0 || (workspace && aligned_to(workspace, 256) && workspace_bytes >= need),
                "scaled_matmul: workspace of %zu bytes (256-byte aligned) needed, got %zu", need, workspace_bytes);
  const int quads = N % 4 == 0 && ldy % 4 == 0 && aligned_to(y, 4 * type_bytes(y_type)) && aligned_to(bias, 16);
  const int rows16 = (ldy * (int64_t)type_bytes(y_type)) % 16 == 0 && aligned_to(y, 16);
  const ProductArgs p = {(const uint8_t *)a, (const uint8_t *)b, lda, ldb, a_scales, b_scales, a_scale_row_stride, a_scale_block_stride,
                         b_scale_row_stride, b_scale_block_stride, bias, y, ldy, (int)M, (int)N, (int)K, (int)((K + kQuantBlock - 1) / kQuantBlock),
                         activation, y_type, quads, rows16};
  const int mode = (y_type == FRCNN_F32 ? kWideF32 : kNarrowF32) + (scale_type == FRCNN_SCALE_E8M0);
  hipStream_t s = (hipStream_t)stream;
  if (mode == kNarrowF32) return launch_product<kNarrowF32>(p, workspace, workspace_bytes, s);
  if (mode == kNarrowE8M0) return launch_product<kNarrowE8M0>(p, workspace, workspace_bytes, s);
  if (mode == kWideF32) return launch_product<kWideF32>(p, workspace, workspace_bytes, s);
  return launch_product<kWideE8M0>(p, workspace, workspace_bytes, s);
}

}  // extern "C"
