// head_norm.hip -- group normalisation of channels-last tensors with an activation, and its gradients.
//
// x (N, S, C), C = G groups of Cg channels; per image n and group g, over the m = S * Cg values:
//   mean, var = E (x - mean)^2, rstd = 1 / sqrt(var + eps), xhat = (x - mean) rstd, z = gamma xhat + beta, y = act(z)
//   dz = dy act'(z), dgamma = sum dz xhat, dbeta = sum dz, d = gamma dz,
//   dx = rstd (d - E d - xhat E (d xhat))          (the expectations over the same m values)
//
// Bound by memory: x read and y written once; x, dy read and dx written once.  A workgroup takes a slab of channels (whole
// groups) of one image and keeps it in registers, so the variance is that of the centred values (no cancellation) and the
// data is read once.  Where a slab of one image does not fit a workgroup's registers the positions are cut into chunks:
// statistics per chunk, joined in a fixed order (Chan, Golub and LeVeque's update), then a second pass over the data.
//
// A thread owns one pack of channels (a column) and walks the positions.  It hands over one number per sum where its pack lies in
// one group, one per channel where it straddles groups; lanes of one wave add a group's.
// No atomics: results do not depend on the order in which workgroups run.
#include "head_common.hpp"

namespace frcnn {

enum { kActNone = FRCNN_ACT_NONE, kActRelu = FRCNN_ACT_RELU, kActSwish = FRCNN_ACT_SWISH };

__device__ __forceinline__ float sigmoid_fast(float z) {  // exp2 and rcp are good to one unit in the last place each
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == kActRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if (ACT == kActSwish) return z * sigmoid_fast(z);
  return z;
}

template <int ACT>
__device__ __forceinline__ float activate_grad(float dy, float z) {
  if (ACT == kActRelu) return z > 0.0f ? dy : 0.0f;
  if (ACT == kActSwish) {
    const float s = sigmoid_fast(z);
    return dy * (s * __builtin_fmaf(z, 1.0f - s, 1.0f));
  }
  return dy;
}

// f(which) with the activation as a constant: one uniform branch around a loop instead of one per element.
template <int A>
struct ActivationIs {
  static constexpr int value = A;
};
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
  if (act == kActRelu) f(ActivationIs<kActRelu>());
  else if (act == kActSwish) f(ActivationIs<kActSwish>());
  else f(ActivationIs<kActNone>());
}

// f(which) with the way of storing as a constant: around a loop, since two stores in the arms of a branch become one plain one.
template <bool P>
struct PastIs {
  static constexpr bool value = P;
};
template <typename F>
__device__ __forceinline__ void with_past(bool past, F f) {
  if (past) f(PastIs<true>());
  else f(PastIs<false>());
}

struct NormShape {
  int N, S, C, G, Cg;
  int slab;    // channels per workgroup, whole groups; the last slab of a row may be shorter
  int slabs;   // ceil(C / slab)
  int chunk;   // positions per workgroup
  int chunks;  // ceil(S / chunk)
  int rows;    // positions a workgroup's threads cover at a time
  bool past;   // results are whole lines: stored past the caches
};

// The workgroup's place.  Slabs that share lines of memory run on one XCD, whose L2 joins their reads and writes: from all XCDs
// (16, 1024, 576) fp32 in slabs of 144 bytes fetches 66 MB instead of 38, and takes 23.5 us instead of 18.6; (64, 196, 576) with
// gradients 62.5 us instead of 53.5.  Where they share nothing this only costs: (8, 3969, 512) fp16 24.4 us to 25.3.
__device__ __forceinline__ unsigned place_of(const NormShape &s) {
  return s.past ? blockIdx.x : (unsigned)xcd_contiguous((int)blockIdx.x, (int)gridDim.x);
}

// ---- reductions inside a workgroup ---------------------------------------------------------------------------------------
// red[rows][slab]: sum over the rows, into row 0.  `row` < rows are the threads that own data; halving keeps the order fixed.
template <int VEC, int K>
__device__ __forceinline__ void rows_to_first(float *red, int rows, int slab, int row, int col, bool active, float (&v)[K][VEC]) {
  // each of the K sums has its own plane of rows * slab floats
  const int plane = rows * slab;
  if (active)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) red[k * plane + row * slab + col + e] = v[k][e];
  int n = rows;
  while (n > 1) {
    const int half = (n + 1) >> 1;
    __syncthreads();
    if (active && row + half < n)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[k][e] += red[k * plane + (row + half) * slab + col + e];
          red[k * plane + row * slab + col + e] = v[k][e];
        }
    n = half;
  }
  __syncthreads();
}

// out[k][g] = the sum of red[k][row][g * width + c] over the rows and c < width, for K sums (planes of red) at once.  P lanes (a
// power of two <= 64) per group, along the longer of the two directions.
template <int K>
__device__ __forceinline__ void groups_of(const float *red, int rows, int columns, int groups, int width, float *out, int stride) {
  const bool down = rows >= width;
  const int along = down ? rows : width, across = down ? width : rows;
  const int step_along = down ? columns : 1, step_across = down ? 1 : columns;
  int P = 1;
  while (P < along && P < 64) P <<= 1;
  const int per = (int)blockDim.x / P;
  const int sub = threadIdx.x & (P - 1), first = threadIdx.x / P;
  for (int base = 0; base < groups; base += per) {
    const int g = base + first;
    float s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = 0.0f;
    if (g < groups)
      for (int i = sub; i < along; i += P) {
        const float *at = red + g * width + i * step_along;
        for (int j = 0; j < across; ++j)
#pragma unroll
          for (int k = 0; k < K; ++k) s[k] += at[k * rows * columns + j * step_across];
      }
    for (int d = P >> 1; d > 0; d >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] += __shfl_xor(s[k], d);
    if (g < groups && sub == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) out[k * stride + g] = s[k];
  }
  __syncthreads();
}

// A pack's groups: one where the pack's width divides Cg (ONE), otherwise one per element.
template <int VEC, bool ONE>
struct Groups {
  static constexpr int N = ONE ? 1 : VEC;
  __device__ __forceinline__ static constexpr int of(int e) { return ONE ? 0 : e; }
};

template <int VEC>
struct Column {  // a thread's place in the slab
  int row, col, rows;  // first row, first channel of its pack inside the slab, rows per pass
  int width;           // channels of this slab
  bool active;
  __device__ __forceinline__ Column(const NormShape &s, int slab_index) {
    width = min(s.slab, s.C - slab_index * s.slab);
    const int vc = s.slab / VEC;  // the same for every slab, also a shorter last one
    rows = s.rows;
    row = (int)threadIdx.x / vc;
    col = ((int)threadIdx.x - row * vc) * VEC;
    active = row < rows && col < width;
  }
};

// out[k][g] = the sums of v[k] over the group's channels and all rows.  With one group per pack a thread hands over one number
// per sum, otherwise one per channel.
template <int VEC, bool ONE, int K>
__device__ __forceinline__ void group_sums(const NormShape &s, const Column<VEC> &me, float *red, const float (&v)[K][VEC], float *out) {
  const int groups = me.width / s.Cg, stride = s.slab / s.Cg;
  const int columns = ONE ? s.slab / VEC : s.slab;
  if (me.active)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float *at = red + (k * s.rows + me.row) * columns + (ONE ? me.col / VEC : me.col);
      if constexpr (ONE) {
        float t = v[k][0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) t += v[k][e];
        *at = t;
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) at[e] = v[k][e];
      }
    }
  __syncthreads();
  groups_of<K>(red, s.rows, columns, groups, ONE ? s.Cg / VEC : s.Cg, out, stride);
}

template <int VEC>
__device__ __forceinline__ void load_parameters(const float *p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = *p;
  } else {
    typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // a four-word load needs four-byte alignment
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const f32x4 v = *reinterpret_cast<const f32x4_any *>(p + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * i + e] = v[e];
    }
  }
}

// ---- forward, a slab of one image (or one chunk of it) in registers --------------------------------------------------------
// WRITE: apply and write y (the whole image is here: chunks == 1).  Otherwise only the chunk's mean and the sum of its
// squared deviations go to `part` (N, chunks, G, 2).
template <typename T, int VEC, bool ONE, int NV, bool WRITE>
__global__ __launch_bounds__(1024) void norm_resident_kernel(const T *__restrict__ x, T *__restrict__ y, const float *__restrict__ gamma,
                                                           const float *__restrict__ beta, float *__restrict__ stats, NormShape s,
                                                           float eps, int act) {
  extern __shared__ float lds[];
  const unsigned place = place_of(s);
  const int slab_index = (int)(place % (unsigned)s.slabs);
  const int rest = (int)(place / (unsigned)s.slabs);
  const int chunk_index = rest % s.chunks, n = rest / s.chunks;
  const Column<VEC> me(s, slab_index);
  const int c0 = slab_index * s.slab + me.col;
  const int p0 = chunk_index * s.chunk;
  const int count = min(s.chunk, s.S - p0);
  const long long base = ((long long)n * s.S + p0) * s.C + c0;
  const int groups = me.width / s.Cg;
  float *red = lds, *gsum = lds + me.rows * s.slab, *grstd = gsum + s.slab / s.Cg;

  Pack<T, VEC> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = me.row + i * me.rows;
    v[i] = (me.active && p < count) ? Pack<T, VEC>::load(x + base + (long long)p * s.C) : Pack<T, VEC>::zero();
  }
  using Gs = Groups<VEC, ONE>;
  int group[Gs::N];
#pragma unroll
  for (int e = 0; e < Gs::N; ++e) group[e] = me.active ? (me.col + e) / s.Cg : 0;

  float sum[1][VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[0][e] = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[VEC];
    v[i].unpack(f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[0][e] += f[e];  // rows beyond the end hold zeros
  }
  group_sums<VEC, ONE, 1>(s, me, red, sum, gsum);
  const float inv = 1.0f / ((float)count * (float)s.Cg);

  float mean[Gs::N];
#pragma unroll
  for (int e = 0; e < Gs::N; ++e) mean[e] = gsum[group[e]] * inv;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[0][e] = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (me.row + i * me.rows < count) {
      float f[VEC];
      v[i].unpack(f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = f[e] - mean[Gs::of(e)];
        sum[0][e] = __builtin_fmaf(d, d, sum[0][e]);
      }
    }
  }
  group_sums<VEC, ONE, 1>(s, me, red, sum, grstd);

  const int g0 = slab_index * s.slab / s.Cg;
  if constexpr (!WRITE) {
    float *part = stats + (((long long)n * s.chunks + chunk_index) * s.G + g0) * 2;
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
      part[2 * g] = gsum[g] * inv;
      part[2 * g + 1] = grstd[g];
    }
  } else {
    if (stats) {
      float *out = stats + ((long long)n * s.G + g0) * 2;
      for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        out[2 * g] = gsum[g] * inv;
        out[2 * g + 1] = 1.0f / __builtin_sqrtf(__builtin_fmaf(grstd[g], inv, eps));
      }
    }
    if (!me.active) return;
    float a[VEC], b[VEC], rstd[Gs::N];
#pragma unroll
    for (int e = 0; e < Gs::N; ++e) rstd[e] = 1.0f / __builtin_sqrtf(__builtin_fmaf(grstd[group[e]], inv, eps));
    load_parameters(gamma + c0, a);
    load_parameters(beta + c0, b);
#pragma unroll
    for (int e = 0; e < VEC; ++e) a[e] *= rstd[Gs::of(e)];
    with_activation(act, [&](auto which) {
      with_past(s.past, [&](auto how) {
        constexpr int ACT = decltype(which)::value;
        constexpr bool PAST = decltype(how)::value;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int p = me.row + i * me.rows;
          if (p < count) {
            float f[VEC];
            v[i].unpack(f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = activate<ACT>(__builtin_fmaf(f[e] - mean[Gs::of(e)], a[e], b[e]));
            Pack<T, VEC>::template store<PAST>(y + base + (long long)p * s.C, f);
          }
        }
      });
    });
  }
}

// Joins the chunks' statistics: one wave per (image, group); the chunks a lane takes and the order of the joins are fixed.
__device__ __forceinline__ void join_stats(float &mean, float &m2, float &have, float mean_b, float m2_b, float count_b) {
  if (count_b == 0.0f) return;
  if (have == 0.0f) {
    mean = mean_b, m2 = m2_b, have = count_b;
    return;
  }
  const float d = mean_b - mean, total = have + count_b, w = count_b / total;
  mean = __builtin_fmaf(d, w, mean);
  m2 += __builtin_fmaf(d * d, have * w, m2_b);
  have = total;
}

__global__ __launch_bounds__(256) void norm_join_kernel(const float *__restrict__ part, float *__restrict__ stats, NormShape s, float eps) {
  const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= (long long)s.N * s.G) return;
  const long long n = i / s.G;
  const int g = (int)(i - n * s.G);
  float mean = 0.0f, m2 = 0.0f, have = 0.0f;
  for (int c = lane_id(); c < s.chunks; c += 64) {
    const f32x2 p = *reinterpret_cast<const f32x2 *>(part + ((n * s.chunks + c) * s.G + g) * 2);
    join_stats(mean, m2, have, p.x, p.y, (float)min(s.chunk, s.S - c * s.chunk) * (float)s.Cg);
  }
  for (int d = 32; d > 0; d >>= 1) {
    const float mean_b = __shfl_xor(mean, d), m2_b = __shfl_xor(m2, d), have_b = __shfl_xor(have, d);
    join_stats(mean, m2, have, mean_b, m2_b, have_b);
  }
  if (lane_id() == 0) {
    stats[2 * i] = mean;
    stats[2 * i + 1] = 1.0f / __builtin_sqrtf(m2 / have + eps);
  }
}

// y from x and the joined statistics; the thread layout of norm_resident_kernel.
template <typename T, int VEC, bool ONE>
__global__ __launch_bounds__(1024) void norm_apply_kernel(const T *__restrict__ x, T *__restrict__ y, const float *__restrict__ gamma,
                                                          const float *__restrict__ beta, const float *__restrict__ stats, NormShape s,
                                                          int act) {
  using Gs = Groups<VEC, ONE>;
  const int slab_index = (int)(blockIdx.x % (unsigned)s.slabs);
  const int rest = (int)(blockIdx.x / (unsigned)s.slabs);
  const int chunk_index = rest % s.chunks, n = rest / s.chunks;
  const Column<VEC> me(s, slab_index);
  if (!me.active) return;
  const int c0 = slab_index * s.slab + me.col;
  const int p0 = chunk_index * s.chunk;
  const int count = min(s.chunk, s.S - p0);
  const long long base = ((long long)n * s.S + p0) * s.C + c0;
  float mean[Gs::N], rstd[Gs::N], a[VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < Gs::N; ++e) {
    const f32x2 st = *reinterpret_cast<const f32x2 *>(stats + ((long long)n * s.G + (c0 + e) / s.Cg) * 2);
    mean[e] = st.x;
    rstd[e] = st.y;
  }
  load_parameters(gamma + c0, a);
  load_parameters(beta + c0, b);
#pragma unroll
  for (int e = 0; e < VEC; ++e) a[e] *= rstd[Gs::of(e)];
  with_activation(act, [&](auto which) {
    with_past(s.past, [&](auto how) {
      constexpr int ACT = decltype(which)::value;
      constexpr bool PAST = decltype(how)::value;
#pragma unroll 4
      for (int p = me.row; p < count; p += me.rows) {
        float f[VEC];
        Pack<T, VEC>::load(x + base + (long long)p * s.C).unpack(f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = activate<ACT>(__builtin_fmaf(f[e] - mean[Gs::of(e)], a[e], b[e]));
        Pack<T, VEC>::template store<PAST>(y + base + (long long)p * s.C, f);
      }
    });
  });
}

// ---- gradients -------------------------------------------------------------------------------------------------------------
template <int VEC, bool ONE>
struct GradCoefficients {
  using Gs = Groups<VEC, ONE>;
  float mean[Gs::N], rstd[Gs::N], gamma[VEC], beta[VEC];
  __device__ __forceinline__ void parameters(const float *__restrict__ g, const float *__restrict__ b, int c0) {
    load_parameters(g + c0, gamma);
    load_parameters(b + c0, beta);
  }
  __device__ __forceinline__ void statistics(const float *__restrict__ stats, const NormShape &s, int n, int c0) {
#pragma unroll
    for (int e = 0; e < Gs::N; ++e) {
      const f32x2 st = *reinterpret_cast<const f32x2 *>(stats + ((long long)n * s.G + (c0 + e) / s.Cg) * 2);
      mean[e] = st.x;
      rstd[e] = st.y;
    }
  }
  __device__ __forceinline__ float xhat(int e, float x) const { return (x - mean[Gs::of(e)]) * rstd[Gs::of(e)]; }
  template <int ACT>
  __device__ __forceinline__ float dz(int e, float xh, float dy) const {
    return activate_grad<ACT>(dy, __builtin_fmaf(xh, gamma[e], beta[e]));
  }
  __device__ __forceinline__ float dx(int e, float xh, float dz, float d1, float d2) const {
    return rstd[Gs::of(e)] * __builtin_fmaf(-xh, d2, __builtin_fmaf(dz, gamma[e], -d1));
  }
};

// A slab of one image's x and dz in registers, x as it is stored and dz in fp32, so that the activation's gradient is computed
// once; each workgroup takes `per` images in turn and leaves its sums for dgamma and dbeta in sums (workgroups along N, C, 2).
template <typename T, int VEC, bool ONE, int NV>
__global__ __launch_bounds__(512) void norm_grad_resident_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                                                                 const float *__restrict__ gamma, const float *__restrict__ beta,
                                                                 const float *__restrict__ stats, T *__restrict__ dx,
                                                                 float *__restrict__ sums, NormShape s, int per, int act) {
  extern __shared__ float lds[];
  using Gs = Groups<VEC, ONE>;
  const unsigned place = place_of(s);
  const int slab_index = (int)(place % (unsigned)s.slabs);
  const int part = (int)(place / (unsigned)s.slabs);
  const Column<VEC> me(s, slab_index);
  const int c0 = slab_index * s.slab + me.col;
  float *red = lds, *first = lds + 2 * me.rows * s.slab, *second = first + s.slab / s.Cg;
  int group[Gs::N];
#pragma unroll
  for (int e = 0; e < Gs::N; ++e) group[e] = me.active ? (me.col + e) / s.Cg : 0;
  GradCoefficients<VEC, ONE> k;
  if (me.active) k.parameters(gamma, beta, c0);
  float total[2][VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) total[0][e] = total[1][e] = 0.0f;
  const float inv = 1.0f / ((float)s.S * (float)s.Cg);

  const int last = min(s.N, (part + 1) * per);
  for (int n = part * per; n < last; ++n) {
    const long long base = (long long)n * s.S * s.C + c0;
    Pack<T, VEC> vx[NV], vd[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int p = me.row + i * me.rows;
      const bool in = me.active && p < s.S;
      vx[i] = in ? Pack<T, VEC>::load(x + base + (long long)p * s.C) : Pack<T, VEC>::zero();
      vd[i] = in ? Pack<T, VEC>::load(dy + base + (long long)p * s.C) : Pack<T, VEC>::zero();
    }
    if (me.active) k.statistics(stats, s, n, c0);
    float sum[2][VEC], dz[NV][VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[0][e] = sum[1][e] = 0.0f;
    with_activation(act, [&](auto which) {
      constexpr int ACT = decltype(which)::value;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        vd[i].unpack(dz[i]);
        if (me.row + i * me.rows < s.S) {
          float fx[VEC];
          vx[i].unpack(fx);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xh = k.xhat(e, fx[e]);
            dz[i][e] = k.template dz<ACT>(e, xh, dz[i][e]);
            sum[0][e] += dz[i][e];
            sum[1][e] = __builtin_fmaf(dz[i][e], xh, sum[1][e]);
          }
        }
      }
    });
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      total[0][e] += sum[0][e];
      total[1][e] += sum[1][e];
      sum[0][e] *= k.gamma[e];
      sum[1][e] *= k.gamma[e];
    }
    group_sums<VEC, ONE, 2>(s, me, red, sum, first);
    if (me.active) {
      float d1[Gs::N], d2[Gs::N];
#pragma unroll
      for (int e = 0; e < Gs::N; ++e) {
        d1[e] = first[group[e]] * inv;
        d2[e] = second[group[e]] * inv;
      }
      with_past(s.past, [&](auto how) {
        constexpr bool PAST = decltype(how)::value;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int p = me.row + i * me.rows;
          if (p < s.S) {
            float f[VEC];
            vx[i].unpack(f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = k.dx(e, k.xhat(e, f[e]), dz[i][e], d1[Gs::of(e)], d2[Gs::of(e)]);
            Pack<T, VEC>::template store<PAST>(dx + base + (long long)p * s.C, f);
          }
        }
      });
    }
    __syncthreads();  // red, first and second are free for the next image
  }
  rows_to_first<VEC, 2>(red, me.rows, s.slab, me.row, me.col, me.active, total);
  if (me.active && me.row == 0)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float *o = sums + ((long long)part * s.C + c0 + e) * 2;
      o[0] = total[0][e];
      o[1] = total[1][e];
    }
}

// Per-channel sums of one chunk of positions, into sums (N, chunks, C, 2).
template <typename T, int VEC, bool ONE>
__global__ __launch_bounds__(512) void norm_grad_sums_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                                                             const float *__restrict__ gamma, const float *__restrict__ beta,
                                                             const float *__restrict__ stats, float *__restrict__ sums, NormShape s,
                                                             int act) {
  extern __shared__ float lds[];
  const int slab_index = (int)(blockIdx.x % (unsigned)s.slabs);
  const int rest = (int)(blockIdx.x / (unsigned)s.slabs);
  const int chunk_index = rest % s.chunks, n = rest / s.chunks;
  const Column<VEC> me(s, slab_index);
  const int c0 = slab_index * s.slab + me.col;
  const int p0 = chunk_index * s.chunk;
  const int count = min(s.chunk, s.S - p0);
  const long long base = ((long long)n * s.S + p0) * s.C + c0;
  float sum[2][VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[0][e] = sum[1][e] = 0.0f;
  if (me.active) {
    GradCoefficients<VEC, ONE> k;
    k.parameters(gamma, beta, c0);
    k.statistics(stats, s, n, c0);
    with_activation(act, [&](auto which) {
      constexpr int ACT = decltype(which)::value;
#pragma unroll 4
      for (int p = me.row; p < count; p += me.rows) {
        float fx[VEC], fd[VEC];
        Pack<T, VEC>::load(x + base + (long long)p * s.C).unpack(fx);
        Pack<T, VEC>::load(dy + base + (long long)p * s.C).unpack(fd);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = k.xhat(e, fx[e]), dz = k.template dz<ACT>(e, xh, fd[e]);
          sum[0][e] += dz;
          sum[1][e] = __builtin_fmaf(dz, xh, sum[1][e]);
        }
      }
    });
  }
  rows_to_first<VEC, 2>(lds, me.rows, s.slab, me.row, me.col, me.active, sum);
  if (me.active && me.row == 0)
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      *reinterpret_cast<f32x2 *>(sums + (((long long)n * s.chunks + chunk_index) * s.C + c0 + e) * 2) = f32x2{sum[0][e], sum[1][e]};
}

// One workgroup per (image, group): the chunks' sums become E d and E (d xhat), and the image's per-channel sums.  Its threads
// form `lanes` columns of channels times 256 / lanes rows of chunks.
__global__ __launch_bounds__(256) void norm_grad_join_kernel(const float *__restrict__ sums, const float *__restrict__ gamma,
                                                             float *__restrict__ image_sums, float *__restrict__ expect, NormShape s) {
  const int g = (int)(blockIdx.x % (unsigned)s.G), n = (int)(blockIdx.x / (unsigned)s.G);
  __shared__ f32x2 red[256];
  int lanes = 1;
  while (lanes < s.Cg && lanes < 256) lanes <<= 1;
  const int lane = (int)threadIdx.x & (lanes - 1), row = (int)threadIdx.x / lanes, rows = 256 / lanes;
  f32x2 d = {0.0f, 0.0f};
  for (int c0 = 0; c0 < s.Cg; c0 += lanes) {
    const int c = c0 + lane, ch = g * s.Cg + c;
    f32x2 v = {0.0f, 0.0f};
    if (c < s.Cg) {
#pragma unroll 8
      for (int k = row; k < s.chunks; k += rows) v += *reinterpret_cast<const f32x2 *>(sums + (((long long)n * s.chunks + k) * s.C + ch) * 2);
    }
    red[threadIdx.x] = v;
    __syncthreads();
    for (int half = rows >> 1; half > 0; half >>= 1) {
      if (row < half) red[threadIdx.x] += red[threadIdx.x + half * lanes];
      __syncthreads();
    }
    if (row == 0 && c < s.Cg) {
      v = red[lane];
      *reinterpret_cast<f32x2 *>(image_sums + ((long long)n * s.C + ch) * 2) = v;
      d += v * gamma[ch];
    }
    __syncthreads();
  }
  red[threadIdx.x] = d;  // zeros but for the first row
  __syncthreads();
  for (int half = 128; half > 0; half >>= 1) {
    if ((int)threadIdx.x < half) red[threadIdx.x] += red[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float m = (float)s.S * (float)s.Cg;
    *reinterpret_cast<f32x2 *>(expect + ((long long)n * s.G + g) * 2) = f32x2{red[0].x / m, red[0].y / m};
  }
}

// dbeta[c], dgamma[c] = the sums of `parts` rows of (C, 2): 8 channels per block, THREADS / 16 threads down the rows of each.
template <int THREADS>
__device__ __forceinline__ void parameter_sums(int block, const float *__restrict__ sums, long long parts, int C, float *__restrict__ dgamma,
                                               float *__restrict__ dbeta) {
  constexpr int DOWN = THREADS / 16;
  __shared__ float red[DOWN][17];
  const int j = threadIdx.x & 15, r = threadIdx.x >> 4;
  const long long at = (long long)block * 16 + j;  // of 2 C
  float s = 0.0f;
  if (at < 2ll * C) {
#pragma unroll 8
    for (long long p = r; p < parts; p += DOWN) s += sums[p * 2 * C + at];
  }
  red[r][j] = s;
  __syncthreads();
  for (int half = DOWN / 2; half > 0; half >>= 1) {
    if (r < half) red[r][j] += red[r + half][j];
    __syncthreads();
  }
  if (r == 0 && at < 2ll * C) ((at & 1) ? dgamma : dbeta)[at >> 1] = red[0][j];
}

static unsigned parameter_blocks(int C) { return (unsigned)((2ll * C + 15) / 16); }

__global__ __launch_bounds__(1024) void norm_grad_params_kernel(const float *__restrict__ sums, long long parts, int C,
                                                                float *__restrict__ dgamma, float *__restrict__ dbeta) {
  parameter_sums<1024>((int)blockIdx.x, sums, parts, C, dgamma, dbeta);
}

// dx; the first `param_blocks` workgroups add up the images' sums for dgamma and dbeta.
template <typename T, int VEC, bool ONE>
__global__ __launch_bounds__(512) void norm_grad_apply_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                                                              const float *__restrict__ gamma, const float *__restrict__ beta,
                                                              const float *__restrict__ stats, const float *__restrict__ expect,
                                                              T *__restrict__ dx, const float *__restrict__ image_sums,
                                                              float *__restrict__ dgamma, float *__restrict__ dbeta,
                                                              unsigned param_blocks, NormShape s, int act) {
  using Gs = Groups<VEC, ONE>;
  if (blockIdx.x < param_blocks) {
    parameter_sums<512>((int)blockIdx.x, image_sums, s.N, s.C, dgamma, dbeta);
    return;
  }
  const unsigned block = blockIdx.x - param_blocks;
  const int slab_index = (int)(block % (unsigned)s.slabs);
  const int rest = (int)(block / (unsigned)s.slabs);
  const int chunk_index = rest % s.chunks, n = rest / s.chunks;
  const Column<VEC> me(s, slab_index);
  if (!me.active) return;
  const int c0 = slab_index * s.slab + me.col;
  const int p0 = chunk_index * s.chunk;
  const int count = min(s.chunk, s.S - p0);
  const long long base = ((long long)n * s.S + p0) * s.C + c0;
  GradCoefficients<VEC, ONE> k;
  k.parameters(gamma, beta, c0);
  k.statistics(stats, s, n, c0);
  float d1[Gs::N], d2[Gs::N];
#pragma unroll
  for (int e = 0; e < Gs::N; ++e) {
    const f32x2 o = *reinterpret_cast<const f32x2 *>(expect + ((long long)n * s.G + (c0 + e) / s.Cg) * 2);
    d1[e] = o.x;
    d2[e] = o.y;
  }
  with_activation(act, [&](auto which) {
    with_past(s.past, [&](auto how) {
      constexpr int ACT = decltype(which)::value;
      constexpr bool PAST = decltype(how)::value;
#pragma unroll 4
      for (int p = me.row; p < count; p += me.rows) {
        float fx[VEC], fd[VEC];
        Pack<T, VEC>::load(x + base + (long long)p * s.C).unpack(fx);
        Pack<T, VEC>::load(dy + base + (long long)p * s.C).unpack(fd);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = k.xhat(e, fx[e]);
          fd[e] = k.dx(e, xh, k.template dz<ACT>(e, xh, fd[e]), d1[Gs::of(e)], d2[Gs::of(e)]);
        }
        Pack<T, VEC>::template store<PAST>(dx + base + (long long)p * s.C, fd);
      }
    });
  });
}

// ---- the choice of a split -------------------------------------------------------------------------------------------------
static const int kNormColumns = 512;   // packs of a slab at most: one row of threads
static const int kNormLine = 128;      // bytes of a slab's row that are worth a read of their own

struct NormPlan {
  NormShape s;
  int vec;      // elements per pack; 0: not supported
  bool one;     // a pack lies in one group
  int threads;
  int nv;       // packs a thread holds
  bool resident;
};

static int gcd_int(int a, int b) { return b ? gcd_int(b, a % b) : a; }

// Threads for a slab of `columns` packs of S positions, `most` packs per thread: the least idle lanes, and near four packs each
// (bytes in flight against registers, that is waves).  0: none fits.
static int norm_threads(int columns, int S, int most, int limit) {
  int best = 0;
  float least = 0;
  for (int t = 64; t <= limit; t += 64) {
    const int rows = t / columns;
    if (!rows) continue;
    const int need = (S + rows - 1) / rows;
    if (need > most) continue;
    const float cost = (float)t * need / ((float)columns * S) + 0.02f * (need > 4 ? need - 4 : 4 - need);
    if (!best || cost < least) best = t, least = cost;
  }
  return best;
}

// Whole images per workgroup where a slab's packs fit its registers, chunks of positions otherwise.  grad: x and dz are held, in up
// to 512 threads of 8 packs; the forward pass holds x, in up to 1024 threads of 16 (12 of 16-bit types).
static NormPlan norm_plan(int N, int S, int C, int G, int elem, bool aligned, bool grad) {
  NormPlan p = {};
  p.s.N = N, p.s.S = S, p.s.C = C, p.s.G = G, p.s.Cg = C / G;
  int vec = aligned && ((long long)C * elem) % 16 == 0 ? 16 / elem : 1;
  long long unit = (long long)p.s.Cg / gcd_int(p.s.Cg, vec) * vec;  // channels: whole groups and whole packs
  if (unit / vec > kNormColumns && vec > 1) {
    vec = 1;
    unit = p.s.Cg;
  }
  if (unit / vec > kNormColumns) return p;
  p.vec = vec;
  p.one = p.s.Cg % vec == 0;
  const long long units = C / unit;
  long long widest = kNormColumns * (long long)vec / unit;  // units per slab
  if (widest > units) widest = units;
  auto threads = [&](long long k, int most, int limit) { return norm_threads((int)(k * unit / vec), S, most, limit); };
  // Packs per thread and threads, in the order in which they are tried.  Small workgroups, of which two or more share a CU and
  // overlap one's loads with another's sums, before large ones: (6000, 49, 512) bf16 forward 125 us with 256 threads and 142 with
  // 448, its gradients 207 and 229; not in
  // fp32, where a narrower slab's shorter rows cost more: (4800, 49, 576) forward 222 us against 204.
  // What registers do not hold goes to chunks too: 16 packs of eight elements in 1024 threads spill ((16, 1024, 720) fp16 forward 57 us,
  // 24 in chunks), and 512 threads of the gradients' 16-bit packs across groups take nearly all registers ((100, 196, 720) bf16
  // 80 us, 64 in chunks; (2000, 196, 720) 1475 and 1050; (600, 196, 720) 305 and 317; others within 2 %; both with the forward call).
  const int choices[3][2] = {{8, elem == 2 ? 256 : 0}, {8, grad && elem == 2 && !p.one ? 0 : 512}, {elem == 2 ? 12 : 16, grad ? 0 : 1024}};
  int most = 0, limit = 0;
  // the widest slab that fits; narrower ones while the chip is not full and a row is still a line
  long long k = widest;
  auto narrow_enough = [&]() {
    for (k = widest;; k = (k + 1) / 2) {
      if (threads(k, most, limit)) return k == units || k * unit * elem >= kNormLine;
      if (k == 1) return false;
    }
  };
  for (const auto &c : choices) {
    most = c[0], limit = c[1];
    p.resident = !knob(kKnobNormChunked, 0) && narrow_enough();
    if (p.resident) break;
  }
  if (p.resident) {
    while (k > 1 && (long long)N * ((units + k - 1) / k) < 1024 && (k + 1) / 2 * unit * elem >= kNormLine && threads((k + 1) / 2, most, limit))
      k = (k + 1) / 2;
    p.threads = threads(k, most, limit);
    p.s.chunk = S;
  } else {
    k = widest;
    p.threads = 512;
  }
  p.s.slab = (int)(k * unit);
  p.s.slabs = (int)((units + k - 1) / k);
  p.s.rows = p.threads / (p.s.slab / vec);
  // Stores past the caches leave them to what is read: (16, 3969, 512) fp32 forward 81 us to 68, (1500, 49, 576) with gradients 187
  // to 171.  Not where neighbouring workgroups share lines: (16, 1024, 576) in slabs of 144 bytes would take 29 us instead of 20.
  p.s.past = p.s.slabs == 1 || ((long long)p.s.slab * elem % kNormLine == 0 && (long long)C * elem % kNormLine == 0);
  if (!p.resident) {
    int per = 8;  // packs per thread and chunk; fewer while the chip is not full, at least four for a chunk's fixed costs
    while (per > 4 && (long long)N * p.s.slabs * ((S + p.s.rows * per - 1) / (p.s.rows * per)) < 400) per /= 2;
    p.s.chunk = p.s.rows * per;
  }
  p.s.chunks = (S + p.s.chunk - 1) / p.s.chunk;
  p.nv = (p.s.chunk + p.s.rows - 1) / p.s.rows;
  if (p.nv > 8) p.nv = p.nv > 12 ? 16 : 12;
  if (vec == 1) p.nv = p.nv > 8 ? 16 : p.nv > 4 ? 8 : p.nv > 1 ? 4 : 1;
  return p;
}

// images per workgroup: about a thousand rows of partial sums are left for the last kernel
static int grad_images_per_group(const NormPlan &p) { return (int)(((long long)p.s.N * p.s.slabs + 1023) / 1024); }

template <typename T, int VEC, bool ONE, int NV, bool WRITE>
static int launch_resident(const NormPlan &p, const void *x, void *y, const float *gamma, const float *beta, float *out, float eps, int act,
                           hipStream_t stream) {
  const size_t lds = ((size_t)p.s.rows * p.s.slab + 2 * (p.s.slab / p.s.Cg)) * sizeof(float);
  const dim3 grid((unsigned)((long long)p.s.N * p.s.chunks * p.s.slabs));
  const int rc = ensure_dynamic_lds((const void *)norm_resident_kernel<T, VEC, ONE, NV, WRITE>, lds, "group_norm");
  if (rc) return rc;
  hipLaunchKernelGGL((norm_resident_kernel<T, VEC, ONE, NV, WRITE>), grid, dim3(p.threads), lds, stream, (const T *)x, (T *)y, gamma, beta,
                     out, p.s, eps, act);
  return check_launch("group_norm");
}

template <typename T, int VEC, bool ONE>
static int launch_norm(const NormPlan &p, const void *x, void *y, const float *gamma, const float *beta, float *stats,
                       float *workspace, float eps, int act, hipStream_t stream) {
#define FRCNN_NORM(NV, W) return launch_resident<T, VEC, ONE, NV, W>(p, x, y, gamma, beta, W ? stats : workspace, eps, act, stream)
  if (p.resident) {
    switch (p.nv) {
      case 1: FRCNN_NORM(1, true);
      case 4: FRCNN_NORM(4, true);
      case 8: FRCNN_NORM(8, true);
    }
    if constexpr (VEC == 1 || sizeof(T) == 4)
      if (p.nv == 16) FRCNN_NORM(16, true);
    if constexpr (VEC > 1) switch (p.nv) {
      case 2: FRCNN_NORM(2, true);
      case 3: FRCNN_NORM(3, true);
      case 5: FRCNN_NORM(5, true);
      case 6: FRCNN_NORM(6, true);
      case 7: FRCNN_NORM(7, true);
      case 12: FRCNN_NORM(12, true);
    }
    return set_error(FRCNN_EUNSUPPORTED, "group_norm: no kernel for %d packs", p.nv);
  }
  auto chunks = [&]() -> int {
    if (p.nv <= 4) FRCNN_NORM(4, false);
    FRCNN_NORM(8, false);
  };
#undef FRCNN_NORM
  int rc = chunks();
  if (rc) return rc;
  const dim3 grid((unsigned)((long long)p.s.N * p.s.chunks * p.s.slabs));
  float *joined = stats ? stats : workspace + (size_t)p.s.N * p.s.chunks * p.s.G * 2;
  hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)(((long long)p.s.N * p.s.G + 3) / 4)), dim3(256), 0, stream, workspace,
                     joined, p.s, eps);
  rc = check_launch("group_norm");
  if (rc) return rc;
  hipLaunchKernelGGL((norm_apply_kernel<T, VEC, ONE>), grid, dim3(p.threads), 0, stream, (const T *)x, (T *)y, gamma, beta, joined, p.s, act);
  return check_launch("group_norm");
}

template <typename T, int VEC, bool ONE, int NV>
static int launch_grad_resident(const NormPlan &p, const void *dy, const void *x, const float *gamma, const float *beta, const float *stats,
                                void *dx, float *sums, int per, long long parts, int act, hipStream_t stream) {
  const NormShape &s = p.s;
  const size_t lds = (2 * (size_t)s.rows * s.slab + 2 * (s.slab / s.Cg)) * sizeof(float);
  const int rc = ensure_dynamic_lds((const void *)norm_grad_resident_kernel<T, VEC, ONE, NV>, lds, "group_norm_grad");
  if (rc) return rc;
  hipLaunchKernelGGL((norm_grad_resident_kernel<T, VEC, ONE, NV>), dim3((unsigned)(parts * s.slabs)), dim3(p.threads), lds, stream,
                     (const T *)dy, (const T *)x, gamma, beta, stats, (T *)dx, sums, s, per, act);
  return check_launch("group_norm_grad");
}

template <typename T, int VEC, bool ONE>
static int launch_norm_grad(const NormPlan &p, const void *dy, const void *x, const float *gamma, const float *beta,
                            const float *stats, void *dx, float *dgamma, float *dbeta, float *workspace, int act,
                            hipStream_t stream) {
  const NormShape &s = p.s;
  int rc;
  if (p.resident) {
    const int per = grad_images_per_group(p);
    const long long parts = (s.N + per - 1) / per;
    auto resident = [&]() -> int {
#define FRCNN_NORM_GRAD(NV) return launch_grad_resident<T, VEC, ONE, NV>(p, dy, x, gamma, beta, stats, dx, workspace, per, parts, act, stream)
      switch (p.nv) {
        case 1: FRCNN_NORM_GRAD(1);
        case 4: FRCNN_NORM_GRAD(4);
        case 8: FRCNN_NORM_GRAD(8);
      }
      if constexpr (VEC > 1) switch (p.nv) {
        case 2: FRCNN_NORM_GRAD(2);
        case 3: FRCNN_NORM_GRAD(3);
        case 5: FRCNN_NORM_GRAD(5);
        case 6: FRCNN_NORM_GRAD(6);
        case 7: FRCNN_NORM_GRAD(7);
      }
#undef FRCNN_NORM_GRAD
      return set_error(FRCNN_EUNSUPPORTED, "group_norm_grad: no kernel for %d packs", p.nv);
    };
    rc = resident();
    if (rc) return rc;
    hipLaunchKernelGGL(norm_grad_params_kernel, dim3(parameter_blocks(s.C)), dim3(1024), 0, stream, workspace, parts, s.C, dgamma, dbeta);
    return check_launch("group_norm_grad");
  } else {
    float *expect = workspace, *image_sums = expect + (size_t)s.N * s.G * 2;
    float *chunk_sums = image_sums + (size_t)s.N * s.C * 2;
    const dim3 grid((unsigned)((long long)s.N * s.chunks * s.slabs));
    const size_t lds = 2 * (size_t)s.rows * s.slab * sizeof(float);
    rc = ensure_dynamic_lds((const void *)norm_grad_sums_kernel<T, VEC, ONE>, lds, "group_norm_grad");
    if (rc) return rc;
    hipLaunchKernelGGL((norm_grad_sums_kernel<T, VEC, ONE>), grid, dim3(p.threads), lds, stream, (const T *)dy, (const T *)x, gamma, beta,
                       stats, chunk_sums, s, act);
    rc = check_launch("group_norm_grad");
    if (rc) return rc;
    hipLaunchKernelGGL(norm_grad_join_kernel, dim3((unsigned)(s.N * s.G)), dim3(256), 0, stream, chunk_sums, gamma, image_sums,
                       expect, s);
    rc = check_launch("group_norm_grad");
    if (rc) return rc;
    const unsigned param_blocks = parameter_blocks(s.C);
    hipLaunchKernelGGL((norm_grad_apply_kernel<T, VEC, ONE>), dim3(grid.x + param_blocks), dim3(p.threads), 0, stream, (const T *)dy,
                       (const T *)x, gamma, beta, stats, expect, (T *)dx, image_sums, dgamma, dbeta, param_blocks, s, act);
    return check_launch("group_norm_grad");
  }
}

// What the two entry points ask of a shape.
static int norm_check(const char *what, int type, int64_t N, int64_t S, int64_t C, int64_t G, int act) {
  FRCNN_REQUIRE(type_known(type), "%s: unknown element type %d", what, type);
  FRCNN_REQUIRE(N >= 0 && S >= 1, "%s: needs at least one position per image (N=%lld, S=%lld)", what, (long long)N, (long long)S);
  FRCNN_REQUIRE(C >= 1 && G >= 1 && C % G == 0, "%s: %lld channels are not a multiple of %lld groups", what, (long long)C, (long long)G);
  FRCNN_REQUIRE(act == FRCNN_ACT_NONE || act == FRCNN_ACT_RELU || act == FRCNN_ACT_SWISH, "%s: unknown activation %d", what, act);
  if (N > (1ll << 30) || S >= (1ll << 24) || C > (1 << 20) || N * G >= (1ll << 31) || N * C >= (1ll << 38))
    return set_error(FRCNN_EUNSUPPORTED, "%s: (%lld, %lld, %lld) is beyond what the kernels index", what, (long long)N, (long long)S, (long long)C);
  return FRCNN_OK;
}

// The plan may depend on the pointers' alignment only through `vec`; workspaces are sized for the larger of the two.
static size_t norm_bytes(int N, int S, int C, int G, int elem, bool grad) {
  size_t most = 0;
  for (int aligned = 0; aligned < 2; ++aligned) {
    const NormPlan p = norm_plan(N, S, C, G, elem, aligned != 0, grad);
    if (!p.vec) continue;
    size_t floats;
    if (!grad) {
      floats = p.resident ? 0 : (size_t)N * (p.s.chunks + 1) * G * 2;
    } else if (p.resident) {
      const int per = grad_images_per_group(p);
      floats = (size_t)((N + per - 1) / per) * C * 2;
    } else {
      floats = (size_t)N * G * 2 + (size_t)N * C * 2 + (size_t)N * p.s.chunks * C * 2;
    }
    if (floats > most) most = floats;
  }
  return most * sizeof(float);
}

}  // namespace frcnn

using namespace frcnn;

extern "C" {

size_t frcnn_group_norm_workspace_bytes(int type, int64_t N, int64_t S, int64_t C, int64_t G) {
  if (norm_check("group_norm", type, N, S, C, G, FRCNN_ACT_NONE) || N == 0) return 0;
  return norm_bytes((int)N, (int)S, (int)C, (int)G, (int)type_bytes(type), false);
}

int frcnn_group_norm(const void *x, int type, int64_t N, int64_t S, int64_t C, int64_t G, const float *gamma, const float *beta,
                     float epsilon, int activation, void *y, float *stats, void *workspace, size_t workspace_bytes,
                     frcnn_stream_t stream) {
  const int bad = norm_check("group_norm", type, N, S, C, G, activation);
  if (bad) return bad;
  FRCNN_REQUIRE(epsilon >= 0.0f, "group_norm: epsilon %g is negative", (double)epsilon);
  if (N == 0) return FRCNN_OK;
  FRCNN_REQUIRE(x && gamma && beta && y, "group_norm: null pointer");
  const int elem = (int)type_bytes(type);
  FRCNN_REQUIRE(aligned_to(x, elem) && aligned_to(y, elem) && aligned_to(gamma, 4) && aligned_to(beta, 4) && aligned_to(stats, 8),
                "group_norm: misaligned pointer");
  const NormPlan p = norm_plan((int)N, (int)S, (int)C, (int)G, elem, aligned_to(x, 16) && aligned_to(y, 16), false);
  if (!p.vec) return set_error(FRCNN_EUNSUPPORTED, "group_norm: %d channels per group", (int)(C / G));
  // images of one launch: workgroups of p.threads, and a wave per group in norm_join_kernel, whose workgroups have four
  const long long threads = (long long)p.s.chunks * p.s.slabs * p.threads, joins = 64ll * G;
  const long long most = (kGridThreads - 255) / (threads > joins ? threads : joins);
  if (most < 1) return set_error(FRCNN_EUNSUPPORTED, "group_norm: (%lld, %lld, %lld) takes too many threads", (long long)N, (long long)S, (long long)C);
  const size_t need = frcnn_group_norm_workspace_bytes(type, N, S, C, G);
  FRCNN_REQUIRE(need == 0 || (workspace && aligned_to(workspace, 256) && workspace_bytes >= need),
                "group_norm: workspace of %zu bytes (256-byte aligned) needed, got %zu", need, workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  float *ws = (float *)workspace;
  for (int64_t first = 0; first < N; first += most) {
    NormPlan part = p;
    part.s.N = (int)(N - first < most ? N - first : most);
    const void *from = (const uint8_t *)x + first * S * C * elem;
    void *to = (uint8_t *)y + first * S * C * elem;
    float *out = stats ? stats + first * G * 2 : nullptr;
#define FRCNN_NORM_T(T)                                                                                                \
  (p.vec == 1 ? launch_norm<T, 1, true>(part, from, to, gamma, beta, out, ws, epsilon, activation, st)                \
   : p.one    ? launch_norm<T, 16 / sizeof(T), true>(part, from, to, gamma, beta, out, ws, epsilon, activation, st)   \
              : launch_norm<T, 16 / sizeof(T), false>(part, from, to, gamma, beta, out, ws, epsilon, activation, st))
    const int rc = type == FRCNN_F32 ? FRCNN_NORM_T(float) : type == FRCNN_F16 ? FRCNN_NORM_T(_Float16) : FRCNN_NORM_T(__bf16);
#undef FRCNN_NORM_T
    if (rc) return rc;
  }
  return FRCNN_OK;
}

size_t frcnn_group_norm_grad_workspace_bytes(int type, int64_t N, int64_t S, int64_t C, int64_t G) {
  if (norm_check("group_norm_grad", type, N, S, C, G, FRCNN_ACT_NONE) || N == 0) return 0;
  return norm_bytes((int)N, (int)S, (int)C, (int)G, (int)type_bytes(type), true);
}

int frcnn_group_norm_grad(const void *dy, const void *x, int type, int64_t N, int64_t S, int64_t C, int64_t G, const float *gamma,
                          const float *beta, const float *stats, int activation, void *dx, float *dgamma, float *dbeta,
                          void *workspace, size_t workspace_bytes, frcnn_stream_t stream) {
  const int bad = norm_check("group_norm_grad", type, N, S, C, G, activation);
  if (bad) return bad;
  FRCNN_REQUIRE(dgamma && dbeta, "group_norm_grad: null pointer");
  FRCNN_REQUIRE(aligned_to(dgamma, 4) && aligned_to(dbeta, 4), "group_norm_grad: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
  if (N == 0) {  // sums over nothing
    hipLaunchKernelGGL(norm_grad_params_kernel, dim3(parameter_blocks((int)C)), dim3(1024), 0, st, (const float *)nullptr, 0ll,
                       (int)C, dgamma, dbeta);
    return check_launch("group_norm_grad");
  }
  FRCNN_REQUIRE(dy && x && gamma && beta && stats && dx, "group_norm_grad: null pointer");
  const int elem = (int)type_bytes(type);
  FRCNN_REQUIRE(aligned_to(dy, elem) && aligned_to(x, elem) && aligned_to(dx, elem) && aligned_to(gamma, 4) && aligned_to(beta, 4) &&
                    aligned_to(stats, 8),
                "group_norm_grad: misaligned pointer");
  const NormPlan p = norm_plan((int)N, (int)S, (int)C, (int)G, elem, aligned_to(x, 16) && aligned_to(dy, 16) && aligned_to(dx, 16), true);
  if (!p.vec) return set_error(FRCNN_EUNSUPPORTED, "group_norm_grad: %d channels per group", (int)(C / G));
  // the form that keeps images in registers takes about a thousand workgroups; the others one per chunk and per group
  if (!p.resident && ((long long)N * p.s.chunks * p.s.slabs + parameter_blocks((int)C) > kGridThreads / 512 || N * G > kGridThreads / 256))
    return set_error(FRCNN_EUNSUPPORTED, "group_norm_grad: (%lld, %lld, %lld) takes too many threads", (long long)N, (long long)S, (long long)C);
  const size_t need = frcnn_group_norm_grad_workspace_bytes(type, N, S, C, G);
  FRCNN_REQUIRE(workspace && aligned_to(workspace, 256) && workspace_bytes >= need,
                "group_norm_grad: workspace of %zu bytes (256-byte aligned) needed, got %zu", need, workspace_bytes);
  float *ws = (float *)workspace;
#define FRCNN_NORM_T(T)                                                                                                        \
  (p.vec == 1 ? launch_norm_grad<T, 1, true>(p, dy, x, gamma, beta, stats, dx, dgamma, dbeta, ws, activation, st)                      \
   : p.one    ? launch_norm_grad<T, 16 / sizeof(T), true>(p, dy, x, gamma, beta, stats, dx, dgamma, dbeta, ws, activation, st)        \
              : launch_norm_grad<T, 16 / sizeof(T), false>(p, dy, x, gamma, beta, stats, dx, dgamma, dbeta, ws, activation, st))
  if (type == FRCNN_F32) return FRCNN_NORM_T(float);
  if (type == FRCNN_F16) return FRCNN_NORM_T(_Float16);
  return FRCNN_NORM_T(__bf16);
#undef FRCNN_NORM_T
}

}  // extern "C"
