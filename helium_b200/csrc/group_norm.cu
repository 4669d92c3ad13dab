// Group normalisation with an activation over channels-last tensors, forward and backward.
//
//   x [N, P, C] (NHWC with the P = H * W positions flattened), G groups of C / G neighbouring channels;
//   mean, var over the P * C / G values of a (picture, group), rstd = 1 / sqrt(var + eps) (biased variance, as in
//   helium's BatchNorm2d, helium/src/modules/batch_norm.rs:38-58, whose statistics run over N, H, W instead)
//   forward    xh = (x - mean) rstd,  z = gamma[c] xh + beta[c],  y = act(z)
//   backward   g = dy act'(z),  dbeta[c] = sum g,  dgamma[c] = sum g xh          (over pictures and positions)
//              dx = rstd (gamma g - m1 - xh m2),  m1 = mean of gamma g, m2 = mean of gamma g xh over the group
//
// Thread layout shared by all kernels here.  A 16-byte vector (V elements) is the unit of every access.  The tensor is
// seen as "super-rows" of f rows, f the smallest factor that makes f * C a multiple of V (1 for the usual channel
// counts, up to 8 for odd ones): a thread owns one vector column j of the super-row and walks super-rows, so the channel
// of each of its V elements never changes -- (j V + i) mod C -- and everything that depends on the channel stays in
// registers.  Where P is no multiple of f a super-row can hold the end of one picture and the start of the next:
// elements outside the picture's range of whole rows are masked (kRagged).
//
// Sums are f32.  The forward moments are taken about a shift of each thread's own (the first value it sees): the
// thread's sum of squares about the group mean m is then q - 2 d s + n d^2 with d = m - shift, whose cancellation is
// bounded by the thread's own spread whatever the tensor's mean is, and partial moments of CTAs meet as
// (count, mean, sum of squares about it) triples.  Every fold runs in a fixed order: results repeat bit for bit.
#include <algorithm>
#include <memory>

#include "device_utils.cuh"
#include "he_internal.h"

namespace he {
namespace {

// ---- element types -----------------------------------------------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<HE_F32> {
  static constexpr int V = 4, kBytes = 4;
  __device__ static void unpack(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <> struct Elem<HE_BF16> {
  static constexpr int V = 8, kBytes = 2;
  __device__ static void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
  }
  __device__ static uint4 pack(const float (&x)[8]) {
    return make_uint4(f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3]), f32x2_to_bf16x2(x[4], x[5]), f32x2_to_bf16x2(x[6], x[7]));
  }
};
template <> struct Elem<HE_F16> {
  static constexpr int V = 8, kBytes = 2;
  __device__ static void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      x[2 * j] = f.x; x[2 * j + 1] = f.y;
    }
  }
  __device__ static uint4 pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// ---- activations -------------------------------------------------------------------------------------------------
// Normal cumulative distribution.  f32 tensors take erfcf; for 16-bit ones Abramowitz & Stegun 7.1.26 gives erfc(|x|) as
// a polynomial times exp(-x^2), used as such on the negative side (no cancellation in the tail), absolute error 1.5e-7.
template <bool kExact> __device__ __forceinline__ float normal_cdf(float z) {
  if (kExact) return 0.5f * erfcf(z * -0.70710678118654752440f);
  const float ax = fabsf(z) * 0.70710678118654752440f;
  const float t = __fdividef(1.0f, fmaf(0.3275911f, ax, 1.0f));
  float poly = fmaf(1.061405429f, t, -1.453152027f);
  poly = fmaf(poly, t, 1.421413741f);
  poly = fmaf(poly, t, -0.284496736f);
  poly = fmaf(poly, t, 0.254829592f);
  const float tail = 0.5f * poly * t * __expf(-ax * ax);
  return z < 0.0f ? tail : 1.0f - tail;
}
// NaN stays NaN in each of them (fmaxf would turn a rectified NaN into 0).
template <int ACT, bool kExact> __device__ __forceinline__ float activate(float z) {
  if (ACT == HE_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if (ACT == HE_ACT_SILU) return __fdividef(z, 1.0f + __expf(-z));
  if (ACT == HE_ACT_GELU) return z * normal_cdf<kExact>(z);
  return z;
}
template <int ACT, bool kExact> __device__ __forceinline__ float slope(float z) {
  if (ACT == HE_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (ACT == HE_ACT_SILU) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-z));
    return fmaf(z * s, 1.0f - s, s);
  }
  if (ACT == HE_ACT_GELU) return fmaf(z * 0.39894228040143267794f, __expf(-0.5f * z * z), normal_cdf<kExact>(z));
  return 1.0f;
}

// ---- geometry ----------------------------------------------------------------------------------------------------
struct GnGeom {
  int N, C, G, cpg;      // pictures, channels, groups, channels per group
  int P;                 // positions
  int f, W;              // rows of a super-row, elements of one (f * C)
  long long total;       // elements of the tensor
  float eps, inv_count;  // 1 / (P * cpg)
  // one CTA's columns: `cols` vector columns from vector column `blk * cols` on, `lanes` super-rows side by side
  int cols, lanes, nblk;
  int per;               // super-rows a CTA walks
};

// The super-rows [first, last) that hold any row of picture n, and the picture's rows [row0, row1).
__device__ __forceinline__ void picture_range(const GnGeom& g, int n, long long& row0, long long& row1, long long& first, long long& last) {
  row0 = (long long)n * g.P;
  row1 = row0 + g.P;
  first = g.f == 1 ? row0 : row0 / g.f;
  last = g.f == 1 ? row1 : (row1 + g.f - 1) / g.f;
}

// Reads the vector at element `e`; elements at or past `limit` (the end of the tensor) read as zero.
template <int DT> __device__ __forceinline__ uint4 load_vec(const void* base, long long e, long long limit) {
  constexpr int V = Elem<DT>::V;
  if (e + V <= limit) return __ldcs(reinterpret_cast<const uint4*>(base) + e / V);
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < V && e + i < limit; ++i) {
    if (V == 4) w[i] = reinterpret_cast<const uint32_t*>(base)[e + i];
    else w[i >> 1] |= (uint32_t) reinterpret_cast<const unsigned short*>(base)[e + i] << (16 * (i & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Writes elements [lo, hi) of the vector at element `e`.
template <int DT> __device__ __forceinline__ void store_vec(void* base, long long e, const uint4& v, int lo, int hi) {
  constexpr int V = Elem<DT>::V;
  if (lo == 0 && hi == V) { __stcs(reinterpret_cast<uint4*>(base) + e / V, v); return; }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i >= lo && i < hi) {
      if (V == 4) reinterpret_cast<uint32_t*>(base)[e + i] = w[i & 3];
      else reinterpret_cast<unsigned short*>(base)[e + i] = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
    }
}

// ---- folds inside a CTA ------------------------------------------------------------------------------------------
// col[e] = sum over the row lanes of val, e < cols * V.  red: blockDim.x * V floats, part: blockDim.x floats.
// threads = parts x columns: every thread adds lanes / parts values, the parts meet in a tree.  Ends with a barrier.
template <int V> __device__ void column_sums(const GnGeom& g, const float (&val)[V], int j, int lane, float* red, float* part, float* col) {
  const int w = g.cols * V, threads = blockDim.x;
  if (lane < g.lanes) {
#pragma unroll
    for (int i = 0; i < V; ++i) red[lane * w + j * V + i] = val[i];
  }
  __syncthreads();
  if (w >= threads) {
    for (int e = threadIdx.x; e < w; e += threads) {
      float s = 0.0f;
      for (int l = 0; l < g.lanes; ++l) s += red[l * w + e];
      col[e] = s;
    }
  } else {
    const int parts = threads / w, p = threadIdx.x / w, e = threadIdx.x - p * w;
    if (p < parts) {
      float s = 0.0f;
      for (int l = p; l < g.lanes; l += parts) s += red[l * w + e];
      part[threadIdx.x] = s;
    }
    __syncthreads();
    for (int h = parts; h > 1;) {
      const int half = (h + 1) >> 1;
      if (p < h - half) part[threadIdx.x] += part[threadIdx.x + half * w];
      __syncthreads();
      h = half;
    }
    if (threadIdx.x < w) col[threadIdx.x] = part[threadIdx.x];
  }
  __syncthreads();
}

__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// =================================================================================================
// Tensors whose (picture, group) slabs are too large for on-chip memory: partial sums of slices, a fold, a second pass.
// =================================================================================================
// Moments of each column of a slice: part[n][slice][e] = (sum, sum of squares about the column's mean in the slice).
template <int DT, bool kRagged>
__global__ void __launch_bounds__(512) gn_moments_kernel(const void* __restrict__ x, float2* __restrict__ part, GnGeom g) {
  constexpr int V = Elem<DT>::V;
  extern __shared__ float sh[];
  float* red = sh;
  float* tree = red + blockDim.x * V;
  float* col = tree + blockDim.x;      // [cols * V] column sums, then column means
  const int n = blockIdx.z, blk = blockIdx.y;
  const int j = threadIdx.x % g.cols, lane = threadIdx.x / g.cols;
  const int vcol = blk * g.cols + j;
  long long row0, row1, first, last;
  picture_range(g, n, row0, row1, first, last);
  const long long s0 = first + (long long)blockIdx.x * g.per, s1 = min(last, s0 + g.per);
  const long long lo = row0 * g.C, hi = row1 * g.C;
  float shift[V], s[V], q[V], cnt[V];
#pragma unroll
  for (int i = 0; i < V; ++i) shift[i] = s[i] = q[i] = cnt[i] = 0.0f;
  if (lane < g.lanes && vcol * V < g.W) {
    bool seen = false;
#pragma unroll 4
    for (long long r = s0 + lane; r < s1; r += g.lanes) {
      const long long e = r * g.W + (long long)vcol * V;
      const uint4 v = load_vec<DT>(x, e, g.total);
      float a[V];
      Elem<DT>::unpack(v, a);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool in = !kRagged || (e + i >= lo && e + i < hi);
        if (kRagged ? (in && cnt[i] == 0.0f) : !seen) shift[i] = a[i];
        const float d = in ? a[i] - shift[i] : 0.0f;
        s[i] += d;
        q[i] = fmaf(d, d, q[i]);
        cnt[i] += in ? 1.0f : 0.0f;
      }
      seen = true;
    }
  }
  // values of column e in this slice: rows of the picture whose place in the super-row is e / C
  auto column_count = [&](int e) -> float {
    if (!kRagged) return (float)max(0ll, s1 - s0);
    const int k = (blk * g.cols * V + e) / g.C;
    const long long a = max(s0 * g.f, row0), b = min(s1 * g.f, row1);
    if (a >= b) return 0.0f;
    return (float)((b - k + g.f - 1) / g.f - (a - k + g.f - 1) / g.f);
  };
  float t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = fmaf(cnt[i], shift[i], s[i]);
  column_sums<V>(g, t, j, lane, red, tree, col);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float cc = lane < g.lanes ? column_count(j * V + i) : 0.0f;
    const float d = cc > 0.0f ? col[j * V + i] / cc - shift[i] : 0.0f;
    t[i] = fmaf(cnt[i] * d, d, fmaf(-2.0f * d, s[i], q[i]));
  }
  __syncthreads();
  float sums[V];
  const int w = g.cols * V;
  // the first fold's totals leave shared memory before the second one overwrites them
  const int base = threadIdx.x;
  float2* out = part + ((size_t)n * gridDim.x + blockIdx.x) * (size_t)(g.nblk * w) + (size_t)blk * w;
  for (int e = base; e < w; e += blockDim.x) out[e].x = col[e];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) sums[i] = t[i];
  column_sums<V>(g, sums, j, lane, red, tree, col);
  for (int e = base; e < w; e += blockDim.x) out[e].y = col[e];
}

// mean and rstd of each (picture, group) from the slices' column moments; one CTA of 128 threads per (picture, group).
__global__ void __launch_bounds__(128) gn_fold_moments_kernel(const float2* __restrict__ part, float* __restrict__ mean, float* __restrict__ rstd,
                                                              GnGeom g, int slices, int pitch) {
  __shared__ float sh[4];
  const int n = blockIdx.x / g.G, k = blockIdx.x % g.G;
  const int per_slice = g.f * g.cpg, items = slices * per_slice;
  const long long row0 = (long long)n * g.P, row1 = row0 + g.P, first = row0 / g.f;
  auto block_sum = [&](float s) {
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
    __syncthreads();
    const float t = (sh[0] + sh[1]) + (sh[2] + sh[3]);
    __syncthreads();
    return t;
  };
  auto item = [&](int i, float& cnt) -> float2 {
    const int sl = i / per_slice, r = i - sl * per_slice, kk = r / g.cpg, c = r - kk * g.cpg;
    const long long s0 = first + (long long)sl * g.per, s1 = min((row1 + g.f - 1) / g.f, s0 + g.per);
    const long long a = max(s0 * g.f, row0), b = min(s1 * g.f, row1);
    cnt = a < b ? (float)((b - kk + g.f - 1) / g.f - (a - kk + g.f - 1) / g.f) : 0.0f;
    return part[((size_t)n * slices + sl) * pitch + (size_t)kk * g.C + (size_t)k * g.cpg + c];
  };
  float s = 0.0f, cnt;
  for (int i = threadIdx.x; i < items; i += 128) {
    const float2 v = item(i, cnt);
    s += v.x;
  }
  const float m = block_sum(s) * g.inv_count;
  float q = 0.0f;
  for (int i = threadIdx.x; i < items; i += 128) {
    const float2 v = item(i, cnt);
    if (cnt > 0.0f) {
      const float d = v.x / cnt - m;
      q += fmaf(cnt * d, d, v.y);
    }
  }
  q = block_sum(q) * g.inv_count;
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = m;
    rstd[blockIdx.x] = 1.0f / sqrtf(q + g.eps);
  }
}

// A thread's per-channel values: channel indices of its V elements.
template <int V> __device__ __forceinline__ void thread_channels(const GnGeom& g, int vcol, int (&c)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = vcol * V + i;
    c[i] = g.f == 1 ? e : e % g.C;
  }
}

// y = act((x - mean) rstd gamma + beta)
template <int DT, int ACT, bool kRagged>
__global__ void __launch_bounds__(512) gn_apply_kernel(const void* __restrict__ x, void* __restrict__ y, const float* __restrict__ gamma,
                                                       const float* __restrict__ beta, const float* __restrict__ mean,
                                                       const float* __restrict__ rstd, GnGeom g) {
  constexpr int V = Elem<DT>::V;
  const int n = blockIdx.z, vcol = blockIdx.y * g.cols + threadIdx.x % g.cols, lane = threadIdx.x / g.cols;
  if (lane >= g.lanes || vcol * V >= g.W) return;
  long long row0, row1, first, last;
  picture_range(g, n, row0, row1, first, last);
  // slices are walked from the last one down: the moments pass ended there, so their values are the likeliest in L2
  const long long s0 = first + (long long)(gridDim.x - 1 - blockIdx.x) * g.per, s1 = min(last, s0 + g.per);
  const long long lo = row0 * g.C, hi = row1 * g.C;
  int c[V];
  thread_channels<V>(g, vcol, c);
  float mu[V], a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const size_t k = (size_t)n * g.G + c[i] / g.cpg;
    mu[i] = mean[k];
    a[i] = gamma[c[i]] * rstd[k];
    b[i] = beta[c[i]];
  }
#pragma unroll 4
  for (long long r = s0 + lane; r < s1; r += g.lanes) {
    const long long e = r * g.W + (long long)vcol * V;
    float v[V];
    Elem<DT>::unpack(load_vec<DT>(x, e, g.total), v);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = activate<ACT, DT == HE_F32>(fmaf(v[i] - mu[i], a[i], b[i]));
    const int p0 = kRagged ? (int)max(0ll, min((long long)V, lo - e)) : 0, p1 = kRagged ? (int)max(0ll, min((long long)V, hi - e)) : V;
    store_vec<DT>(y, e, Elem<DT>::pack(v), p0, p1);
  }
}

// part[n][slice][0..1][e] = sums over the slice's column e of g and of g xh
template <int DT, int ACT, bool kRagged>
__global__ void __launch_bounds__(512) gn_grad_sums_kernel(const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ gamma,
                                                           const float* __restrict__ beta, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, float* __restrict__ part, GnGeom g) {
  constexpr int V = Elem<DT>::V;
  extern __shared__ float sh[];
  float* red = sh;
  float* tree = red + blockDim.x * V;
  float* col = tree + blockDim.x;
  const int n = blockIdx.z, blk = blockIdx.y;
  const int j = threadIdx.x % g.cols, lane = threadIdx.x / g.cols, vcol = blk * g.cols + j;
  long long row0, row1, first, last;
  picture_range(g, n, row0, row1, first, last);
  const long long s0 = first + (long long)blockIdx.x * g.per, s1 = min(last, s0 + g.per);
  const long long lo = row0 * g.C, hi = row1 * g.C;
  float sb[V], sw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sb[i] = sw[i] = 0.0f;
  if (lane < g.lanes && vcol * V < g.W) {
    int c[V];
    thread_channels<V>(g, vcol, c);
    float mu[V], rs[V], ga[V], be[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const size_t k = (size_t)n * g.G + c[i] / g.cpg;
      mu[i] = mean[k]; rs[i] = rstd[k];
      ga[i] = gamma[c[i]]; be[i] = beta[c[i]];
    }
#pragma unroll 2
    for (long long r = s0 + lane; r < s1; r += g.lanes) {
      const long long e = r * g.W + (long long)vcol * V;
      float xv[V], dv[V];
      Elem<DT>::unpack(load_vec<DT>(x, e, g.total), xv);
      Elem<DT>::unpack(load_vec<DT>(dy, e, g.total), dv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (xv[i] - mu[i]) * rs[i];
        float t = dv[i] * slope<ACT, DT == HE_F32>(fmaf(xh, ga[i], be[i]));
        const bool in = !kRagged || (e + i >= lo && e + i < hi);
        sb[i] += in ? t : 0.0f;
        sw[i] += in ? t * xh : 0.0f;
      }
    }
  }
  const int w = g.cols * V;
  float* out = part + ((size_t)n * gridDim.x + blockIdx.x) * 2 * (size_t)(g.nblk * w) + (size_t)blk * w;
  column_sums<V>(g, sb, j, lane, red, tree, col);
  for (int e = threadIdx.x; e < w; e += blockDim.x) out[e] = col[e];
  __syncthreads();
  column_sums<V>(g, sw, j, lane, red, tree, col);
  for (int e = threadIdx.x; e < w; e += blockDim.x) out[(size_t)g.nblk * w + e] = col[e];
}

// Channel sums of a picture, nc[n][0..1][c], and the two means of each of its groups, coef[n][k] = (m1, m2).
// One CTA of 256 threads per (picture, group).
__global__ void __launch_bounds__(256) gn_fold_grads_kernel(const float* __restrict__ part, const float* __restrict__ gamma, float* __restrict__ nc,
                                                            float2* __restrict__ coef, GnGeom g, int slices, int pitch) {
  __shared__ float sh[2][8];
  const int n = blockIdx.x / g.G, k = blockIdx.x % g.G;
  const int warp = threadIdx.x >> 5, ln = threadIdx.x & 31;
  float m[2] = {0.0f, 0.0f};
  // a warp per channel: its lanes add the slices
  for (int cc = warp; cc < g.cpg; cc += 8) {
    const int c = k * g.cpg + cc;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float s = 0.0f;
      for (int i = ln; i < slices * g.f; i += 32) {
        const int sl = i / g.f, r = i - sl * g.f;
        s += part[(((size_t)n * slices + sl) * 2 + h) * pitch + (size_t)r * g.C + c];
      }
      s = warp_sum(s);
      if (ln == 0) nc[((size_t)n * 2 + h) * g.C + c] = s;
      m[h] = fmaf(gamma[c], s, m[h]);
    }
  }
  if (ln == 0) { sh[0][warp] = m[0]; sh[1][warp] = m[1]; }
  __syncthreads();
  if (threadIdx.x == 0) {
    float a = 0.0f, b = 0.0f;
    for (int i = 0; i < 8; ++i) { a += sh[0][i]; b += sh[1][i]; }
    coef[blockIdx.x] = make_float2(a * g.inv_count, b * g.inv_count);
  }
}

// dgamma[c] = sum over pictures of nc[n][1][c], dbeta[c] of nc[n][0][c]; 32 channels x 32 picture lanes per CTA
__global__ void __launch_bounds__(1024) gn_param_grads_kernel(const float* __restrict__ nc, float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                              int N, int C) {
  __shared__ float sh[32][33];
  const int i = blockIdx.x * 32 + threadIdx.x;   // over [2][C]
  float s = 0.0f;
  if (i < 2 * C)
    for (int n = threadIdx.y; n < N; n += 32) s += nc[(size_t)n * 2 * C + i];
  sh[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && i < 2 * C) {
    float t = 0.0f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += sh[r][threadIdx.x];
    if (i < C) dbeta[i] = t;
    else dgamma[i - C] = t;
  }
}

// dx = rstd (gamma g - m1 - xh m2)
template <int DT, int ACT, bool kRagged>
__global__ void __launch_bounds__(512) gn_grad_apply_kernel(const void* __restrict__ dy, const void* __restrict__ x, void* __restrict__ dx,
                                                            const float* __restrict__ gamma, const float* __restrict__ beta,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            const float2* __restrict__ coef, GnGeom g) {
  constexpr int V = Elem<DT>::V;
  const int n = blockIdx.z, vcol = blockIdx.y * g.cols + threadIdx.x % g.cols, lane = threadIdx.x / g.cols;
  if (lane >= g.lanes || vcol * V >= g.W) return;
  long long row0, row1, first, last;
  picture_range(g, n, row0, row1, first, last);
  const long long s0 = first + (long long)(gridDim.x - 1 - blockIdx.x) * g.per, s1 = min(last, s0 + g.per);
  const long long lo = row0 * g.C, hi = row1 * g.C;
  int c[V];
  thread_channels<V>(g, vcol, c);
  float mu[V], rs[V], ga[V], be[V], m1[V], m2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const size_t k = (size_t)n * g.G + c[i] / g.cpg;
    mu[i] = mean[k]; rs[i] = rstd[k];
    ga[i] = gamma[c[i]]; be[i] = beta[c[i]];
    const float2 m = coef[k];
    m1[i] = m.x; m2[i] = m.y;
  }
#pragma unroll 2
  for (long long r = s0 + lane; r < s1; r += g.lanes) {
    const long long e = r * g.W + (long long)vcol * V;
    float xv[V], dv[V];
    Elem<DT>::unpack(load_vec<DT>(x, e, g.total), xv);
    Elem<DT>::unpack(load_vec<DT>(dy, e, g.total), dv);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float xh = (xv[i] - mu[i]) * rs[i];
      const float t = dv[i] * slope<ACT, DT == HE_F32>(fmaf(xh, ga[i], be[i]));
      dv[i] = rs[i] * (fmaf(ga[i], t, -m1[i]) - xh * m2[i]);
    }
    const int p0 = kRagged ? (int)max(0ll, min((long long)V, lo - e)) : 0, p1 = kRagged ? (int)max(0ll, min((long long)V, hi - e)) : V;
    store_vec<DT>(dx, e, Elem<DT>::pack(dv), p0, p1);
  }
}

// ---- plan --------------------------------------------------------------------------------------------------------
struct GroupNormPlan : he_plan {
  int direction = 0, dtype = HE_BF16, act = HE_ACT_NONE;
  bool ragged = false;
  GnGeom g{};
  int threads = 512, slices = 1;
  int32_t launch(const void* const* inputs, void* const* outputs, void* workspace, cudaStream_t stream) override;
  template <int DT, int ACT, bool R> int32_t run(const void* const* in, void* const* out, void* ws, cudaStream_t st);
  template <int DT, int ACT> int32_t pick_ragged(const void* const* in, void* const* out, void* ws, cudaStream_t st) {
    return ragged ? run<DT, ACT, true>(in, out, ws, st) : run<DT, ACT, false>(in, out, ws, st);
  }
  template <int DT> int32_t pick_act(const void* const* in, void* const* out, void* ws, cudaStream_t st) {
    switch (act) {
      case HE_ACT_RELU: return pick_ragged<DT, HE_ACT_RELU>(in, out, ws, st);
      case HE_ACT_SILU: return pick_ragged<DT, HE_ACT_SILU>(in, out, ws, st);
      case HE_ACT_GELU: return pick_ragged<DT, HE_ACT_GELU>(in, out, ws, st);
      default: return pick_ragged<DT, HE_ACT_NONE>(in, out, ws, st);
    }
  }
};

template <int DT, int ACT, bool R>
int32_t GroupNormPlan::run(const void* const* in, void* const* out, void* ws, cudaStream_t st) {
  constexpr int V = Elem<DT>::V;
  const dim3 grid((unsigned)slices, (unsigned)g.nblk, (unsigned)g.N);
  const int w = g.cols * V, pitch = g.nblk * w;
  const size_t smem = (size_t)(threads * V + threads + w) * sizeof(float);
  if (direction == HE_GN_FORWARD) {
    const void* x = in[0];
    const float* gamma = (const float*)in[1]; const float* beta = (const float*)in[2];
    float* mean = (float*)out[1]; float* rstd = (float*)out[2];
    gn_moments_kernel<DT, R><<<grid, threads, smem, st>>>(x, (float2*)ws, g);
    HE_CUDA(cudaGetLastError());
    gn_fold_moments_kernel<<<g.N * g.G, 128, 0, st>>>((const float2*)ws, mean, rstd, g, slices, pitch);
    HE_CUDA(cudaGetLastError());
    gn_apply_kernel<DT, ACT, R><<<grid, threads, 0, st>>>(x, out[0], gamma, beta, mean, rstd, g);
    HE_CUDA(cudaGetLastError());
    last_launches = 3;
    return HE_OK;
  }
  const float* gamma = (const float*)in[2]; const float* beta = (const float*)in[3];
  const float* mean = (const float*)in[4]; const float* rstd = (const float*)in[5];
  float* nc = (float*)ws;                                         // [N][2][C]
  float2* coef = (float2*)(nc + (size_t)g.N * 2 * g.C);           // [N][G]
  float* part = (float*)(coef + (size_t)g.N * g.G);               // [N][slices][2][pitch]
  gn_grad_sums_kernel<DT, ACT, R><<<grid, threads, smem, st>>>(in[0], in[1], gamma, beta, mean, rstd, part, g);
  HE_CUDA(cudaGetLastError());
  gn_fold_grads_kernel<<<g.N * g.G, 256, 0, st>>>(part, gamma, nc, coef, g, slices, pitch);
  HE_CUDA(cudaGetLastError());
  gn_param_grads_kernel<<<(2 * g.C + 31) / 32, dim3(32, 32), 0, st>>>(nc, (float*)out[1], (float*)out[2], g.N, g.C);
  HE_CUDA(cudaGetLastError());
  gn_grad_apply_kernel<DT, ACT, R><<<grid, threads, 0, st>>>(in[0], in[1], out[0], gamma, beta, mean, rstd, coef, g);
  HE_CUDA(cudaGetLastError());
  last_launches = 4;
  return HE_OK;
}

int32_t GroupNormPlan::launch(const void* const* in, void* const* out, void* ws, cudaStream_t st) {
  const int n_in = direction == HE_GN_FORWARD ? 3 : 6;
  if (!in || !out) HE_FAIL(HE_ERR_INVALID, "group norm: null operand list");
  for (int i = 0; i < n_in; ++i)
    if (!in[i]) HE_FAIL(HE_ERR_INVALID, "group norm: input %d is null", i);
  for (int i = 0; i < 3; ++i)
    if (!out[i]) HE_FAIL(HE_ERR_INVALID, "group norm: output %d is null", i);
  const int n_big = direction == HE_GN_FORWARD ? 1 : 2;
  const size_t bytes = (size_t)g.total * dtype_bytes(dtype);
  const uintptr_t o = (uintptr_t)out[0];
  for (int i = 0; i < n_big; ++i) {
    const uintptr_t p = (uintptr_t)in[i];
    if (p & 15) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: tensors must be 16-byte aligned");
    if (p < o + bytes && o < p + bytes) HE_FAIL(HE_ERR_INVALID, "group norm: the output overlaps input %d", i);
  }
  if (o & 15) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: tensors must be 16-byte aligned");
  for (int i = n_big; i < n_in; ++i)
    if ((uintptr_t)in[i] & 3) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: f32 vectors must be 4-byte aligned");
  if (((uintptr_t)out[1] | (uintptr_t)out[2]) & 3) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: f32 vectors must be 4-byte aligned");
  switch (dtype) {
    case HE_F16: return pick_act<HE_F16>(in, out, ws, st);
    case HE_BF16: return pick_act<HE_BF16>(in, out, ws, st);
    default: return pick_act<HE_F32>(in, out, ws, st);
  }
}

int32_t plan_group_norm(he_ctx* ctx, int32_t direction, const he_group_norm_params* prm, he_plan** out) {
  if (!prm || !out) HE_FAIL(HE_ERR_INVALID, "group norm: null argument");
  *out = nullptr;
  if (direction != HE_GN_FORWARD && direction != HE_GN_BACKWARD) HE_FAIL(HE_ERR_INVALID, "group norm: unknown direction %d", direction);
  if (prm->dtype != HE_F16 && prm->dtype != HE_BF16 && prm->dtype != HE_F32)
    HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: tensors must be f16, bf16 or f32");
  if (prm->activation < HE_ACT_NONE || prm->activation > HE_ACT_GELU) HE_FAIL(HE_ERR_INVALID, "group norm: unknown activation %d", prm->activation);
  if (prm->batch <= 0 || prm->positions <= 0 || prm->channels <= 0) HE_FAIL(HE_ERR_INVALID, "group norm: empty tensor");
  if (prm->groups <= 0 || prm->channels % prm->groups != 0)
    HE_FAIL(HE_ERR_INVALID, "group norm: %d channels do not divide into %d groups", prm->channels, prm->groups);
  if (!(prm->eps >= 0.0f) || prm->eps > 3.4e38f) HE_FAIL(HE_ERR_INVALID, "group norm: eps must be finite and not negative");
  if (prm->batch > 65535) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: more than 65535 pictures");
  if (prm->positions >= (1ll << 31)) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: more than 2^31 - 1 positions");
  if (prm->channels > (1 << 16)) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: more than 65536 channels");
  if ((int64_t)prm->batch * prm->groups >= (1ll << 31)) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: 2^31 or more statistics");
  if ((double)prm->batch * prm->positions * prm->channels > 9e15) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: tensor too large");
  std::unique_ptr<GroupNormPlan> plan(new GroupNormPlan);
  plan->ctx = ctx;
  plan->direction = direction; plan->dtype = prm->dtype; plan->act = prm->activation;
  GnGeom& g = plan->g;
  const int V = prm->dtype == HE_F32 ? 4 : 8;
  g.N = prm->batch; g.P = (int)prm->positions; g.C = prm->channels; g.G = prm->groups; g.cpg = g.C / g.G;
  int gcd = V;
  while (g.C % gcd != 0) gcd >>= 1;
  g.f = V / gcd;
  g.W = g.f * g.C;
  g.total = (long long)g.N * g.P * g.C;
  g.eps = prm->eps;
  g.inv_count = (float)(1.0 / ((double)g.P * g.cpg));
  plan->ragged = g.P % g.f != 0;
  const int sms = ctx_sm_count(ctx);
  const int vcols = g.W / V;
  plan->threads = 512;
  g.cols = std::min(vcols, plan->threads);
  g.nblk = (vcols + g.cols - 1) / g.cols;
  g.lanes = plan->threads / g.cols;
  // slices: about four CTAs of 512 threads for each SM, at least 16 super-rows a thread (the folds' cost is per CTA)
  const long long srows = ((long long)g.P + g.f - 1) / g.f + (plan->ragged ? 1 : 0);
  const long long per_min = (long long)g.lanes * 16;
  long long want = std::max<long long>(1, (long long)sms * 4 / std::max<long long>(1, (long long)g.N * g.nblk));
  want = std::min(want, std::max<long long>(1, srows / per_min));
  g.per = (int)((srows + want - 1) / want);
  plan->slices = (int)((srows + g.per - 1) / g.per);
  const size_t pitch = (size_t)g.nblk * g.cols * V;
  plan->workspace_bytes = direction == HE_GN_FORWARD
                              ? (size_t)g.N * plan->slices * pitch * sizeof(float2)
                              : ((size_t)g.N * 2 * g.C + (size_t)g.N * g.G * 2 + (size_t)g.N * plan->slices * 2 * pitch) * sizeof(float);
  static const char* const kActs[] = {"none", "relu", "silu", "gelu"};
  char desc[256];
  snprintf(desc, sizeof desc, "group norm %s: %s [%d,%d,%d] in %d groups, activation %s, two passes over %d slices a picture",
           direction == HE_GN_FORWARD ? "forward" : "backward", dtype_name(prm->dtype), g.N, g.P, g.C, g.G, kActs[plan->act], plan->slices);
  plan->description = desc;
  *out = plan.release();
  return HE_OK;
}

}  // namespace
}  // namespace he

extern "C" int32_t he_plan_group_norm(he_ctx* ctx, int32_t direction, const he_group_norm_params* params, he_plan** out) {
  try {
    return he::plan_group_norm(ctx, direction, params, out);
  } catch (const std::exception& e) {
    HE_FAIL(HE_ERR_INVALID, "group norm: %s", e.what());
  }
}
