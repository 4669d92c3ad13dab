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
// Sums are f32.  The forward moments are taken about a shift: in the two-pass kernels one of each thread's own (the first
// value it sees, then the mean of the first 8, 64, 512 ... of them: Moments), whose sums become the thread's about the group
// mean m by q - 2 d s + n d^2 with d = m - shift; in the slab kernels the group's first value, and where that (or zero) lies
// far from the mean a second round over the tile, which is on chip, takes the mean instead.  Either way the cancellation is
// bounded whatever the tensor's mean and its first values are.  Every fold runs in a fixed order: results repeat bit for bit.
#include <algorithm>
#include <cmath>
#include <memory>

#include "device_utils.cuh"
#include "he_internal.h"
#include "sm100_ptx.cuh"

namespace he {
namespace {

// ---- packed pairs ------------------------------------------------------------------------------------------------
// All arithmetic runs on pairs of neighbouring channels with sm_100's f32x2 instructions (two IEEE-rounded f32 operations
// per issue slot): with one instruction per value the issue slots, not HBM, set the pace (31 instructions a value took 93 us
// for the [64, 3136, 256] bf16 forward pass, whose traffic is worth 31 us).
typedef unsigned long long f2;
__device__ __forceinline__ f2 pk(float a, float b) { return ptx::f2_pack(a, b); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { return ptx::f2_mul(a, b); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { return ptx::f2_fma(a, b, c); }
__device__ __forceinline__ void un(f2 v, float& a, float& b) { ptx::f2_unpack(v, a, b); }

// ---- element types -----------------------------------------------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<HE_F32> {
  static constexpr int V = 4;
  __device__ static void unpack(const uint4& v, f2 (&x)[2]) {
    x[0] = pk(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = pk(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  __device__ static uint4 pack(const f2 (&x)[2]) {
    float a, b, c, d;
    un(x[0], a, b);
    un(x[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
  }
};
template <> struct Elem<HE_BF16> {
  static constexpr int V = 8;
  __device__ static void unpack(const uint4& v, f2 (&x)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = pk(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
  }
  __device__ static uint4 pack(const f2 (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      un(x[j], a, b);
      w[j] = f32x2_to_bf16x2(a, b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Elem<HE_F16> {
  static constexpr int V = 8;
  __device__ static void unpack(const uint4& v, f2 (&x)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      x[j] = pk(f.x, f.y);
    }
  }
  __device__ static uint4 pack(const f2 (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, b;
      un(x[j], a, b);
      const __half2 h = __floats2half2_rn(a, b);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// ---- activations -------------------------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ f2 reciprocals(f2 v) {
  float a, b;
  un(v, a, b);
  return pk(rcp(a), rcp(b));
}
// 1 / (1 + exp(-z)).  One reciprocal serves a pair, b / (a b) and a / (a b): the special-function unit, 8 cycles a warp, is all
// but the bound here (two passes backward over a [2,512,512,128] tensor: 128 -> 121 us).  a = 2^-63 (1 + exp(-z)) with exp held
// at 2^126.4, so that a lies between 2^-63 and 2^63.4 and the product and its reciprocal in f32's range; the sigmoid is right down
// to 2^-126 and below that flushed to zero (z < -87.6; a NaN's too, z times which is a NaN again).  (A branch to two reciprocals
// where a product of unscaled terms overflows: 50.2 -> 56.4 us for [64,3136,256] bf16 forward.  GELU, which waits for other
// things, was 2 % slower with one.)
__device__ __forceinline__ f2 sigmoid2(f2 z) {
  const f2 scale = pk(1.0842021724855044e-19f, 1.0842021724855044e-19f);   // 2^-63
  float a, b;
  un(mul2(z, pk(-1.4426950408889634f, -1.4426950408889634f)), a, b);
  un(fma2(pk(ex2(fminf(a, 126.4f)), ex2(fminf(b, 126.4f))), scale, scale), a, b);
  const float r = rcp(a * b);
  const f2 v = mul2(pk(b, a), pk(r, r));
  f2 s;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(s) : "l"(v), "l"(scale));
  return s;
}
// Normal cumulative distribution, and exp(-z^2 / 2) beside it: half of erfc(|z| / sqrt 2) on the negative side (no
// cancellation in the tail), one minus that on the other.  f32 tensors take the Chebyshev form of Numerical Recipes
// ("erfcc": t exp(-x^2 + a polynomial in t), relative error 1.2e-7; erff and erfcf of the library took most of the kernel's time),
// 16-bit ones Abramowitz & Stegun 7.1.26 (a polynomial in t times exp(-x^2), absolute error 1.5e-7).  |x| is capped at 20, where
// erfc is 0 in f32.
template <bool kExact> __device__ __forceinline__ f2 normal_cdf2(f2 z, f2& bell) {
  float za, zb;
  un(z, za, zb);
  const f2 ax = pk(fminf(fabsf(za) * 0.70710678118654752440f, 20.0f), fminf(fabsf(zb) * 0.70710678118654752440f, 20.0f));
  auto c2 = [](float c) { return pk(c, c); };
  const f2 log2e = c2(1.4426950408889634f), nsq = mul2(mul2(ax, ax), c2(-1.0f));
  float ea, eb, ta, tb;
  un(mul2(nsq, log2e), ea, eb);
  bell = pk(ex2(ea), ex2(eb));
  f2 half;
  if (kExact) {
    const f2 t = reciprocals(fma2(ax, c2(0.5f), c2(1.0f)));
    f2 p = fma2(c2(0.17087277f), t, c2(-0.82215223f));
    p = fma2(p, t, c2(1.48851587f));
    p = fma2(p, t, c2(-1.13520398f));
    p = fma2(p, t, c2(0.27886807f));
    p = fma2(p, t, c2(-0.18628806f));
    p = fma2(p, t, c2(0.09678418f));
    p = fma2(p, t, c2(0.37409196f));
    p = fma2(p, t, c2(1.00002368f));
    p = fma2(p, t, c2(-1.26551223f));
    un(mul2(add2(nsq, p), log2e), ea, eb);
    half = mul2(mul2(t, c2(0.5f)), pk(ex2(ea), ex2(eb)));
  } else {
    const f2 t = reciprocals(fma2(ax, c2(0.3275911f), c2(1.0f)));
    f2 p = fma2(c2(1.061405429f), t, c2(-1.453152027f));
    p = fma2(p, t, c2(1.421413741f));
    p = fma2(p, t, c2(-0.284496736f));
    p = fma2(p, t, c2(0.254829592f));
    half = mul2(mul2(p, mul2(t, c2(0.5f))), bell);
  }
  un(half, ta, tb);
  return pk(za < 0.0f ? ta : 1.0f - ta, zb < 0.0f ? tb : 1.0f - tb);
}
// NaN stays NaN in each of them (fmaxf would turn a rectified NaN into 0).
template <int ACT, bool kExact> __device__ __forceinline__ f2 activate2(f2 z) {
  if (ACT == HE_ACT_RELU) {
    float a, b;
    un(z, a, b);
    return pk(a < 0.0f ? 0.0f : a, b < 0.0f ? 0.0f : b);
  }
  if (ACT == HE_ACT_SILU) return mul2(z, sigmoid2(z));
  if (ACT == HE_ACT_GELU) {
    f2 bell;
    return mul2(z, normal_cdf2<kExact>(z, bell));
  }
  return z;
}
template <int ACT, bool kExact> __device__ __forceinline__ f2 slope2(f2 z) {
  if (ACT == HE_ACT_RELU) {
    float a, b;
    un(z, a, b);
    return pk(a > 0.0f ? 1.0f : 0.0f, b > 0.0f ? 1.0f : 0.0f);
  }
  if (ACT == HE_ACT_SILU) {   // s + z s (1 - s)
    const f2 s = sigmoid2(z), one = pk(1.0f, 1.0f);
    return mul2(s, fma2(z, fma2(s, pk(-1.0f, -1.0f), one), one));
  }
  if (ACT == HE_ACT_GELU) {
    f2 bell;
    const f2 cdf = normal_cdf2<kExact>(z, bell);
    return fma2(mul2(z, pk(0.39894228040143267794f, 0.39894228040143267794f)), bell, cdf);
  }
  return pk(1.0f, 1.0f);
}

// ---- geometry ----------------------------------------------------------------------------------------------------
struct GnGeom {
  int N, C, G, cpg;      // pictures, channels, groups, channels per group
  int P;                 // positions
  int f, W;              // rows of a super-row, elements of one (f * C)
  long long total;       // elements of the tensor
  float eps, inv_count;  // 1 / (P * cpg)
  FastDiv div_c, div_cpg;
  // one CTA's columns: `cols` vector columns from vector column `blk * cols` on, `lanes` super-rows side by side
  int cols, lanes, nblk;
  int per;               // super-rows a CTA walks
};

// A CTA's share of a picture: super-rows [s0, s1).  Those in [f0, f1) lie inside the picture; with kRagged one more may
// stand at either end that holds rows of the neighbouring picture (or nothing), of which elements [lo, hi) of the tensor
// are the picture's.
struct Share {
  long long row0, row1, s0, s1, f0, f1, lo, hi;
};
__device__ __forceinline__ Share share_of(const GnGeom& g, int n, long long part) {
  Share h;
  h.row0 = (long long)n * g.P;
  h.row1 = h.row0 + g.P;
  long long first, last, in0, in1;
  if (g.f == 1) { first = in0 = h.row0; last = in1 = h.row1; }
  else {
    first = h.row0 / g.f; last = (h.row1 + g.f - 1) / g.f;
    in0 = (h.row0 + g.f - 1) / g.f; in1 = h.row1 / g.f;
  }
  h.s0 = first + part * g.per;
  h.s1 = min(last, h.s0 + g.per);
  h.f0 = max(h.s0, in0);
  h.f1 = min(h.s1, in1);
  h.lo = h.row0 * g.C; h.hi = h.row1 * g.C;
  return h;
}
// rows of the picture in the share
__device__ __forceinline__ float share_rows(const GnGeom& g, const Share& h) {
  return (float)max(0ll, min(h.s1 * g.f, h.row1) - max(h.s0 * g.f, h.row0));
}
// Calls fn(super-row) for the picture's edge super-rows that fall to this row lane.
template <class F> __device__ __forceinline__ void edge_rows(const GnGeom& g, const Share& h, int lane, F fn) {
  // the first and the last super-row of the share, where they are not inside; they may be one and the same
  const bool head = h.s0 < h.s1 && h.s0 < h.f0, tail = h.s0 < h.s1 && h.s1 > h.f1 && !(head && h.s1 - h.s0 == 1);
  if (head && lane == 0) fn(h.s0);
  if (tail && lane == g.lanes - 1) fn(h.s1 - 1);
}

// Reads the vector at element `e`; elements outside the tensor read as zero.
template <int DT> __device__ __forceinline__ uint4 load_edge(const void* base, long long e, long long limit) {
  constexpr int V = Elem<DT>::V;
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e + i < limit) {
      if (V == 4) w[i & 3] = reinterpret_cast<const uint32_t*>(base)[e + i];
      else w[i >> 1] |= (uint32_t) reinterpret_cast<const unsigned short*>(base)[e + i] << (16 * (i & 1));
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Writes the elements of the vector at element `e` that lie in [lo, hi).
template <int DT> __device__ __forceinline__ void store_edge(void* base, long long e, const uint4& v, long long lo, long long hi) {
  constexpr int V = Elem<DT>::V;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e + i >= lo && e + i < hi) {
      if (V == 4) reinterpret_cast<uint32_t*>(base)[e + i] = w[i & 3];
      else reinterpret_cast<unsigned short*>(base)[e + i] = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
    }
}

// ---- what happens to a vector ------------------------------------------------------------------------------------
// Moments of a thread's columns about a shift of its own: the first value it sees, then the mean of the first n for n = 8, 64,
// 512 ... .  With S(n) the sum of squares of n values about their own mean, what is added between two such points is at most
// S(8n) + 8n (mean(n) - mean(8n))^2 <= 9 S(8n): whichever values come first, no more than nine times the result cancels.
// (About the first value alone, 230 values behind one 10^4 deviations away left rstd up to 3200 u off.)
template <int DT, bool kRagged> struct Moments {
  static constexpr int V = Elem<DT>::V, H = V / 2;
  f2 nshift[H], s[H], q[H];
  float inner;                     // vectors seen inside the picture
  float extra[kRagged ? V : 1];    // values seen in the edge super-rows
  __device__ void clear() {
#pragma unroll
    for (int h = 0; h < H; ++h) nshift[h] = s[h] = q[h] = pk(0.0f, 0.0f);
    inner = 0.0f;
#pragma unroll
    for (int i = 0; i < (kRagged ? V : 1); ++i) extra[i] = 0.0f;
  }
  __device__ void start(const uint4& v) {
    f2 x[H];
    Elem<DT>::unpack(v, x);
#pragma unroll
    for (int h = 0; h < H; ++h) nshift[h] = mul2(x[h], pk(-1.0f, -1.0f));
  }
  // from the sums of n values about the shift to those about their mean, e further: s + n e and q + e (s + (s + n e))
  __device__ void rebase(float n) {
    const f2 ninv = pk(-1.0f / n, -1.0f / n), n2 = pk(n, n), neg = pk(-1.0f, -1.0f);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const f2 c = fma2(s[h], ninv, nshift[h]), e = fma2(nshift[h], neg, c), t = fma2(e, n2, s[h]);
      q[h] = fma2(e, add2(s[h], t), q[h]);
      s[h] = t;
      nshift[h] = c;
    }
  }
  __device__ __forceinline__ void add(const uint4& v) {
    f2 x[H];
    Elem<DT>::unpack(v, x);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const f2 d = add2(x[h], nshift[h]);
      s[h] = add2(s[h], d);
      q[h] = fma2(d, d, q[h]);
    }
  }
  __device__ void add_edge(const uint4& v, long long e, long long lo, long long hi) {
    f2 x[H];
    Elem<DT>::unpack(v, x);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float xv[2], ns[2], sv[2], qv[2];
      un(x[h], xv[0], xv[1]); un(nshift[h], ns[0], ns[1]); un(s[h], sv[0], sv[1]); un(q[h], qv[0], qv[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = 2 * h + k;
        if (e + i >= lo && e + i < hi) {
          float& n = extra[kRagged ? i : 0];
          if (inner + n == 0.0f) ns[k] = -xv[k];
          const float d = xv[k] + ns[k];
          sv[k] += d;
          qv[k] = fmaf(d, d, qv[k]);
          n += 1.0f;
        }
      }
      nshift[h] = pk(ns[0], ns[1]); s[h] = pk(sv[0], sv[1]); q[h] = pk(qv[0], qv[1]);
    }
  }
  __device__ float count(int i) const { return inner + extra[kRagged ? i : 0]; }
  __device__ void sums(float (&t)[V]) const {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float a, b, c, d;
      un(nshift[h], a, b);
      un(s[h], c, d);
      t[2 * h] = fmaf(-count(2 * h), a, c);
      t[2 * h + 1] = fmaf(-count(2 * h + 1), b, d);
    }
  }
  // sums of squares about `mean` of each column
  __device__ void squares(const float (&mean)[V], float (&t)[V]) const {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float n[2], sv[2], qv[2];
      un(nshift[h], n[0], n[1]); un(s[h], sv[0], sv[1]); un(q[h], qv[0], qv[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = 2 * h + k;
        const float c = count(i), d = mean[i] + n[k];
        t[i] = c > 0.0f ? fmaf(c * d, d, fmaf(-2.0f * d, sv[k], qv[k])) : 0.0f;
      }
    }
  }
};

// y = act((x - mean) scale + beta), scale = gamma rstd
template <int DT, int ACT> struct Normalise {
  static constexpr int V = Elem<DT>::V, H = V / 2;
  f2 nmu[H], sc[H], be[H];
  __device__ __forceinline__ uint4 operator()(const uint4& v) const {
    f2 x[H];
    Elem<DT>::unpack(v, x);
#pragma unroll
    for (int h = 0; h < H; ++h) x[h] = activate2<ACT, DT == HE_F32>(fma2(add2(x[h], nmu[h]), sc[h], be[h]));
    return Elem<DT>::pack(x);
  }
};

// xh = (x - mean) rstd and g = dy act'(gamma xh + beta)
template <int DT, int ACT> struct Gradient {
  static constexpr int V = Elem<DT>::V, H = V / 2;
  f2 nmu[H], rs[H], ga[H], be[H];
  __device__ __forceinline__ void operator()(const uint4& vx, const uint4& vd, f2 (&xh)[H], f2 (&t)[H]) const {
    Elem<DT>::unpack(vx, xh);
    Elem<DT>::unpack(vd, t);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      xh[h] = mul2(add2(xh[h], nmu[h]), rs[h]);
      if (ACT != HE_ACT_NONE) t[h] = mul2(t[h], slope2<ACT, DT == HE_F32>(fma2(xh[h], ga[h], be[h])));
    }
  }
  __device__ void load(const GnGeom& g, int n, const int (&c)[V], const float* gamma, const float* beta, const float* mean, const float* rstd) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const size_t k0 = (size_t)n * g.G + c[2 * h] / g.cpg, k1 = (size_t)n * g.G + c[2 * h + 1] / g.cpg;
      nmu[h] = pk(-mean[k0], -mean[k1]);
      rs[h] = pk(rstd[k0], rstd[k1]);
      ga[h] = pk(gamma[c[2 * h]], gamma[c[2 * h + 1]]);
      be[h] = pk(beta[c[2 * h]], beta[c[2 * h + 1]]);
    }
  }
};
// sums over a thread's vectors of g and of g xh, by column
template <int DT, int ACT> struct GradSums {
  static constexpr int V = Elem<DT>::V, H = V / 2;
  f2 b[H], w[H];
  __device__ void clear() {
#pragma unroll
    for (int h = 0; h < H; ++h) b[h] = w[h] = pk(0.0f, 0.0f);
  }
  __device__ __forceinline__ void add(const f2 (&xh)[H], const f2 (&t)[H]) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      b[h] = add2(b[h], t[h]);
      w[h] = fma2(t[h], xh[h], w[h]);
    }
  }
  __device__ void add_edge(const f2 (&xh)[H], const f2 (&t)[H], long long e, long long lo, long long hi) {
    f2 x2[H], t2[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float xa, xb, ta, tb;
      un(xh[h], xa, xb);
      un(t[h], ta, tb);
      const bool ia = e + 2 * h >= lo && e + 2 * h < hi, ib = e + 2 * h + 1 >= lo && e + 2 * h + 1 < hi;
      x2[h] = pk(ia ? xa : 0.0f, ib ? xb : 0.0f);
      t2[h] = pk(ia ? ta : 0.0f, ib ? tb : 0.0f);
    }
    add(x2, t2);
  }
  __device__ static void unpack(const f2 (&v)[H], float (&t)[V]) {
#pragma unroll
    for (int h = 0; h < H; ++h) un(v[h], t[2 * h], t[2 * h + 1]);
  }
};
// dx = rstd (gamma g - m1 - xh m2), the factor rstd multiplied into the others
template <int DT, int ACT> struct GradApply {
  static constexpr int V = Elem<DT>::V, H = V / 2;
  f2 gr[H], n1[H], n2[H];
  __device__ void set(const Gradient<DT, ACT>& p, const float (&m1)[V], const float (&m2)[V]) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      gr[h] = mul2(p.ga[h], p.rs[h]);
      n1[h] = mul2(pk(-m1[2 * h], -m1[2 * h + 1]), p.rs[h]);
      n2[h] = mul2(pk(-m2[2 * h], -m2[2 * h + 1]), p.rs[h]);
    }
  }
  __device__ __forceinline__ uint4 operator()(const f2 (&xh)[H], const f2 (&t)[H]) const {
    f2 o[H];
#pragma unroll
    for (int h = 0; h < H; ++h) o[h] = fma2(gr[h], t[h], fma2(xh[h], n2[h], n1[h]));
    return Elem<DT>::pack(o);
  }
};

// ---- folds inside a CTA ------------------------------------------------------------------------------------------
// col[e] = sum over the row lanes of val, e < cols * R (R values a thread).  red: blockDim.x * R floats, part: blockDim.x
// floats.  threads = parts x columns: every thread adds lanes / parts values, the parts meet in a tree.  Ends with a barrier.
template <int R> __device__ void column_sums(const GnGeom& g, const float (&val)[R], int j, int lane, float* red, float* part, float* col) {
  const int w = g.cols * R, threads = blockDim.x;
  if (lane < g.lanes) {
#pragma unroll
    for (int i = 0; i < R; ++i) red[lane * w + j * R + i] = val[i];
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
    float s = 0.0f;
    if (p < parts)
      for (int l = p; l < g.lanes; l += parts) s += red[l * w + e];
    if (parts == 1) {
      if (threadIdx.x < w) col[threadIdx.x] = s;
    } else {
      part[threadIdx.x] = s;
      __syncthreads();
      for (int h = parts; h > 2;) {
        const int half = (h + 1) >> 1;
        if (p < h - half) part[threadIdx.x] += part[threadIdx.x + half * w];
        __syncthreads();
        h = half;
      }
      if (threadIdx.x < w) col[threadIdx.x] = part[threadIdx.x] + part[threadIdx.x + w];
    }
  }
  __syncthreads();
}
__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
// Channels of a thread's V elements.
template <int V> __device__ __forceinline__ void thread_channels(const GnGeom& g, int vcol, int (&c)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t e = (uint32_t)(vcol * V + i);
    c[i] = g.f == 1 ? (int)e : (int)(e - g.div_c.div(e) * (uint32_t)g.C);
  }
}

// 16 bytes from global to shared memory without passing through registers; a thread reads only what it copied itself
__device__ __forceinline__ void copy16(const void* dst_shared, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst_shared)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until at most `n` of the thread's latest groups are in flight
__device__ __forceinline__ void copy_wait(int n) {
  if (n >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
// Walks a thread's vectors of T tensors in order, `kDepth` of each in flight: copies into a ring of its own in shared
// memory ([place][tensor][thread], so no two threads share any of it).  With two or four loads held in registers instead,
// the passes over a [2,512,512,128] tensor ran at 3.1 and 3.8 TB/s.
constexpr int kDepth = 8;
template <int T, class F>
__device__ __forceinline__ void stream_vectors(const uint4* (&src)[T], size_t step, int count, uint4* ring, F fn) {
  uint4* const mine = ring + threadIdx.x;
  const int place = T * blockDim.x;
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) {
    if (i < count)
#pragma unroll
      for (int t = 0; t < T; ++t) copy16(mine + i * place + t * blockDim.x, src[t] + i * step);
    copy_commit();
  }
  for (int i = 0; i < count; ++i) {
    if (i + kDepth - 1 < count)
#pragma unroll
      for (int t = 0; t < T; ++t)
        copy16(mine + ((i + kDepth - 1) % kDepth) * place + t * blockDim.x, src[t] + (size_t)(i + kDepth - 1) * step);
    copy_commit();
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    uint4 v[T];
#pragma unroll
    for (int t = 0; t < T; ++t) v[t] = mine[(i % kDepth) * place + t * blockDim.x];
    fn(i, v);
  }
}

// =================================================================================================
// Tensors whose (picture, group) slabs are too large for on-chip memory: partial sums of slices, a fold, a second pass.
// =================================================================================================
// Moments of each column of a slice: part[n][slice][e] = (sum, sum of squares about the column's mean in the slice).
// 80 registers: three CTAs of 256 threads an SM (82 that the compiler would take, with two of them: [2,262144,128] bf16 forward
// 87.9 us, with three 84.1 us).
template <int DT, bool kRagged>
__global__ void __maxnreg__(80) gn_moments_kernel(const void* __restrict__ x, float2* __restrict__ part, GnGeom g) {
  constexpr int V = Elem<DT>::V;
  extern __shared__ float sh[];        // the ring, then (behind the barrier of the first fold's caller) the folds' space
  float* red = sh;
  float* tree = red + blockDim.x * V;
  float* col = tree + blockDim.x;      // [cols * V]
  const int n = blockIdx.z, blk = blockIdx.y;
  const int j = threadIdx.x % g.cols, lane = threadIdx.x / g.cols;
  const int vcol = blk * g.cols + j;
  const Share h = share_of(g, n, blockIdx.x);
  ptx::grid_release();
  Moments<DT, kRagged> m;
  m.clear();
  if (lane < g.lanes && vcol * V < g.W) {
    const int pitch = g.W / V;
    const uint4* src[1] = {reinterpret_cast<const uint4*>(x) + (h.f0 + lane) * pitch + vcol};
    const int rows = (int)max(0ll, h.f1 - h.f0 - lane), count = (rows + g.lanes - 1) / g.lanes;
    unsigned next = 8;
    stream_vectors<1>(src, (size_t)g.lanes * pitch, count, reinterpret_cast<uint4*>(sh), [&](int i, const uint4 (&v)[1]) {
      if (i == 0) m.start(v[0]);
      m.add(v[0]);
      if ((unsigned)i + 1 == next) {
        m.rebase((float)next);
        next *= 8;
      }
    });
    m.inner = (float)count;
    if (kRagged)
      edge_rows(g, h, lane, [&](long long row) {
        const long long e = row * g.W + (long long)vcol * V;
        m.add_edge(load_edge<DT>(x, e, g.total), e, h.lo, h.hi);
      });
  }
  float t[V], mean[V];
  m.sums(t);
  __syncthreads();                     // every thread is through with its ring
  column_sums<V>(g, t, j, lane, red, tree, col);
  const int w = g.cols * V;
  if (g.nblk == 1) {
    // all columns are here: (sum, sum of squares about the slice's mean) of each group
    float* grp = col + w;              // [G]
    float2* out = part + ((size_t)n * gridDim.x + blockIdx.x) * (size_t)g.G;
    const int ln = threadIdx.x & 31;
    auto fold = [&](auto put) {
      for (int k = threadIdx.x >> 5; k < g.G; k += blockDim.x >> 5) {
        float s = 0.0f;
        for (int r = 0; r < g.f; ++r)
          for (int c = ln; c < g.cpg; c += 32) s += col[r * g.C + k * g.cpg + c];
        s = warp_sum(s);
        if (ln == 0) put(k, s);
      }
      __syncthreads();
    };
    const float count = share_rows(g, h) * g.cpg;
    fold([&](int k, float s) {
      out[k].x = s;
      grp[k] = count > 0.0f ? s / count : 0.0f;
    });
    int c[V];
    thread_channels<V>(g, lane < g.lanes ? j : 0, c);
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = grp[g.div_cpg.div((uint32_t)c[i])];
    m.squares(mean, t);
    column_sums<V>(g, t, j, lane, red, tree, col);
    fold([&](int k, float s) { out[k].y = s; });
    return;
  }
  // values of column e in this slice: rows of the picture whose place in the super-row is e / C
  auto column_count = [&](int e) -> float {
    if (!kRagged) return (float)max(0ll, h.s1 - h.s0);
    const int k = (blk * g.cols * V + e) / g.C;
    const long long a = max(h.s0 * g.f, h.row0), b = min(h.s1 * g.f, h.row1);
    if (a >= b) return 0.0f;
    return (float)((b - k + g.f - 1) / g.f - (a - k + g.f - 1) / g.f);
  };
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float cc = lane < g.lanes ? column_count(j * V + i) : 0.0f;
    mean[i] = cc > 0.0f ? col[j * V + i] / cc : 0.0f;
  }
  m.squares(mean, t);
  // the first fold's totals leave shared memory before the second one overwrites them
  float2* out = part + ((size_t)n * gridDim.x + blockIdx.x) * (size_t)(g.nblk * w) + (size_t)blk * w;
  for (int e = threadIdx.x; e < w; e += blockDim.x) out[e].x = col[e];
  __syncthreads();
  column_sums<V>(g, t, j, lane, red, tree, col);
  for (int e = threadIdx.x; e < w; e += blockDim.x) out[e].y = col[e];
}

// mean and rstd of each (picture, group) from the slices' moments, of the group (one item a slice) or, where a slice is cut
// into column blocks, of its columns; one CTA of 256 threads per (picture, group).
__global__ void __launch_bounds__(256) gn_fold_moments_kernel(const float2* __restrict__ part, float* __restrict__ mean, float* __restrict__ rstd,
                                                              GnGeom g, int slices, int pitch) {
  __shared__ float sh[8];
  const int n = blockIdx.x / g.G, k = blockIdx.x % g.G;
  const bool whole = g.nblk == 1;
  const int per_slice = whole ? 1 : g.f * g.cpg, items = slices * per_slice;
  const long long row0 = (long long)n * g.P, row1 = row0 + g.P, first = row0 / g.f;
  auto block_sum = [&](float s) {
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
    __syncthreads();
    const float t = ((sh[0] + sh[1]) + (sh[2] + sh[3])) + ((sh[4] + sh[5]) + (sh[6] + sh[7]));
    __syncthreads();
    return t;
  };
  auto item = [&](int i, float& cnt) -> float2 {
    const int sl = whole ? i : i / per_slice, r = i - sl * per_slice, kk = whole ? 0 : r / g.cpg, c = r - kk * g.cpg;
    const long long s0 = first + (long long)sl * g.per, s1 = min((row1 + g.f - 1) / g.f, s0 + g.per);
    const long long a = max(s0 * g.f, row0), b = min(s1 * g.f, row1);
    if (whole) {
      cnt = (float)max(0ll, b - a) * g.cpg;
      return __ldcg(part + ((size_t)n * slices + sl) * g.G + k);
    }
    cnt = a < b ? (float)((b - kk + g.f - 1) / g.f - (a - kk + g.f - 1) / g.f) : 0.0f;
    return __ldcg(part + ((size_t)n * slices + sl) * pitch + (size_t)kk * g.C + (size_t)k * g.cpg + c);
  };
  ptx::grid_wait();
  float s = 0.0f, cnt;
  for (int i = threadIdx.x; i < items; i += 256) s += item(i, cnt).x;
  const float m = block_sum(s) * g.inv_count;
  float q = 0.0f;
  for (int i = threadIdx.x; i < items; i += 256) {
    const float2 v = item(i, cnt);
    if (cnt > 0.0f) {
      const float d = v.x / cnt - m;
      q += fmaf(cnt * d, d, v.y);
    }
  }
  q = block_sum(q) * g.inv_count;
  q = q < 0.0f ? 0.0f : q;   // by rounding; NaN stays
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = m;
    rstd[blockIdx.x] = 1.0f / sqrtf(q + g.eps);
  }
}

// y = act((x - mean) rstd gamma + beta)
template <int DT, int ACT, bool kRagged>
__global__ void __launch_bounds__(512, 1) gn_apply_kernel(const void* __restrict__ x, void* __restrict__ y, const float* __restrict__ gamma,
                                                       const float* __restrict__ beta, const float* __restrict__ mean,
                                                       const float* __restrict__ rstd, GnGeom g) {
  constexpr int V = Elem<DT>::V, H = V / 2;
  const int n = blockIdx.z, vcol = blockIdx.y * g.cols + threadIdx.x % g.cols, lane = threadIdx.x / g.cols;
  if (lane >= g.lanes || vcol * V >= g.W) return;
  // a picture's slices are taken from the last one down: with one picture the moments pass ended there, so its values are the
  // likeliest in L2 (with several it ended in the last picture, and this pass begins with the first: no reuse is counted on)
  const Share h = share_of(g, n, gridDim.x - 1 - blockIdx.x);
  int c[V];
  thread_channels<V>(g, vcol, c);
  Normalise<DT, ACT> f;
#pragma unroll
  for (int i = 0; i < H; ++i) {
    const size_t k0 = (size_t)n * g.G + c[2 * i] / g.cpg, k1 = (size_t)n * g.G + c[2 * i + 1] / g.cpg;
    f.nmu[i] = pk(-mean[k0], -mean[k1]);
    f.sc[i] = pk(gamma[c[2 * i]] * rstd[k0], gamma[c[2 * i + 1]] * rstd[k1]);
    f.be[i] = pk(beta[c[2 * i]], beta[c[2 * i + 1]]);
  }
  const int pitch = g.W / V;
  extern __shared__ float4 ring4[];
  const uint4* src[1] = {reinterpret_cast<const uint4*>(x) + (h.f0 + lane) * pitch + vcol};
  uint4* dst = reinterpret_cast<uint4*>(y) + (h.f0 + lane) * pitch + vcol;
  const int rows = (int)max(0ll, h.f1 - h.f0 - lane);
  const size_t step = (size_t)g.lanes * pitch;
  stream_vectors<1>(src, step, (rows + g.lanes - 1) / g.lanes, reinterpret_cast<uint4*>(ring4), [&](int, const uint4 (&v)[1]) {
    __stcs(dst, f(v[0]));
    dst += step;
  });
  if (kRagged)
    edge_rows(g, h, lane, [&](long long row) {
      const long long e = row * g.W + (long long)vcol * V;
      store_edge<DT>(y, e, f(load_edge<DT>(x, e, g.total)), h.lo, h.hi);
    });
}

// part[n][slice][0..1][e] = sums over the slice's column e of g and of g xh
template <int DT, int ACT, bool kRagged>
__global__ void __launch_bounds__(512, 1) gn_grad_sums_kernel(const void* __restrict__ dy, const void* __restrict__ x, const float* __restrict__ gamma,
                                                           const float* __restrict__ beta, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, float* __restrict__ part, GnGeom g) {
  constexpr int V = Elem<DT>::V, H = V / 2;
  extern __shared__ float sh[];        // the ring, then the folds' space
  float* red = sh;
  float* tree = red + blockDim.x * V;
  float* col = tree + blockDim.x;
  const int n = blockIdx.z, blk = blockIdx.y;
  const int j = threadIdx.x % g.cols, lane = threadIdx.x / g.cols, vcol = blk * g.cols + j;
  const Share h = share_of(g, n, blockIdx.x);
  ptx::grid_release();
  GradSums<DT, ACT> sum;
  sum.clear();
  if (lane < g.lanes && vcol * V < g.W) {
    int c[V];
    thread_channels<V>(g, vcol, c);
    Gradient<DT, ACT> f;
    f.load(g, n, c, gamma, beta, mean, rstd);
    const int pitch = g.W / V;
    const size_t at = (size_t)(h.f0 + lane) * pitch + vcol, step = (size_t)g.lanes * pitch;
    const uint4* src[2] = {reinterpret_cast<const uint4*>(x) + at, reinterpret_cast<const uint4*>(dy) + at};
    const int rows = (int)max(0ll, h.f1 - h.f0 - lane);
    f2 xh[H], t[H];
    stream_vectors<2>(src, step, (rows + g.lanes - 1) / g.lanes, reinterpret_cast<uint4*>(sh), [&](int, const uint4 (&v)[2]) {
      f(v[0], v[1], xh, t);
      sum.add(xh, t);
    });
    if (kRagged)
      edge_rows(g, h, lane, [&](long long row) {
        const long long e = row * g.W + (long long)vcol * V;
        f(load_edge<DT>(x, e, g.total), load_edge<DT>(dy, e, g.total), xh, t);
        sum.add_edge(xh, t, e, h.lo, h.hi);
      });
  }
  // columns of the slice; where one CTA has them all the f places of a channel meet here
  const int w = g.cols * V, channels = g.nblk == 1 ? g.C : w, pitch = g.nblk == 1 ? g.C : g.nblk * w;
  float* out = part + ((size_t)n * gridDim.x + blockIdx.x) * 2 * (size_t)pitch + (size_t)blk * w;
  float v[V];
  GradSums<DT, ACT>::unpack(sum.b, v);
  __syncthreads();                     // every thread is through with its ring
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    column_sums<V>(g, v, j, lane, red, tree, col);
    for (int e = threadIdx.x; e < channels; e += blockDim.x) {
      float s = col[e];
      if (g.nblk == 1)
        for (int k = 1; k < g.f; ++k) s += col[e + k * g.C];
      out[(size_t)half * pitch + e] = s;
    }
    __syncthreads();
    GradSums<DT, ACT>::unpack(sum.w, v);
  }
}

// Channel sums of a picture, nc[n][0..1][c], from the slices': 32 channels x 32 slice lanes per CTA.
__global__ void __launch_bounds__(1024) gn_fold_grads_kernel(const float* __restrict__ part, float* __restrict__ nc, GnGeom g, int slices, int pitch) {
  __shared__ float sh[32][33];
  const int n = blockIdx.y, i = blockIdx.x * 32 + threadIdx.x, h = i >= g.C ? 1 : 0, c = i - h * g.C;   // over [2][C]
  ptx::grid_release();
  ptx::grid_wait();
  float s = 0.0f;
  if (i < 2 * g.C) {
    const float* p = part + ((size_t)n * slices * 2 + h) * pitch + c;
    const int places = g.nblk == 1 ? 1 : g.f;
#pragma unroll 4
    for (int sl = threadIdx.y; sl < slices; sl += 32)
      for (int k = 0; k < places; ++k) s += __ldcg(p + (size_t)sl * 2 * pitch + (size_t)k * g.C);
  }
  sh[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && i < 2 * g.C) {
    float t = 0.0f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += sh[r][threadIdx.x];
    nc[(size_t)n * 2 * g.C + i] = t;
  }
}

// dgamma[c] = sum over pictures of nc[n][1][c], dbeta[c] of nc[n][0][c]: 32 channels x 32 picture lanes per CTA.  CTAs behind
// the first `param_ctas`: the two means of the groups, coef[n][k] = (m1, m2), one warp each.
__global__ void __launch_bounds__(1024) gn_param_grads_kernel(const float* __restrict__ nc, float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                              const float* __restrict__ gamma, float2* __restrict__ coef, GnGeom g, int param_ctas) {
  __shared__ float sh[32][33];
  ptx::grid_wait();
  if ((int)blockIdx.x >= param_ctas) {
    const int k = ((int)blockIdx.x - param_ctas) * 32 + threadIdx.y;   // (picture, group)
    if (k >= g.N * g.G) return;
    const int n = k / g.G, c0 = (k - n * g.G) * g.cpg;
    const float* b = nc + (size_t)n * 2 * g.C + c0;
    float m1 = 0.0f, m2 = 0.0f;
    for (int c = threadIdx.x; c < g.cpg; c += 32) {
      const float w = gamma[c0 + c];
      m1 = fmaf(w, __ldcg(b + c), m1);
      m2 = fmaf(w, __ldcg(b + g.C + c), m2);
    }
    m1 = warp_sum(m1);
    m2 = warp_sum(m2);
    if (threadIdx.x == 0) coef[k] = make_float2(m1 * g.inv_count, m2 * g.inv_count);
    return;
  }
  const int i = blockIdx.x * 32 + threadIdx.x;   // over [2][C]
  float s = 0.0f;
  if (i < 2 * g.C)
    for (int n = threadIdx.y; n < g.N; n += 32) s += __ldcg(nc + (size_t)n * 2 * g.C + i);
  sh[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && i < 2 * g.C) {
    float t = 0.0f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += sh[r][threadIdx.x];
    if (i < g.C) dbeta[i] = t;
    else dgamma[i - g.C] = t;
  }
}

// dx = rstd (gamma g - m1 - xh m2)
template <int DT, int ACT, bool kRagged>
__global__ void __launch_bounds__(512, 1) gn_grad_apply_kernel(const void* __restrict__ dy, const void* __restrict__ x, void* __restrict__ dx,
                                                            const float* __restrict__ gamma, const float* __restrict__ beta,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            const float2* __restrict__ coef, GnGeom g) {
  constexpr int V = Elem<DT>::V, H = V / 2;
  const int n = blockIdx.z, vcol = blockIdx.y * g.cols + threadIdx.x % g.cols, lane = threadIdx.x / g.cols;
  if (lane >= g.lanes || vcol * V >= g.W) return;
  const Share h = share_of(g, n, gridDim.x - 1 - blockIdx.x);   // backwards, as in gn_apply_kernel
  int c[V];
  thread_channels<V>(g, vcol, c);
  Gradient<DT, ACT> f;
  f.load(g, n, c, gamma, beta, mean, rstd);
  float m1[V], m2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 m = coef[(size_t)n * g.G + c[i] / g.cpg];
    m1[i] = m.x; m2[i] = m.y;
  }
  GradApply<DT, ACT> a;
  a.set(f, m1, m2);
  const int pitch = g.W / V;
  const size_t at = (size_t)(h.f0 + lane) * pitch + vcol, step = (size_t)g.lanes * pitch;
  extern __shared__ float4 ring4[];
  const uint4* src[2] = {reinterpret_cast<const uint4*>(x) + at, reinterpret_cast<const uint4*>(dy) + at};
  uint4* dst = reinterpret_cast<uint4*>(dx) + at;
  const int rows = (int)max(0ll, h.f1 - h.f0 - lane);
  f2 xh[H], t[H];
  stream_vectors<2>(src, step, (rows + g.lanes - 1) / g.lanes, reinterpret_cast<uint4*>(ring4), [&](int, const uint4 (&v)[2]) {
    f(v[0], v[1], xh, t);
    __stcs(dst, a(xh, t));
    dst += step;
  });
  if (kRagged)
    edge_rows(g, h, lane, [&](long long row) {
      const long long e = row * g.W + (long long)vcol * V;
      f(load_edge<DT>(x, e, g.total), load_edge<DT>(dy, e, g.total), xh, t);
      store_edge<DT>(dx, e, a(xh, t), h.lo, h.hi);
    });
}

// =================================================================================================
// One pass: a cluster of CTAs holds a slab -- one picture, `cols` vector columns of whole groups -- in its shared
// memory, exchanges the groups' sums through distributed shared memory and finishes the slab from there.  The tensor is
// read once and the result written once.
// =================================================================================================
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the float at the address of `p` in the shared memory of CTA `rank` of this cluster
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
  return v;
}

constexpr int kPieces = 4;   // a thread's vectors arrive in this many groups

// A cluster's place: grid (cluster size, column blocks, pictures).
struct Slab {
  int n, blk, j, lane, vcol, groups, channels;
  uint32_t rank, size;
  bool active;
  int rows, piece;       // this thread's vectors inside the picture, and how many rows of the lane grid a piece spans
  Share h;
};
template <int V> __device__ __forceinline__ Slab slab_of(const GnGeom& g) {
  Slab b;
  b.n = blockIdx.z; b.blk = blockIdx.y;
  b.size = gridDim.x;
  b.rank = b.size > 1 ? cluster_rank() : 0;
  b.lane = threadIdx.x / g.cols; b.j = threadIdx.x - b.lane * g.cols;
  b.vcol = b.blk * g.cols + b.j;
  b.groups = g.G / g.nblk;
  b.channels = b.groups * g.cpg;
  b.h = share_of(g, b.n, b.rank);
  b.active = b.lane < g.lanes;
  b.rows = b.active ? (int)max(0ll, b.h.f1 - b.h.f0 - b.lane) : 0;
  b.piece = (b.rows + kPieces * g.lanes - 1) / (kPieces * g.lanes) * g.lanes;
  return b;
}

// How a thread's V columns meet the groups.  R = 1: a group is whole vectors, R = 2: whole halves of vectors (4 channels a
// group in 16-bit types); both have rows of whole vectors.  R = V: anything else.
__host__ __device__ inline int fold_values(int V, int f, int cpg) { return f > 1 ? V : cpg % V == 0 ? 1 : cpg % (V / 2) == 0 ? 2 : V; }
template <int V, int R> struct Cols {
  static constexpr int H = V / 2, NG = R, NP = R == V ? H : R;   // groups of a thread, and pairs that differ by group
  int c[R == V ? V : 1];   // channels within the block (whole vectors: the first)
  int k[NG];               // groups within the block
  __device__ __forceinline__ void set(const GnGeom& g, const Slab& b) {
    if (R == V) {
      int cc[V];
      thread_channels<V>(g, b.j, cc);
#pragma unroll
      for (int i = 0; i < V; ++i) { c[R == V ? i : 0] = cc[i]; k[R == V ? i : 0] = (int)g.div_cpg.div((uint32_t)cc[i]); }
    } else {
      c[0] = b.j * V;
#pragma unroll
      for (int i = 0; i < NG; ++i) k[i] = (int)g.div_cpg.div((uint32_t)(b.j * V + i * (V / R)));
    }
  }
  __device__ static constexpr int pair(int h) { return R == V ? h : h * R / H; }   // which of the NP pairs column pair h uses
  // a value of every group as pairs
  template <class F> __device__ __forceinline__ void by_group(f2 (&o)[NP], F f) const {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (R == V) o[i] = pk(f(k[R == V ? 2 * i : 0]), f(k[R == V ? 2 * i + 1 : 0]));
      else {
        const float v = f(k[i]);
        o[i] = pk(v, v);
      }
    }
  }
  // the V values of a channel vector that starts with the block's channel 0 at `p`
  __device__ __forceinline__ void by_channel(f2 (&o)[H], const float* __restrict__ p) const {
    if (R == V) {
#pragma unroll
      for (int h = 0; h < H; ++h) o[h] = pk(__ldg(p + c[R == V ? 2 * h : 0]), __ldg(p + c[R == V ? 2 * h + 1 : 0]));
    } else {
#pragma unroll
      for (int h = 0; h < H; h += 2) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + c[0]) + h / 2);
        o[h] = pk(v.x, v.y);
        o[h + 1] = pk(v.z, v.w);
      }
    }
  }
};

// Two sums of a thread's columns at once, folded over the CTA by group: out[k], out[groups + k].  R values a thread:
// neighbouring columns of one group meet in the thread first.  A warp, or several where groups are few, adds a group's
// columns of all row lanes.  red: 2 * lanes * (cols * R | 1) floats (odd rows keep the warps' reads apart in the banks),
// part: 2 * max(groups, warps) floats.
template <int R, int V> __device__ __forceinline__ void fold_groups(const GnGeom& g, const Slab& b, const f2 (&s2)[V / 2], const f2 (&q2)[V / 2],
                                                                    float* red, float* part, float* out) {
  constexpr int run = V / R;
  const int w = (g.cols * R) | 1;
  float* red_q = red + g.lanes * w;
  if (b.active) {
    float s[V], q[V];
#pragma unroll
    for (int h = 0; h < V / 2; ++h) { un(s2[h], s[2 * h], s[2 * h + 1]); un(q2[h], q[2 * h], q[2 * h + 1]); }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float a = s[i * run], c = q[i * run];
#pragma unroll
      for (int k = 1; k < run; ++k) { a += s[i * run + k]; c += q[i * run + k]; }
      red[b.lane * w + b.j * R + i] = a;
      red_q[b.lane * w + b.j * R + i] = c;
    }
  }
  __syncthreads();
  const int per = g.cpg / run, pitch = b.channels / run;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, ln = threadIdx.x & 31;
  const int share = warps > b.groups ? warps / b.groups : 1;   // warps of a group
  const int packed = per < 32 ? 32 / per : 1;                  // row lanes a warp takes side by side
  const int l0 = per < 32 ? ln / per : 0, c0 = per < 32 ? ln - l0 * per : ln;
  const int slot = warp % share;
  for (int k = warp / share; k < b.groups; k += max(1, warps / share)) {
    float a = 0.0f, c = 0.0f;
    if (l0 < packed)
      for (int r = 0; r < (R == V ? g.f : 1); ++r)
        for (int l = slot * packed + l0; l < g.lanes; l += share * packed)
          for (int e = c0; e < per; e += 32) {
            const int at = l * w + r * pitch + k * per + e;
            a += red[at];
            c += red_q[at];
          }
    a = warp_sum(a);
    c = warp_sum(c);
    if (ln == 0) { part[2 * (k * share + slot)] = a; part[2 * (k * share + slot) + 1] = c; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * b.groups; i += blockDim.x) {
    const int k = i >> 1;
    float v = 0.0f;
    for (int t = 0; t < share; ++t) v += part[2 * (k * share + t) + (i & 1)];
    out[(i & 1) * b.groups + k] = v;
  }
}

// Sums of x and of (x - shift)^2.  The shift of a group is one of its values, the picture's first: all CTAs of the cluster
// take the same one, so their sums simply add up.  x itself is added, not x - shift, whose mean would carry the rounding of
// |mean - shift| where the mean is next to nothing.  The second round, whose shift is the mean, adds x - shift (kAbout).
template <int DT, int R> struct ShiftedSums {
  static constexpr int V = Elem<DT>::V, H = V / 2;
  typedef Cols<V, R> C;
  f2 nshift[C::NP], s[H], q[H];
  __device__ void clear() {
#pragma unroll
    for (int h = 0; h < H; ++h) s[h] = q[h] = pk(0.0f, 0.0f);
  }
  template <bool kAbout> __device__ __forceinline__ void add(const uint4& v) {
    f2 x[H];
    Elem<DT>::unpack(v, x);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const f2 d = add2(x[h], nshift[C::pair(h)]);
      s[h] = add2(s[h], kAbout ? d : x[h]);
      q[h] = fma2(d, d, q[h]);
    }
  }
  template <bool kAbout> __device__ void add_edge(const uint4& v, long long e, long long lo, long long hi) {
    f2 x[H];
    Elem<DT>::unpack(v, x);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const bool ia = e + 2 * h >= lo && e + 2 * h < hi, ib = e + 2 * h + 1 >= lo && e + 2 * h + 1 < hi;
      float xa, xb, da, db;
      un(x[h], xa, xb);
      un(add2(x[h], nshift[C::pair(h)]), da, db);
      const f2 d = pk(ia ? da : 0.0f, ib ? db : 0.0f);
      s[h] = add2(s[h], kAbout ? d : pk(ia ? xa : 0.0f, ib ? xb : 0.0f));
      q[h] = fma2(d, d, q[h]);
    }
  }
};

template <int DT, int ACT, int R, bool kRagged>
__global__ void __launch_bounds__(512, 2) gn_forward_slab_kernel(const void* __restrict__ x, void* __restrict__ y, const float* __restrict__ gamma,
                                                                 const float* __restrict__ beta, float* __restrict__ mean_out,
                                                                 float* __restrict__ rstd_out, GnGeom g) {
  constexpr int V = Elem<DT>::V, H = V / 2;
  typedef Cols<V, R> C;
  extern __shared__ float4 sh4[];
  uint4* tile = reinterpret_cast<uint4*>(sh4);                       // [per][cols]
  const Slab b = slab_of<V>(g);
  const Share& h = b.h;
  float* own = reinterpret_cast<float*>(tile + (size_t)g.per * g.cols);   // [2][groups] this CTA's sums, for the cluster
  float* own2 = own + 2 * b.groups;                                  // the same of the second round
  float* mean_s = own2 + 2 * b.groups;
  float* rstd_s = mean_s + b.groups;
  float* part = rstd_s + b.groups;                                   // [2 * max(groups, warps)]
  float* red = part + 2 * max(b.groups, (int)(blockDim.x >> 5));
  const int pitch = g.W / V;
  const size_t step = (size_t)g.lanes * pitch;
  const int tstep = g.lanes * g.cols;
  const size_t at = (size_t)(h.f0 + b.lane) * pitch + b.vcol;
  uint4* const mine = tile + (size_t)(h.f0 - h.s0 + b.lane) * g.cols + b.j;

  // all of the thread's copies leave at once, in pieces that are waited for one after the other
  {
    const uint4* src = reinterpret_cast<const uint4*>(x) + at;
    uint4* dst = mine;
    int r = 0;
#pragma unroll
    for (int k = 1; k <= kPieces; ++k) {
      const int end = min(b.rows, k * b.piece);
      for (; r < end; r += g.lanes, src += step, dst += tstep) copy16(dst, src);
      copy_commit();
    }
  }
  C cols;
  cols.set(g, b);
  const long long corner = h.lo + (long long)b.blk * b.channels;     // the picture's first position, this block's channels
  ShiftedSums<DT, R> m;
  m.clear();
  Normalise<DT, ACT> f;
  if (b.active) {
    cols.by_group(m.nshift, [&](int k) { return -load_param_as_f32(x, DT, corner + k * g.cpg); });
    cols.by_channel(f.sc, gamma + b.blk * b.channels);
    cols.by_channel(f.be, beta + b.blk * b.channels);
    if (kRagged)
      edge_rows(g, h, b.lane, [&](long long row) {
        const long long e = row * g.W + (long long)b.vcol * V;
        const uint4 v = load_edge<DT>(x, e, g.total);
        tile[(size_t)(row - h.s0) * g.cols + b.j] = v;
        m.template add_edge<false>(v, e, h.lo, h.hi);
      });
  }
  {
    const uint4* src = mine;
    int r = 0;
#pragma unroll
    for (int k = 1; k <= kPieces; ++k) {
      copy_wait(kPieces - k);
      const int end = min(b.rows, k * b.piece);
#pragma unroll 2
      for (; r < end; r += g.lanes, src += tstep) m.template add<false>(*src);
    }
  }
  // Totals of the cluster, and the variance from them.  Where the shift turns out to be far from the mean (its square 16 times
  // the variance) the squares have cancelled too much, and where the mean is as far from zero its rounding is too much for
  // the variance: then a second round over the tile takes the mean as its shift.  (By the root-mean-square and the largest
  // error of rstd in half steps of f32: mean at 4 deviations 3.7 and 20, at 7 5.9 and 48, after a second round 0.8 and 2.4.
  // It takes [64,3136,256] from 50 to 65 us.)  Every CTA of the cluster sees the same totals, so they agree on it.
  const float count = (float)g.P * (float)g.cpg;
  for (int round = 0; round < 2; ++round) {
    float* sums = round ? own2 : own;
    fold_groups<R, V>(g, b, m.s, m.q, red, part, sums);
    if (b.size > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();
    bool again = false;
    for (int k = threadIdx.x; k < b.groups; k += blockDim.x) {
      float ts, tq;
      if (b.size > 1) {
        float vs[8], vq[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r) {
          vs[r] = r < b.size ? peer_float(sums + k, r) : 0.0f;
          vq[r] = r < b.size ? peer_float(sums + b.groups + k, r) : 0.0f;
        }
        ts = ((vs[0] + vs[1]) + (vs[2] + vs[3])) + ((vs[4] + vs[5]) + (vs[6] + vs[7]));
        tq = ((vq[0] + vq[1]) + (vq[2] + vq[3])) + ((vq[4] + vq[5]) + (vq[6] + vq[7]));
      } else {
        ts = sums[k];
        tq = sums[b.groups + k];
      }
      const float shift = round ? mean_s[k] : load_param_as_f32(x, DT, corner + k * g.cpg);
      const float of_sum = ts * g.inv_count, mean = round ? shift + of_sum : of_sum, d = round ? of_sum : of_sum - shift;
      const float sq = fmaf(-d * count, d, tq), rstd = 1.0f / sqrtf((sq < 0.0f ? 0.0f : sq) * g.inv_count + g.eps);
      mean_s[k] = mean;
      rstd_s[k] = rstd;
      const bool more = round == 0 && (sq * 16.0f < tq || mean * mean * count > 16.0f * sq);
      again = again || more;
      if (b.rank == 0) {   // written again by a second round
        const size_t out = (size_t)b.n * g.G + (size_t)b.blk * b.groups + k;
        mean_out[out] = mean;
        rstd_out[out] = rstd;
      }
    }
    if (!__syncthreads_or(again)) break;
    // every thread reads the means here; the next round's writes are behind fold_groups' barriers
    m.clear();
    if (b.active) {
      cols.by_group(m.nshift, [&](int k) { return -mean_s[k]; });
      const uint4* src = mine;
      for (int r = 0; r < b.rows; r += g.lanes, src += tstep) m.template add<true>(*src);
      if (kRagged)
        edge_rows(g, h, b.lane, [&](long long row) {
          m.template add_edge<true>(tile[(size_t)(row - h.s0) * g.cols + b.j], row * g.W + (long long)b.vcol * V, h.lo, h.hi);
        });
    }
  }
  if (b.size > 1) cluster_arrive();   // done with the peers' shared memory
  if (b.active) {
    f2 nm[C::NP], rs[C::NP];
    cols.by_group(nm, [&](int k) { return -mean_s[k]; });
    cols.by_group(rs, [&](int k) { return rstd_s[k]; });
#pragma unroll
    for (int i = 0; i < H; ++i) {
      f.nmu[i] = nm[C::pair(i)];
      f.sc[i] = mul2(f.sc[i], rs[C::pair(i)]);
    }
    const uint4* src = mine;
    uint4* dst = reinterpret_cast<uint4*>(y) + at;
#pragma unroll 2
    for (int r = 0; r < b.rows; r += g.lanes, src += tstep, dst += step) __stcs(dst, f(*src));
    if (kRagged)
      edge_rows(g, h, b.lane, [&](long long row) {
        store_edge<DT>(y, row * g.W + (long long)b.vcol * V, f(tile[(size_t)(row - h.s0) * g.cols + b.j]), h.lo, h.hi);
      });
  }
  if (b.size > 1) cluster_wait();
}

// col[e] and col[w + e]: sums over the row lanes of two values of each column, e < w = cols * V.  red: lanes * 2 w floats,
// part: blockDim.x floats.  Ends with a barrier.
template <int V> __device__ void fold_columns(const GnGeom& g, const Slab& b, const f2 (&s2)[V / 2], const f2 (&q2)[V / 2], float* red, float* part,
                                              float* col) {
  const int w2 = 2 * g.cols * V, threads = blockDim.x;
  if (b.active) {
    float4* d = reinterpret_cast<float4*>(red + b.lane * w2 + b.j * V);
    float4* e = reinterpret_cast<float4*>(red + b.lane * w2 + w2 / 2 + b.j * V);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      float4 a, c;
      un(s2[2 * i], a.x, a.y); un(s2[2 * i + 1], a.z, a.w);
      un(q2[2 * i], c.x, c.y); un(q2[2 * i + 1], c.z, c.w);
      d[i] = a;
      e[i] = c;
    }
  }
  __syncthreads();
  const int parts = threads / w2;
  if (parts <= 1) {
    for (int e = threadIdx.x; e < w2; e += threads) {
      float v = 0.0f;
      for (int l = 0; l < g.lanes; ++l) v += red[l * w2 + e];
      col[e] = v;
    }
  } else {
    const int p = threadIdx.x / w2, e = threadIdx.x - p * w2;
    float v = 0.0f;
    if (p < parts)
      for (int l = p; l < g.lanes; l += parts) v += red[l * w2 + e];
    part[threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.x < w2) {
      v = 0.0f;
      for (int k = 0; k < parts; ++k) v += part[k * w2 + threadIdx.x];
      col[threadIdx.x] = v;
    }
  }
  __syncthreads();
}

template <int DT, int ACT, int R, bool kRagged>
__global__ void __launch_bounds__(512, 1) gn_backward_slab_kernel(const void* __restrict__ dy, const void* __restrict__ x, void* __restrict__ dx,
                                                                  const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                  float* __restrict__ nc, GnGeom g) {
  constexpr int V = Elem<DT>::V, H = V / 2;
  typedef Cols<V, R> C;
  extern __shared__ float4 sh4[];
  uint4* tile_x = reinterpret_cast<uint4*>(sh4);                     // [per][cols]
  uint4* tile_d = tile_x + (size_t)g.per * g.cols;                   // [per][cols]
  const Slab b = slab_of<V>(g);
  const Share& h = b.h;
  float* red = reinterpret_cast<float*>(tile_d + (size_t)g.per * g.cols);   // [lanes][2 cols V]
  float* part = red + g.lanes * 2 * g.cols * V;
  float* col = part + blockDim.x;                                    // [2][cols * V] sums of g and of g xh
  float* m1_s = col + 2 * g.cols * V;
  float* m2_s = m1_s + b.groups;
  float* chan = m2_s + b.groups;                                     // [2][channels]
  const int pitch = g.W / V;
  const size_t step = (size_t)g.lanes * pitch;
  const int tstep = g.lanes * g.cols;
  const size_t at = (size_t)(h.f0 + b.lane) * pitch + b.vcol;
  const size_t tile_at = (size_t)(h.f0 - h.s0 + b.lane) * g.cols + b.j;
  {
    const uint4* px = reinterpret_cast<const uint4*>(x) + at;
    const uint4* pd = reinterpret_cast<const uint4*>(dy) + at;
    uint4* tx = tile_x + tile_at;
    uint4* td = tile_d + tile_at;
    int r = 0;
#pragma unroll
    for (int k = 1; k <= kPieces; ++k) {
      const int end = min(b.rows, k * b.piece);
      for (; r < end; r += g.lanes, px += step, pd += step, tx += tstep, td += tstep) {
        copy16(tx, px);
        copy16(td, pd);
      }
      copy_commit();
    }
  }
  ptx::grid_release();
  C cols;
  cols.set(g, b);
  f2 nmu[C::NP], rs[C::NP], ga[H], be[H];
  GradSums<DT, ACT> sum;
  sum.clear();
  if (b.active) {
    const size_t k0 = (size_t)b.n * g.G + (size_t)b.blk * b.groups;
    cols.by_group(nmu, [&](int k) { return -mean[k0 + k]; });
    cols.by_group(rs, [&](int k) { return rstd[k0 + k]; });
    cols.by_channel(ga, gamma + b.blk * b.channels);
    cols.by_channel(be, beta + b.blk * b.channels);
  }
  auto normal = [&](const uint4& v, f2 (&xh)[H]) {
    Elem<DT>::unpack(v, xh);
#pragma unroll
    for (int i = 0; i < H; ++i) xh[i] = mul2(add2(xh[i], nmu[C::pair(i)]), rs[C::pair(i)]);
  };
  auto grad = [&](const uint4& v, const f2 (&xh)[H], f2 (&t)[H]) {
    Elem<DT>::unpack(v, t);
    if (ACT != HE_ACT_NONE)
#pragma unroll
      for (int i = 0; i < H; ++i) t[i] = mul2(t[i], slope2<ACT, DT == HE_F32>(fma2(xh[i], ga[i], be[i])));
  };
  f2 xh[H], t[H];
  if (kRagged && b.active)
    edge_rows(g, h, b.lane, [&](long long row) {
      const long long e = row * g.W + (long long)b.vcol * V;
      const uint4 vx = load_edge<DT>(x, e, g.total), vd = load_edge<DT>(dy, e, g.total);
      const size_t k = (size_t)(row - h.s0) * g.cols + b.j;
      tile_x[k] = vx;
      normal(vx, xh);
      grad(vd, xh, t);
      tile_d[k] = vd;
      sum.add_edge(xh, t, e, h.lo, h.hi);
    });
  {
    const uint4* tx = tile_x + tile_at;
    const uint4* td = tile_d + tile_at;
    int r = 0;
#pragma unroll
    for (int k = 1; k <= kPieces; ++k) {
      copy_wait(kPieces - k);
      const int end = min(b.rows, k * b.piece);
      for (; r < end; r += g.lanes, tx += tstep, td += tstep) {
        normal(*tx, xh);
        grad(*td, xh, t);
        sum.add(xh, t);
      }
    }
  }
  fold_columns<V>(g, b, sum.b, sum.w, red, part, col);
  if (b.size > 1) { cluster_arrive(); cluster_wait(); }
  // channel sums of the picture over the cluster's CTAs and the f places of a channel (every CTA makes its own copy);
  // rank 0 hands them on for the parameters' gradients
  for (int i = threadIdx.x; i < 2 * b.channels; i += blockDim.x) {
    const int half = i >= b.channels ? 1 : 0, c = i - half * b.channels;
    const float* src = col + half * g.cols * V + c;
    float s = 0.0f;
    for (int k = 0; k < g.f; ++k) {
      if (b.size > 1) {
        float v[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r) v[r] = r < b.size ? peer_float(src + k * b.channels, r) : 0.0f;
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      } else {
        s += src[k * b.channels];
      }
    }
    if (b.rank == 0) nc[((size_t)b.n * 2 + half) * g.C + (size_t)b.blk * b.channels + c] = s;
    chan[i] = s;
  }
  __syncthreads();
  if (b.size > 1) cluster_arrive();
  {
    const int ln = threadIdx.x & 31;
    for (int k = threadIdx.x >> 5; k < b.groups; k += blockDim.x >> 5) {
      float v1 = 0.0f, v2 = 0.0f;
      for (int c = ln; c < g.cpg; c += 32) {
        const float w = __ldg(gamma + b.blk * b.channels + k * g.cpg + c);
        v1 = fmaf(w, chan[k * g.cpg + c], v1);
        v2 = fmaf(w, chan[b.channels + k * g.cpg + c], v2);
      }
      v1 = warp_sum(v1);
      v2 = warp_sum(v2);
      if (ln == 0) { m1_s[k] = v1 * g.inv_count; m2_s[k] = v2 * g.inv_count; }
    }
  }
  __syncthreads();
  if (b.active) {
    // dx = rstd (gamma g - m1 - xh m2), the factor rstd multiplied into the others
    f2 n1[C::NP], n2[C::NP], gr[H];
    cols.by_group(n1, [&](int k) { return -m1_s[k]; });
    cols.by_group(n2, [&](int k) { return -m2_s[k]; });
#pragma unroll
    for (int i = 0; i < C::NP; ++i) { n1[i] = mul2(n1[i], rs[i]); n2[i] = mul2(n2[i], rs[i]); }
#pragma unroll
    for (int i = 0; i < H; ++i) gr[i] = mul2(ga[i], rs[C::pair(i)]);
    auto result = [&](const uint4& vx, const uint4& vd) {
      normal(vx, xh);
      grad(vd, xh, t);
#pragma unroll
      for (int i = 0; i < H; ++i) t[i] = fma2(gr[i], t[i], fma2(xh[i], n2[C::pair(i)], n1[C::pair(i)]));
      return Elem<DT>::pack(t);
    };
    const uint4* tx = tile_x + tile_at;
    const uint4* td = tile_d + tile_at;
    uint4* dst = reinterpret_cast<uint4*>(dx) + at;
#pragma unroll 2
    for (int r = 0; r < b.rows; r += g.lanes, tx += tstep, td += tstep, dst += step) __stcs(dst, result(*tx, *td));
    if (kRagged)
      edge_rows(g, h, b.lane, [&](long long row) {
        const size_t k = (size_t)(row - h.s0) * g.cols + b.j;
        store_edge<DT>(dx, row * g.W + (long long)b.vcol * V, result(tile_x[k], tile_d[k]), h.lo, h.hi);
      });
  }
  if (b.size > 1) cluster_wait();
}

constexpr int kMaxSmem = 232448 - 1024;   // dynamic shared memory a CTA may ask for (with room for what kernels declare)
// Bytes of shared memory of a slab CTA.
size_t slab_smem(int direction, int dt, int values, int threads, int per, int cols, int groups, int channels) {
  const size_t tile = (size_t)per * cols * 16, lanes = (size_t)threads / cols;
  const int V = dt == HE_F32 ? 4 : 8;
  if (direction == HE_GN_FORWARD)
    return tile + 4 * (6 * (size_t)groups + 2 * (size_t)std::max(groups, threads / 32) + 2 * lanes * ((size_t)(cols * values) | 1));
  return 2 * tile +
         4 * (lanes * 2 * cols * V + (size_t)threads + 2 * (size_t)cols * V + 2 * (size_t)groups + 2 * (size_t)channels);
}

// ---- plan --------------------------------------------------------------------------------------------------------
struct GroupNormPlan : he_plan {
  int direction = 0, dtype = HE_BF16, act = HE_ACT_NONE;
  bool ragged = false;
  GnGeom g{};
  int threads = 512, slices = 1;
  int cluster = 0;         // CTAs of a slab's cluster; 0: the two-pass kernels
  size_t smem = 0;
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

// The folds start behind the kernel in front of them (launch_behind): a few small CTAs that are in place when its last one ends
// (slabs backward [3,437,320] 9.2 -> 8.4 us, two passes backward [1,200000,77] 48.4 -> 45.2 us).  The second passes, and the
// products of muon.cu, do not: started early, their many CTAs take the room of those still running (two passes forward
// [2,262144,128] 84 -> 93 us, the conv net's filters 292 -> 299 us).
template <int DT, int ACT, bool R>
int32_t GroupNormPlan::run(const void* const* in, void* const* out, void* ws, cudaStream_t st) {
  constexpr int V = Elem<DT>::V;
  if (cluster) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)cluster, (unsigned)g.nblk, (unsigned)g.N);
    lc.blockDim = dim3((unsigned)threads, 1, 1);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    lc.attrs = &attr;
    lc.numAttrs = 1;
    const int values = fold_values(V, g.f, g.cpg);
    static SmemLimit limits[2][3];
    SmemLimit& limit = limits[direction][!R && values == 1 ? 0 : !R && values == 2 ? 1 : 2];
    if (direction == HE_GN_FORWARD) {
      auto kernel = gn_forward_slab_kernel<DT, ACT, V, R>;
      if (!R && values == 1) kernel = gn_forward_slab_kernel<DT, ACT, 1, false>;
      if (!R && values == 2) kernel = gn_forward_slab_kernel<DT, ACT, 2, false>;
      HE_TRY(limit.raise(kernel, ctx->device, kMaxSmem));
      HE_CUDA(cudaLaunchKernelEx(&lc, kernel, in[0], out[0], (const float*)in[1], (const float*)in[2], (float*)out[1], (float*)out[2], g));
      last_launches = 1;
      return HE_OK;
    }
    auto kernel = gn_backward_slab_kernel<DT, ACT, V, R>;
    if (!R && values == 1) kernel = gn_backward_slab_kernel<DT, ACT, 1, false>;
    if (!R && values == 2) kernel = gn_backward_slab_kernel<DT, ACT, 2, false>;
    HE_TRY(limit.raise(kernel, ctx->device, kMaxSmem));
    HE_CUDA(cudaLaunchKernelEx(&lc, kernel, in[0], in[1], out[0], (const float*)in[2], (const float*)in[3], (const float*)in[4],
                               (const float*)in[5], (float*)ws, g));
    const int param_ctas = (2 * g.C + 31) / 32;
    HE_TRY(launch_behind(gn_param_grads_kernel, dim3((unsigned)param_ctas), dim3(32, 32), 0, st, (const float*)ws, (float*)out[1], (float*)out[2],
                         (const float*)nullptr, (float2*)nullptr, g, param_ctas));
    last_launches = 2;
    return HE_OK;
  }
  const dim3 grid((unsigned)slices, (unsigned)g.nblk, (unsigned)g.N);
  const int w = g.cols * V, pitch = g.nblk * w;
  const int tensors = direction == HE_GN_FORWARD ? 1 : 2;
  const size_t ring = (size_t)kDepth * tensors * threads * 16, folds = (size_t)(threads * V + threads + w + (g.nblk == 1 ? g.G : 0)) * sizeof(float);
  const size_t smem = std::max(ring, folds);
  static SmemLimit limits2[4];
  if (direction == HE_GN_FORWARD) {
    const void* x = in[0];
    const float* gamma = (const float*)in[1]; const float* beta = (const float*)in[2];
    float* mean = (float*)out[1]; float* rstd = (float*)out[2];
    HE_TRY(limits2[0].raise(gn_moments_kernel<DT, R>, ctx->device, kMaxSmem));
    HE_TRY(limits2[1].raise(gn_apply_kernel<DT, ACT, R>, ctx->device, kMaxSmem));
    gn_moments_kernel<DT, R><<<grid, threads, smem, st>>>(x, (float2*)ws, g);
    HE_CUDA(cudaGetLastError());
    HE_TRY(launch_behind(gn_fold_moments_kernel, dim3((unsigned)(g.N * g.G)), dim3(256), 0, st, (const float2*)ws, mean, rstd, g, slices, pitch));
    gn_apply_kernel<DT, ACT, R><<<grid, threads, ring, st>>>(x, out[0], gamma, beta, mean, rstd, g);
    HE_CUDA(cudaGetLastError());
    last_launches = 3;
    return HE_OK;
  }
  const float* gamma = (const float*)in[2]; const float* beta = (const float*)in[3];
  const float* mean = (const float*)in[4]; const float* rstd = (const float*)in[5];
  float* nc = (float*)ws;                                         // [N][2][C]
  float2* coef = (float2*)(nc + (size_t)g.N * 2 * g.C);           // [N][G]
  float* part = (float*)(coef + (size_t)g.N * g.G);               // [N][slices][2][pitch]
  HE_TRY(limits2[2].raise(gn_grad_sums_kernel<DT, ACT, R>, ctx->device, kMaxSmem));
  HE_TRY(limits2[3].raise(gn_grad_apply_kernel<DT, ACT, R>, ctx->device, kMaxSmem));
  gn_grad_sums_kernel<DT, ACT, R><<<grid, threads, smem, st>>>(in[0], in[1], gamma, beta, mean, rstd, part, g);
  HE_CUDA(cudaGetLastError());
  const int param_ctas = (2 * g.C + 31) / 32, coef_ctas = (g.N * g.G + 31) / 32;
  HE_TRY(launch_behind(gn_fold_grads_kernel, dim3((unsigned)param_ctas, (unsigned)g.N), dim3(32, 32), 0, st, (const float*)part, nc, g, slices,
                       g.nblk == 1 ? g.C : pitch));
  HE_TRY(launch_behind(gn_param_grads_kernel, dim3((unsigned)(param_ctas + coef_ctas)), dim3(32, 32), 0, st, (const float*)nc, (float*)out[1],
                       (float*)out[2], gamma, coef, g, param_ctas));
  gn_grad_apply_kernel<DT, ACT, R><<<grid, threads, ring, st>>>(in[0], in[1], out[0], gamma, beta, mean, rstd, coef, g);
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
  // No output overlaps an input or another output: later kernels of a launch read what earlier ones would have written over.
  const size_t big = (size_t)g.total * dtype_bytes(dtype), param = (size_t)g.C * 4, stat = (size_t)g.N * g.G * 4;
  auto in_bytes = [&](int i) { return i < n_big ? big : i < n_big + 2 ? param : stat; };
  auto out_bytes = [&](int i) { return i == 0 ? big : direction == HE_GN_FORWARD ? stat : param; };
  auto meet = [](const void* p, size_t np, const void* q, size_t nq) {
    return (uintptr_t)p < (uintptr_t)q + nq && (uintptr_t)q < (uintptr_t)p + np;
  };
  for (int o = 0; o < 3; ++o) {
    for (int i = 0; i < n_in; ++i)
      if (meet(out[o], out_bytes(o), in[i], in_bytes(i))) HE_FAIL(HE_ERR_INVALID, "group norm: output %d overlaps input %d", o, i);
    for (int i = 0; i < o; ++i)
      if (meet(out[o], out_bytes(o), out[i], out_bytes(i))) HE_FAIL(HE_ERR_INVALID, "group norm: output %d overlaps output %d", o, i);
  }
  for (int i = 0; i < n_big; ++i)
    if ((uintptr_t)in[i] & 15) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: tensors must be 16-byte aligned");
  if ((uintptr_t)out[0] & 15) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: tensors must be 16-byte aligned");
  for (int i = n_big; i < n_in; ++i) {
    const bool vectors = i < n_big + 2;   // gamma and beta are read as vectors
    if ((uintptr_t)in[i] & (vectors ? 15 : 3)) HE_FAIL(HE_ERR_UNSUPPORTED, "group norm: %s must be %d-byte aligned", vectors ? "gamma and beta" : "mean and rstd", vectors ? 16 : 4);
  }
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
  g.div_c = FastDiv((uint32_t)g.C);
  g.div_cpg = FastDiv((uint32_t)g.cpg);
  g.inv_count = (float)(1.0 / ((double)g.P * g.cpg));
  plan->ragged = g.P % g.f != 0;
  const int sms = ctx_sm_count(ctx);
  const int vcols = g.W / V;
  plan->threads = 512;
  static const char* const kActs[] = {"none", "relu", "silu", "gelu"};
  char desc[256];
  // One pass where a slab fits the shared memory of a cluster.  Candidates: column blocks of whole groups and vectors (only
  // where a row is whole vectors), clusters of up to 8 CTAs (the portable size), CTAs of 128 to 512 threads.  Their time is
  // estimated from what was measured on a B200: a CTA's life is a fixed part (issue, folds, exchange: 4 us, with a
  // cluster 1.5 us more) and a part for each of its vectors; shared memory says how many live on an SM at once, gangs of
  // CTAs fill it to some 85 %; an SM issues 18 (backward 40) instructions a value; row segments below 64 bytes waste half
  // of DRAM's sectors.  ([64,3136,256] bf16 silu forward: 64-byte segments in clusters of 8 x 128 threads 50 us, 512-byte
  // ones in clusters of 8 x 512 threads 98 us; [128,784,128] backward: 32 us and 47 us.)
  const long long srows = ((long long)g.P + g.f - 1) / g.f + (plan->ragged ? 1 : 0);
  const bool fwd = direction == HE_GN_FORWARD;
  const int es = dtype_bytes(prm->dtype);
  double best = 1e30;
  for (int nblk = 1; nblk <= g.G; ++nblk) {
    if (g.G % nblk != 0 || (g.f > 1 && nblk > 1)) continue;
    const int ch = g.C / nblk;
    if ((g.f == 1 && ch % V != 0) || (nblk > 1 && ch * es < 32)) continue;
    const int cols = ch * g.f / V;
    for (int threads = 128; threads <= 512; threads *= 2) {
      if (cols > threads) continue;
      for (int cs = 1; cs <= 8; cs *= 2) {
        const long long per = (srows + cs - 1) / cs;
        if (cs > 1 && per * (cs - 1) >= srows) continue;   // a CTA of the cluster would be left without rows
        if (per * cols * 16 > 232448) continue;
        const size_t sm = slab_smem(direction, prm->dtype, fold_values(V, g.f, g.cpg), threads, (int)per, cols, g.G / nblk, ch);
        if (sm > kMaxSmem) continue;
        const int resident = std::max(1, std::min((int)(233472 / (sm + 1024)), (fwd ? 1024 : 512) / threads));
        const double ctas = (double)g.N * nblk * cs;
        const double vectors = std::ceil((double)per / (threads / cols));
        const double life = 4.0 + (cs > 1 ? 1.5 : 0.0) + vectors * (fwd ? 0.25 : 0.45) + threads * 0.002;
        const double rounds = std::max(1.0, ctas / (sms * resident * (cs > 1 ? 0.85 : 1.0)));
        const double issue = (double)g.total / std::min<double>(sms, ctas) * (fwd ? 18.0 : 40.0) / 243e3;
        const double narrow = nblk == 1 || ch * es >= 64 ? 1.0 : 1.3;
        const double memory = (double)g.total * es * (fwd ? 2 : 3) / 6.5e6 * narrow;
        const double us = std::max(rounds * life, std::max(issue, memory));
        if (us < best) {
          best = us;
          plan->cluster = cs;
          plan->smem = sm;
          plan->threads = threads;
          g.nblk = nblk; g.cols = cols; g.per = (int)per;
        }
      }
    }
  }
  // Against two passes over all of it (three launches forward, four backward, 5.6 TB/s): worth it for the largest tensors
  // only, where the slabs' folds and exchanges add up ([64,3136,256] bf16: backward 102 us in two passes, 129 us in slabs,
  // forward 73 and 50 us; [128,784,128] backward 41 and 32 us).  The constants were fitted to 16-bit types.  f32 backward, slabs and
  // two passes: [128,784,128] 44 and 54 us, [128,196,256] 21 and 34, [16,1024,320] 25 and 27 -- and five shapes where the estimate
  // takes slabs and two passes are the faster: [64,3136,256] 204 and 183 us, [128,3136,64] 105 and 95, [32,3136,64] 31 and 28,
  // [4,4096,512] 36 and 33, [8,4096,128] 23 and 20.  bf16 has one such, [32,3136,64] backward, 28 and 26 us; forward has none.
  const double two_us = (fwd ? 18.0 : 22.0) + (double)g.total * es * (fwd ? 3 : 5) / 5.6e6;
  if (plan->cluster && 6.0 + 1.25 * best > two_us) plan->cluster = 0;
  if (plan->cluster) {
    g.lanes = plan->threads / g.cols;
    plan->workspace_bytes = direction == HE_GN_FORWARD ? 0 : (size_t)g.N * 2 * g.C * sizeof(float);
    snprintf(desc, sizeof desc, "group norm %s: %s [%d,%d,%d] in %d groups, activation %s, one pass: slabs of %d channels in clusters of %d x %d threads",
             direction == HE_GN_FORWARD ? "forward" : "backward", dtype_name(prm->dtype), g.N, g.P, g.C, g.G, kActs[plan->act], g.C / g.nblk,
             plan->cluster, plan->threads);
    plan->description = desc;
    *out = plan.release();
    return HE_OK;
  }
  // Two passes: CTAs of 256 threads, or as many more as a row's vectors take
  plan->threads = vcols > 256 ? 512 : 256;
  g.cols = std::min(vcols, plan->threads);
  g.nblk = (vcols + g.cols - 1) / g.cols;
  g.lanes = plan->threads / g.cols;
  // slices: as many CTAs as shared memory has rings for, 6 an SM forward and 3 backward of 256 threads, and at least 16 super-rows
  // a thread (the folds' cost is per CTA).  Registers let fewer live: 3 of the moments pass (80), 2 or 3 of the others (16-bit types:
  // gn_apply_kernel 72-96, gn_grad_sums_kernel 78-126, gn_grad_apply_kernel 94-126), so a grid is two or three waves forward and one
  // and a half backward.
  const long long per_min = (long long)g.lanes * 16;
  long long want = std::max<long long>(1, (long long)sms * (fwd ? 6 : 3) * 256 / plan->threads / std::max<long long>(1, (long long)g.N * g.nblk));
  want = std::min(want, std::max<long long>(1, srows / per_min));
  g.per = (int)((srows + want - 1) / want);
  plan->slices = (int)((srows + g.per - 1) / g.per);
  // partial sums of a slice: of the groups or the channels, or of all columns where they are cut into blocks
  const size_t columns = (size_t)g.nblk * g.cols * V;
  plan->workspace_bytes = fwd ? (size_t)g.N * plan->slices * (g.nblk == 1 ? g.G : columns) * sizeof(float2)
                              : ((size_t)g.N * 2 * g.C + (size_t)g.N * g.G * 2 + (size_t)g.N * plan->slices * 2 * (g.nblk == 1 ? g.C : columns)) * sizeof(float);
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
