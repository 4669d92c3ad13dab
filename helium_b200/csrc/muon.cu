// The Muon optimiser's update: the momentum average of a weight gradient, orthogonalised by Newton-Schulz products.
//
//   avg' = m avg + (1 - m) g                              (helium's exponential average, helium/src/optimizer/sgd.rs:47-62)
//   d    = m avg' + (1 - m) g  (Nesterov)  or  avg'       (no momentum: d = g)
//   X    = d / (|d|_F + eps), transposed where d has more rows than columns: m x n with m <= n
//   steps times:  S = X X^T,  B = b S + c S^2,  X <- a X + B X
//   update = scale X
// so every singular value v of d / |d| is mapped by a v + b v^3 + c v^5 once per step.  helium builds optimisers from
// pointwise ops and matmuls (helium/src/optimizer); the products here are three tcgen05 GEMMs a step over the whole list of
// matrices at once, of which the symmetric ones (S and S^2) compute the tiles on and below the diagonal only.
//
// Numbers.  The operands are f16, each matrix scaled by a power of two: X by sx ~ sqrt(m n), which makes its
// root-mean-square 1 at the start and keeps |X| below 65504 (|X| <= 1.3 sx), S by 2^12, B by 2^10.  X itself is kept as a
// pair hi + lo of f16 (22 bits): the products read hi, the term a X adds the pair, so the rounding of hi is not multiplied
// by a = 3.4 step after step, and B's diagonal, by far its largest values, stays f32 and is applied to the pair too.
// Simulated against 64 bits, the update is 4e-4 .. 9e-4 off (relative, 2-norm), half a bf16 rounding of the result;
// bf16 operands were 4e-3 .. 2e-2 off, f16 without the pair 2e-3 .. 5e-3.
//
// Layout.  The workspace holds every matrix as blocks of 128 rows x 64 columns, 128 bytes a row, block after block: one
// tensor map over the whole workspace serves all operands of all matrices, whatever their shapes.  A block is a K-major
// operand of S = X X^T and, read as 64-row halves, an MN-major operand of B X.
#include <algorithm>
#include <cmath>
#include <memory>
#include <vector>

#include "device_utils.cuh"
#include "he_internal.h"
#include "sm100_ptx.cuh"

namespace he {
namespace {

constexpr int kMaxMats = 64;        // matrices of one round of launches (their table travels in the kernel parameters)
constexpr int kBlockRows = 128, kBlockCols = 64;
constexpr float kScaleS = 4096.0f, kScaleB = 1024.0f;
constexpr int kSumThreads = 256;

struct MuonMat {
  const void* g;
  const float* avg;
  float* avg_out;
  void* out;
  long long x[2], xlo, s, b;   // first rows of the blocks in the arena (128-byte rows)
  long long diag;              // first of m f32 values behind the table
  long long chunk;             // elements a CTA of the first pass sums
  int m, n, tall;              // m <= n; tall: the gradient is [n, m]
  int mt, nt;                  // 128-row and 128-column tiles
  int part0, chunks;           // partial sums of squares
  int sym0, x0, pack0;         // first tile of this matrix in the symmetric, product and packing grids
  float sx, out_scale;
};
struct MuonTable {
  int count;
  MuonMat mat[kMaxMats];
};
struct MuonStep {
  float momentum, rest;        // m and 1 - m
  int has_momentum, nesterov, grad_dt, out_dt;
  float a, b, c, eps;
};

__device__ __forceinline__ long long x_block(const MuonMat& m, int buf_row_block, int col_block) {
  return ((long long)buf_row_block * (2 * m.nt) + col_block) * kBlockRows;
}
__device__ __forceinline__ long long s_block(const MuonMat& m, int row_block, int col_block) {
  return ((long long)row_block * (2 * m.mt) + col_block) * kBlockRows;
}

// The matrix a tile belongs to: the last one whose first tile is not behind it.
template <class F> __device__ __forceinline__ int find_matrix(int count, int tile, F first) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(mid) <= tile) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float load_grad(const void* g, int dt, long long i) { return load_param_as_f32(g, dt, i); }
__device__ __forceinline__ float direction(const MuonStep& st, float g, float avg) {
  return st.nesterov ? fmaf(st.momentum, avg, st.rest * g) : avg;
}

// ---- first pass: the average, and partial sums of squares of the direction ------------------------------------------
// Squares are added in 64 bits: gradients as large as 1e30 and as small as 1e-25 keep their norm.
__global__ void __launch_bounds__(kSumThreads) muon_average_kernel(const __grid_constant__ MuonTable t, const __grid_constant__ MuonStep st,
                                                                  MuonTable* __restrict__ table_out, double* __restrict__ parts) {
  if (blockIdx.x == 0) {   // the later kernels read the table from memory
    const uint32_t* src = reinterpret_cast<const uint32_t*>(&t);
    uint32_t* dst = reinterpret_cast<uint32_t*>(table_out);
    for (int i = threadIdx.x; i < (int)(sizeof(MuonTable) / 4); i += kSumThreads) dst[i] = src[i];
  }
  const int k = find_matrix(t.count, blockIdx.x, [&](int i) { return t.mat[i].part0; });
  const MuonMat& m = t.mat[k];
  const long long total = (long long)m.m * m.n;
  const long long e0 = (long long)(blockIdx.x - m.part0) * m.chunk, e1 = min(total, e0 + m.chunk);
  double sum = 0.0;
  for (long long e = e0 + threadIdx.x * 4; e < e1; e += kSumThreads * 4) {
    float g[4], av[4];
    const int nv = (int)min(4ll, e1 - e);
    if (nv == 4) {
      if (st.grad_dt == HE_F32) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(m.g) + e));
        g[0] = v.x; g[1] = v.y; g[2] = v.z; g[3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(m.g) + e));
        const uint32_t w[2] = {v.x, v.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          g[2 * i] = st.grad_dt == HE_BF16 ? bf16_bits_to_f32(w[i] & 0xffffu) : f16_bits_to_f32(w[i] & 0xffffu);
          g[2 * i + 1] = st.grad_dt == HE_BF16 ? bf16_bits_to_f32(w[i] >> 16) : f16_bits_to_f32(w[i] >> 16);
        }
      }
      if (st.has_momentum) {
        const float4 v = *reinterpret_cast<const float4*>(m.avg + e);
        av[0] = v.x; av[1] = v.y; av[2] = v.z; av[3] = v.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) av[i] = fmaf(st.momentum, av[i], st.rest * g[i]);
        *reinterpret_cast<float4*>(m.avg_out + e) = make_float4(av[0], av[1], av[2], av[3]);
      }
    } else {
      for (int i = 0; i < nv; ++i) {
        g[i] = load_grad(m.g, st.grad_dt, e + i);
        if (st.has_momentum) {
          av[i] = fmaf(st.momentum, m.avg[e + i], st.rest * g[i]);
          m.avg_out[e + i] = av[i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < nv) {
        const double d = st.has_momentum ? direction(st, g[i], av[i]) : g[i];
        sum = fma(d, d, sum);
      }
  }
  __shared__ double sh[kSumThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < kSumThreads / 32; ++i) s += sh[i];
    parts[blockIdx.x] = s;
  }
}

// hi + lo of two neighbouring values as two packed words
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// ---- second pass: the direction, scaled and split, into the blocks of the workspace; zeros behind its edges ----------
__global__ void __launch_bounds__(256) muon_pack_kernel(const MuonTable* __restrict__ tp, const __grid_constant__ MuonStep st,
                                                        const double* __restrict__ parts, uint8_t* __restrict__ arena) {
  __shared__ float tile[64][65];
  __shared__ float scale_sh;
  const MuonTable& t = *tp;
  const int k = find_matrix(t.count, blockIdx.x, [&](int i) { return t.mat[i].pack0; });
  const MuonMat& m = t.mat[k];
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < m.chunks; i += 32) s += parts[m.part0 + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) scale_sh = (float)((double)m.sx / (sqrt(s) + (double)st.eps));
  }
  const int p = blockIdx.x - m.pack0, cb = p % (2 * m.nt), rb = p / (2 * m.nt);   // 64 x 64 piece
  const int r0 = rb * 64, c0 = cb * 64;
  __syncthreads();
  const float scale = scale_sh;
  // the gradient's own rows run along X's columns, or along its rows where it is tall
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int u = i >> 6, v = i & 63;
    const int r = m.tall ? r0 + v : r0 + u, c = m.tall ? c0 + u : c0 + v;
    float d = 0.0f;
    if (r < m.m && c < m.n) {
      const long long e = m.tall ? (long long)c * m.m + r : (long long)r * m.n + c;
      if (!st.has_momentum) d = load_grad(m.g, st.grad_dt, e);
      else d = st.nesterov ? direction(st, load_grad(m.g, st.grad_dt, e), m.avg_out[e]) : m.avg_out[e];
      d *= scale;
    }
    tile[r - r0][c - c0] = d;
  }
  __syncthreads();
  const long long row = x_block(m, r0 / kBlockRows, cb) + (r0 % kBlockRows);
  for (int i = threadIdx.x; i < 64 * 8; i += 256) {
    const int r = i >> 3, q = (i & 7) * 8;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_pair(tile[r][q + 2 * j], tile[r][q + 2 * j + 1], hi[j], lo[j]);
    const long long at = (row + r) * 128 + q * 2;
    *reinterpret_cast<uint4*>(arena + m.x[0] * 128 + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(arena + m.xlo * 128 + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// ---- the products -----------------------------------------------------------------------------------------------
enum Phase { PH_S = 0, PH_B = 1, PH_X = 2 };
constexpr int kTile = 128, kKBlock = 64;
constexpr int kStages = 3;                                  // 96 KB: two CTAs fit an SM, one's epilogue under the other's products
constexpr int kOperandBytes = kTile * kKBlock * 2;          // 16 KB
constexpr int kGemmThreads = 192;                           // producer warp, MMA warp, four epilogue warps
constexpr int kGemmSmem = kStages * 2 * kOperandBytes + (2 * kStages + 2) * 8 + 16 + 1024;

struct GemmArgs {
  const MuonTable* table;
  uint8_t* arena;
  float* diag;
  DeviceStatus* status;
  unsigned wait_limit_us;
  int withhold_loads;
  int cur;           // buffer of X that the step reads
  int last;          // the step writes the update
  float b, c, a;
  int out_dt;
};

// 64 bytes; not through the read-only path, since the lo values are rewritten in place by the thread that read them
__device__ __forceinline__ void load_chunk(const uint8_t* p, uint32_t (&w)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[8 * h]), "=r"(w[8 * h + 1]), "=r"(w[8 * h + 2]), "=r"(w[8 * h + 3]), "=r"(w[8 * h + 4]), "=r"(w[8 * h + 5]),
                   "=r"(w[8 * h + 6]), "=r"(w[8 * h + 7])
                 : "l"(p + 32 * h)
                 : "memory");
}
__device__ __forceinline__ void store_chunk(uint8_t* p, const uint32_t (&w)[16]) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = w[i];
  ptx::st_global_256(p, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = w[8 + i];
  ptx::st_global_256(p + 32, r);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ unsigned short out_bits(float v, int dt) {
  return (unsigned short)(dt == HE_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
}

template <int PH>
__global__ void __launch_bounds__(kGemmThreads) muon_gemm_kernel(const __grid_constant__ CUtensorMap map128,
                                                                 const __grid_constant__ CUtensorMap map64, const __grid_constant__ GemmArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t base = ptx::smem_u32(smem);
  const uint32_t bars = base + kStages * 2 * kOperandBytes;
  auto bar_full = [&](int s) { return bars + 8u * s; };
  auto bar_empty = [&](int s) { return bars + 8u * (kStages + s); };
  const uint32_t bar_done = bars + 8u * (2 * kStages), bar_drain = bar_done + 8u;
  volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(smem + kStages * 2 * kOperandBytes + (2 * kStages + 2) * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // the tile: row block i, column block j (the symmetric products: j <= i)
  const MuonTable& t = *p.table;
  const int mi = find_matrix(t.count, blockIdx.x, [&](int q) { return PH == PH_X ? t.mat[q].x0 : t.mat[q].sym0; });
  const MuonMat& m = t.mat[mi];
  int i, j;
  if (PH == PH_X) {
    const int q = blockIdx.x - m.x0;
    j = q / m.mt;      // neighbours share X's columns
    i = q - j * m.mt;
  } else {
    const int q = blockIdx.x - m.sym0;
    i = (int)((sqrtf(8.0f * q + 1.0f) - 1.0f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= q) ++i;
    while (i * (i + 1) / 2 > q) --i;
    j = q - i * (i + 1) / 2;
  }
  const bool same = PH != PH_X && i == j;    // both operands are one block row: loaded once
  const int k_blocks = PH == PH_S ? (m.n + kKBlock - 1) / kKBlock : (m.m + kKBlock - 1) / kKBlock;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(bar_full(s), 1);
      ptx::mbar_init(bar_empty(s), 1);
    }
    ptx::mbar_init(bar_done, 1);
    ptx::mbar_init(bar_drain, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_holder)), kTile);
    ptx::tmem_relinquish();
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0 && !p.withhold_loads) {
      int kb = 0;
      bool alive = true;
      for (; kb < k_blocks; ++kb) {
        const int s = kb % kStages;
        const uint32_t ph = (uint32_t)(kb / kStages) & 1u;
        if (!ptx::mbar_wait(bar_empty(s), ph ^ 1u, abort_flag, p.status, 1, s, p.wait_limit_us)) { alive = false; break; }
        const uint32_t a_dst = base + s * 2 * kOperandBytes, b_dst = a_dst + kOperandBytes;
        ptx::mbar_arrive_expect_tx(bar_full(s), same ? kOperandBytes : 2 * kOperandBytes);
        if (PH == PH_S) {
          ptx::tma_load_3d(a_dst, &map128, bar_full(s), 0, (int)(m.x[p.cur] + x_block(m, i, kb)), 0);
          if (!same) ptx::tma_load_3d(b_dst, &map128, bar_full(s), 0, (int)(m.x[p.cur] + x_block(m, j, kb)), 0);
        } else if (PH == PH_B) {
          ptx::tma_load_3d(a_dst, &map128, bar_full(s), 0, (int)(m.s + s_block(m, i, kb)), 0);
          if (!same) ptx::tma_load_3d(b_dst, &map128, bar_full(s), 0, (int)(m.s + s_block(m, j, kb)), 0);
        } else {
          ptx::tma_load_3d(a_dst, &map128, bar_full(s), 0, (int)(m.b + s_block(m, i, kb)), 0);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            ptx::tma_load_3d(b_dst + h * (kOperandBytes / 2), &map64, bar_full(s), 0,
                             (int)(m.x[p.cur] + x_block(m, kb >> 1, 2 * j + h) + (kb & 1) * 64), 0);
        }
      }
      // a tile that was given up: the copies in flight still land in this CTA's memory
      if (!alive)
        for (int b = kb > kStages ? kb - kStages : 0; b < kb; ++b) {
          int never = 0;
          ptx::mbar_wait(bar_full(b % kStages), (uint32_t)(b / kStages) & 1u, &never, p.status, 7, b % kStages, p.wait_limit_us);
        }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr bool kBMn = PH == PH_X;
      const uint32_t idesc = ptx::make_idesc_f16(0, 0, kBMn ? 1 : 0, kTile, kTile);
      constexpr uint32_t b_lbo = kBMn ? kOperandBytes / 2 : 16, b_kadv = kBMn ? 2048 : 32;
      bool alive = true;
      for (int kb = 0; kb < k_blocks; ++kb) {
        const int s = kb % kStages;
        if (!ptx::mbar_wait(bar_full(s), (uint32_t)(kb / kStages) & 1u, abort_flag, p.status, 3, s, p.wait_limit_us)) { alive = false; break; }
        ptx::tcgen05_fence_after();
        const uint32_t a_addr = base + s * 2 * kOperandBytes, b_addr = same ? a_addr : a_addr + kOperandBytes;
#pragma unroll
        for (int k = 0; k < kKBlock / 16; ++k)
          ptx::umma_f16(tmem, ptx::make_smem_desc_sw128(a_addr + k * 32, 16, 1024), ptx::make_smem_desc_sw128(b_addr + k * b_kadv, b_lbo, 1024),
                        idesc, (kb | k) != 0 ? 1u : 0u);
        ptx::umma_commit(bar_empty(s));
      }
      ptx::umma_commit(alive ? bar_done : bar_drain);
      if (!alive) {   // nothing may still write tensor memory when it is freed
        int never = 0;
        ptx::mbar_wait(bar_drain, 0, &never, p.status, 8, 0, p.wait_limit_us);
      }
    }
  } else {
    const bool ok = ptx::mbar_wait(bar_done, 0, abort_flag, p.status, 4, 0, p.wait_limit_us);
    if (__all_sync(0xffffffffu, ok)) {
      ptx::tcgen05_fence_after();
      const int quadrant = warp & 3, r = quadrant * 32 + lane;
      const int grow = i * kTile + r;
      const float inv_x2 = kScaleS / (m.sx * m.sx);
      float dg = 0.0f;
      if (PH == PH_X) dg = p.a + p.diag[m.diag + grow];
#pragma unroll 1
      for (int c0 = 0; c0 < kTile; c0 += 32) {
        uint32_t acc[32];
        ptx::tmem_ld_32x32(tmem + ((uint32_t)(quadrant * 32) << 16) + (uint32_t)c0, acc);
        // this thread's 32 columns in block (i, 2 j + c0 / 64): 64 bytes
        const long long sym_at = (s_block(m, i, 2 * j + (c0 >> 6)) + r) * 128 + (c0 & 32) * 2;
        const long long x_at = (x_block(m, i, 2 * j + (c0 >> 6)) + r) * 128 + (c0 & 32) * 2;
        uint32_t w0[16], w1[16];
        if (PH == PH_B) load_chunk(p.arena + m.s * 128 + sym_at, w0);
        if (PH == PH_X) {
          load_chunk(p.arena + m.x[p.cur] * 128 + x_at, w0);
          load_chunk(p.arena + m.xlo * 128 + x_at, w1);
        }
        ptx::tmem_ld_wait_regs(acc);
        float v[32];
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(acc[q]);
        if (PH == PH_S) {
#pragma unroll
          for (int q = 0; q < 32; ++q) v[q] *= inv_x2;
        } else if (PH == PH_B) {
          const float kb = p.b * (kScaleB / kScaleS), kc = p.c * (kScaleB / (kScaleS * kScaleS));
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 s = unpack_half2(w0[q]);
            v[2 * q] = fmaf(kc, v[2 * q], kb * s.x);
            v[2 * q + 1] = fmaf(kc, v[2 * q + 1], kb * s.y);
          }
          if (i == j) {   // the diagonal stays f32
#pragma unroll
            for (int q = 0; q < 32; ++q)
              if (c0 + q == r) {
                p.diag[m.diag + grow] = v[q] * (1.0f / kScaleB);
                v[q] = 0.0f;
              }
          }
        } else {
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 h = unpack_half2(w0[q]), l = unpack_half2(w1[q]);
            v[2 * q] = fmaf(dg, h.x + l.x, v[2 * q] * (1.0f / kScaleB));
            v[2 * q + 1] = fmaf(dg, h.y + l.y, v[2 * q + 1] * (1.0f / kScaleB));
          }
        }
        if (PH != PH_X) {
          uint8_t* dst = p.arena + (PH == PH_S ? m.s : m.b) * 128;
#pragma unroll
          for (int q = 0; q < 16; ++q) w0[q] = pack_half2(v[2 * q], v[2 * q + 1]);
          store_chunk(dst + sym_at, w0);
          if (i != j) {   // the mirrored tile: lanes are neighbouring columns of it
            unsigned short* mir = reinterpret_cast<unsigned short*>(dst + (s_block(m, j, 2 * i + (r >> 6)) + c0) * 128) + (r & 63);
#pragma unroll
            for (int q = 0; q < 32; ++q) mir[q * 64] = (unsigned short)(w0[q >> 1] >> (16 * (q & 1)));
          }
        } else if (!p.last) {
#pragma unroll
          for (int q = 0; q < 16; ++q) split_pair(v[2 * q], v[2 * q + 1], w0[q], w1[q]);
          store_chunk(p.arena + m.x[p.cur ^ 1] * 128 + x_at, w0);
          store_chunk(p.arena + m.xlo * 128 + x_at, w1);
        } else if (grow < m.m) {
          const float scale = m.out_scale / m.sx;
          unsigned short* out = reinterpret_cast<unsigned short*>(m.out);
          const int gcol = j * kTile + c0;
          if (m.tall) {
#pragma unroll
            for (int q = 0; q < 32; ++q)
              if (gcol + q < m.n) out[(long long)(gcol + q) * m.m + grow] = out_bits(v[q] * scale, p.out_dt);
          } else {
            unsigned short* o = out + (long long)grow * m.n + gcol;
            if ((m.n & 7) == 0 && gcol + 32 <= m.n) {
#pragma unroll
              for (int q = 0; q < 32; q += 8) {
                uint32_t w[4];
#pragma unroll
                for (int h = 0; h < 4; ++h)
                  w[h] = out_bits(v[q + 2 * h] * scale, p.out_dt) | ((uint32_t)out_bits(v[q + 2 * h + 1] * scale, p.out_dt) << 16);
                *reinterpret_cast<uint4*>(o + q) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (gcol + q < m.n) o[q] = out_bits(v[q] * scale, p.out_dt);
            }
          }
        }
      }
    }
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem, kTile);
  }
}

// ---- plan --------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}
int32_t encode_arena(CUtensorMap* map, void* arena, long long rows, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) HE_FAIL(HE_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[3] = {kBlockCols, (cuuint64_t)rows, 1};
  const cuuint64_t strides[2] = {128, (cuuint64_t)rows * 128};
  const cuuint32_t box[3] = {kBlockCols, (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, arena, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) HE_FAIL(HE_ERR_CUDA, "cuTensorMapEncodeTiled (muon workspace) failed with CUresult %d", (int)r);
  return HE_OK;
}

struct MuonPlan : he_plan {
  struct Round {
    int first;                 // first matrix of the list
    MuonTable table;           // pointers are filled in at launch
    int sum_ctas, sym_ctas, x_ctas, pack_ctas;
    size_t off_parts, off_diag, off_arena;
    long long arena_rows;
  };
  std::vector<Round> rounds;
  int count = 0, steps = 5;
  MuonStep st{};
  unsigned wait_limit_us = ptx::kDefaultWaitLimitUs;
  int withhold = 0;
  int32_t set_fault_injection(uint32_t limit, int32_t w) override {
    wait_limit_us = limit ? limit : ptx::kDefaultWaitLimitUs;
    withhold = w;
    return HE_OK;
  }
  int32_t launch(const void* const* in, void* const* out, void* ws, cudaStream_t stream) override;
  int32_t check_overlap(const void* const* in, void* const* out) const;
};

// No output may share memory with another operand, but for an average that is updated in place.
int32_t MuonPlan::check_overlap(const void* const* in, void* const* out) const {
  struct Span {
    uintptr_t lo, hi;
    bool written;
  };
  std::vector<Span> v;
  v.reserve(4 * count);
  for (const Round& r : rounds)
    for (int i = 0; i < r.table.count; ++i) {
      const int k = r.first + i;
      const uintptr_t n = (uintptr_t)r.table.mat[i].m * r.table.mat[i].n;
      auto add = [&](const void* p, uintptr_t bytes, bool w) { v.push_back({(uintptr_t)p, (uintptr_t)p + bytes, w}); };
      add(in[k], n * dtype_bytes(st.grad_dt), false);
      add(out[k], n * dtype_bytes(st.out_dt), true);
      if (st.has_momentum) {
        add(out[count + k], n * 4, true);
        if (in[count + k] != out[count + k]) add(in[count + k], n * 4, false);
      }
    }
  std::sort(v.begin(), v.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t read_end = 0, write_end = 0;   // ends of what starts at or before the current span
  for (const Span& s : v) {
    if (s.lo < write_end || (s.written && s.lo < read_end)) HE_FAIL(HE_ERR_INVALID, "muon: an output overlaps another operand");
    (s.written ? write_end : read_end) = std::max(s.written ? write_end : read_end, s.hi);
  }
  return HE_OK;
}

template <int PH> int32_t launch_gemm(const CUtensorMap& m128, const CUtensorMap& m64, const GemmArgs& a, int ctas, cudaStream_t stream) {
  static bool configured = false;   // benign race: the attribute call is idempotent
  if (!configured) {
    HE_CUDA(cudaFuncSetAttribute(muon_gemm_kernel<PH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem));
    configured = true;
  }
  muon_gemm_kernel<PH><<<ctas, kGemmThreads, kGemmSmem, stream>>>(m128, m64, a);
  HE_CUDA(cudaGetLastError());
  return HE_OK;
}

int32_t MuonPlan::launch(const void* const* in, void* const* out, void* ws, cudaStream_t stream) try {
  if (!in || !out) HE_FAIL(HE_ERR_INVALID, "muon: null operand list");
  const int per = st.has_momentum ? 2 : 1;
  for (int i = 0; i < per * count; ++i) {
    if (!in[i] || !out[i]) HE_FAIL(HE_ERR_INVALID, "muon: operand %d is null", i);
    if (((uintptr_t)in[i] | (uintptr_t)out[i]) & 15) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: tensors must be 16-byte aligned");
  }
  HE_TRY(check_overlap(in, out));
  for (const Round& r : rounds) {
    MuonTable t = r.table;   // a copy: the plan is not changed by a launch
    for (int i = 0; i < t.count; ++i) {
      MuonMat& m = t.mat[i];
      const int k = r.first + i;
      m.g = in[k];
      m.out = out[k];
      m.avg = st.has_momentum ? (const float*)in[count + k] : nullptr;
      m.avg_out = st.has_momentum ? (float*)out[count + k] : nullptr;
    }
    uint8_t* w = (uint8_t*)ws;
    MuonTable* table = (MuonTable*)w;
    double* parts = (double*)(w + r.off_parts);
    uint8_t* arena = w + r.off_arena;
    CUtensorMap m128, m64;
    HE_TRY(encode_arena(&m128, arena, r.arena_rows, 128));
    HE_TRY(encode_arena(&m64, arena, r.arena_rows, 64));
    muon_average_kernel<<<r.sum_ctas, kSumThreads, 0, stream>>>(t, st, table, parts);
    HE_CUDA(cudaGetLastError());
    muon_pack_kernel<<<r.pack_ctas, 256, 0, stream>>>(table, st, parts, arena);
    HE_CUDA(cudaGetLastError());
    GemmArgs a{};
    a.table = table; a.arena = arena; a.diag = (float*)(w + r.off_diag);
    a.status = ctx->d_status; a.wait_limit_us = wait_limit_us; a.withhold_loads = withhold;
    a.a = st.a; a.b = st.b; a.c = st.c; a.out_dt = st.out_dt;
    for (int s = 0; s < steps; ++s) {
      a.cur = s & 1;
      a.last = s == steps - 1;
      HE_TRY(launch_gemm<PH_S>(m128, m64, a, r.sym_ctas, stream));
      HE_TRY(launch_gemm<PH_B>(m128, m64, a, r.sym_ctas, stream));
      HE_TRY(launch_gemm<PH_X>(m128, m64, a, r.x_ctas, stream));
    }
    last_launches += 2 + 3 * steps;
  }
  return HE_OK;
} catch (const std::exception& e) {
  HE_FAIL(HE_ERR_INVALID, "muon: %s", e.what());
}

int32_t plan_muon(he_ctx* ctx, const he_muon_params* prm, he_plan** out) {
  if (!prm || !out) HE_FAIL(HE_ERR_INVALID, "muon: null argument");
  *out = nullptr;
  if (prm->count <= 0 || !prm->rows || !prm->cols) HE_FAIL(HE_ERR_INVALID, "muon: no matrices");
  if (prm->count > 4096) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: more than 4096 matrices in one plan");
  if (prm->grad_dtype != HE_F16 && prm->grad_dtype != HE_BF16 && prm->grad_dtype != HE_F32)
    HE_FAIL(HE_ERR_UNSUPPORTED, "muon: gradients must be f16, bf16 or f32");
  if (prm->out_dtype != HE_F16 && prm->out_dtype != HE_BF16) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: updates are f16 or bf16");
  if (prm->steps < 1 || prm->steps > 64) HE_FAIL(HE_ERR_INVALID, "muon: %d steps (1 to 64)", prm->steps);
  for (int i = 0; i < 3; ++i)
    if (!std::isfinite(prm->coef[i])) HE_FAIL(HE_ERR_INVALID, "muon: coefficients must be finite");
  if (!(prm->eps >= 0.0f) || !std::isfinite(prm->eps)) HE_FAIL(HE_ERR_INVALID, "muon: eps must be finite and not negative");
  if (!(prm->momentum >= 0.0f && prm->momentum < 1.0f)) HE_FAIL(HE_ERR_INVALID, "muon: momentum must be in [0, 1)");
  std::unique_ptr<MuonPlan> plan(new MuonPlan);
  plan->ctx = ctx;
  plan->count = prm->count;
  plan->steps = prm->steps;
  MuonStep& st = plan->st;
  st.momentum = prm->momentum;
  st.rest = (float)(1.0 - (double)prm->momentum);
  st.has_momentum = prm->use_momentum != 0;
  st.nesterov = prm->nesterov != 0;
  st.grad_dt = prm->grad_dtype;
  st.out_dt = prm->out_dtype;
  st.a = prm->coef[0]; st.b = prm->coef[1]; st.c = prm->coef[2];
  st.eps = prm->eps;
  for (int first = 0; first < prm->count; first += kMaxMats) {
    MuonPlan::Round r{};
    r.first = first;
    r.table.count = std::min(kMaxMats, prm->count - first);
    long long rows = 0, diag = 0, sym = 0, xt = 0, pack = 0, parts = 0;
    for (int i = 0; i < r.table.count; ++i) {
      MuonMat& m = r.table.mat[i];
      const int64_t h = prm->rows[first + i], w = prm->cols[first + i];
      if (h <= 0 || w <= 0) HE_FAIL(HE_ERR_INVALID, "muon: matrix %d is empty", first + i);
      if (std::min(h, w) > 32768 || std::max(h, w) > (1 << 20)) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: matrix %d is larger than 32768 x 1048576", first + i);
      m.tall = h > w;
      m.m = (int)std::min(h, w);
      m.n = (int)std::max(h, w);
      m.mt = (m.m + 127) / 128;
      m.nt = (m.n + 127) / 128;
      m.out_scale = prm->scales ? prm->scales[first + i] : 1.0f;
      if (!std::isfinite(m.out_scale)) HE_FAIL(HE_ERR_INVALID, "muon: scale of matrix %d is not finite", first + i);
      const double side = std::sqrt((double)m.m * m.n);
      m.sx = (float)std::ldexp(1.0, std::min(15, (int)std::floor(std::log2(side))));
      const long long xrows = (long long)m.mt * 2 * m.nt * kBlockRows, srows = (long long)m.mt * 2 * m.mt * kBlockRows;
      m.x[0] = rows; rows += xrows;
      m.x[1] = rows; rows += xrows;
      m.xlo = rows; rows += xrows;
      m.s = rows; rows += srows;
      m.b = rows; rows += srows;
      m.diag = diag; diag += (long long)m.mt * 128;
      m.sym0 = (int)sym; sym += (long long)m.mt * (m.mt + 1) / 2;
      m.x0 = (int)xt; xt += (long long)m.mt * m.nt;
      m.pack0 = (int)pack; pack += (long long)m.mt * 2 * 2 * m.nt;
      // partial sums: CTAs of at least 4096 elements, at most 512 of them
      const long long total = (long long)m.m * m.n;
      long long chunks = std::min<long long>(512, (total + 4095) / 4096);
      m.chunk = (total + chunks - 1) / chunks;
      m.chunk = (m.chunk + 3) / 4 * 4;
      m.chunks = (int)((total + m.chunk - 1) / m.chunk);
      m.part0 = (int)parts; parts += m.chunks;
      if (rows >= (1ll << 31) || pack >= (1ll << 31)) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: the matrices of a plan exceed 2^31 workspace rows");
    }
    r.sum_ctas = (int)parts; r.sym_ctas = (int)sym; r.x_ctas = (int)xt; r.pack_ctas = (int)pack;
    r.arena_rows = rows;
    auto align = [](size_t v) { return (v + 1023) / 1024 * 1024; };
    r.off_parts = align(sizeof(MuonTable));
    r.off_diag = align(r.off_parts + (size_t)parts * sizeof(double));
    r.off_arena = align(r.off_diag + (size_t)diag * sizeof(float));
    plan->workspace_bytes = std::max(plan->workspace_bytes, r.off_arena + (size_t)rows * 128);
    plan->rounds.push_back(r);
  }
  char desc[256];
  snprintf(desc, sizeof desc, "muon: %d matri%s, %s gradients%s, %d Newton-Schulz steps on tcgen05 (f16 operands, hi + lo pair), %s updates", prm->count,
           prm->count == 1 ? "x" : "ces", dtype_name(st.grad_dt), st.has_momentum ? (st.nesterov ? ", Nesterov momentum" : ", momentum") : "",
           plan->steps, dtype_name(st.out_dt));
  plan->description = desc;
  *out = plan.release();
  return HE_OK;
}

}  // namespace
}  // namespace he

extern "C" int32_t he_plan_muon(he_ctx* ctx, const he_muon_params* params, he_plan** out) {
  try {
    return he::plan_muon(ctx, params, out);
  } catch (const std::exception& e) {
    HE_FAIL(HE_ERR_INVALID, "muon: %s", e.what());
  }
}
