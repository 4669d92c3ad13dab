// The Muon optimiser's update: the momentum average of a weight gradient, orthogonalised by Newton-Schulz products.
//
//   avg' = m avg + (1 - m) g                              (helium's exponential average, helium/src/optimizer/sgd.rs:47-62)
//   d    = m avg' + (1 - m) g  (Nesterov)  or  avg'       (no momentum: d = g)
//   X    = d / (|d|_F + eps), transposed where d has more rows than columns: m x n with m <= n
//   steps times:  S = X X^T,  B = b S + c S^2,  X <- a X + B X
//   update = scale X
// so every singular value v of d / |d| is mapped by a v + b v^3 + c v^5 once per step.  helium builds optimisers from
// pointwise ops and matmuls (helium/src/optimizer); the products here are three tcgen05 GEMMs a step over the whole list of
// matrices, of which the symmetric ones (S and S^2) compute the tiles on and below the diagonal only.
//
// Numbers.  The operands are f16, each matrix scaled by a power of two: X by sx ~ sqrt(m n), which makes its
// root-mean-square 1 at the start and keeps |X| below 65504 (|X| <= 1.3 sx with the usual coefficients; others are checked
// when a call is planned), S by 2^12, B by 2^10.  X itself is kept as a pair hi + lo of f16 (22 bits): the products read
// hi, the term a X adds the pair, so the rounding of hi is not multiplied by a = 3.4 step after step, and B's diagonal, by
// far its largest values, stays f32 and is applied to the pair too.
// Measured against 64 bits (the update's own rounding taken out), an update of five steps is 3e-4 .. 1.1e-3 off (relative, 2-norm)
// where m >= 64 (64 x 576 6.8e-4, 512 x 2304 6.4e-4, 4096 x 4096 6.0e-4), up to 2e-3 from 16 rows and up to 3e-3 below, where few
// singular values average less; six steps are a third more.  A bf16 update's rounding alone is 1.7e-3.  In a simulation bf16 operands were 4e-3 .. 2e-2 off, f16 without the pair 2e-3 .. 5e-3.
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
#include "gemm_sm100_2cta.cuh"
#include "tensor_map.h"

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
  int mt, nt;                  // 128-row and 128-column blocks (even numbers of them where CTA pairs work)
  long long partial;           // first f32 of the split tiles of S (splits > 1)
  int part0, chunks;           // partial sums of squares
  int s0, b0, x0, pack0;       // first item of this matrix in a step's list, first piece of the packing grid
  int splits, split_blocks;    // S: slices of n, and 64-column blocks of one
  int arrive0;                 // first arrival counter of the tiles of S
  float sx, out_scale;
};
struct MuonTable {
  int count;
  int items_s, items_b, items; // of a step: the first phase, the first two, all three
  MuonMat mat[kMaxMats];
};
// Counters of a launch, zeroed by its first kernel; they only ever grow.
struct MuonSync {
  unsigned next;               // next item of the list
  unsigned pad[31];
  unsigned done[kMaxMats][4];  // tiles of S, B and X finished, by matrix, over all steps
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

// 4 elements from e on (e a multiple of 4, tensors start on 16 bytes); those at or behind `total` are not read
__device__ __forceinline__ void load_grad4(const void* g, int dt, long long e, long long total, float (&v)[4], bool read_only = true) {
  if (e + 4 <= total) {
    if (dt == HE_F32) {
      const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(g) + e);
      const float4 a = read_only ? __ldg(p) : *p;
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(g) + e));
      const uint32_t w[2] = {a.x, a.y};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[2 * i] = dt == HE_BF16 ? bf16_bits_to_f32(w[i] & 0xffffu) : f16_bits_to_f32(w[i] & 0xffffu);
        v[2 * i + 1] = dt == HE_BF16 ? bf16_bits_to_f32(w[i] >> 16) : f16_bits_to_f32(w[i] >> 16);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = e + i >= total ? 0.0f : dt == HE_F32 && !read_only ? reinterpret_cast<const float*>(g)[e + i] : load_grad(g, dt, e + i);
  }
}

// ---- first pass: the average, and partial sums of squares of the direction ------------------------------------------
// Squares are added in 64 bits: gradients as large as 1e30 and as small as 1e-25 keep their norm.
__global__ void __launch_bounds__(kSumThreads, 8) muon_average_kernel(const __grid_constant__ MuonTable t, const __grid_constant__ MuonStep st,
                                                                  MuonTable* __restrict__ table_out, double* __restrict__ parts,
                                                                  unsigned* __restrict__ sync, int sync_words) {
  if (blockIdx.x == 0) {   // the later kernels read the table from memory
    const uint32_t* src = reinterpret_cast<const uint32_t*>(&t);
    uint32_t* dst = reinterpret_cast<uint32_t*>(table_out);
    for (int i = threadIdx.x; i < (int)(sizeof(MuonTable) / 4); i += kSumThreads) dst[i] = src[i];
    for (int i = threadIdx.x; i < sync_words; i += kSumThreads) sync[i] = 0;
  }
  const int k = find_matrix(t.count, blockIdx.x, [&](int i) { return t.mat[i].part0; });
  const MuonMat& m = t.mat[k];
  const long long total = (long long)m.m * m.n;
  const long long e0 = (long long)(blockIdx.x - m.part0) * m.chunk, e1 = min(total, e0 + m.chunk);
  double sum = 0.0;
  constexpr int U = 2;     // vectors of 4 elements a thread keeps in flight (conv net's filters: 4 299 us; 1 and 2, 293 and 291 us, are within 1 %)
  for (long long e = e0 + threadIdx.x * 4; e < e1; e += U * kSumThreads * 4) {
    float g[U][4], av[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) load_grad4(m.g, st.grad_dt, e + u * kSumThreads * 4, e1, g[u]);
    if (st.has_momentum)
#pragma unroll
      for (int u = 0; u < U; ++u) load_grad4(m.avg, HE_F32, e + u * kSumThreads * 4, e1, av[u], false);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long at = e + u * kSumThreads * 4;
      if (st.has_momentum) {
#pragma unroll
        for (int i = 0; i < 4; ++i) av[u][i] = fmaf(st.momentum, av[u][i], st.rest * g[u][i]);
        if (at + 4 <= e1) *reinterpret_cast<float4*>(m.avg_out + at) = make_float4(av[u][0], av[u][1], av[u][2], av[u][3]);
        else
          for (int i = 0; i < 4 && at + i < e1; ++i) m.avg_out[at + i] = av[u][i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {      // what lies behind the end came as zeros
        const double d = st.has_momentum ? (at + i < e1 ? direction(st, g[u][i], av[u][i]) : 0.0f) : g[u][i];
        sum = fma(d, d, sum);
      }
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

// The factor sx / (|d| + eps) of the direction as two, `pre` a power of two: for |d| + eps below 1e-34 it leaves f32's range
// (denormal gradients, or a zero one with a tiny eps, which has to come out as zero).  pre d is at most 2^15 there.
__device__ __forceinline__ float direction_scale(double sum_of_squares, float sx, float eps, float& pre) {
  const double f = (double)sx / (sqrt(sum_of_squares) + (double)eps);
  const bool far = f > 0x1p96;
  pre = far ? 0x1p96f : 1.0f;
  return (float)(far ? f * 0x1p-96 : f);
}

// ---- second pass: the direction, scaled and split, into the blocks of the workspace; zeros behind its edges ----------
// A CTA fills one block of 128 rows x 64 columns.  Where the gradient's rows run along X's and are whole vectors a thread
// reads 8 columns and writes them; otherwise the block goes through shared memory, read along the gradient's own rows.
__device__ __forceinline__ void load_grad8(const void* g, int dt, long long e, float (&v)[8]) {   // e * size is a multiple of 16
  if (dt == HE_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(g) + e));
    const float4 b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(g) + e) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned short*>(g) + e));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = dt == HE_BF16 ? bf16_bits_to_f32(w[i] & 0xffffu) : f16_bits_to_f32(w[i] & 0xffffu);
      v[2 * i + 1] = dt == HE_BF16 ? bf16_bits_to_f32(w[i] >> 16) : f16_bits_to_f32(w[i] >> 16);
    }
  }
}
// the direction at 8 elements from e on
__device__ __forceinline__ void direction8(const MuonMat& m, const MuonStep& st, long long e, float (&v)[8]) {
  if (!st.has_momentum || st.nesterov) load_grad8(m.g, st.grad_dt, e, v);
  if (st.has_momentum) {
    const float4 a = *reinterpret_cast<const float4*>(m.avg_out + e), b = *reinterpret_cast<const float4*>(m.avg_out + e + 4);
    const float av[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = direction(st, v[i], av[i]);
  }
}
__device__ __forceinline__ float direction1(const MuonMat& m, const MuonStep& st, long long e) {
  if (!st.has_momentum) return load_grad(m.g, st.grad_dt, e);
  return direction(st, st.nesterov ? load_grad(m.g, st.grad_dt, e) : 0.0f, m.avg_out[e]);
}
constexpr int kPackPitch = 65;
__global__ void __launch_bounds__(256) muon_pack_kernel(const __grid_constant__ MuonTable t, const __grid_constant__ MuonStep st,
                                                        const double* __restrict__ parts, uint8_t* __restrict__ arena) {
  __shared__ float tile[kBlockRows * kPackPitch];
  __shared__ double sums[8];
  const int k = find_matrix(t.count, blockIdx.x, [&](int i) { return t.mat[i].pack0; });
  const MuonMat& m = t.mat[k];
  const int piece = blockIdx.x - m.pack0, cb = piece % (2 * m.nt), rb = piece / (2 * m.nt);
  const int r0 = rb * kBlockRows, c0 = cb * kBlockCols;
  // the norm, from the partial sums in a fixed order
  double s = 0.0;
  for (int i = threadIdx.x; i < m.chunks; i += 256) s += parts[m.part0 + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  const bool direct = !m.tall && (m.n & 7) == 0, across = m.tall && (m.m & 7) == 0;
  uint8_t* const hi_at = arena + (m.x[0] + x_block(m, rb, cb)) * 128;
  uint8_t* const lo_at = arena + (m.xlo + x_block(m, rb, cb)) * 128;
  if (!direct) {
    if (across) {
      for (int i = threadIdx.x; i < kBlockCols * 16; i += 256) {
        const int c = i >> 4, r = (i & 15) * 8;
        float v[8] = {};
        if (c0 + c < m.n && r0 + r < m.m) direction8(m, st, (long long)(c0 + c) * m.m + r0 + r, v);
#pragma unroll
        for (int q = 0; q < 8; ++q) tile[(r + q) * kPackPitch + c] = v[q];
      }
    } else {
      for (int i = threadIdx.x; i < kBlockRows * kBlockCols; i += 256) {
        const int r = m.tall ? i & 127 : i >> 6, c = m.tall ? i >> 7 : i & 63;
        float d = 0.0f;
        if (r0 + r < m.m && c0 + c < m.n)
          d = direction1(m, st, m.tall ? (long long)(c0 + c) * m.m + r0 + r : (long long)(r0 + r) * m.n + c0 + c);
        tile[r * kPackPitch + c] = d;
      }
    }
  }
  __syncthreads();
  s = ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
  float pre;
  const float scale = direction_scale(s, m.sx, st.eps, pre);
#pragma unroll
  for (int i = 0; i < kBlockRows * 8 / 256; ++i) {
    const int r = (threadIdx.x >> 3) + 32 * i, q = (threadIdx.x & 7) * 8;
    float v[8] = {};
    if (!direct) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = tile[r * kPackPitch + q + j];
    } else if (r0 + r < m.m && c0 + q < m.n) {
      direction8(m, st, (long long)(r0 + r) * m.n + c0 + q, v);
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_pair(v[2 * j] * pre * scale, v[2 * j + 1] * pre * scale, hi[j], lo[j]);
    *reinterpret_cast<uint4*>(hi_at + r * 128 + q * 2) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(lo_at + r * 128 + q * 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// ---- the products -----------------------------------------------------------------------------------------------
// One kernel for all steps.  The work is one list of items -- for every step the tiles of S, then of B, then of the new X,
// each over all matrices -- and CTAs (or CTA pairs) take the next item from a counter.  An item waits for the counters of
// its own matrix (S: the X of the step before is whole; B: S is; X: B is), which only items earlier in the list raise, and
// those are in the hands of CTAs that run already: whatever the order and number of the CTAs, every wait ends.  A matrix's
// phases follow one another without a launch or a grid-wide barrier between them, and other matrices fill the gaps.
// The long sum of S (n columns, few tiles) is split into slices whose f32 tiles the last slice to arrive adds up, in the
// order of the slices: results do not depend on who it was.
//
// PAIR = false: one CTA, 128 x 128 tiles.  PAIR = true: a cluster of two CTAs on 256 x 256 tiles (cta_group::2), each with
// 128 rows and half of the column operand: half the bytes from L2 for the same products, which is what bounds 128 x 128
// tiles (350 ns for the 32 KB of a 64-deep block, 13.5 TB/s over the chip, where the products take 140 ns).
//
// Warps: 0 items and loads, 1 products, 2 and 3 stores, 4 .. 19 epilogue: four teams of four warps, each on 32 of every 128
// columns.  Behind a tile's operands the same ring hands the epilogue one stage for every 64 columns: TMA brings what it
// reads there (S, or X's two halves), the results replace it in place and TMA takes them out, the mirrored tile of a
// symmetric product too.
// What follows a store (its completion, the count) is the store warps' business: an epilogue that waited for them itself took
// 5.8 us a tile of the conv net's X, whose products take 3.8.
// (A thread owns a row.  Its own 32-byte loads and stores touch a line of its own each: 6 us a 128 x 128 tile with both, 3.2 us
// with TMA loads and the stores as they were.)
enum Phase { PH_S = 0, PH_B = 1, PH_X = 2 };
constexpr int kTile = 128, kKBlock = 64;
constexpr int kStages = 6;
constexpr int kOperandBytes = kTile * kKBlock * 2;          // 16 KB
constexpr int kEpiThreads = 512;
constexpr int kGemmThreads = 128 + kEpiThreads;
constexpr int kSlots = 4;                                   // items in flight in a CTA

struct Item {
  int phase, mat, i, j, k0, k_blocks, split, step;
};
struct IterShared {
  MuonTable table;
  Item item[kSlots];
  uint64_t full[kStages], empty[kStages], item_full[kSlots], item_empty[kSlots], acc_full[2], acc_empty[2], epi_full[kSlots][4], written[kSlots][4], drain;
  uint32_t tmem;
  int abort_flag;
  int last_split;
  int unfinished[kSlots][2];   // the item's tile waits for other slices; for either store warp
};
constexpr int kOffShared = kStages * 2 * kOperandBytes;
constexpr int kIterSmem = kOffShared + (int)sizeof(IterShared) + 1024;
static_assert(kIterSmem <= 232448, "shared memory budget of sm_100 exceeded");

struct IterArgs {
  const MuonTable* table;
  MuonSync* sync;
  unsigned* arrive;  // a counter for every tile of S and CTA of its pair
  uint8_t* arena;
  float* diag;
  float* partial;
  DeviceStatus* status;
  unsigned wait_limit_us;
  int withhold_loads;
  int steps;
  float a, b, c;
  int out_dt;
};

// 16 columns of row r (c0 a multiple of 16) of a 128 x 64 block in shared memory, 128-byte swizzle
__device__ __forceinline__ void load_block_row(const uint8_t* block, int r, int c0, uint32_t (&w)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 v = *reinterpret_cast<const uint4*>(block + r * 128 + ((((c0 >> 3) + h) ^ (r & 7)) << 4));
    w[4 * h] = v.x; w[4 * h + 1] = v.y; w[4 * h + 2] = v.z; w[4 * h + 3] = v.w;
  }
}
__device__ __forceinline__ void store_block_row(uint8_t* block, int r, int c0, const uint32_t (&w)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    *reinterpret_cast<uint4*>(block + r * 128 + ((((c0 >> 3) + h) ^ (r & 7)) << 4)) = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ unsigned short out_bits(float v, int dt) {
  return (unsigned short)(dt == HE_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v));
}
__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// orders what was acquired before it against this thread's TMA loads
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }

// Waits until *p >= want.  Bounded like every wait here.
__device__ __forceinline__ bool wait_count(const unsigned* p, unsigned want, volatile int* abort_flag, DeviceStatus* status, uint32_t limit_us) {
  if (load_acquire(p) >= want) return true;
  const uint64_t t0 = ptx::globaltimer_ns();
  while (load_acquire(p) < want) {
    if (*abort_flag) return false;
    if (ptx::globaltimer_ns() - t0 > (uint64_t)limit_us * 1000ull) {
      *abort_flag = 1;
      if (status && atomicCAS(&status->code, 0u, (9u << 16) | (want & 0xffffu)) == 0u) { status->block = blockIdx.x; status->aux0 = want; }
      return false;
    }
  }
  return true;
}

// Named barrier of `threads` threads that tells each of them whether all of them said yes.
__device__ __forceinline__ bool barrier_all(uint32_t id, uint32_t threads, bool yes) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)yes)
      : "memory");
  return r != 0;
}

template <bool PAIR> __device__ __forceinline__ Item decode_item(const MuonTable& t, unsigned id, int steps) {
  Item w;
  w.step = (int)(id / (unsigned)t.items);
  if (w.step >= steps) { w.phase = -1; return w; }
  const int r = (int)(id - (unsigned)w.step * (unsigned)t.items);
  w.phase = r < t.items_s ? PH_S : r < t.items_b ? PH_B : PH_X;
  const int phase = w.phase;
  w.mat = find_matrix(t.count, r, [&](int q) { return phase == PH_S ? t.mat[q].s0 : phase == PH_B ? t.mat[q].b0 : t.mat[q].x0; });
  const MuonMat& m = t.mat[w.mat];
  w.split = 0;
  w.k0 = 0;
  w.k_blocks = (m.m + kKBlock - 1) / kKBlock;
  if (phase == PH_X) {
    const int q = r - m.x0, ti = PAIR ? m.mt >> 1 : m.mt;
    w.j = q / ti;        // neighbours in the list share X's columns
    w.i = q - w.j * ti;
    return w;
  }
  int q = r - (phase == PH_S ? m.s0 : m.b0);
  if (phase == PH_S) {
    w.k_blocks = (m.n + kKBlock - 1) / kKBlock;
    if (m.splits > 1) {
      w.split = q % m.splits;
      q /= m.splits;
      w.k0 = w.split * m.split_blocks;
      w.k_blocks = min(m.split_blocks, w.k_blocks - w.k0);
    }
  }
  w.i = (int)((sqrtf(8.0f * q + 1.0f) - 1.0f) * 0.5f);
  while ((w.i + 1) * (w.i + 2) / 2 <= q) ++w.i;
  while (w.i * (w.i + 1) / 2 > q) --w.i;
  w.j = q - w.i * (w.i + 1) / 2;
  return w;
}

// 128 rows x 64 columns of the finished update from shared memory (128-byte swizzle) by 256 threads, lanes along the rows.
__device__ __forceinline__ void copy_update(const MuonMat& m, const uint8_t* block, int row0, int col0, int tid) {
  unsigned short* out = reinterpret_cast<unsigned short*>(m.out);
  if ((m.n & 7) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (tid >> 3) + 32 * i, q = tid & 7;
      if (row0 + r < m.m && col0 + 8 * q < m.n)
        *reinterpret_cast<uint4*>(out + (long long)(row0 + r) * m.n + col0 + 8 * q) = *reinterpret_cast<const uint4*>(block + r * 128 + ((q ^ (r & 7)) << 4));
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < 32; ++i) {
      const int r = (tid >> 6) + 4 * i, c = tid & 63;
      if (row0 + r < m.m && col0 + c < m.n)
        out[(long long)(row0 + r) * m.n + col0 + c] = *reinterpret_cast<const unsigned short*>(block + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
    }
  }
}

// TMA store of a box of the arena from this CTA's shared memory
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int row) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row),
               "r"(0), "r"(src)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }   // the source may be reused
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }             // the writes are made

// store to the same place of CTA `rank`'s shared memory
__device__ __forceinline__ void store_peer(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void arrive_peer_release(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void fence_cluster_acquire() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }

template <bool PAIR>
__global__ void __launch_bounds__(kGemmThreads, 1) muon_iterate_kernel(const __grid_constant__ CUtensorMap map128,
                                                                       const __grid_constant__ CUtensorMap map64,
                                                                       const __grid_constant__ IterArgs p) {
  constexpr int kN = PAIR ? 256 : 128;        // columns of a tile
  constexpr int kGroups = kN / 64;
  constexpr int kCtas = PAIR ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  IterShared& sh = *reinterpret_cast<IterShared*>(smem + kOffShared);
  const uint32_t base = ptx::smem_u32(smem);
  auto bar = [](uint64_t& b) { return ptx::smem_u32(&b); };
  volatile int* abort_flag = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? ptx::cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  // a barrier of the leader, seen from either CTA
  auto lead = [&](uint64_t& b) { return PAIR ? ptx::mapa(bar(b), 0) : bar(b); };
  auto arrive_lead = [&](uint64_t& b) {
    if (PAIR) ptx::mbar_arrive_cluster(ptx::mapa(bar(b), 0));
    else ptx::mbar_arrive(bar(b));
  };

  if (threadIdx.x == 0) {
    sh.abort_flag = 0;
    for (int s = 0; s < kStages; ++s) { ptx::mbar_init(bar(sh.full[s]), 1); ptx::mbar_init(bar(sh.empty[s]), 1); }
    for (int s = 0; s < kSlots; ++s) { ptx::mbar_init(bar(sh.item_full[s]), 1); ptx::mbar_init(bar(sh.item_empty[s]), kCtas * (kEpiThreads / 32 + 2)); }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(bar(sh.acc_full[s]), 1);
      ptx::mbar_init(bar(sh.acc_empty[s]), kCtas * (kEpiThreads / 32));
    }
    for (int s = 0; s < kSlots * 4; ++s) { ptx::mbar_init(bar(sh.epi_full[s >> 2][s & 3]), 1); ptx::mbar_init(bar(sh.written[s >> 2][s & 3]), 8); }
    ptx::mbar_init(bar(sh.drain), 1);
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    if (PAIR) {
      ptx::tmem_alloc_2cta(ptx::smem_u32(&sh.tmem), 2 * kN);
      ptx::tmem_relinquish_2cta();
    } else {
      ptx::tmem_alloc(ptx::smem_u32(&sh.tmem), 2 * kN);
      ptx::tmem_relinquish();
    }
  }
  {
    const uint32_t* src = reinterpret_cast<const uint32_t*>(p.table);
    uint32_t* dst = reinterpret_cast<uint32_t*>(&sh.table);
    const int words = (int)((sizeof(MuonTable) - sizeof(MuonMat) * (kMaxMats - p.table->count)) / 4);
    for (int i = threadIdx.x; i < words; i += kGemmThreads) dst[i] = src[i];
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (PAIR) ptx::cluster_sync();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);
  const MuonTable& t = sh.table;

  if (warp == 0) {
    // ===================== items and operand loads =====================
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      unsigned filled = 0, any = 0;                  // operand fills of each stage: parity, and whether there were any
      unsigned epi_filled = 0, epi_any = 0;          // the same of each epilogue barrier
      const uint32_t full0 = bar(sh.full[0]), empty0 = bar(sh.empty[0]);
      auto bar_full = [&](int s) { return full0 + 8u * s; };
      auto bar_empty = [&](int s) { return empty0 + 8u * s; };
      DeviceStatus* const status = p.status;
      const uint32_t wait_us = p.wait_limit_us;
      bool alive = true;
      for (int n = 0; alive; ++n) {
        const int slot = n % kSlots;
        Item w;
        if (leader) {
          // taken when the loads of the one before are out, no earlier: a CTA that waits must not sit on a second item
          w = decode_item<PAIR>(t, atomicAdd(&p.sync->next, 1u), p.steps);
          if (!ptx::mbar_wait(bar(sh.item_empty[slot]), ((uint32_t)(n / kSlots) & 1u) ^ 1u, abort_flag, p.status, 1, slot, p.wait_limit_us)) { alive = false; break; }
          if (w.phase >= 0) {
            const MuonMat& m = t.mat[w.mat];
            const unsigned* done = p.sync->done[w.mat];
            const unsigned ti = (unsigned)(PAIR ? m.mt >> 1 : m.mt), tj = (unsigned)(PAIR ? m.nt >> 1 : m.nt), sym = ti * (ti + 1) / 2 * (2 * kCtas);   // two store warps a CTA
            if (w.phase == PH_S) alive = wait_count(done + PH_X, (unsigned)w.step * ti * tj * (2 * kCtas), abort_flag, p.status, p.wait_limit_us);
            else alive = wait_count(done + (w.phase == PH_B ? PH_S : PH_B), (unsigned)(w.step + 1) * sym, abort_flag, p.status, p.wait_limit_us);
            if (!alive) break;
          }
          sh.item[slot] = w;
          if (PAIR) {
            const uint32_t peer = ptx::mapa(ptx::smem_u32(&sh.item[slot]), 1);
            const uint32_t* words = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
            for (int i = 0; i < (int)(sizeof(Item) / 4); ++i) store_peer(peer + 4 * i, words[i]);
            arrive_peer_release(ptx::mapa(bar(sh.item_full[slot]), 1));
          }
          ptx::mbar_arrive(bar(sh.item_full[slot]));
        } else {
          if (!ptx::mbar_wait(bar(sh.item_full[slot]), (uint32_t)(n / kSlots) & 1u, abort_flag, p.status, 3, slot, 2 * p.wait_limit_us)) { alive = false; break; }
          fence_cluster_acquire();
          w = sh.item[slot];
        }
        if (w.phase < 0) break;
        fence_proxy_async_all();
        if (p.withhold_loads) continue;
        const MuonMat& m = t.mat[w.mat];
        const bool same = w.phase != PH_X && w.i == w.j;   // both operands are one block row: loaded once
        const int ri = PAIR ? 2 * w.i + (int)rank : w.i, rj = PAIR ? 2 * w.j + (int)rank : w.j;
        const int xcur = (int)m.x[w.step & 1], x_pitch = 2 * m.nt * kBlockRows, s_pitch = 2 * m.mt * kBlockRows;
        // Rows of the arena that the next block of each operand starts at.  One thread paces the ring: what it computes for
        // a block is two additions (with the addresses worked out from the tile each time a block took 350 ns).
        int row_a = (w.phase == PH_S ? xcur + ri * x_pitch : (w.phase == PH_B ? (int)m.s : (int)m.b) + ri * s_pitch) + w.k0 * kBlockRows;
        int row_b = w.phase == PH_S ? xcur + rj * x_pitch + w.k0 * kBlockRows : w.phase == PH_B ? (int)m.s + rj * s_pitch : xcur + 2 * rj * kBlockRows;
        const uint32_t bytes = (same ? 1 : 2) * kCtas * kOperandBytes;
        auto fill = [&](auto load_b) {
          for (int kb = 0; kb < w.k_blocks; ++kb) {
            if (!ptx::mbar_wait(bar_empty(stage), phase ^ 1u, abort_flag, status, 2, stage, wait_us)) { alive = false; break; }
            const uint32_t a_dst = base + stage * 2 * kOperandBytes, fb = PAIR ? ptx::mapa(bar_full(stage), 0) : bar_full(stage);
            if (leader) ptx::mbar_arrive_expect_tx(bar_full(stage), bytes);
            filled ^= 1u << stage;
            any |= 1u << stage;
            if (PAIR) ptx::tma_load_3d_2cta(a_dst, &map128, fb, 0, row_a, 0);
            else ptx::tma_load_3d(a_dst, &map128, fb, 0, row_a, 0);
            load_b(a_dst + kOperandBytes, fb, kb);
            row_a += kBlockRows;
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
          }
        };
        if (w.phase == PH_X) {
          fill([&](uint32_t dst, uint32_t fb, int kb) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (PAIR) ptx::tma_load_3d_2cta(dst + h * (kOperandBytes / 2), &map64, fb, 0, row_b + h * kBlockRows, 0);
              else ptx::tma_load_3d(dst + h * (kOperandBytes / 2), &map64, fb, 0, row_b + h * kBlockRows, 0);
            }
            row_b += kb & 1 ? x_pitch - 64 : 64;    // X's rows, 64 at a time
          });
        } else {
          fill([&](uint32_t dst, uint32_t fb, int) {
            if (!same) {
              if (PAIR) ptx::tma_load_3d_2cta(dst, &map128, fb, 0, row_b, 0);
              else ptx::tma_load_3d(dst, &map128, fb, 0, row_b, 0);
            }
            row_b += kBlockRows;
          });
        }
        if (!alive) break;
        // the epilogue's stages, each CTA its own rows (S: room only)
        int row = (w.phase == PH_X ? xcur + ri * x_pitch : (int)m.s + ri * s_pitch) + kGroups * w.j * kBlockRows;
        const int lo = (int)m.xlo - xcur;
        for (int g = 0; g < kGroups; ++g, row += kBlockRows) {
          if (!ptx::mbar_wait(bar_empty(stage), phase ^ 1u, abort_flag, status, 2, stage, wait_us)) { alive = false; break; }
          const uint32_t dst = base + stage * 2 * kOperandBytes, eb = bar(sh.epi_full[slot][g]);
          if (w.phase == PH_S) {
            ptx::mbar_arrive(eb);
          } else {
            ptx::mbar_arrive_expect_tx(eb, (w.phase == PH_X ? 2 : 1) * kOperandBytes);
            ptx::tma_load_3d(dst, &map128, eb, 0, row, 0);
            if (w.phase == PH_X) ptx::tma_load_3d(dst + kOperandBytes, &map128, eb, 0, row + lo, 0);
          }
          epi_filled ^= 1u << (4 * slot + g);
          epi_any |= 1u << (4 * slot + g);
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // an item that was given up: the copies in flight still land in this CTA's memory (the operands' count is the leader's)
      if (!alive) {
        int never = 0;
        if (leader)
          for (int s = 0; s < kStages; ++s)
            if (any >> s & 1u) ptx::mbar_wait(bar(sh.full[s]), (filled >> s & 1u) ^ 1u, &never, p.status, 7, s, p.wait_limit_us);
        for (int k = 0; k < kSlots * 4; ++k)
          if (epi_any >> k & 1u) ptx::mbar_wait(bar(sh.epi_full[k >> 2][k & 3]), (epi_filled >> k & 1u) ^ 1u, &never, p.status, 11, k, p.wait_limit_us);
      }
    }
  } else if (warp == 1) {
    // ===================== products =====================
    if (lane == 0 && leader) {
      int stage = 0;
      unsigned full_parity = 0;      // bit s: parity of the next operand fill of stage s (tiles of the epilogue fill others)
      const uint32_t full0 = bar(sh.full[0]), empty0 = bar(sh.empty[0]), empty1 = PAIR ? ptx::mapa(empty0, 1) : 0u;
      DeviceStatus* const status = p.status;
      const uint32_t wait_us = p.wait_limit_us;
      const uint64_t a_desc0 = ptx::make_smem_desc_sw128(base, 16, 1024);
      bool alive = true;
      for (int n = 0; alive; ++n) {
        const int slot = n % kSlots, acc = n & 1;
        if (!ptx::mbar_wait(bar(sh.item_full[slot]), (uint32_t)(n / kSlots) & 1u, abort_flag, status, 3, slot, 2 * wait_us)) { alive = false; break; }
        const int phase = sh.item[slot].phase, k_blocks = sh.item[slot].k_blocks;
        if (phase < 0) break;
        const bool same = phase != PH_X && sh.item[slot].i == sh.item[slot].j;
        if (!ptx::mbar_wait(bar(sh.acc_empty[acc]), ((uint32_t)(n >> 1) & 1u) ^ 1u, abort_flag, status, 4, acc, wait_us)) { alive = false; break; }
        ptx::tcgen05_fence_after();
        const bool b_mn = phase == PH_X;
        const uint32_t idesc = ptx::make_idesc_f16(0, 0, b_mn ? 1 : 0, kCtas * kTile, kN);
        // descriptors of stage 0; a stage, and 16 values of k within it, are additions to the address field
        const uint64_t b_desc0 = ptx::make_smem_desc_sw128(base + (same ? 0 : kOperandBytes), b_mn ? kOperandBytes / 2 : 16, 1024);
        const uint32_t b_step = b_mn ? 2048 >> 4 : 32 >> 4;
        const uint32_t d = tmem + (uint32_t)(acc * kN);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!ptx::mbar_wait(full0 + 8u * stage, full_parity >> stage & 1u, abort_flag, status, 5, stage, wait_us)) { alive = false; break; }
          full_parity ^= 1u << stage;
          ptx::tcgen05_fence_after();
          const uint64_t ad = a_desc0 + (uint32_t)(stage * (2 * kOperandBytes >> 4)), bd = b_desc0 + (uint32_t)(stage * (2 * kOperandBytes >> 4));
#pragma unroll
          for (int k = 0; k < kKBlock / 16; ++k) {
            if (PAIR) ptx::umma_f16_2cta(d, ad + 2 * k, bd + b_step * k, idesc, (kb | k) != 0 ? 1u : 0u);
            else ptx::umma_f16(d, ad + 2 * k, bd + b_step * k, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          if (PAIR) {
            ptx::umma_commit_2cta(empty0 + 8u * stage);
            ptx::umma_commit_2cta(empty1 + 8u * stage);
          } else {
            ptx::umma_commit(empty0 + 8u * stage);
          }
          if (++stage == kStages) stage = 0;
        }
        stage = (stage + kGroups) % kStages;   // the epilogue's
        if (alive) {
          if (PAIR) {
            ptx::umma_commit_2cta(bar(sh.acc_full[acc]));
            ptx::umma_commit_2cta(ptx::mapa(bar(sh.acc_full[acc]), 1));
          } else {
            ptx::umma_commit(bar(sh.acc_full[acc]));
          }
        }
      }
      if (!alive) {   // nothing may still write tensor memory when it is freed
        int never = 0;
        if (PAIR) ptx::umma_commit_2cta(bar(sh.drain));
        else ptx::umma_commit(bar(sh.drain));
        ptx::mbar_wait(bar(sh.drain), 0, &never, p.status, 8, 0, p.wait_limit_us);
      }
    }
  } else if (warp < 4) {
    // ===================== stores: warp 2 + buf, the 64-column blocks of its parity =====================
    if (lane == 0) {
      const int buf = warp - 2;
      int first_stage = 0;
      unsigned parity = 0;           // of the next use of each `written` barrier
      for (int n = 0;; ++n) {
        const int slot = n % kSlots;
        if (!ptx::mbar_wait(bar(sh.item_full[slot]), (uint32_t)(n / kSlots) & 1u, abort_flag, p.status, 3, slot, 2 * p.wait_limit_us)) break;
        if (PAIR) fence_cluster_acquire();
        const Item w = sh.item[slot];
        if (w.phase < 0) break;
        const MuonMat& m = t.mat[w.mat];
        const int ri = PAIR ? 2 * w.i + (int)rank : w.i, cb0 = kGroups * w.j;
        const bool mirror = w.phase != PH_X && w.i != w.j, direct = w.phase == PH_X && w.step == p.steps - 1;
        int out_row, lo_row = 0, mir_row = 0;    // rows of the arena: of the tile's first block, of its low half, of the mirrored tile
        if (w.phase == PH_X) {
          const int at = (int)x_block(m, ri, cb0);
          out_row = (int)m.x[(w.step & 1) ^ 1] + at;
          lo_row = (int)m.xlo + at;
        } else {
          const int into = (int)(w.phase == PH_S ? m.s : m.b);
          out_row = into + (int)s_block(m, ri, cb0);
          mir_row = into + (int)s_block(m, cb0 >> 1, 2 * ri);
        }
        const int mir_pitch = 2 * m.mt * kBlockRows;   // from one block row to the next
        bool alive = true, finish = true;
        for (int g = buf; g < kGroups; g += 2) {
          const int k = 4 * slot + g, stage = (first_stage + w.k_blocks + g) % kStages;
          if (!ptx::mbar_wait(bar(sh.written[slot][g]), parity >> k & 1u, abort_flag, p.status, 14, k, 2 * p.wait_limit_us)) { alive = false; break; }
          parity ^= 1u << k;
          finish = sh.unfinished[slot][buf] == 0;
          if (finish && !direct) {
            const uint32_t src = base + stage * 2 * kOperandBytes;
            tma_store_3d(&map128, src, out_row + g * kBlockRows);
            if (w.phase == PH_X) tma_store_3d(&map128, src + kOperandBytes, lo_row + g * kBlockRows);
            if (mirror) {
              const int row = mir_row + (g >> 1) * mir_pitch + (g & 1) * 64;
              tma_store_3d(&map64, src + kOperandBytes, row);
              tma_store_3d(&map64, src + kOperandBytes + kOperandBytes / 2, row + kBlockRows);
            }
            tma_store_commit();
            tma_store_wait_read();
          }
          ptx::mbar_arrive(bar(sh.empty[stage]));
        }
        tma_store_wait();
        if (!alive) break;
        if (finish) {   // this half of the tile is in memory: only then does the count say so
          __threadfence();
          atomicAdd(&p.sync->done[w.mat][w.phase], 1u);
        }
        first_stage = (first_stage + w.k_blocks + kGroups) % kStages;
        arrive_lead(sh.item_empty[slot]);
      }
    }
  } else {
    // ===================== epilogue: thread = row of the tile, team = 32 columns of every 128 =====================
    const int quadrant = warp & 3, team = (warp - 4) >> 2, buf = team >> 1, r = quadrant * 32 + lane;
    const int tid = threadIdx.x - 128;
    int first_stage = 0;           // of the item
    unsigned epi_parity = 0;       // of the next fill of each epilogue barrier
    for (int n = 0;; ++n) {
      const int slot = n % kSlots, acc = n & 1;
      // the warps go on or give up together: they share barriers below
      bool ok = ptx::mbar_wait(bar(sh.item_full[slot]), (uint32_t)(n / kSlots) & 1u, abort_flag, p.status, 3, slot, 2 * p.wait_limit_us);
      if (PAIR) fence_cluster_acquire();
      const Item w = sh.item[slot];
      // What depends on the item alone is worked out while its products run.
      const MuonMat& m = t.mat[ok && w.phase >= 0 ? w.mat : 0];
      const int ri = PAIR ? 2 * w.i + (int)rank : w.i;   // block row of this CTA
      const int grow = ri * kTile + r, cb0 = kGroups * w.j;
      const bool last = w.step == p.steps - 1;
      const bool split = w.phase == PH_S && m.splits > 1;
      const float s_scale = kScaleS / (m.sx * m.sx), o_scale = m.out_scale / m.sx;
      float dg = 0.0f;         // B's diagonal at this row
      const bool mirror = w.phase != PH_X && w.i != w.j;
      if (ok && w.phase == PH_X) dg = p.a + __ldcg(p.diag + m.diag + grow);
      float* part = nullptr;   // split tiles: slices side by side, each [column / 4][row][4]
      if (split) part = p.partial + m.partial + (size_t)((w.i * (w.i + 1) / 2 + w.j) * kCtas + (int)rank) * m.splits * (kTile * kN) + r * 4;
      if (ok && w.phase >= 0) ok = ptx::mbar_wait(bar(sh.acc_full[acc]), (uint32_t)(n >> 1) & 1u, abort_flag, p.status, 6, acc, p.wait_limit_us);
      if (!barrier_all(1, kEpiThreads, ok && w.phase >= 0)) break;
      ptx::tcgen05_fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(quadrant * 32) << 16) + (uint32_t)(acc * kN);
      auto release = [&]() {   // the accumulator
        ptx::tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) arrive_lead(sh.acc_empty[acc]);
      };
      bool finish = true;      // this CTA completes the tile
      if (split) {
        float* mine = part + (size_t)w.split * (kTile * kN);
#pragma unroll 1
        for (int c0 = team * 32; c0 < kN; c0 += 128) {
          uint32_t v[32];
          ptx::tmem_ld_32x32(taddr + (uint32_t)c0, v);
          ptx::tmem_ld_wait_regs(v);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<uint4*>(mine + (size_t)(c0 / 4 + q) * (4 * kTile)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
        release();
        ptx::named_barrier_sync(1, kEpiThreads);
        if (tid == 0) {
          __threadfence();
          const unsigned before = atomicAdd(p.arrive + m.arrive0 + (w.i * (w.i + 1) / 2 + w.j) * kCtas + (int)rank, 1u);
          sh.last_split = (before + 1) % (unsigned)m.splits == 0;
          __threadfence();
        }
        ptx::named_barrier_sync(1, kEpiThreads);
        finish = sh.last_split != 0;
      }
      if ((tid & 255) == 0) sh.unfinished[slot][buf] = finish ? 0 : 1;
      const int c0 = (team & 1) * 32;           // this team's columns of a 64-column block
#pragma unroll 1
      for (int g = buf; g < kGroups; g += 2) {
        const int stage = (first_stage + w.k_blocks + g) % kStages;
        uint8_t* const epi = smem + stage * 2 * kOperandBytes;    // in: S, or X's high half; out: the result's
        uint8_t* const epi2 = epi + kOperandBytes;                // in: X's low half; out: that of the result, or the mirrored tile
        uint32_t acc_v[32];
        if (!split) ptx::tmem_ld_32x32(taddr + (uint32_t)(g * 64 + c0), acc_v);
        {
          // (a wait that runs out leaves stale values behind, and the abort flag: the item loop ends at its next wait)
          const int k = 4 * slot + g;
          ptx::mbar_wait(bar(sh.epi_full[slot][g]), epi_parity >> k & 1u, abort_flag, p.status, 12, k, p.wait_limit_us);
          epi_parity ^= 1u << k;
          __syncwarp();
        }
        if (finish) {
          if (split) {
            const float* src = part + (size_t)((g * 64 + c0) / 4) * (4 * kTile);
#pragma unroll
            for (int q = 0; q < 32; ++q) acc_v[q] = 0u;
            for (int k = 0; k < m.splits; ++k, src += kTile * kN) {
              float4 u[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) u[q] = __ldcg(reinterpret_cast<const float4*>(src + q * (4 * kTile)));
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                acc_v[4 * q] = __float_as_uint(__uint_as_float(acc_v[4 * q]) + u[q].x);
                acc_v[4 * q + 1] = __float_as_uint(__uint_as_float(acc_v[4 * q + 1]) + u[q].y);
                acc_v[4 * q + 2] = __float_as_uint(__uint_as_float(acc_v[4 * q + 2]) + u[q].z);
                acc_v[4 * q + 3] = __float_as_uint(__uint_as_float(acc_v[4 * q + 3]) + u[q].w);
              }
            }
          } else {
            ptx::tmem_ld_wait_regs(acc_v);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int c = c0 + 16 * half;
            float v[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(acc_v[16 * half + q]);
            uint32_t w0[8], w1[8];
            if (w.phase != PH_X) {
              if (w.phase == PH_S) {
#pragma unroll
                for (int q = 0; q < 16; ++q) v[q] *= s_scale;
              } else {
                load_block_row(epi, r, c, w0);
                const float kb = p.b * (kScaleB / kScaleS), kc = p.c * (kScaleB / (kScaleS * kScaleS));
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                  const float2 s = unpack_half2(w0[q]);
                  v[2 * q] = fmaf(kc, v[2 * q], kb * s.x);
                  v[2 * q + 1] = fmaf(kc, v[2 * q + 1], kb * s.y);
                }
                const int dq = grow - ((cb0 + g) * 64 + c);
                if ((unsigned)dq < 16u) {   // the diagonal stays f32
                  float d = 0.0f;
#pragma unroll
                  for (int q = 0; q < 16; ++q) {
                    d = q == dq ? v[q] : d;
                    v[q] = q == dq ? 0.0f : v[q];
                  }
                  p.diag[m.diag + grow] = d * (1.0f / kScaleB);
                }
              }
#pragma unroll
              for (int q = 0; q < 8; ++q) w0[q] = pack_half2(v[2 * q], v[2 * q + 1]);
              store_block_row(epi, r, c, w0);
              if (mirror) {   // two pieces of 64 x 64, by the half of the rows; lanes are neighbouring columns of them
                uint8_t* const to = epi2 + (r >> 6) * (kOperandBytes / 2) + (r & 7) * 2;
                const int chunk = (r & 63) >> 3;
#pragma unroll
                for (int q = 0; q < 16; ++q)
                  *reinterpret_cast<unsigned short*>(to + (c + q) * 128 + ((chunk ^ (q & 7)) << 4)) = (unsigned short)(w0[q >> 1] >> (16 * (q & 1)));
              }
            } else {
              load_block_row(epi, r, c, w0);
              load_block_row(epi2, r, c, w1);
              const unsigned long long dg2 = ptx::f2_pack(dg, dg), one2 = ptx::f2_pack(1.0f, 1.0f), inv2 = ptx::f2_pack(1.0f / kScaleB, 1.0f / kScaleB);
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const float2 h = unpack_half2(w0[q]), l = unpack_half2(w1[q]);
                const unsigned long long x = ptx::f2_fma(ptx::f2_pack(h.x, h.y), one2, ptx::f2_pack(l.x, l.y));
                ptx::f2_unpack(ptx::f2_fma(dg2, x, ptx::f2_mul(ptx::f2_pack(v[2 * q], v[2 * q + 1]), inv2)), v[2 * q], v[2 * q + 1]);
              }
              if (!last) {
#pragma unroll
                for (int q = 0; q < 8; ++q) split_pair(v[2 * q], v[2 * q + 1], w0[q], w1[q]);
                store_block_row(epi, r, c, w0);
                store_block_row(epi2, r, c, w1);
              } else if (!m.tall) {
#pragma unroll
                for (int q = 0; q < 8; ++q) w0[q] = out_bits(v[2 * q] * o_scale, p.out_dt) | ((uint32_t)out_bits(v[2 * q + 1] * o_scale, p.out_dt) << 16);
                store_block_row(epi, r, c, w0);
              } else if (grow < m.m) {   // lanes are neighbouring columns of the tall update
                unsigned short* out = reinterpret_cast<unsigned short*>(m.out) + grow;
                const int gcol = (cb0 + g) * 64 + c;
#pragma unroll
                for (int q = 0; q < 16; ++q)
                  if (gcol + q < m.n) out[(long long)(gcol + q) * m.m] = (unsigned short)out_bits(v[q] * o_scale, p.out_dt);
              }
            }
          }
          ptx::fence_proxy_async_smem();
          if (w.phase == PH_X && last && !m.tall) {
            ptx::named_barrier_sync(2 + buf, kEpiThreads / 2);   // the block is whole
            copy_update(m, epi, ri * kTile, (cb0 + g) * 64, tid & 255);
          }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(sh.written[slot][g]));
      }
      if (!split) release();
      first_stage = (first_stage + w.k_blocks + kGroups) % kStages;
      __syncwarp();
      if (lane == 0) arrive_lead(sh.item_empty[slot]);
    }
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (PAIR) ptx::cluster_sync();   // the peer may still be signalling this CTA's barriers or reading its memory
  if (warp == 1) {
    ptx::tcgen05_fence_after();
    if (PAIR) ptx::tmem_dealloc_2cta(tmem, 2 * kN);
    else ptx::tmem_dealloc(tmem, 2 * kN);
  }
}

// ---- small matrices: one CTA each, everything on chip ------------------------------------------------------------
// Up to 128 x 320 the pair hi + lo of X (160 KB), S and B (32 KB each) stay in one SM's shared memory for the whole call:
// average, norm, all steps and the update in one launch, with block barriers where the list of tiles has counters in memory
// (5 us a phase there, 1.5 us here; a 64 x 288 filter takes 88 us by tiles).  The layout is the arena's: blocks of 128 rows x
// 64 columns, 128-byte swizzle.  16 warps: thread = row, a warp's team 32 columns (of S, B) or 16 (of each block of X).
constexpr int kSmallBlocks = 5, kSmallThreads = 512;
struct SmallShared {
  uint64_t done;
  uint32_t tmem;
  int abort_flag;
  float diag[128];
  double sums[kSmallThreads / 32];
};
constexpr int kOffSmallLo = kSmallBlocks * kOperandBytes, kOffSmallS = 2 * kOffSmallLo, kOffSmallB = kOffSmallS + 2 * kOperandBytes;
constexpr int kOffSmallShared = kOffSmallB + 2 * kOperandBytes;
constexpr int kSmallSmem = kOffSmallShared + (int)sizeof(SmallShared) + 1024;
static_assert(kSmallSmem <= 232448, "shared memory budget of sm_100 exceeded");
static_assert(128 * (64 * kSmallBlocks + 4) * 4 <= kOffSmallShared, "the f32 direction fits in front of the barriers");

struct SmallArgs {
  DeviceStatus* status;
  unsigned wait_limit_us;
  int withhold;
  int steps;
};

__global__ void __launch_bounds__(kSmallThreads, 1) muon_small_kernel(const __grid_constant__ MuonTable t, const __grid_constant__ MuonStep st,
                                                                      const __grid_constant__ SmallArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  SmallShared& sh = *reinterpret_cast<SmallShared*>(smem + kOffSmallShared);
  const uint32_t base = ptx::smem_u32(smem), bar = ptx::smem_u32(&sh.done);
  const MuonMat& m = t.mat[blockIdx.x];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quadrant = warp & 3, team = warp >> 2, r = quadrant * 32 + lane;
  const int blocks = (m.n + 63) / 64;
  if (tid == 0) {
    sh.abort_flag = 0;
    ptx::mbar_init(bar, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 0) {
    ptx::tmem_alloc(ptx::smem_u32(&sh.tmem), 512);
    ptx::tmem_relinquish();
  }
  // the average and the direction, as f32 [row][pitch] over the space of X, S and B
  float* const d32 = reinterpret_cast<float*>(smem);
  const int pitch = 64 * blocks + 4, total = m.m * m.n, inner = m.tall ? m.m : m.n;
  for (int i = tid; i < 128 * pitch / 4; i += kSmallThreads) reinterpret_cast<float4*>(d32)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __syncthreads();
  double sum = 0.0;
  constexpr int U = 5;     // vectors of 4 elements a thread keeps in flight: one at a time, loading took 10 us of 49
  for (int v0 = tid; v0 * 4 < total; v0 += U * kSmallThreads) {
    float g[U][4], av[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) load_grad4(m.g, st.grad_dt, 4ll * (v0 + u * kSmallThreads), total, g[u]);
    if (st.has_momentum)
#pragma unroll
      for (int u = 0; u < U; ++u) load_grad4(m.avg, HE_F32, 4ll * (v0 + u * kSmallThreads), total, av[u], false);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e0 = 4 * (v0 + u * kSmallThreads);
      int o = e0 / inner, i = e0 - o * inner;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (e0 + q < total) {
          float d = g[u][q];
          if (st.has_momentum) {
            av[u][q] = fmaf(st.momentum, av[u][q], st.rest * d);
            m.avg_out[e0 + q] = av[u][q];
            d = direction(st, d, av[u][q]);
          }
          d32[m.tall ? i * pitch + o : o * pitch + i] = d;
          sum = fma((double)d, (double)d, sum);
        }
        if (++i == inner) { i = 0; ++o; }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sh.sums[warp] = sum;
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);
  sum = 0.0;
  for (int i = 0; i < kSmallThreads / 32; ++i) sum += sh.sums[i];
  float pre;
  const float scale = direction_scale(sum, m.sx, st.eps, pre);
  // scaled and split into the blocks
  {
    float v[kSmallBlocks][16];
#pragma unroll
    for (int b = 0; b < kSmallBlocks; ++b)
      if (b < blocks)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 f = *reinterpret_cast<const float4*>(d32 + r * pitch + b * 64 + team * 16 + 4 * q);
          v[b][4 * q] = f.x; v[b][4 * q + 1] = f.y; v[b][4 * q + 2] = f.z; v[b][4 * q + 3] = f.w;
        }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < kSmallBlocks; ++b)
      if (b < blocks) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) split_pair(v[b][2 * q] * pre * scale, v[b][2 * q + 1] * pre * scale, hi[q], lo[q]);
        store_block_row(smem + b * kOperandBytes, r, team * 16, hi);
        store_block_row(smem + kOffSmallLo + b * kOperandBytes, r, team * 16, lo);
      }
  }
  const float s_scale = kScaleS / (m.sx * m.sx), o_scale = m.out_scale / m.sx;
  const float kb = st.b * (kScaleB / kScaleS), kc = st.c * (kScaleB / (kScaleS * kScaleS));
  const uint32_t taddr = tmem + ((uint32_t)(quadrant * 32) << 16);
  uint8_t* const s_tile = smem + kOffSmallS;
  uint8_t* const b_tile = smem + kOffSmallB;
  // Rows and columns behind the matrix are zeros from the start and stay so: their warps write S and B once.
  const bool no_row = quadrant * 32 >= m.m, no_col = team * 32 >= m.m;
  uint32_t parity = 0;
  // Ends a phase's writes to shared memory and tensor memory reads, lets thread 0 issue the next products and waits for them.
  auto products = [&](auto issue) {
    ptx::fence_proxy_async_smem();
    ptx::tcgen05_fence_before();
    __syncthreads();
    if (tid == 0 && !p.withhold) {
      ptx::tcgen05_fence_after();
      issue();
      ptx::umma_commit(bar);
    }
    const bool ok = ptx::mbar_wait(bar, parity, &sh.abort_flag, p.status, 13, 0, p.wait_limit_us);
    parity ^= 1u;
    const bool all = __syncthreads_and(ok);
    ptx::tcgen05_fence_after();
    return all;
  };
  bool alive = true;
  for (int step = 0; step < p.steps; ++step) {
    // S = X X^T
    alive = products([&] {
      const uint32_t idesc = ptx::make_idesc_f16(0, 0, 0, 128, 128);
      for (int b = 0; b < blocks; ++b) {
        const uint64_t d = ptx::make_smem_desc_sw128(base + b * kOperandBytes, 16, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) ptx::umma_f16(tmem, d + 2 * k, d + 2 * k, idesc, (b | k) != 0 ? 1u : 0u);
      }
    });
    if (!alive) break;
    if (step == 0 || !(no_row || no_col)) {
      uint32_t a[32], w[8];
      ptx::tmem_ld_32x32(taddr + team * 32, a);
      ptx::tmem_ld_wait_regs(a);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = pack_half2(__uint_as_float(a[16 * h + 2 * q]) * s_scale, __uint_as_float(a[16 * h + 2 * q + 1]) * s_scale);
        store_block_row(s_tile + (team >> 1) * kOperandBytes, r, (team & 1) * 32 + 16 * h, w);
      }
    }
    // B = b S + c S^2, its diagonal apart
    alive = products([&] {
      const uint32_t idesc = ptx::make_idesc_f16(0, 0, 0, 128, 128);
      for (int b = 0; b < 2; ++b) {
        const uint64_t d = ptx::make_smem_desc_sw128(base + kOffSmallS + b * kOperandBytes, 16, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) ptx::umma_f16(tmem + 128, d + 2 * k, d + 2 * k, idesc, (b | k) != 0 ? 1u : 0u);
      }
    });
    if (!alive) break;
    if (step == 0 || !(no_row || no_col)) {
      uint32_t a[32], w[8];
      ptx::tmem_ld_32x32(taddr + 128 + team * 32, a);
      ptx::tmem_ld_wait_regs(a);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[16];
        load_block_row(s_tile + (team >> 1) * kOperandBytes, r, (team & 1) * 32 + 16 * h, w);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float2 s = unpack_half2(w[q]);
          v[2 * q] = fmaf(kc, __uint_as_float(a[16 * h + 2 * q]), kb * s.x);
          v[2 * q + 1] = fmaf(kc, __uint_as_float(a[16 * h + 2 * q + 1]), kb * s.y);
        }
        const int dq = r - (team * 32 + 16 * h);
        if ((unsigned)dq < 16u) {
          float d = 0.0f;
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            d = q == dq ? v[q] : d;
            v[q] = q == dq ? 0.0f : v[q];
          }
          sh.diag[r] = d * (1.0f / kScaleB);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = pack_half2(v[2 * q], v[2 * q + 1]);
        store_block_row(b_tile + (team >> 1) * kOperandBytes, r, (team & 1) * 32 + 16 * h, w);
      }
    }
    // X <- a X + B X, in place
    alive = products([&] {
      // up to four blocks an instruction: the issuing thread spends some 65 cycles on each whatever its width
      for (int b = 0; b < blocks; b += 4) {
        const uint32_t idesc = ptx::make_idesc_f16(0, 0, 1, 128, 64 * min(4, blocks - b));
        const uint64_t x = ptx::make_smem_desc_sw128(base + b * kOperandBytes, kOperandBytes, 1024);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint64_t a = ptx::make_smem_desc_sw128(base + kOffSmallB + (k >> 2) * kOperandBytes, 16, 1024) + 2 * (k & 3);
          ptx::umma_f16(tmem + b * 64, a, x + k * (2048 >> 4), idesc, k != 0 ? 1u : 0u);
        }
      }
    });
    if (!alive) break;
    const float dg = st.a + sh.diag[r];
    const bool last = step == p.steps - 1;
    if (!no_row) {
#pragma unroll
      for (int b0 = 0; b0 < kSmallBlocks; b0 += 2) {   // two blocks' loads before the first one's arithmetic
        if (b0 >= blocks) break;
        uint32_t a[2][16], w0[2][8], w1[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (b0 + u < blocks) {
            const uint8_t* const hi = smem + (b0 + u) * kOperandBytes;
            ptx::tmem_ld_32x16(taddr + (b0 + u) * 64 + team * 16, a[u]);
            load_block_row(hi, r, team * 16, w0[u]);
            load_block_row(hi + kOffSmallLo, r, team * 16, w1[u]);
          }
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (b0 + u < blocks) {
            uint8_t* const hi = smem + (b0 + u) * kOperandBytes;
            ptx::tmem_ld_wait_regs(a[u]);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float2 h = unpack_half2(w0[u][q]), l = unpack_half2(w1[u][q]);
              const float x = fmaf(dg, h.x + l.x, __uint_as_float(a[u][2 * q]) * (1.0f / kScaleB));
              const float y = fmaf(dg, h.y + l.y, __uint_as_float(a[u][2 * q + 1]) * (1.0f / kScaleB));
              if (!last) split_pair(x, y, w0[u][q], w1[u][q]);
              else w0[u][q] = out_bits(x * o_scale, st.out_dt) | ((uint32_t)out_bits(y * o_scale, st.out_dt) << 16);
            }
            store_block_row(hi, r, team * 16, w0[u]);
            if (!last) store_block_row(hi + kOffSmallLo, r, team * 16, w1[u]);
          }
      }
    }
  }
  __syncthreads();
  if (alive) {
    unsigned short* out = reinterpret_cast<unsigned short*>(m.out);
#pragma unroll 2
    for (int v = tid; v * 4 < total; v += kSmallThreads) {
      const int e0 = 4 * v;
      int o = e0 / inner, i = e0 - o * inner;
      uint32_t h[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = m.tall ? i : o, c = m.tall ? o : i;
        h[q] = e0 + q < total ? *reinterpret_cast<const unsigned short*>(smem + (c >> 6) * kOperandBytes + row * 128 +
                                                                        ((((c & 63) >> 3) ^ (row & 7)) << 4) + (c & 7) * 2) : 0u;
        if (++i == inner) { i = 0; ++o; }
      }
      if (e0 + 4 <= total) *reinterpret_cast<uint2*>(out + e0) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
      else
        for (int q = 0; q < 4 && e0 + q < total; ++q) out[e0 + q] = (unsigned short)h[q];
    }
  } else if (tid == 0 && !p.withhold) {   // products in flight may not write tensor memory that is freed
    int never = 0;
    ptx::mbar_wait(bar, parity ^ 1u, &never, p.status, 8, 0, p.wait_limit_us);
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---- plan --------------------------------------------------------------------------------------------------------
int32_t encode_arena(CUtensorMap* map, void* arena, long long rows, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
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
    std::vector<int> index;    // the table's matrices in the caller's list
    bool small;                // every matrix fits an SM: muon_small_kernel
    bool pair;                 // CTA pairs on 256 x 256 tiles
    MuonTable table;           // pointers are filled in at launch
    int sum_ctas, pack_ctas, iter_ctas, sync_words;
    size_t off_sync, off_parts, off_diag, off_partial, off_arena;
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
      const int k = r.index[i];
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

template <bool PAIR>
int32_t launch_iterate(const CUtensorMap& m128, const CUtensorMap& m64, const IterArgs& a, int ctas, int device, cudaStream_t stream) {
  auto kernel = muon_iterate_kernel<PAIR>;
  static SmemLimit limit;
  HE_TRY(limit.raise(kernel, device, kIterSmem));
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((unsigned)ctas, 1, 1);
  lc.blockDim = dim3(kGemmThreads, 1, 1);
  lc.dynamicSmemBytes = kIterSmem;
  lc.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = PAIR ? 2 : 1; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  lc.attrs = &attr;
  lc.numAttrs = 1;
  HE_CUDA(cudaLaunchKernelEx(&lc, kernel, m128, m64, a));
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
      const int k = r.index[i];
      m.g = in[k];
      m.out = out[k];
      m.avg = st.has_momentum ? (const float*)in[count + k] : nullptr;
      m.avg_out = st.has_momentum ? (float*)out[count + k] : nullptr;
    }
    if (r.small) {
      static SmemLimit limit;
      HE_TRY(limit.raise(muon_small_kernel, ctx->device, kSmallSmem));
      const SmallArgs sa{ctx->d_status, wait_limit_us, withhold, steps};
      muon_small_kernel<<<t.count, kSmallThreads, kSmallSmem, stream>>>(t, st, sa);
      HE_CUDA(cudaGetLastError());
      last_launches += 1;
      continue;
    }
    uint8_t* w = (uint8_t*)ws;
    MuonTable* table = (MuonTable*)w;
    double* parts = (double*)(w + r.off_parts);
    uint8_t* arena = w + r.off_arena;
    CUtensorMap m128, m64;
    HE_TRY(encode_arena(&m128, arena, r.arena_rows, 128));
    HE_TRY(encode_arena(&m64, arena, r.arena_rows, 64));
    MuonSync* sync = (MuonSync*)(w + r.off_sync);
    muon_average_kernel<<<r.sum_ctas, kSumThreads, 0, stream>>>(t, st, table, parts, (unsigned*)sync, r.sync_words);
    HE_CUDA(cudaGetLastError());
    muon_pack_kernel<<<r.pack_ctas, 256, 0, stream>>>(t, st, parts, arena);
    HE_CUDA(cudaGetLastError());
    IterArgs a{};
    a.table = table; a.sync = sync; a.arrive = (unsigned*)(sync + 1);
    a.arena = arena; a.diag = (float*)(w + r.off_diag); a.partial = (float*)(w + r.off_partial);
    a.status = ctx->d_status; a.wait_limit_us = wait_limit_us; a.withhold_loads = withhold;
    a.steps = steps; a.a = st.a; a.b = st.b; a.c = st.c; a.out_dt = st.out_dt;
    HE_TRY(r.pair ? launch_iterate<true>(m128, m64, a, r.iter_ctas, ctx->device, stream)
                  : launch_iterate<false>(m128, m64, a, r.iter_ctas, ctx->device, stream));
    last_launches += 3;
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
  // The products' f16 operands have room for |X| < 65504 / 2^15 and |b S + c S^2| < 65504 / 2^10 (an entry is at most the
  // largest singular value): the map of the singular values, which start in [0, 1], is followed step by step.
  for (int i = 0; i <= 4096; ++i) {
    double v = i / 4096.0;
    for (int step = 0; step < prm->steps; ++step) {
      const double q = v * v;
      if (!(std::fabs(v) < 1.9) || !(std::fabs((double)prm->coef[1]) * q + std::fabs((double)prm->coef[2]) * q * q < 60.0))
        HE_FAIL(HE_ERR_UNSUPPORTED, "muon: after %d steps these coefficients take a singular value of %.4f to %g, beyond the products' range", step,
                i / 4096.0, v);
      v = v * (prm->coef[0] + q * (prm->coef[1] + q * (double)prm->coef[2]));
    }
  }
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
  // Smallest products first: at every border of a phase the small matrices' items, whose own phase is over by then, come
  // before those of the large ones, which have to wait (the conv net's filters: 297 us, largest first 322 us).
  std::vector<int> order((size_t)prm->count);
  for (int i = 0; i < prm->count; ++i) order[i] = i;
  auto weight = [&](int i) { return (double)std::min(prm->rows[i], prm->cols[i]) * (double)prm->rows[i] * (double)prm->cols[i]; };
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return weight(a) < weight(b); });
  for (int first = 0; first < prm->count; first += kMaxMats) {
    MuonPlan::Round r{};
    r.table.count = std::min(kMaxMats, prm->count - first);
    r.index.assign(order.begin() + first, order.begin() + first + r.table.count);
    const int sms = ctx_sm_count(ctx);
    // Every matrix of this part of the list fits an SM.  Where only some do, all go by tiles: the small ones' tiles find room
    // beside the others' (32 of 64 x 288 with one 64 x 576 100 us in one list, 139 us in two, 43 of them the small ones' kernel; 40 of
    // them with one 512 x 4608 177 and 213 us).
    r.small = true;
    for (int i = 0; i < r.table.count; ++i) {
      const int64_t h = prm->rows[r.index[i]], w = prm->cols[r.index[i]];
      r.small = r.small && h > 0 && w > 0 && std::min(h, w) <= 128 && std::max(h, w) <= 64 * kSmallBlocks;
    }
    // Which tiles: a phase lasts as long as its deepest tile and a fixed part (waits, first loads, epilogue), or as its
    // whole work spread over the workers, if that is longer.  Measured on a B200: 0.35 us a 64-deep block and 5 us fixed for
    // 128 x 128 tiles, 0.41 us and 8 us for 256 x 256 tiles of a pair.  (A 1024 x 1024 matrix takes 166 us on single CTAs and
    // 222 us on pairs, 2048 x 8192 851 and 767, 4096 x 4096 1790 and 1257.)  One size for the whole list: 4096 x 4096 with 16 of
    // 512 x 512 takes 1307 us so, in two lists with a size each 1450 us; with the conv net's filters 1449 and 1588 us.
    long long s_blocks1 = 0, s_blocks2 = 0;
    for (int i = 0; i < r.table.count; ++i) {
      const int64_t h = prm->rows[r.index[i]], w = prm->cols[r.index[i]];
      if (h <= 0 || w <= 0) HE_FAIL(HE_ERR_INVALID, "muon: matrix %d is empty", r.index[i]);
      if (std::min(h, w) > 32768 || std::max(h, w) > (1 << 20)) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: matrix %d is larger than 32768 x 1048576", r.index[i]);
    }
    auto step_us = [&](long long tile, int workers, double block_us, double fixed_us, long long* s_blocks) {
      double work_s = 0, work_b = 0, work_x = 0, deep = 0;
      for (int i = 0; i < r.table.count; ++i) {
        const long long h = prm->rows[r.index[i]], w = prm->cols[r.index[i]], mm = std::min(h, w), nn = std::max(h, w);
        const long long km = (mm + 63) / 64, kn = (nn + 63) / 64, ti = (mm + tile - 1) / tile, tj = (nn + tile - 1) / tile, sym = ti * (ti + 1) / 2;
        work_s += (double)sym * kn;
        work_b += (double)sym * km;
        work_x += (double)ti * tj * km;
        deep = std::max(deep, (double)km);
      }
      *s_blocks = (long long)work_s;
      // S's sums are split where tiles are few
      return block_us * (std::max(work_s / workers, std::min(deep, 16.0)) + std::max(work_b / workers, deep) + std::max(work_x / workers, deep)) + 3 * fixed_us;
    };
    r.pair = step_us(256, sms / 2, 0.41, 8.0, &s_blocks2) < step_us(128, sms, 0.35, 5.0, &s_blocks1);
    const int unit = r.pair ? 2 : 1;
    // S is split along n until a step's list of S items keeps every CTA (pair) busy, at 16 or more blocks of 64 columns a slice
    // (a slice costs the write and the read of its f32 tile; 512 x 4608: 8 blocks 223 us, 16 198 us, 24 205 us)
    const long long s_blocks = r.pair ? s_blocks2 : s_blocks1, workers = sms / unit;
    const long long slice = std::max<long long>(16, (s_blocks + workers - 1) / workers);
    long long rows = 0, diag = 0, items_s = 0, items_b = 0, items_x = 0, pack = 0, parts = 0, arrive = 0, partial = 0;
    for (int i = 0; i < r.table.count; ++i) {
      MuonMat& m = r.table.mat[i];
      const int64_t h = prm->rows[r.index[i]], w = prm->cols[r.index[i]];
      m.tall = h > w;
      m.m = (int)std::min(h, w);
      m.n = (int)std::max(h, w);
      m.mt = (m.m + 128 * unit - 1) / (128 * unit) * unit;
      m.nt = (m.n + 128 * unit - 1) / (128 * unit) * unit;
      m.out_scale = prm->scales ? prm->scales[r.index[i]] : 1.0f;
      if (!std::isfinite(m.out_scale)) HE_FAIL(HE_ERR_INVALID, "muon: scale of matrix %d is not finite", r.index[i]);
      const double side = std::sqrt((double)m.m * m.n);
      m.sx = (float)std::ldexp(1.0, std::min(15, (int)std::floor(std::log2(side))));
      const long long xrows = (long long)m.mt * 2 * m.nt * kBlockRows, srows = (long long)m.mt * 2 * m.mt * kBlockRows;
      m.x[0] = rows; rows += xrows;
      m.x[1] = rows; rows += xrows;
      m.xlo = rows; rows += xrows;
      m.s = rows; rows += srows;
      m.b = rows; rows += srows;
      m.diag = diag; diag += (long long)m.mt * 128;
      const long long ti = m.mt / unit, tj = m.nt / unit, tiles = ti * (ti + 1) / 2, blocks = (m.n + 63) / 64;
      m.splits = (int)std::min<long long>(16, (blocks + slice - 1) / slice);
      m.split_blocks = (int)((blocks + m.splits - 1) / m.splits);
      m.splits = (int)((blocks + m.split_blocks - 1) / m.split_blocks);
      m.arrive0 = (int)arrive; arrive += tiles * unit;
      m.partial = partial;
      if (m.splits > 1) partial += tiles * unit * m.splits * kTile * kTile * unit;
      m.s0 = (int)items_s; items_s += tiles * m.splits;
      m.b0 = (int)items_b; items_b += tiles;
      m.x0 = (int)items_x; items_x += ti * tj;
      m.pack0 = (int)pack; pack += (long long)m.mt * 2 * m.nt;
      // partial sums: CTAs of at least 4096 elements, at most 2048 of them (512 or 2048 are within 1 % for 4096 x 4096)
      const long long total = (long long)m.m * m.n;
      long long chunks = std::min<long long>(2048, (total + 4095) / 4096);
      m.chunk = (total + chunks - 1) / chunks;
      m.chunk = (m.chunk + 3) / 4 * 4;
      m.chunks = (int)((total + m.chunk - 1) / m.chunk);
      m.part0 = (int)parts; parts += m.chunks;
      if (rows >= (1ll << 31) || pack >= (1ll << 31)) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: the matrices of a plan exceed 2^31 workspace rows");
    }
    if ((items_s + items_b + items_x) * (prm->steps + 1) + 4096 >= (1ll << 31)) HE_FAIL(HE_ERR_UNSUPPORTED, "muon: 2^31 or more work items");
    for (int i = 0; i < r.table.count; ++i) {   // one list: S, then B, then X
      r.table.mat[i].b0 += (int)items_s;
      r.table.mat[i].x0 += (int)(items_s + items_b);
    }
    r.table.items_s = (int)items_s;
    r.table.items_b = (int)(items_s + items_b);
    r.table.items = (int)(items_s + items_b + items_x);
    r.sum_ctas = (int)parts; r.pack_ctas = (int)pack;
    r.iter_ctas = unit * (int)std::min<long long>(workers, std::max(items_s, items_x));
    r.sync_words = (int)(sizeof(MuonSync) / 4 + arrive);
    r.arena_rows = rows;
    auto align = [](size_t v) { return (v + 1023) / 1024 * 1024; };
    r.off_sync = align(sizeof(MuonTable));
    r.off_parts = align(r.off_sync + (size_t)r.sync_words * 4);
    r.off_diag = align(r.off_parts + (size_t)parts * sizeof(double));
    r.off_partial = align(r.off_diag + (size_t)diag * sizeof(float));
    r.off_arena = align(r.off_partial + (size_t)partial * sizeof(float));
    if (!r.small) plan->workspace_bytes = std::max(plan->workspace_bytes, r.off_arena + (size_t)rows * 128);
    plan->rounds.push_back(std::move(r));
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
