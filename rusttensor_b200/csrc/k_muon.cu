// Muon: an optimizer step whose update is the momentum with its singular values brought near one.
//
//   m = mu m + s g      u = m, or s g + mu m (nesterov)      p = (1 - lr wd) p - lr sqrt(max(1, cols / rows)) O(u)
//
// O(u) comes from Newton-Schulz steps on X = u / (|u| + 1e-7): X <- (a I + b G + c G^2) X with G = X X^T, which takes every singular value x to
// a x + b x^3 + c x^5, with 3.4445, -4.7750, 2.0315, the coefficients published with Muon (K. Jordan, 2024): five steps bring values between 0.002 and
// 1 to between 0.7 and 1.2.  G is taken on the shorter side; a matrix with more rows than columns is transposed for the steps.
//
// A step is three products, each of which has to wait for the one before: G = X X^T and b G + c G^2, both symmetric, of which the lower half is
// computed and written twice, and a X + (b G + c G^2) X.  Errors of early steps grow (small singular values by 3.4 a step), so the products
// keep fp32's precision: an operand is held as two fp16 parts, hi = fp16(2^15 x) and lo = fp16(2^15 x - hi), 22 bits, and a product is three
// tcgen05.mma of kind::f16: hi lo, lo hi and hi hi.  No element of X, G or the polynomial is beyond 1.21, 1.46 and 2.81 (bounds of their singular
// values; the polynomial takes 2^14), so the scale is fixed.  Below 2^-18, where lo has fewer than 11 bits left, an element is off by
// 2^-40 at most, of G and the polynomial together by 2^-37.2 in its share of the result: that is 2^-19 of a row or column of k elements as long as its
// norm is sqrt(max(k, 64)) 2^-21 or more.  Rows whose norms differ by exp(N(0, 1)) stay above that up to some 10000 x 10000.  Where a row or a
// column that is not zero lies below, the matrix is wide: its operands are three bf16 parts, 24 bits of fp32's range, and a product is six MMAs
// (all but the three smallest), so that every row and column is as near as in fp32 against its own size: what a step adds up for one has that
// size as a factor.  (With two parts alone, at 2^12, rows 2^-16 of the others were 9e-5 off and rows 2^-32 of them not updated at all.)  Rows
// and columns shrink by no more than a third over all steps (singular values up to 1 end above 0.68), so this is decided once.
//
// A product's epilogue adds what the formula adds and writes the parts that the next product reads, as they lie: X [m][n] is an operand with n as
// the reduction, and with m, by tensor maps and MMA descriptors of either kind.  All matrices of a call go through every product together, and all
// products are one cooperative launch, whose blocks wait for one another between two products (15 launches for five steps were 4 us each
// besides the work).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

#include <cuda_bf16.h>

#include "parts_common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr double kEpsilon = 1e-7;
constexpr int kNormBlocks = 256;

struct Update {
  const float* x;  // what is orthogonalised; with a gradient: made of it and the momentum
  const float* g;
  float* m;
  float mu, scale;
  int nesterov;
};
__device__ __forceinline__ float momentum_at(const Update& u, int64_t i) { return u.mu * u.m[i] + u.scale * __ldg(u.g + i); }
// From the old momentum.
__device__ __forceinline__ float update_at(const Update& u, int64_t i) {
  if (!u.g) return __ldg(u.x + i);
  const float m = momentum_at(u, i);
  return u.nesterov ? u.scale * __ldg(u.g + i) + u.mu * m : m;
}
// The new momentum, if it is to be written by now, and the sum of the squares of the update, block by block in 64 bits: squares of large fp32 values have no room in 32.  A
// matrix has kNormBlocks blocks.  Bound by memory: 4096 x 4096 takes 17 us (236 with one value at a time in 128 blocks).
constexpr int kGroup = 12;  // matrices of a launch
struct Squares {
  Update u[kGroup];
  int64_t n[kGroup];
  int write;
  double* sums;  // [matrix][block]
  unsigned long long* zero;  // what later launches begin with zeros
  int64_t zeros;
};
template <bool VEC>
__device__ __forceinline__ double sum_of_squares(const Update& u, int64_t n, bool write) {
  constexpr int kAhead = 4, V = VEC ? 4 : 1;
  double sum = 0.0;
  const int64_t step = (int64_t)kNormBlocks * kThreads * V;
  for (int64_t i0 = ((int64_t)(blockIdx.x % kNormBlocks) * kThreads + threadIdx.x) * V; i0 < n; i0 += kAhead * step) {
    float g[kAhead][V], m[kAhead][V];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * step;
#pragma unroll
      for (int j = 0; j < V; ++j) g[k][j] = m[k][j] = 0.f;
      if (i >= n) continue;
      const float *from = (u.g ? u.g : u.x) + i, *old = u.m + i;
      if (VEC) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(from));
        g[k][0] = q.x; g[k][V / 4] = q.y; g[k][V / 2] = q.z; g[k][V - 1] = q.w;
        if (u.g) {
          const float4 r = *reinterpret_cast<const float4*>(old);
          m[k][0] = r.x; m[k][V / 4] = r.y; m[k][V / 2] = r.z; m[k][V - 1] = r.w;
        }
      } else {
        g[k][0] = __ldg(from);
        if (u.g) m[k][0] = *old;
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * step;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        double v = g[k][j];
        if (u.g) {
          m[k][j] = u.mu * m[k][j] + u.scale * g[k][j];
          v = u.nesterov ? u.scale * g[k][j] + u.mu * m[k][j] : m[k][j];
        }
        sum += v * v;
      }
      if (write && i < n) {
        if (VEC) *reinterpret_cast<float4*>(u.m + i) = make_float4(m[k][0], m[k][V / 4], m[k][V / 2], m[k][V - 1]);
        else u.m[i] = m[k][0];
      }
    }
  }
  return sum;
}
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Squares p) {
  RT_PDL_ENTRY();
  __shared__ double of_warp[kThreads / 32];
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < p.zeros; i += (int64_t)gridDim.x * kThreads) p.zero[i] = 0;
  const int q = blockIdx.x / kNormBlocks;
  const Update u = p.u[q];
  const int64_t n = p.n[q];
  const bool vec = n % 4 == 0 && (((uintptr_t)u.x | (uintptr_t)u.g | (uintptr_t)u.m) & 15) == 0;
  const bool write = p.write && u.g;
  double sum = vec ? sum_of_squares<true>(u, n, write) : sum_of_squares<false>(u, n, write);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) sum += of_warp[w];
    p.sums[blockIdx.x] = sum;
  }
}
// 1 / (norm + epsilon), in every thread of a warp, as a product of two numbers: of the largest matrices it has no room among the normal numbers of
// 32 bits.  The first one is a power of two.
__device__ __forceinline__ float2 one_over_norm(const double* __restrict__ sums) {
  double sum = 0.0;
#pragma unroll
  for (int b = 0; b < kNormBlocks; b += 32) sum += __ldg(sums + b + (threadIdx.x & 31));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const double by = 1.0 / (sqrt(sum) + kEpsilon);
  return by < 0x1p-100 ? make_float2(0x1p-64f, (float)(by * 0x1p64)) : make_float2(1.f, (float)by);
}
// X: the update divided by its norm, its shorter side first.
__global__ void __launch_bounds__(kThreads) normalise_kernel(const Update u, int64_t rows, int64_t cols, const double* __restrict__ sums, float* __restrict__ x) {
  RT_PDL_ENTRY();
  const float2 by = one_over_norm(sums);
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / cols, c = i - r * cols;
    x[rows > cols ? c * rows + r : i] = update_at(u, i) * by.x * by.y;
  }
}
// s = a I + b g + c s
__global__ void __launch_bounds__(kThreads) polynomial_kernel(const float* __restrict__ g, int64_t m, float* __restrict__ s) {
  RT_PDL_ENTRY();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < m * m; i += (int64_t)gridDim.x * kThreads)
    s[i] = kB * __ldg(g + i) + kC * s[i] + (i / m == i % m ? kA : 0.f);
}
// out = keep * out - step * x, or out = x; and the new momentum
__global__ void __launch_bounds__(kThreads) apply_kernel(const float* __restrict__ x, int64_t rows, int64_t cols, float* __restrict__ out, int update, float keep,
                                                         float step, const Update u) {
  RT_PDL_ENTRY();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / cols, c = i - r * cols;
    const float o = __ldg(x + (rows > cols ? c * rows + r : i));
    out[i] = update ? keep * out[i] - step * o : o;
    if (u.g) u.m[i] = momentum_at(u, i);
  }
}

struct Matrix {
  Update u;
  int64_t rows, cols;
  float* out;
  int update;
  float keep, step;
};

rt_status launch_squares(rt_ctx* ctx, const Matrix* list, int count, int write, double* sums, unsigned long long* zero = nullptr, int64_t zeros = 0) {
  Squares p{};
  for (int q = 0; q < count; ++q) {
    p.u[q] = list[q].u;
    p.n[q] = list[q].rows * list[q].cols;
  }
  p.write = write;
  p.sums = sums;
  p.zero = zero;
  p.zeros = zeros;
  rt_launch(ctx, squares_kernel, kNormBlocks * count, kThreads, 0, p);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

// ---- the products on the tensor cores -----------------------------------------------------------------------------------------------
using namespace tc;
namespace cg = cooperative_groups;
using parts::kBox;

constexpr float kScale = 32768.f, kScaleS = 16384.f;  // of the two parts of X and G; of the polynomial
constexpr int kPlanes = 3;
constexpr int kTileM = 128, kBlockK = 64;  // rows of a tile; elements of the reduction that a stage holds
constexpr uint32_t kSecond = 256;          // tensor-memory column of the second accumulator
enum { kGram, kSquare, kApply, kResult };  // kResult: the last kApply, whose result goes to `out`

struct Item {
  int m, n;              // m <= n
  int ldx, ldm;          // halves between rows of X, of G and the polynomial
  uint16_t *x[2], *g, *s; // kPlanes each: hi, lo; or, of a wide matrix, the middle one, the first, the last.  X begins in x[0], of a wide matrix in x[1]
  int first[3], splits[3];  // by product: first work item of the matrix, CTAs that share a tile's reduction
  int first_part[3];        // partial sums of the matrices before, in tiles
  int first_ticket[3];
  // the result
  float* out;
  int tall, update, vec; // X is transposed against out; 128-bit accesses to out
  float keep, step;
};
struct Product {
  // X, G and the polynomial, two planes in a box: 128 rows high as left operands, as right ones as many as a CTA brings in, X 64 as the right operand
  // whose rows are the reduction.
  CUtensorMap x_left[2][kGroup], x_right[2][kGroup], x_apply[2][kGroup], g_left[kGroup], g_right[kGroup], s_left[kGroup];
  Item item[kGroup];
  int count, steps;
  int items[3];
  const unsigned* wide;  // a bit for each matrix
  float* sums;           // partial sums of tiles, [columns][128 rows] each
  unsigned* tickets;     // zero
  unsigned* arrived;     // zero; blocks that have done their part, of all products
  uint32_t polls;        // looks at that for each product
  int* status;
};
constexpr unsigned kGaveUp = 1u << 31;  // in `arrived`: a wait has run out somewhere
// Results are finished by slabs of 64 columns.
constexpr int kSlab = 64;
// A tile of W columns has 128 rows and belongs to a CTA, or (PAIR) 256 rows and belongs to two CTAs of a cluster: each has 128 of the rows and
// brings in half of the right operand, which the MMAs of a pair read from both.
template <int W, bool PAIR>
struct Layout {
  static constexpr int rows = PAIR ? 2 * kTileM : kTileM;
  static constexpr int right = PAIR ? W / 2 : W;   // columns of the right operand that a CTA brings in
  static constexpr int warps = 16;                 // that finish results; then one for TMA, one for the MMAs
  static constexpr int tma = warps, mma = warps + 1, threads = (warps + 2) * 32;
  static constexpr int cols = W * 4 / warps;       // of a warp
  static constexpr uint32_t stage = (2 * kTileM + 2 * right) / 64 * kBox, stages = right == 128 ? 3 : 4;
  static constexpr uint32_t slab = stages * stage;
  static constexpr uint32_t bars = slab + kTileM * kSlab * 4, bytes = bars + (2 * stages + 5) * 8 + 16;
  static_assert(bytes <= 232448, "shared memory");
  static_assert(W == rows || W == rows / 2, "tiles of the lower half");
};
struct Tile {
  int q, row, col, k0, k1, split, index;  // K-blocks k0 .. k1; index: among the matrix's tiles
};
// K-blocks that an accumulator sums before it is emptied into registers, because it adds with truncation.  After two a long reduction is nearer to the
// exact result than one in fp32 (five steps of 4096 x 4096: 1.6e-6 and 4.9e-6 off); a short one needs the half of that (784 x 128: 1.7e-6, 1.6e-6 in
// fp32), where it costs little.  Wide matrices take one, whose small products come first.
template <int W>
__device__ __forceinline__ int chunk_of(int depth, bool wide) { return wide || (W == 64 && depth < 1024) ? 1 : 2; }
template <int W, bool PAIR>
__device__ __forceinline__ Tile tile_of(const Product& p, int phase, int i) {
  constexpr int rows = Layout<W, PAIR>::rows;
  int q = 0;
  while (q + 1 < p.count && i >= p.item[q + 1].first[phase]) ++q;
  const Item& a = p.item[q];
  Tile t;
  t.q = q;
  const int local = i - a.first[phase], splits = a.splits[phase];
  t.split = local % splits;
  t.index = local / splits;
  const int m_tiles = (a.m + rows - 1) / rows;
  if (phase == kApply) {
    t.row = t.index % m_tiles * rows;
    t.col = t.index / m_tiles * W;
  } else if (W == rows) {  // the lower half, row by row: 1 + 2 + 3 + ... tiles
    int r = (int)((sqrtf(8.f * t.index + 1.f) - 1.f) * 0.5f);
    while (r * (r + 1) / 2 > t.index) --r;
    while ((r + 1) * (r + 2) / 2 <= t.index) ++r;
    t.row = r * rows;
    t.col = (t.index - r * (r + 1) / 2) * W;
  } else {  // 2 + 4 + 6 + ...
    int r = (int)((sqrtf(4.f * t.index + 1.f) - 1.f) * 0.5f);
    while (r * (r + 1) > t.index) --r;
    while ((r + 1) * (r + 2) <= t.index) ++r;
    t.row = r * rows;
    t.col = (t.index - r * (r + 1)) * W;
  }
  const int k_blocks = ((phase == kGram ? a.n : a.m) + kBlockK - 1) / kBlockK;
  t.k0 = (int)((int64_t)k_blocks * t.split / splits);
  t.k1 = (int)((int64_t)k_blocks * (t.split + 1) / splits);
  return t;
}
// With PAIR the barrier is the one of the cluster's first CTA at the same place.
template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar & 0xFEFFFFFFu)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
// The MMAs before are done: for this CTA, or for both of a pair.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred pe;\n\t.reg .b16 m;\n\t"
        "elect.sync _|pe, 0xffffffff;\n\t"
        "mov.u16 m, 3;\n\t"
        "@pe tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar)
        : "memory");
  else
    umma_commit_elect(bar);
}
// At the barrier of the CTA that issues the MMAs.
template <bool PAIR>
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .b32 r;\n\t"
        "mapa.shared::cluster.u32 r, %0, 0;\n\t"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n\t}" ::"r"(bar)
        : "memory");
  else
    mbar_arrive(bar);
}
template <bool PAIR>
__device__ __forceinline__ void allocate(uint32_t slot) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(slot, 512);
  }
}
template <bool PAIR>
__device__ __forceinline__ void release(uint32_t tmem) {
  if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  else tmem_dealloc(tmem, 512);
}
// The MMAs of a K-block, in one statement: what they need is then moved to where they take it from all at once (one by one each took 71 cycles to
// issue).  A slot of 16 of the reduction is 2 further in the left descriptor, `step_b` in the right one.  hi lo and lo hi come first: what is cut off of
// them in an empty accumulator is as small as they are.  One elected lane of a converged warp issues.
template <bool PAIR>
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t a, uint32_t a_lo, uint32_t b, uint32_t b_lo, uint32_t step_b, uint32_t desc_hi, uint32_t idesc,
                                          uint32_t more) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred pe, pm, pt;\n\t"
        ".reg .b32 a1, a2, a3, b1, b2, b3, x1, x2, x3, y1, y2, y3;\n\t"
        ".reg .b64 A0, A1, A2, A3, B0, B1, B2, B3, X0, X1, X2, X3, Y0, Y1, Y2, Y3;\n\t"
        "elect.sync _|pe, 0xffffffff;\n\t"
        "setp.ne.b32 pm, %8, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "add.u32 a1, %1, 2;\n\tadd.u32 a2, %1, 4;\n\tadd.u32 a3, %1, 6;\n\t"
        "add.u32 x1, %2, 2;\n\tadd.u32 x2, %2, 4;\n\tadd.u32 x3, %2, 6;\n\t"
        "add.u32 b1, %3, %5;\n\tadd.u32 b2, b1, %5;\n\tadd.u32 b3, b2, %5;\n\t"
        "add.u32 y1, %4, %5;\n\tadd.u32 y2, y1, %5;\n\tadd.u32 y3, y2, %5;\n\t"
        "mov.b64 A0, {%1, %6};\n\tmov.b64 A1, {a1, %6};\n\tmov.b64 A2, {a2, %6};\n\tmov.b64 A3, {a3, %6};\n\t"
        "mov.b64 X0, {%2, %6};\n\tmov.b64 X1, {x1, %6};\n\tmov.b64 X2, {x2, %6};\n\tmov.b64 X3, {x3, %6};\n\t"
        "mov.b64 B0, {%3, %6};\n\tmov.b64 B1, {b1, %6};\n\tmov.b64 B2, {b2, %6};\n\tmov.b64 B3, {b3, %6};\n\t"
        "mov.b64 Y0, {%4, %6};\n\tmov.b64 Y1, {y1, %6};\n\tmov.b64 Y2, {y2, %6};\n\tmov.b64 Y3, {y3, %6};\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A0, Y0, %7, pm;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], X0, B0, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A1, Y1, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], X1, B1, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A2, Y2, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], X2, B2, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A3, Y3, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], X3, B3, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A0, B0, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A1, B1, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A2, B2, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], A3, B3, %7, pt;\n\t}" ::"r"(d),
        "r"(a), "r"(a_lo), "r"(b), "r"(b_lo), "r"(step_b), "r"(desc_hi), "r"(idesc), "r"(more)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred pe, pm, pt;\n\t"
        ".reg .b32 a1, a2, a3, b1, b2, b3, x1, x2, x3, y1, y2, y3;\n\t"
        ".reg .b64 A0, A1, A2, A3, B0, B1, B2, B3, X0, X1, X2, X3, Y0, Y1, Y2, Y3;\n\t"
        "elect.sync _|pe, 0xffffffff;\n\t"
        "setp.ne.b32 pm, %8, 0;\n\t"
        "setp.eq.b32 pt, 0, 0;\n\t"
        "add.u32 a1, %1, 2;\n\tadd.u32 a2, %1, 4;\n\tadd.u32 a3, %1, 6;\n\t"
        "add.u32 x1, %2, 2;\n\tadd.u32 x2, %2, 4;\n\tadd.u32 x3, %2, 6;\n\t"
        "add.u32 b1, %3, %5;\n\tadd.u32 b2, b1, %5;\n\tadd.u32 b3, b2, %5;\n\t"
        "add.u32 y1, %4, %5;\n\tadd.u32 y2, y1, %5;\n\tadd.u32 y3, y2, %5;\n\t"
        "mov.b64 A0, {%1, %6};\n\tmov.b64 A1, {a1, %6};\n\tmov.b64 A2, {a2, %6};\n\tmov.b64 A3, {a3, %6};\n\t"
        "mov.b64 X0, {%2, %6};\n\tmov.b64 X1, {x1, %6};\n\tmov.b64 X2, {x2, %6};\n\tmov.b64 X3, {x3, %6};\n\t"
        "mov.b64 B0, {%3, %6};\n\tmov.b64 B1, {b1, %6};\n\tmov.b64 B2, {b2, %6};\n\tmov.b64 B3, {b3, %6};\n\t"
        "mov.b64 Y0, {%4, %6};\n\tmov.b64 Y1, {y1, %6};\n\tmov.b64 Y2, {y2, %6};\n\tmov.b64 Y3, {y3, %6};\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A0, Y0, %7, pm;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], X0, B0, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A1, Y1, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], X1, B1, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A2, Y2, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], X2, B2, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A3, Y3, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], X3, B3, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A0, B0, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A1, B1, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A2, B2, %7, pt;\n\t"
        "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], A3, B3, %7, pt;\n\t}" ::"r"(d),
        "r"(a), "r"(a_lo), "r"(b), "r"(b_lo), "r"(step_b), "r"(desc_hi), "r"(idesc), "r"(more)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_one(uint32_t d, uint32_t a, uint32_t b, uint32_t desc_hi, uint32_t idesc, uint32_t more) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred pa, pe;\n\t.reg .b64 da, db;\n\t"
        "elect.sync _|pe, 0xffffffff;\n\t"
        "setp.ne.b32 pa, %5, 0;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "@pe tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, pa;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(desc_hi), "r"(idesc), "r"(more)
        : "memory");
  else
    parts::mma(d, a, desc_hi, b, desc_hi, idesc, more);
}
// Two neighbouring values as parts.
__device__ __forceinline__ void split2(float a, float b, float scale, uint32_t& hi, uint32_t& lo) {
  a *= scale;
  b *= scale;
  const __half2 h = __floats2half2_rn(a, b);
  const float2 back = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - back.x, b - back.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ float2 join2(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi)), l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return make_float2((h.x + l.x) * (1.f / kScale), (h.y + l.y) * (1.f / kScale));
}
__device__ __forceinline__ float2 of_bf16(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t to_bf16(float2& v) {  // leaves the rest
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
  const float2 back = of_bf16(w);
  v.x -= back.x;
  v.y -= back.y;
  return w;
}
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[kPlanes]) {
  float2 v = make_float2(a, b);
  w[1] = to_bf16(v);
  w[0] = to_bf16(v);
  w[2] = to_bf16(v);
}
__device__ __forceinline__ float2 join3(uint32_t middle, uint32_t first, uint32_t last) {
  const float2 m = of_bf16(middle), h = of_bf16(first), l = of_bf16(last);
  return make_float2(h.x + m.x + l.x, h.y + m.y + l.y);
}
// A CTA's 128 x 64 results in shared memory, four columns a piece; where a row has its pieces keeps apart what is accessed together: the same
// piece of eight rows in a row, and of every fourth one.
__device__ __forceinline__ int piece_at(int row, int piece) { return row * kSlab + ((piece ^ ((row ^ row >> 2) & 7)) << 2); }
// A slab: adds what the formula adds and writes it, a warp eight rows, 128 bytes of the parts of a row in an access (a warp that has the 32 rows
// that it takes out of tensor memory touches 32 lines in every access).  Columns are written as rows where a result lies turned and, of
// symmetric matrices, what is below their diagonal blocks of 32 x 32.  (Those are written as they come: two results that mirror one
// another have the same terms.)  Rows of parts are padded to eight values, and what is written there nobody reads.
template <int PHASE>
struct Slab {
  static constexpr bool kSymmetric = PHASE == kGram || PHASE == kSquare;
  static constexpr float kOut = PHASE == kSquare ? kScaleS : kScale;
  int r, c;  // the lane's first row and column of eight; its second row is four behind
  uint4 hi[2], lo[2];
  __device__ __forceinline__ Slab(int row, int col, int warp, int lane) : r(row + warp * 8 + (lane >> 3)), c(col + (lane & 7) * 8) {}
  __device__ __forceinline__ bool in(const Item& q, int k) const {
    return r + 4 * k < q.m && c < (kSymmetric ? q.m : q.n) && (!kSymmetric || (c & ~31) <= (r & ~31));  // both rows are in one block of 32
  }
  __device__ __forceinline__ void fetch(const Item& q, int from) {
    if (PHASE == kGram) return;
    const int ld = kSymmetric ? q.ldm : q.ldx;
    const uint16_t* more = (PHASE == kSquare ? q.g : (from ? q.x[1] : q.x[0])) + (int64_t)r * ld + c;
    const int64_t plane = (int64_t)q.m * ld;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      hi[k] = lo[k] = make_uint4(0u, 0u, 0u, 0u);
      if (in(q, k)) {
        hi[k] = __ldcg(reinterpret_cast<const uint4*>(more + (int64_t)4 * k * ld));  // written by other SMs meanwhile
        lo[k] = __ldcg(reinterpret_cast<const uint4*>(more + (int64_t)4 * k * ld + plane));
      }
    }
  }
  // What is added has been fetched; the sums are in the slab.  row0, col0: of the slab.
  __device__ __forceinline__ void rows(const Item& q, int from, bool wide, float* slab, int row0) {
    const int ld = kSymmetric ? q.ldm : q.ldx;
    uint16_t* to = (PHASE == kGram ? q.g : (PHASE == kSquare ? q.s : (from ? q.x[0] : q.x[1]))) + (int64_t)r * ld + c;
    const int64_t plane = (int64_t)q.m * ld;
    const bool turned = PHASE == kResult ? q.tall : kSymmetric;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int y = r + 4 * k - row0, piece = (threadIdx.x & 7) * 2;
      float4* at[2] = {reinterpret_cast<float4*>(slab + piece_at(y, piece)), reinterpret_cast<float4*>(slab + piece_at(y, piece + 1))};
      const float4 s0 = *at[0], s1 = *at[1];
      float v[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
      constexpr float f = PHASE == kSquare ? kC : 1.f, g = PHASE == kSquare ? kB : kA, scale = kScale * (PHASE == kGram || PHASE == kSquare ? kScale : kScaleS);
      if (!wide) {
        const uint32_t hs[4] = {hi[k].x, hi[k].y, hi[k].z, hi[k].w}, ls[4] = {lo[k].x, lo[k].y, lo[k].z, lo[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] *= f / scale;
          v[2 * j + 1] *= f / scale;
          if (PHASE != kGram) {
            const float2 w = join2(hs[j], ls[j]);
            v[2 * j] += g * w.x;
            v[2 * j + 1] += g * w.y;
          }
        }
      } else if (PHASE != kGram && in(q, k)) {
        const uint16_t* more = (PHASE == kSquare ? q.g : (from ? q.x[1] : q.x[0])) + (int64_t)(r + 4 * k) * ld + c;
        uint32_t parts[kPlanes][4];
#pragma unroll
        for (int i = 0; i < kPlanes; ++i) {
          const uint4 w = __ldcg(reinterpret_cast<const uint4*>(more + i * plane));
          parts[i][0] = w.x; parts[i][1] = w.y; parts[i][2] = w.z; parts[i][3] = w.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 w = join3(parts[0][j], parts[1][j], parts[2][j]);
          v[2 * j] = f * v[2 * j] + g * w.x;
          v[2 * j + 1] = f * v[2 * j + 1] + g * w.y;
        }
      }
      if (turned) {
        *at[0] = make_float4(v[0], v[1], v[2], v[3]);
        *at[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
      if (PHASE == kResult) {
        if (!turned && in(q, k)) {
          float* o = q.out + (int64_t)(r + 4 * k) * q.n + c;
          put(q, o, make_float4(v[0], v[1], v[2], v[3]), q.n - c);
          put(q, o + 4, make_float4(v[4], v[5], v[6], v[7]), q.n - c - 4);
        }
      } else if (in(q, k) && !wide) {
        uint4 h, l;
        split2(v[0], v[1], kOut, h.x, l.x);
        split2(v[2], v[3], kOut, h.y, l.y);
        split2(v[4], v[5], kOut, h.z, l.z);
        split2(v[6], v[7], kOut, h.w, l.w);
        *reinterpret_cast<uint4*>(to + (int64_t)4 * k * ld) = h;
        *reinterpret_cast<uint4*>(to + (int64_t)4 * k * ld + plane) = l;
      } else if (in(q, k)) {
        uint32_t w[4][kPlanes];
#pragma unroll
        for (int j = 0; j < 4; ++j) split3(v[2 * j], v[2 * j + 1], w[j]);
#pragma unroll
        for (int i = 0; i < kPlanes; ++i) *reinterpret_cast<uint4*>(to + (int64_t)4 * k * ld + i * plane) = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
      }
    }
  }
  // A warp writes four columns as rows, a lane four values of each.
  __device__ __forceinline__ void columns(const Item& q, bool wide, const float* slab, int row0, int col0, int warp, int lane) {
    const int y = lane * 4, first = row0 + y, left = q.m - first, width = kSymmetric ? q.m : q.n;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int x = warp * 4 + k, col = col0 + x;
      if (left <= 0 || col >= width || (kSymmetric && (col & ~31) >= (first & ~31))) continue;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = slab[piece_at(y + j, x >> 2) + (x & 3)];
      if (kSymmetric) {
        uint16_t* o = (PHASE == kGram ? q.g : q.s) + (int64_t)col * q.ldm + first;
        const int64_t plane = (int64_t)q.m * q.ldm;
        if (!wide) {
          uint2 h, l;
          split2(v[0], v[1], kOut, h.x, l.x);
          split2(v[2], v[3], kOut, h.y, l.y);
          *reinterpret_cast<uint2*>(o) = h;
          *reinterpret_cast<uint2*>(o + plane) = l;
        } else {
          uint32_t w[2][kPlanes];
          split3(v[0], v[1], w[0]);
          split3(v[2], v[3], w[1]);
#pragma unroll
          for (int i = 0; i < kPlanes; ++i) *reinterpret_cast<uint2*>(o + i * plane) = make_uint2(w[0][i], w[1][i]);
        }
      } else {
        put(q, q.out + (int64_t)col * q.m + first, make_float4(v[0], v[1], v[2], v[3]), left);
      }
    }
  }
  // `left` of four results, none or less too
  static __device__ __forceinline__ void put(const Item& q, float* o, const float4& w, int left) {
    if (left <= 0) return;
    const float keep = q.keep, step = q.step;
    const bool update = q.update;
    if (q.vec) {
      float4 v = w;
      if (update) {
        const float4 old = *reinterpret_cast<const float4*>(o);
        v = make_float4(keep * old.x - step * w.x, keep * old.y - step * w.y, keep * old.z - step * w.z, keep * old.w - step * w.w);
      }
      *reinterpret_cast<float4*>(o) = v;
      return;
    }
    const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) o[j] = update ? keep * o[j] - step * v[j] : v[j];
  }
};

// What a warp that finishes results keeps from tile to tile.
struct Accumulators {
  uint32_t sums, full, empty;  // tensor memory; barriers, of the first of two
  uint32_t chunks;             // so far
  bool ok;
  volatile int *abort, *drawn;
  float* slab;
  int quad, group, lane, rank;
  unsigned wide;
};
template <int PHASE, int W, bool PAIR, bool WIDE_ONES>
__device__ __forceinline__ void finish_tiles(const Product& p, Accumulators& acc, int step) {
  using M = Layout<W, PAIR>;
  constexpr int cols = M::cols;
  constexpr int phase = PHASE == kResult ? kApply : PHASE;
  const int items = p.items[phase];
  for (int i = blockIdx.x >> PAIR; i < items; i += gridDim.x >> PAIR) {  // to the end also if a wait has run out: the warps meet at barriers
    const Tile t = tile_of<W, PAIR>(p, phase, i);
    const int splits = p.item[t.q].splits[phase];
    const Item q = p.item[t.q];  // of its own: what is left in the parameters is read again after every store
    const int row0 = t.row + acc.rank * kTileM, warp = threadIdx.x >> 5, width = PHASE == kGram || PHASE == kSquare ? q.m : q.n;
    const bool wide = WIDE_ONES && (acc.wide >> t.q & 1);
    const int from = (step ^ (int)wide) & 1;
    constexpr bool early = W == 64;  // what is added is on its way during the product: elsewhere there are no registers for it
    Slab<PHASE> slab(row0, t.col, warp, acc.lane);
    if (early && !wide) slab.fetch(q, from);
    const int chunk = chunk_of<W>(phase == kGram ? q.n : q.m, wide), chunks = (t.k1 - t.k0 + chunk - 1) / chunk;
    float sum[cols];
#pragma unroll
    for (int j = 0; j < cols; ++j) sum[j] = 0.f;
    for (int ch = 0; ch < chunks && acc.ok; ++ch, ++acc.chunks) {
      const uint32_t second = acc.chunks & 1;
      acc.ok = __all_sync(0xffffffffu, parts::wait(acc.full + 8 * second, acc.chunks >> 1 & 1, p.status, 96, acc.abort));
      if (!acc.ok) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < cols; c += 16) {
        uint32_t v[16];
        tmem_ld16_nowait(acc.sums + kSecond * second + c, v);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(v[j]);
      }
      tc_fence_before();
      __syncwarp();
      if (acc.lane == 0) arrive_first<PAIR>(acc.empty + 8 * second);
    }
    if (splits > 1) {
      const int64_t size = (int64_t)W * kTileM;
      float* mine = p.sums + (int64_t)((p.item[t.q].first_part[phase] + t.index * splits << PAIR) + acc.rank * splits) * size + (int64_t)acc.group * cols * kTileM + acc.quad * 32 + acc.lane;
#pragma unroll
      for (int j = 0; j < cols; ++j) __stcg(mine + t.split * size + j * kTileM, sum[j]);
      __threadfence();
      asm volatile("bar.sync 1, %0;" ::"n"(M::warps * 32) : "memory");
      if (threadIdx.x == 0) {
        unsigned* ticket = p.tickets + (p.item[t.q].first_ticket[phase] + t.index << PAIR) + acc.rank;
        const int d = *acc.abort ? -1 : (int)atomicAdd(ticket, 1u);  // with a share missing, nobody finishes the tile
        if (d == splits - 1) *ticket = 0;
        *acc.drawn = d;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(M::warps * 32) : "memory");
      const bool mine_to_finish = *acc.drawn == splits - 1;
      asm volatile("bar.sync 1, %0;" ::"n"(M::warps * 32) : "memory");  // `drawn` has been read
      if (!mine_to_finish) continue;
      __threadfence();
#pragma unroll
      for (int j = 0; j < cols; ++j) sum[j] = 0.f;
      for (int o = 0; o < splits; ++o)
#pragma unroll
        for (int j = 0; j < cols; ++j) sum[j] += __ldcg(mine + o * size + j * kTileM);
    }
#pragma unroll 1
    for (int k = 0; k < W / kSlab; ++k) {
      const int col0 = t.col + k * kSlab;
      if (row0 >= q.m || col0 >= width || (Slab<PHASE>::kSymmetric && col0 >= row0 + kTileM)) break;  // the same for all warps
      if (!early || k > 0) {
        slab = Slab<PHASE>(row0, col0, warp, acc.lane);
        if (!wide) slab.fetch(q, from);
      }
      if (acc.group * cols / kSlab == k) {
#pragma unroll
        for (int j = 0; j < cols; j += 4)
          *reinterpret_cast<float4*>(acc.slab + piece_at(acc.quad * 32 + acc.lane, (acc.group * cols % kSlab + j) / 4)) = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(M::warps * 32) : "memory");
      const int out = *acc.abort ? 1 << 30 : 0;  // if a wait has run out, results lie outside
      slab.c += out;
      slab.rows(q, from, wide, acc.slab, row0);
      if (Slab<PHASE>::kSymmetric || (PHASE == kResult && q.tall)) {
        asm volatile("bar.sync 1, %0;" ::"n"(M::warps * 32) : "memory");
        slab.columns(q, wide, acc.slab, row0 + out, col0, warp, acc.lane);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(M::warps * 32) : "memory");
    }
  }
}

// All products of all steps.  Roles of a CTA, one per SM, that walks over tiles: a TMA warp some K-blocks of 64 ahead, an MMA warp (of a pair's first
// CTA), and 16 warps that empty the accumulators into registers and write the result.  Where the
// tiles are fewer than the SMs, several CTAs share a tile's reduction: each leaves its sums in memory, and the one that draws the last ticket
// adds them up in their order.  A K-block takes 12 MMAs, of a wide matrix 24 on two stages: the first and last parts, then the middle and first
// (4096 x 4096 7.2 ms instead of 3.6 - 3.9, 512 x 512 205 us instead of 159).  What bounds large products otherwise is what all SMs together bring in
// from the L2 cache (some 37 bytes a cycle and SM): a pair with W = 256 takes 64 KB a K-block and CTA for 128 x 256 results, one CTA alone would take 96.
// Between two products a block's warps count the block as done when they have written their results, and its TMA warp waits for all blocks
// before it brings in what the next product reads and lets the block's others go on.  Every wait is bounded; on expiry the kernel records
// a code in the status word, raises a flag that all other waits poll, lets its own copies land, frees tensor memory and returns.  From then on the
// block writes no result and does not count as done, so that no other one goes on to the next product: `out`, which the last one writes, is
// what it was unless the wait was that one's.
template <int W, bool PAIR>
__global__ void __launch_bounds__(Layout<W, PAIR>::threads, 1) newton_schulz_kernel(const __grid_constant__ Product p) {
  using M = Layout<W, PAIR>;
  constexpr int kStages = M::stages;
  extern __shared__ __align__(1024) char smem[];  // and none besides: it starts where shared memory does
  const uint32_t base = smem_u32(smem);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = PAIR ? blockIdx.x & 1 : 0, unit = blockIdx.x >> PAIR, units = gridDim.x >> PAIR;
  const uint32_t bars = base + M::bars;
  auto full = [&](int i) { return bars + 8 * i; };
  auto empty = [&](int i) { return bars + 8 * (kStages + i); };
  const uint32_t acc_full = bars + 16 * kStages, acc_empty = acc_full + 16, go = acc_full + 32;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + M::bars + (2 * kStages + 5) * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, M::warps << PAIR);
    }
    mbar_init(go, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == M::mma) allocate<PAIR>(smem_u32(tmem_slot));
  tc_fence_before();
  if (PAIR) cg::this_cluster().sync();  // the barriers, too, are there
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const unsigned wide_ones = *p.wide;
  // Whether any matrix is wide is compiled for itself: what wide ones need would take registers from the others (five layers 457 us instead of 383).
  auto run = [&](auto any) {
    constexpr bool WIDE_ONES = decltype(any)::value;
    bool ok = true;
    if (warp == M::tma) {
      if (lane == 0) {
        int it = 0;
        for (int product = 0; product < 3 * p.steps && ok; ++product) {
          const int phase = product % 3, items = p.items[phase];
          Tile t = tile_of<W, PAIR>(p, phase, unit);  // before the wait: a thousand cycles
          if (product > 0) {
            const unsigned all = gridDim.x * (unsigned)product;
            unsigned there = 0;
            for (uint32_t k = 0; k < p.polls && there < all && !*abort_flag; ++k)
              asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(p.arrived) : "memory");
            if (there < all || there >= kGaveUp) {
              if (there < all && !*abort_flag) record_status(p.status, 97);
              *abort_flag = 1;
              ok = false;
              break;
            }
            mbar_arrive(go);
          }
          asm volatile("fence.proxy.async.global;" ::: "memory");  // the parts were written by ordinary stores
          for (int i = unit; i < items && ok; i += units) {
            if (i != unit) t = tile_of<W, PAIR>(p, phase, i);
            const int wide = WIDE_ONES ? wide_ones >> t.q & 1 : 0, from = product / 3 + wide & 1;
            const CUtensorMap* map_a = phase == kGram ? &p.x_left[from][t.q] : (phase == kSquare ? &p.g_left[t.q] : &p.s_left[t.q]);
            const CUtensorMap* map_b = phase == kGram ? &p.x_right[from][t.q] : (phase == kSquare ? &p.g_right[t.q] : &p.x_apply[from][t.q]);
            for (int kb = t.k0, z = wide; kb < t.k1 && ok; ++it) {  // from plane z on
              const int st = it % kStages;
              if (it >= kStages) ok = parts::wait(empty(st), (it / kStages - 1) & 1, p.status, 91, abort_flag);
              if (!ok) break;
              const uint32_t dst = base + st * M::stage;
              if (rank == 0) mbar_expect_tx(full(st), M::stage << PAIR);
              load_3d<PAIR>(dst, map_a, kb * kBlockK, t.row + rank * kTileM, z, full(st));
              const int col = t.col + rank * M::right;
              if (phase == kApply) {
  #pragma unroll
                for (int j = 0; j < M::right / 64; ++j) load_3d<PAIR>(dst + (4 + 2 * j) * kBox, map_b, col + j * 64, kb * kBlockK, z, full(st));
              } else {
                load_3d<PAIR>(dst + 4 * kBox, map_b, kb * kBlockK, col, z, full(st));
              }
              if (z == 0) {
                ++kb;
                z = wide;
              } else {
                z = 0;
              }
            }
          }
        }
        if (!ok) asm volatile("red.relaxed.gpu.global.or.b32 [%0], %1;" ::"l"(p.arrived), "r"(kGaveUp) : "memory");
        // what the MMA warp tells of the last stages has arrived before the CTA may leave, and copies that nobody has waited for have landed
        for (int i = it > kStages ? it - kStages : 0; ok && i < it; ++i) ok = parts::wait(empty(i % kStages), (i / kStages) & 1, p.status, 99, abort_flag);
        if (!ok && rank == 0)
          for (int i = it > kStages ? it - kStages : 0; i < it; ++i) mbar_wait(full(i % kStages), (i / kStages) & 1, p.status, 92);
      }
    } else if (warp == M::mma) {
      if (rank == 0) {
      // Descriptors as in parts_common.cuh: groups of 8 rows (of 8 K) 1024 bytes apart, 128-byte swizzle; where the columns lie side by side instead of
      // the reduction, groups of 64 columns, both planes of them, 2 * kBox apart.
      constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
      constexpr uint32_t lbo = (2 * kBox >> 4) << 16, slot_a = 32 >> 4;  // mma_block has the latter as 2
      int it = 0;
      uint32_t chunks = 0;
      for (int product = 0; product < 3 * p.steps && ok; ++product) {
        const int phase = product % 3, items = p.items[phase];
        const uint32_t slot_b = phase == kApply ? 2048 >> 4 : 32 >> 4;
        const uint32_t idesc_f16 = (1u << 4) | (uint32_t)(phase == kApply) << 16 | (uint32_t)(M::rows >> 4) << 24 | (uint32_t)(W >> 3) << 17;
        for (int i = unit; i < items && ok; i += units) {
          const Tile t = tile_of<W, PAIR>(p, phase, i);
          const bool wide = WIDE_ONES && (wide_ones >> t.q & 1);
          const int depth = phase == kGram ? p.item[t.q].n : p.item[t.q].m, chunk = chunk_of<W>(depth, wide);
          const uint32_t idesc = idesc_f16 | (wide ? 1u << 7 | 1u << 10 : 0u);
          for (int kb = t.k0, z = wide, in_chunk = 0; kb < t.k1 && ok; ++it) {
            const int st = it % kStages;
            const bool first = in_chunk == 0, last = z == 0 && (wide || in_chunk + 1 == chunk || kb + 1 == t.k1);
            in_chunk = last ? 0 : in_chunk + 1;
            const uint32_t a = ((base + st * M::stage) >> 4 & 0x3FFF) | lbo, b = ((base + st * M::stage + 4 * kBox) >> 4 & 0x3FFF) | lbo;
            const uint32_t a_lo = a + (2 * kBox >> 4), b_lo = b + ((phase == kApply ? 1 : M::right / 64) * kBox >> 4), second = chunks & 1;
            const uint32_t d = tmem + kSecond * second, more = !first;
            const int slots = min(kBlockK, depth - kb * kBlockK + 15) / 16;  // what is behind the reduction is zeros
            ok = parts::wait(full(st), (it / kStages) & 1, p.status, 93, abort_flag);
            if (ok && first && chunks > 1) ok = parts::wait(acc_empty + 8 * second, ((chunks >> 1) - 1) & 1, p.status, 94, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            if (wide) {  // a, a_lo: the first and last parts, or the middle and first
              if (z == 0)
                for (int k = 0; k < slots; ++k) mma_one<PAIR>(d, a + k * slot_a, b + k * slot_b, desc_hi, idesc, 1);
              for (int k = 0; k < slots; ++k) {
                mma_one<PAIR>(d, a + k * slot_a, b_lo + k * slot_b, desc_hi, idesc, more | (uint32_t)(k > 0));
                mma_one<PAIR>(d, a_lo + k * slot_a, b + k * slot_b, desc_hi, idesc, 1);
              }
              if (z == 0)
                for (int k = 0; k < slots; ++k) mma_one<PAIR>(d, a_lo + k * slot_a, b_lo + k * slot_b, desc_hi, idesc, 1);
            } else if (slots == kBlockK / 16) {
              mma_block<PAIR>(d, a, a_lo, b, b_lo, slot_b, desc_hi, idesc, more);
            } else {
              for (int k = 0; k < slots; ++k) {
                mma_one<PAIR>(d, a + k * slot_a, b_lo + k * slot_b, desc_hi, idesc, more | (uint32_t)(k > 0));
                mma_one<PAIR>(d, a_lo + k * slot_a, b + k * slot_b, desc_hi, idesc, 1);
              }
              for (int k = 0; k < slots; ++k) mma_one<PAIR>(d, a + k * slot_a, b + k * slot_b, desc_hi, idesc, 1);
            }
            kb += z == 0;
            z = z == 0 && wide;
            commit<PAIR>(empty(st));
            if (last) {
              commit<PAIR>(acc_full + 8 * second);
              ++chunks;
            }
          }
        }
      }
      }
    } else {
      Accumulators acc;
      acc.rank = rank;
      acc.quad = warp & 3;
      acc.group = warp >> 2;
      acc.lane = lane;
      acc.sums = tmem + ((uint32_t)(acc.quad * 32) << 16) + acc.group * M::cols;
      acc.full = acc_full;
      acc.empty = acc_empty;
      acc.chunks = 0;
      acc.ok = true;
      acc.wide = wide_ones;
      acc.abort = abort_flag;
      acc.drawn = reinterpret_cast<volatile int*>(tmem_slot + 2);
      acc.slab = reinterpret_cast<float*>(smem + M::slab);
      for (int step = 0; step < p.steps; ++step) {
  #pragma unroll 1
        for (int phase = 0; phase < 3; ++phase) {
          const int product = 3 * step + phase;
          if (product > 0 && acc.ok) acc.ok = __all_sync(0xffffffffu, parts::wait(go, (product - 1) & 1, p.status, 98, abort_flag));
          if (phase == kGram) finish_tiles<kGram, W, PAIR, WIDE_ONES>(p, acc, step);
          else if (phase == kSquare) finish_tiles<kSquare, W, PAIR, WIDE_ONES>(p, acc, step);
          else if (step + 1 < p.steps) finish_tiles<kApply, W, PAIR, WIDE_ONES>(p, acc, step);
          else finish_tiles<kResult, W, PAIR, WIDE_ONES>(p, acc, step);
          if (product + 1 == 3 * p.steps) break;
          asm volatile("bar.sync 1, %0;" ::"n"(M::warps * 32) : "memory");
          if (threadIdx.x == 0 && !*abort_flag) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p.arrived) : "memory");
        }
      }
    }
  };
  if (wide_ones == 0) run(std::false_type());
  else run(std::true_type());
  tc_fence_before();
  if (PAIR) cg::this_cluster().sync();  // neither leaves while the other still uses its memory
  else __syncthreads();
  if (warp == M::mma) {
    tc_fence_after();
    release<PAIR>(tmem);
  }
}

__device__ __forceinline__ unsigned long long faint_below(int64_t elements) { return (unsigned long long)max(elements, (int64_t)64) << 18; }  // (sqrt(k) 2^-21)^2 2^60
__device__ __forceinline__ void add_size(unsigned long long* to, float sum, int64_t elements) {
  if (sum > 0.f && __ldcg(to) < faint_below(elements)) atomicAdd(to, max(1ull, (unsigned long long)(sum * 0x1p60f)));
}
// X as parts, of either kind: the update divided by its norm, its shorter side first.  Tiles of 64 x 64, turned in shared memory where that is
// the columns.  And the sums of the squares of X's rows and columns, in units of 2^-60 (the sum of all is 1), so that the order in which tiles are
// added does not matter; one that is not zero counts one unit at least, and one that is known not to be faint is left as it is (adding on and on to few
// rows: 64 x 500000 took 0.1 ms more).
struct Parts {
  Update u[kGroup];
  int64_t rows[kGroup], cols[kGroup];
  const double* sums[kGroup];
  uint16_t *x[kGroup], *x_wide[kGroup];
  unsigned long long* sizes[kGroup];  // of the rows, then the columns of X
  int ldx[kGroup];
  unsigned first[kGroup + 1];  // tiles of the matrices before
  int count;
  unsigned *tickets, tickets_end;
};
__global__ void __launch_bounds__(kThreads) parts_kernel(const __grid_constant__ Parts p) {
  RT_PDL_ENTRY();
  __shared__ float tile[64][65];
  __shared__ float2 by;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < p.tickets_end; i += gridDim.x * kThreads) p.tickets[i] = 0;
  int q = 0;
  while (blockIdx.x >= p.first[q + 1]) ++q;
  const Update u = p.u[q];
  const int64_t rows = p.rows[q], cols = p.cols[q];
  const unsigned local = blockIdx.x - p.first[q], tiles_c = (unsigned)((cols + 63) / 64);
  const int64_t r0 = (int64_t)(local / tiles_c) * 64, c0 = (int64_t)(local % tiles_c) * 64;
  if (threadIdx.x < 32) {
    const float2 f = one_over_norm(p.sums[q]);
    if (threadIdx.x == 0) by = f;
  }
  const int lane = threadIdx.x & 63, row = threadIdx.x >> 6;
  float v[16];
  const int64_t at = (r0 + row) * cols + c0 + lane, jump = 4 * cols;
  const int left = c0 + lane < cols ? (int)min((int64_t)64, rows - r0) - row : 0;
  const float* from = (u.g ? (u.nesterov ? u.g : u.m) : u.x) + at;  // of the update, what there is one of (update_at)
#pragma unroll
  for (int k = 0; k < 16; ++k, from += jump) v[k] = 4 * k < left ? *from : 0.f;
  if (u.g && u.nesterov) {
    const float* m = u.m + at;
#pragma unroll
    for (int k = 0; k < 16; ++k, m += jump) v[k] = u.scale * v[k] + (4 * k < left ? u.mu * *m : 0.f);
  }
  __syncthreads();
  const bool tall = rows > cols;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float w = v[k] * by.x * by.y;
    if (tall) tile[lane][row + 4 * k] = w;
    else tile[row + 4 * k][lane] = w;
  }
  __syncthreads();
  const int64_t m = tall ? cols : rows, n = tall ? rows : cols, y0 = tall ? c0 : r0, x0 = tall ? r0 : c0, ld = p.ldx[q], plane = m * ld;
  {  // four threads a row, four a column; what is outside is zeros, or NaN if the norm is
    const int line = threadIdx.x >> 2, k0 = (threadIdx.x & 3) * 16;
    float of_row = 0.f, of_col = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float a = tile[line][k0 + k], b = tile[k0 + k][line];
      of_row += a != 0.f ? fmaxf(a * a, 0x1p-100f) : 0.f;
      of_col += b != 0.f ? fmaxf(b * b, 0x1p-100f) : 0.f;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      of_row += __shfl_xor_sync(0xffffffffu, of_row, o);
      of_col += __shfl_xor_sync(0xffffffffu, of_col, o);
    }
    if (k0 == 0 && y0 + line < m) add_size(p.sizes[q] + y0 + line, of_row, n);
    if (k0 == 0 && x0 + line < n) add_size(p.sizes[q] + m + x0 + line, of_col, m);
  }
  const int pair = threadIdx.x & 31, y = threadIdx.x >> 5, high = x0 + 2 * pair < ld ? (int)min((int64_t)64, m - y0) - y : 0;  // the padding of a row: zeros
  const int64_t at_o = (y0 + y) * ld + x0 + 2 * pair;
  uint16_t *o = p.x[q] + at_o, *o_wide = p.x_wide[q] + at_o;
#pragma unroll
  for (int k = 0; k < 8; ++k, o += 8 * ld, o_wide += 8 * ld) {
    if (8 * k >= high) break;
    const float a = tile[y + 8 * k][2 * pair], b = tile[y + 8 * k][2 * pair + 1];
    uint32_t hi, lo, w[kPlanes];
    split2(a, b, kScale, hi, lo);
    *reinterpret_cast<uint32_t*>(o) = hi;
    *reinterpret_cast<uint32_t*>(o + plane) = lo;
    split3(a, b, w);
#pragma unroll
    for (int i = 0; i < kPlanes; ++i) *reinterpret_cast<uint32_t*>(o_wide + i * plane) = w[i];
  }
}
// Which matrices have a row or column that is too faint for two parts (see above).  3 us by itself, 2 in a row with the others.
struct Faint {
  const unsigned long long* sizes[kGroup];
  int64_t m[kGroup], n[kGroup];
  unsigned* wide;
};
__global__ void __launch_bounds__(kThreads) faint_kernel(const __grid_constant__ Faint p) {
  RT_PDL_ENTRY();
  const int q = blockIdx.y;
  const unsigned long long* sizes = p.sizes[q];
  const int64_t m = p.m[q], n = p.n[q];
  bool faint = false;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < m + n; i += (int64_t)gridDim.x * kThreads) {
    const unsigned long long v = __ldg(sizes + i);
    faint |= v != 0 && v < faint_below(i < m ? n : m);
  }
  if (__syncthreads_or(faint) && threadIdx.x == 0) atomicOr(p.wide, 1u << q);
}

// [kPlanes][rows][cols] 16-bit values, rows ld apart, boxes of 64 columns and `height` rows of two planes, zeros outside.
bool map_planes(CUtensorMap* map, uint16_t* t, int64_t cols, int64_t rows, int64_t ld, int height) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, kPlanes}, strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(ld * rows) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)height, 2}, one[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, t, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How the tiles are laid out over the SMs: their width (64: of one CTA, 128 and 256: of a pair), and into how many parts the reduction of each
// matrix's tiles is split, by product.
struct Plan {
  int width, splits[3][kGroup];
};
int rows_of_tile(int width) { return width == 64 ? kTileM : 2 * kTileM; }
int64_t tiles_of(int phase, int width, int64_t m, int64_t n) {
  const int64_t height = rows_of_tile(width), rows = (m + height - 1) / height;
  if (phase == kApply) return rows * ((n + width - 1) / width);
  if (width == height) return rows * (rows + 1) / 2;
  const int64_t all = rows * (rows + 1);
  return (rows - 1) * height + width >= m ? all - 1 : all;  // the last one has no columns
}
// What a tile takes in cycles: for a K-block, besides, if its reduction is shared, and for each CTA that shares it.  A product takes as many rounds as its
// work items need at one per CTA or pair, of the time that they take on average.  Fitted to 55 measurements, from 64 x 64 to 4096 x 4096 and 300 x 20000 and
// lists of up to 12, with each of the widths and two ways to share reductions: within 5 to 7 % (root of the mean square).  Microseconds with 64,
// 128 and 256 columns: 512 x 512 158, 206 and 340; 1400 x 1400 378, 378 and 553; 2048 x 2048 929, 638 and 756; 3000 x 3500 3227, 2477 and
// 2297; five matrices up to 2048 wide 501, 369 and 630.
struct Cost {
  double block, rest, shared, share;
};
constexpr Cost kCosts[3] = {{1140, 7600, 3600, 500}, {1400, 12600, 7000, 950}, {2230, 23900, 12200, 3900}};
Plan plan_products(const int (&fit)[3], int count, const Item* items) {
  Plan best{};
  double least = 1e300;
  for (int width = 64; width <= 256; width *= 2) {
    Plan p{};
    p.width = width;
    double sum = 0;
    const Cost& cost = kCosts[width / 128];
    const int units = fit[width / 128];
    if (units == 0) continue;
    for (int phase = 0; phase < 3; ++phase) {
      double least_here = 1e300;
      int deepest = 1;
      for (int q = 0; q < count; ++q)
        while (deepest < ((phase == kGram ? items[q].n : items[q].m) + kBlockK - 1) / kBlockK) deepest *= 2;
      for (int most = deepest; most >= 1; most /= 2) {  // K-blocks of a tile at most, where that needs it split
        int splits[kGroup];
        double work = 0, tiles = 0, longest = 0;
        for (int q = 0; q < count; ++q) {
          const int blocks = ((phase == kGram ? items[q].n : items[q].m) + kBlockK - 1) / kBlockK;
          splits[q] = (blocks + most - 1) / most;
          const double one = cost.block * ((blocks + splits[q] - 1) / splits[q]) + cost.rest + (splits[q] > 1 ? cost.shared + cost.share * splits[q] : 0);
          const double all = (double)tiles_of(phase, width, items[q].m, items[q].n) * splits[q];
          work += one * all;
          tiles += all;
          longest = std::max(longest, one);
        }
        const double time = std::max(longest, std::ceil(tiles / units) * work / tiles);
        if (time < least_here) {
          least_here = time;
          std::copy(splits, splits + count, p.splits[phase]);
        }
      }
      sum += least_here;
    }
    if (sum < least) {
      least = sum;
      best = p;
    }
  }
  return best;
}
template <int W, bool PAIR>
cudaLaunchConfig_t config(const rt_ctx* ctx, unsigned blocks, cudaLaunchAttribute (&at)[2]) {
  using M = Layout<W, PAIR>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
  cfg.blockDim = M::threads;
  cfg.dynamicSmemBytes = M::bytes;
  cfg.stream = ctx->stream;
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = PAIR ? 2 : 1;
  return cfg;
}
// How many CTAs or pairs the device runs at once, which is what waits for one another; asked once.
template <int W, bool PAIR>
rt_status units_of(rt_ctx* ctx, int* units) {
  if (*units >= 0) return RT_OK;
  using M = Layout<W, PAIR>;
  static RtDeviceOnce once;
  RT_CUDA(ctx, once([] { return cudaFuncSetAttribute(newton_schulz_kernel<W, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)M::bytes); }));
  int n = 0;
  if (PAIR) {
    cudaLaunchAttribute at[2];
    cudaLaunchConfig_t cfg = config<W, PAIR>(ctx, 2, at);
    cfg.attrs = at + 1;
    cfg.numAttrs = 1;
    RT_CUDA(ctx, cudaOccupancyMaxActiveClusters(&n, newton_schulz_kernel<W, PAIR>, &cfg));
  } else {
    RT_CUDA(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, newton_schulz_kernel<W, PAIR>, M::threads, M::bytes));
    n *= ctx->sm_count;
  }
  *units = std::min(n, ctx->sm_count >> PAIR);
  return RT_OK;
}
template <int W, bool PAIR>
rt_status launch_products(rt_ctx* ctx, const Product& p) {
  const int items = std::max(p.items[0], std::max(p.items[1], p.items[2]));
  cudaLaunchAttribute at[2];
  const cudaLaunchConfig_t cfg = config<W, PAIR>(ctx, (unsigned)std::min(items, ctx->muon_units[W / 128]) << PAIR, at);
  RT_CUDA(ctx, cudaLaunchKernelEx(&cfg, newton_schulz_kernel<W, PAIR>, p));
  RT_LAUNCHED(ctx);
  return RT_OK;
}

// Up to kGroup matrices together.  What may fail comes before the first launch: sizes, room and tensor maps.
struct Group {
  Product p{};
  Parts x{};
  Faint f{};
  Plan plan{};
  const Matrix* list = nullptr;
  int count = 0;
  size_t halves = 0, sizes = 0, partials = 0, tickets = 0, at[kGroup] = {};
  double* squares = nullptr;
  size_t bytes() const {
    return sizeof(uint16_t) * halves + sizeof(float) * partials + sizeof(double) * kNormBlocks * count + sizeof(unsigned long long) * (sizes + 1) +
           sizeof(unsigned) * (tickets + 1);
  }
};
void lay_out(const rt_ctx* ctx, const Matrix* list, int count, int steps, Group* group) {
  Product& p = group->p;
  group->list = list;
  group->count = p.count = group->x.count = count;
  p.status = ctx->device_status;
  p.polls = ctx->sequence_polls;
  p.steps = steps;
  for (int q = 0; q < count; ++q) {
    Item& i = p.item[q];
    i.m = (int)std::min(list[q].rows, list[q].cols);
    i.n = (int)std::max(list[q].rows, list[q].cols);
    i.ldx = (i.n + 7) / 8 * 8;
    i.ldm = (i.m + 7) / 8 * 8;
    group->at[q] = group->halves;
    group->halves += ((size_t)2 * kPlanes * i.m * (i.ldx + i.ldm) + 63) / 64 * 64;
    group->sizes += (size_t)(i.m + i.n);
    i.out = list[q].out;
    i.tall = list[q].rows > list[q].cols;
    i.update = list[q].update;
    i.vec = list[q].cols % 4 == 0 && rt_aligned16(i.out);
    i.keep = list[q].keep;
    i.step = list[q].step;
  }
  const Plan& plan = group->plan = plan_products(ctx->muon_units, count, p.item);
  for (int phase = 0; phase < 3; ++phase) {
    int items = 0, first_part = 0, first_ticket = 0;
    for (int q = 0; q < count; ++q) {
      Item& i = p.item[q];
      const int tiles = (int)tiles_of(phase, plan.width, i.m, i.n), splits = plan.splits[phase][q];
      i.splits[phase] = splits;
      i.first[phase] = items;
      i.first_part[phase] = first_part;
      i.first_ticket[phase] = first_ticket;
      items += tiles * splits;
      if (splits > 1) {
        first_part += tiles * splits;
        first_ticket += tiles;
      }
    }
    p.items[phase] = items;
    group->partials = std::max(group->partials, (size_t)first_part * plan.width * rows_of_tile(plan.width));
    group->tickets = std::max(group->tickets, (size_t)first_ticket * 2);
  }
}
// False if a tensor map cannot be had.
bool place(Group* group, void* memory) {
  Product& p = group->p;
  Parts& x = group->x;
  uint16_t* halves = static_cast<uint16_t*>(memory);
  p.sums = reinterpret_cast<float*>(halves + group->halves);
  group->squares = reinterpret_cast<double*>(p.sums + group->partials);
  unsigned long long *const zeros = reinterpret_cast<unsigned long long*>(group->squares + (size_t)kNormBlocks * group->count), *size = zeros + 1;
  p.wide = group->f.wide = reinterpret_cast<unsigned*>(zeros);
  p.tickets = reinterpret_cast<unsigned*>(zeros + 1 + group->sizes);
  p.arrived = p.tickets + group->tickets;
  unsigned tiles = 0;
  const int right = group->plan.width == 64 ? 64 : group->plan.width / 2;  // columns that a CTA brings in
  for (int q = 0; q < group->count; ++q) {
    const Matrix& of = group->list[q];
    Item& i = p.item[q];
    const size_t of_x = (size_t)kPlanes * i.m * i.ldx, of_g = (size_t)kPlanes * i.m * i.ldm;
    i.x[0] = halves + group->at[q];
    i.x[1] = i.x[0] + of_x;
    i.g = i.x[1] + of_x;
    i.s = i.g + of_g;
    bool mapped = map_planes(&p.g_left[q], i.g, i.m, i.m, i.ldm, kTileM) && map_planes(&p.g_right[q], i.g, i.m, i.m, i.ldm, right) &&
                  map_planes(&p.s_left[q], i.s, i.m, i.m, i.ldm, kTileM);
    for (int k = 0; k < 2; ++k)
      mapped = mapped && map_planes(&p.x_left[k][q], i.x[k], i.n, i.m, i.ldx, kTileM) && map_planes(&p.x_right[k][q], i.x[k], i.n, i.m, i.ldx, right) &&
               map_planes(&p.x_apply[k][q], i.x[k], i.n, i.m, i.ldx, 64);
    if (!mapped) return false;
    x.u[q] = of.u;
    x.rows[q] = of.rows;
    x.cols[q] = of.cols;
    x.sums[q] = group->squares + (size_t)kNormBlocks * q;
    x.x[q] = i.x[0];
    x.x_wide[q] = i.x[1];
    group->f.sizes[q] = x.sizes[q] = size;
    size += i.m + i.n;
    group->f.m[q] = i.m;
    group->f.n[q] = i.n;
    x.ldx[q] = i.ldx;
    x.first[q] = tiles;
    tiles += (unsigned)((of.rows + 63) / 64 * ((of.cols + 63) / 64));
  }
  x.first[group->count] = tiles;
  x.tickets = p.tickets;
  x.tickets_end = (unsigned)group->tickets + 1;  // and the count of the blocks
  return true;
}
rt_status launch(rt_ctx* ctx, const Group& group) {
  rt_status st = launch_squares(ctx, group.list, group.count, 1, group.squares, group.x.sizes[0] - 1, (int64_t)group.sizes + 1);
  if (st != RT_OK) return st;
  rt_launch(ctx, parts_kernel, group.x.first[group.count], kThreads, 0, group.x);
  RT_LAUNCHED(ctx);
  int longest = 0;
  for (int q = 0; q < group.count; ++q) longest = std::max(longest, group.p.item[q].m + group.p.item[q].n);
  rt_launch(ctx, faint_kernel, dim3(rt_grid_for(ctx, longest, kThreads), group.count), kThreads, 0, group.f);
  RT_LAUNCHED(ctx);
  const int width = group.plan.width;
  return width == 256 ? launch_products<256, true>(ctx, group.p) : (width == 128 ? launch_products<128, true>(ctx, group.p) : launch_products<64, false>(ctx, group.p));
}

// ---- by the framework's other products: without tensor cores, or with no steps ------------------------------------------------------------
size_t bytes_otherwise(const Matrix& q) {
  const size_t m = (size_t)std::min(q.rows, q.cols), n = (size_t)std::max(q.rows, q.cols);
  return sizeof(double) * kNormBlocks + sizeof(float) * (2 * m * n + 2 * m * m);
}
// The momentum is written with the result: a product may not find room for itself.
rt_status orthogonalize(rt_ctx* ctx, const Matrix& q, int steps, void* memory) {
  const int64_t m = std::min(q.rows, q.cols), n = std::max(q.rows, q.cols), all = m * n;
  double* sums = static_cast<double*>(memory);
  float *x = reinterpret_cast<float*>(sums + kNormBlocks), *y = x + all, *g = y + all, *s = g + m * m;
  rt_status st = launch_squares(ctx, &q, 1, 0, sums);
  if (st != RT_OK) return st;
  rt_launch(ctx, normalise_kernel, rt_grid_for(ctx, all, kThreads), kThreads, 0, q.u, q.rows, q.cols, sums, x);
  RT_LAUNCHED(ctx);
  for (int k = 0; k < steps; ++k) {
    if ((st = rt_gemm(ctx, 0, 1, m, m, n, x, n, x, n, g, m, 0)) != RT_OK) return st;
    if ((st = rt_gemm(ctx, 0, 0, m, m, m, g, m, g, m, s, m, 0)) != RT_OK) return st;
    rt_launch(ctx, polynomial_kernel, rt_grid_for(ctx, m * m, kThreads), kThreads, 0, g, m, s);
    RT_LAUNCHED(ctx);
    if ((st = rt_gemm(ctx, 0, 0, m, n, m, s, m, x, n, y, n, 0)) != RT_OK) return st;
    std::swap(x, y);
  }
  rt_launch(ctx, apply_kernel, rt_grid_for(ctx, all, kThreads), kThreads, 0, x, q.rows, q.cols, q.out, q.update, q.keep, q.step, q.u);
  RT_LAUNCHED(ctx);
  return RT_OK;
}
// Everything is ready before the first launch, which changes momenta.
rt_status orthogonalize_all(rt_ctx* ctx, const std::vector<Matrix>& list, int steps) {
  if (list.empty()) return RT_OK;
  rt_status st = RT_OK;
  bool together = steps > 0 && ctx->use_tensor_cores;
  int(&units)[3] = ctx->muon_units;
  if (together) {
    if ((st = units_of<64, false>(ctx, &units[0])) != RT_OK || (st = units_of<128, true>(ctx, &units[1])) != RT_OK ||
        (st = units_of<256, true>(ctx, &units[2])) != RT_OK)
      return st;
    together = units[0] || units[1] || units[2];
  }
  if (together) {
    RtScratch work(ctx);
    std::vector<Group> groups((list.size() + kGroup - 1) / kGroup);
    size_t bytes = 0;
    for (size_t k = 0; k < groups.size(); ++k) {
      lay_out(ctx, &list[k * kGroup], (int)std::min<size_t>(kGroup, list.size() - k * kGroup), steps, &groups[k]);
      bytes = std::max(bytes, groups[k].bytes());
    }
    if ((st = work.alloc(bytes)) != RT_OK) return st;
    for (Group& g : groups) together = together && place(&g, work.ptr);
    for (size_t k = 0; together && st == RT_OK && k < groups.size(); ++k) st = launch(ctx, groups[k]);
    if (together) return st;
  }
  RtScratch work(ctx);
  size_t bytes = 0;
  for (const Matrix& q : list) bytes = std::max(bytes, bytes_otherwise(q));
  if ((st = work.alloc(bytes)) != RT_OK) return st;
  for (const Matrix& q : list)
    if ((st = orthogonalize(ctx, q, steps, work.ptr)) != RT_OK) return st;
  return RT_OK;
}

rt_status check_sizes(rt_ctx* ctx, const char* who, int count, const int64_t* rows, const int64_t* cols, int steps) {
  if (count < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: %d matrices", who, count);
  if (steps < 0 || steps > 64) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: between 0 and 64 steps, got %d", who, steps);
  if (count == 0) return RT_OK;
  RT_CHECK_PTR(ctx, rows);
  RT_CHECK_PTR(ctx, cols);
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 0 || cols[i] < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: negative size", who);
    if (rows[i] >= (1 << 24) || cols[i] >= (1 << 24) || std::min(rows[i], cols[i]) > 65536) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: size out of range", who);
  }
  return RT_OK;
}
struct Block {
  uintptr_t begin, end;
  bool written;
};
Block block_of(const float* p, int64_t n, bool written) { return {(uintptr_t)p, (uintptr_t)(p + n), written}; }
// Whether nothing that is written overlaps anything else.
bool apart(std::vector<Block> blocks) {
  std::sort(blocks.begin(), blocks.end(), [](const Block& a, const Block& b) { return a.begin < b.begin; });
  uintptr_t end = 0, written = 0;  // of all blocks so far, of those that are written
  for (size_t i = 0; i < blocks.size(); ++i) {
    const Block& b = blocks[i];
    if (b.begin < (b.written ? end : written)) return false;
    end = std::max(end, b.end);
    if (b.written) written = std::max(written, b.end);
  }
  return true;
}

}  // namespace

extern "C" {

rt_status rt_orthogonalize_list(rt_ctx* ctx, int count, const float* const* xs, const int64_t* rows, const int64_t* cols, int steps, float* const* outs) {
  RT_CHECK_CTX(ctx);
  rt_status st = check_sizes(ctx, "rt_orthogonalize_list", count, rows, cols, steps);
  if (st != RT_OK || count == 0) return st;
  RT_CHECK_PTR(ctx, xs);
  RT_CHECK_PTR(ctx, outs);
  try {
    std::vector<Matrix> list;
    std::vector<Block> blocks;
    for (int i = 0; i < count; ++i) {
      if (rows[i] == 0 || cols[i] == 0) continue;
      RT_CHECK_PTR(ctx, xs[i]);
      RT_CHECK_PTR(ctx, outs[i]);
      if (xs[i] != outs[i]) blocks.push_back(block_of(xs[i], rows[i] * cols[i], false));  // in place: nobody else's
      blocks.push_back(block_of(outs[i], rows[i] * cols[i], true));
      Matrix q{};
      q.u.x = xs[i];
      q.rows = rows[i];
      q.cols = cols[i];
      q.out = outs[i];
      list.push_back(q);
    }
    if (!apart(blocks)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_orthogonalize_list: a result overlaps another or another's matrix");
    RtOnDevice here(ctx);
    if ((st = orthogonalize_all(ctx, list, steps)) != RT_OK) return st;
  } catch (const std::bad_alloc&) {
    RT_FAIL(ctx, RT_ERR_OOM, "rt_orthogonalize_list: out of host memory");
  }
  return RT_OK;
}

rt_status rt_muon_step_multi(rt_ctx* ctx, int n_tensors, float* const* params, const float* const* grads, float* const* momenta, const int64_t* rows,
                             const int64_t* cols, float lr, float momentum, int nesterov, float weight_decay, int steps, float grad_scale) {
  RT_CHECK_CTX(ctx);
  rt_status st = check_sizes(ctx, "rt_muon_step_multi", n_tensors, rows, cols, steps);
  if (st != RT_OK || n_tensors == 0) return st;
  RT_CHECK_PTR(ctx, params);
  RT_CHECK_PTR(ctx, grads);
  RT_CHECK_PTR(ctx, momenta);
  try {
    std::vector<Matrix> list;
    std::vector<Block> blocks;
    for (int i = 0; i < n_tensors; ++i) {
      if (rows[i] == 0 || cols[i] == 0) continue;
      RT_CHECK_PTR(ctx, params[i]);
      RT_CHECK_PTR(ctx, grads[i]);
      RT_CHECK_PTR(ctx, momenta[i]);
      blocks.push_back(block_of(params[i], rows[i] * cols[i], true));
      blocks.push_back(block_of(grads[i], rows[i] * cols[i], false));
      blocks.push_back(block_of(momenta[i], rows[i] * cols[i], true));
      Matrix q{};
      q.u = {nullptr, grads[i], momenta[i], momentum, grad_scale, nesterov};
      q.rows = rows[i];
      q.cols = cols[i];
      q.out = params[i];
      q.update = 1;
      q.keep = 1.f - lr * weight_decay;
      q.step = (float)(lr * std::sqrt(std::max(1.0, (double)cols[i] / (double)rows[i])));
      list.push_back(q);
    }
    if (!apart(blocks)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_muon_step_multi: a parameter or momentum overlaps another or a gradient");
    RtOnDevice here(ctx);
    if ((st = orthogonalize_all(ctx, list, steps)) != RT_OK) return st;
  } catch (const std::bad_alloc&) {
    RT_FAIL(ctx, RT_ERR_OOM, "rt_muon_step_multi: out of host memory");
  }
  return RT_OK;
}

}  // extern "C"
