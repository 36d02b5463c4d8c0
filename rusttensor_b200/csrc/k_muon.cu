// Muon: an optimizer step whose update is the momentum with its singular values brought near one.
//
//   m = mu m + s g      u = m, or s g + mu m (nesterov)      p = (1 - lr wd) p - lr sqrt(max(1, cols / rows)) O(u)
//
// O(u) comes from Newton-Schulz steps on X = u / (|u| + 1e-7): X <- (a I + b G + c G^2) X with G = X X^T, which takes every singular value x to
// a x + b x^3 + c x^5, with the published coefficients 3.4445, -4.7750, 2.0315: five steps bring values between 0.002 and 1 to between 0.7 and
// 1.2.  G is taken on the shorter side; a matrix with more rows than columns is transposed for the steps.
//
// A step is three products, each of which has to wait for the one before: G = X X^T and b G + c G^2, both symmetric, of which the lower half is
// computed and written twice, and a X + (b G + c G^2) X.  Errors of early steps grow (small singular values by 3.4 a step), so the products
// keep fp32's precision: an operand is held as two fp16 parts, hi = fp16(2^12 x) and lo = fp16(2^11 (2^12 x - hi)), 22 bits, and a product is
// three tcgen05.mma of kind::f16, hi hi to one accumulator, hi lo and lo hi to another.  No element of X, G or the polynomial is beyond 3 (their
// singular values are at most 1.21, 1.46 and 2.81), so the scale is fixed and nothing is looked at beforehand.  A product's epilogue adds what
// the formula adds and writes the parts that the next product reads, as they lie: X [m][n] is an operand with n as the reduction, and with
// m, by tensor maps and MMA descriptors of either kind.  All matrices of a call go through every product together, as tiles of one launch.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "parts_common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr double kEpsilon = 1e-7;
constexpr int kNormBlocks = 128;

struct Update {
  const float* x;  // what is orthogonalised; with a gradient: made of it and the momentum
  const float* g;
  float* m;
  float mu, scale;
  int nesterov;
};
__device__ __forceinline__ float update_at(const Update& u, int64_t i) {
  if (!u.g) return __ldg(u.x + i);
  return u.nesterov ? u.scale * __ldg(u.g + i) + u.mu * u.m[i] : u.m[i];
}
// The new momentum, and the sum of the squares of the update, block by block in 64 bits: squares of large fp32 values have no room in 32.
__global__ void __launch_bounds__(kThreads) squares_kernel(const Update u, int64_t n, double* __restrict__ sums) {
  RT_PDL_ENTRY();
  __shared__ double of_warp[kThreads / 32];
  double sum = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    if (u.g) u.m[i] = u.mu * u.m[i] + u.scale * __ldg(u.g + i);
    const double v = update_at(u, i);
    sum += v * v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) sum += of_warp[w];
    sums[blockIdx.x] = sum;
  }
}
// X: the update divided by its norm, its shorter side first.
__global__ void __launch_bounds__(kThreads) normalise_kernel(const Update u, int64_t rows, int64_t cols, const double* __restrict__ sums, float* __restrict__ x) {
  RT_PDL_ENTRY();
  double sum = 0.0;
  for (int b = 0; b < kNormBlocks; ++b) sum += __ldg(sums + b);
  const float by = (float)(1.0 / (sqrt(sum) + kEpsilon));
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / cols, c = i - r * cols;
    x[rows > cols ? c * rows + r : i] = update_at(u, i) * by;
  }
}
// s = a I + b g + c s
__global__ void __launch_bounds__(kThreads) polynomial_kernel(const float* __restrict__ g, int64_t m, float* __restrict__ s) {
  RT_PDL_ENTRY();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < m * m; i += (int64_t)gridDim.x * kThreads)
    s[i] = kB * __ldg(g + i) + kC * s[i] + (i / m == i % m ? kA : 0.f);
}
// out = keep * out - step * x, or out = x
__global__ void __launch_bounds__(kThreads) apply_kernel(const float* __restrict__ x, int64_t rows, int64_t cols, float* __restrict__ out, int update, float keep,
                                                         float step) {
  RT_PDL_ENTRY();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / cols, c = i - r * cols;
    const float o = __ldg(x + (rows > cols ? c * rows + r : i));
    out[i] = update ? keep * out[i] - step * o : o;
  }
}

struct Matrix {
  Update u;
  int64_t rows, cols;
  float* out;
  int update;
  float keep, step;
};

// ---- the products on the tensor cores -----------------------------------------------------------------------------------------------
using namespace tc;
using parts::kBox;

constexpr int kGroup = 16;                 // matrices of a launch
constexpr float kScale = 4096.f, kLow = 2048.f;
constexpr int kTileM = 128, kBlockK = 64;  // rows of a tile; elements of the reduction that a stage holds
constexpr int kProductThreads = 320, kEpilogueWarps = 8, kTmaWarp = 8, kMmaWarp = 9;
constexpr uint32_t kCross = 256;           // tensor-memory column of the cross terms
enum { kGram, kSquare, kApply };

struct Item {
  int m, n;              // m <= n
  int ldx, ldm;          // halves between rows of X, of G and the polynomial
  uint16_t *x[2], *g, *s;
  int first, splits;     // of this product: first work item of the matrix, CTAs that share a tile's reduction
  int first_part;        // tile partial sums of matrices before, in tiles
  int first_ticket;
  // the result
  float* out;
  int tall, update;      // X is transposed against out
  float keep, step;
};
struct Product {
  CUtensorMap x[2][kGroup], g[kGroup], s[kGroup];
  Item item[kGroup];
  int count, items;
  int from;              // which of the two X is read
  int last;              // the result goes to `out`
  int chunk;             // K-blocks that the accumulator of hi * hi sums before it is emptied: it adds with truncation
  float* sums;           // partial sums of tiles, [128 columns or 256][128 rows] each
  unsigned* tickets;     // zero between launches
  int* status;
};
template <int W>
struct Smem {
  static constexpr uint32_t stage = (2 * kTileM + 2 * W) / 64 * kBox, stages = W == 256 ? 2 : 3;
  static constexpr uint32_t bars = stages * stage, bytes = bars + (2 * stages + 3) * 8 + 16 + 1024;
  static_assert(bytes <= 232448, "shared memory");
};
struct Tile {
  int q, row, col, k0, k1, split, index;  // K-blocks k0 .. k1; index: among the matrix's tiles
};
template <int PHASE, int W>
__device__ __forceinline__ Tile tile_of(const Product& p, int i) {
  int q = 0;
  while (q + 1 < p.count && i >= p.item[q + 1].first) ++q;
  const Item& a = p.item[q];
  Tile t;
  t.q = q;
  const int local = i - a.first;
  t.split = local % a.splits;
  t.index = local / a.splits;
  const int m_tiles = (a.m + kTileM - 1) / kTileM;
  if (PHASE == kApply) {
    t.row = t.index % m_tiles * kTileM;
    t.col = t.index / m_tiles * W;
  } else if (W == kTileM) {  // the lower half, row by row: 1 + 2 + 3 + ... tiles
    int r = (int)((sqrtf(8.f * t.index + 1.f) - 1.f) * 0.5f);
    while (r * (r + 1) / 2 > t.index) --r;
    while ((r + 1) * (r + 2) / 2 <= t.index) ++r;
    t.row = r * kTileM;
    t.col = (t.index - r * (r + 1) / 2) * W;
  } else {  // 1 + 1 + 2 + 2 + 3 + 3 + ...
    int r = (int)((sqrtf(4.f * t.index + 1.f) - 1.f) * 0.5f);
    while (r * (r + 1) > t.index) --r;
    while ((r + 1) * (r + 2) <= t.index) ++r;
    const int in = t.index - r * (r + 1);
    t.row = (2 * r + (in > r)) * kTileM;
    t.col = (in > r ? in - r - 1 : in) * W;
  }
  const int k_blocks = ((PHASE == kGram ? a.n : a.m) + kBlockK - 1) / kBlockK;
  t.k0 = (int)((int64_t)k_blocks * t.split / a.splits);
  t.k1 = (int)((int64_t)k_blocks * (t.split + 1) / a.splits);
  return t;
}
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
// Two neighbouring values as parts.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  a *= kScale;
  b *= kScale;
  const __half2 h = __floats2half2_rn(a, b);
  const float2 back = __half22float2(h);
  const __half2 l = __floats2half2_rn((a - back.x) * kLow, (b - back.y) * kLow);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ float2 join2(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi)), l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return make_float2((h.x + l.x * (1.f / kLow)) * (1.f / kScale), (h.y + l.y * (1.f / kLow)) * (1.f / kScale));
}
// What of eight values of a row is added to the product: `by` times what the parts at p (hi; lo a plane behind) hold.
__device__ __forceinline__ void add_parts(float (&v)[8], const uint16_t* p, int64_t plane, float by) {
  const uint4 h = *reinterpret_cast<const uint4*>(p), l = *reinterpret_cast<const uint4*>(p + plane);
  const uint32_t hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = join2(hs[k], ls[k]);
    v[2 * k] += by * f.x;
    v[2 * k + 1] += by * f.y;
  }
}
// Eight values of row r, columns c .. c + 7, of a symmetric matrix [m][m], of which those up to the diagonal are to be written, here and mirrored.
// The lanes of the warp have 32 rows one after the other.
__device__ __forceinline__ void write_symmetric(uint16_t* p, int64_t plane, int ld, int m, int r, int c, const float (&v)[8]) {
  if (r >= m) return;
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) split2(v[2 * k], v[2 * k + 1], hi[k], lo[k]);
  uint16_t* at = p + (int64_t)r * ld + c;
  const bool whole = c + 7 <= r;
  if (whole) {
    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(at + plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint16_t h = (uint16_t)(hi[k / 2] >> (k & 1) * 16), l = (uint16_t)(lo[k / 2] >> (k & 1) * 16);
    if (!whole && c + k <= r) {
      at[k] = h;
      at[k + plane] = l;
    }
    if (c + k < r) {
      uint16_t* mirror = p + (int64_t)(c + k) * ld + r;
      mirror[0] = h;
      mirror[plane] = l;
    }
  }
}

// Roles of a CTA, one per SM, that walks over tiles of 128 x W: a TMA warp some K-blocks of 64 ahead, an MMA warp, eight warps that empty the
// accumulators into registers and write the result.  Where the tiles are fewer than the SMs, several CTAs share a tile's reduction: each leaves its
// sums in memory, and the one that draws the last ticket adds them up in their order.  A K-block takes 12 MMAs; for W = 128 what crosses the
// shared memory bounds them (107 cycles each instead of 64), for W = 256 it is 160 instead of 128.  Every wait is bounded; on expiry the kernel records
// a code in the status word, raises a flag that all other waits poll, lets its own copies land, frees tensor memory and returns.
template <int PHASE, int W>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ Product p) {
  RT_PDL_ENTRY();
  using M = Smem<W>;
  constexpr int kStages = M::stages;
  extern __shared__ char smem_raw[];
  __shared__ volatile int abort_flag;
  __shared__ int drawn;
  const uint32_t raw_base = smem_u32(smem_raw), base = (raw_base + 1023) & ~1023u;
  char* smem = smem_raw + (base - raw_base);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t bars = base + M::bars;
  auto full = [&](int i) { return bars + 8 * i; };
  auto empty = [&](int i) { return bars + 8 * (kStages + i); };
  const uint32_t acc_full = bars + 16 * kStages, acc_empty = acc_full + 8, cross_empty = acc_full + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + M::bars + (2 * kStages + 3) * 8);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, kEpilogueWarps);
    mbar_init(cross_empty, kEpilogueWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) tmem_alloc(smem_u32(tmem_slot), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  bool ok = true;

  if (warp == kTmaWarp) {
    if (lane == 0) {
      asm volatile("fence.proxy.async.global;" ::: "memory");  // the parts were written by ordinary stores
      int it = 0;
      for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
        const Tile t = tile_of<PHASE, W>(p, i);
        const CUtensorMap* map_a = PHASE == kGram ? &p.x[p.from][t.q] : (PHASE == kSquare ? &p.g[t.q] : &p.s[t.q]);
        const CUtensorMap* map_b = PHASE == kSquare ? &p.g[t.q] : &p.x[p.from][t.q];
        const int boxes = (min(W, (PHASE == kApply ? p.item[t.q].n : p.item[t.q].m) - t.col) + 63) / 64;
        for (int kb = t.k0; kb < t.k1 && ok; ++kb, ++it) {
          const int st = it % kStages;
          if (it >= kStages) ok = parts::wait(empty(st), (it / kStages - 1) & 1, p.status, 91, &abort_flag);
          if (!ok) break;
          const uint32_t dst = base + st * M::stage;
          mbar_expect_tx(full(st), (4 + 2 * boxes) * kBox);
          for (int z = 0; z < 2; ++z) {
            for (int j = 0; j < 2; ++j) load_3d(dst + (2 * z + j) * kBox, map_a, kb * kBlockK, t.row + j * 64, z, full(st));
            for (int j = 0; j < boxes; ++j) {
              const int n = t.col + j * 64;
              load_3d(dst + (4 + z * (W / 64) + j) * kBox, map_b, PHASE == kApply ? n : kb * kBlockK, PHASE == kApply ? kb * kBlockK : n, z, full(st));
            }
          }
        }
      }
      // copies that nobody has waited for must have landed before the CTA may leave
      if (!ok)
        for (int i = it > kStages ? it - kStages : 0; i < it; ++i) mbar_wait(full(i % kStages), (i / kStages) & 1, p.status, 92);
    }
  } else if (warp == kMmaWarp) {
    // descriptors as in parts_common.cuh: groups of 8 rows (of 8 K) 1024 bytes apart, 128-byte swizzle; where the columns lie side by side instead of
    // the reduction, groups of 64 columns a box apart
    constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    constexpr uint32_t lbo = (kBox >> 4) << 16, slot_a = 32 >> 4, slot_b = PHASE == kApply ? 2048 >> 4 : 32 >> 4;
    constexpr uint32_t idesc0 = (1u << 4) | (uint32_t)(PHASE == kApply) << 16 | (uint32_t)(kTileM >> 4) << 24;
    int it = 0, chunks = 0, tiles = 0;
    for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
      const Tile t = tile_of<PHASE, W>(p, i);
      const int width = (PHASE == kApply ? p.item[t.q].n : p.item[t.q].m) - t.col, depth = PHASE == kGram ? p.item[t.q].n : p.item[t.q].m;
      const uint32_t idesc = idesc0 | (uint32_t)(min(W, (width + 15) & ~15) >> 3) << 17;
      for (int kb = t.k0, in_chunk = 0; kb < t.k1 && ok; ++kb, ++it) {
        const int st = it % kStages;
        const bool first = in_chunk == 0, last = ++in_chunk == p.chunk || kb + 1 == t.k1;
        if (last) in_chunk = 0;
        ok = parts::wait(full(st), (it / kStages) & 1, p.status, 93, &abort_flag);
        if (ok && kb == t.k0 && tiles > 0) ok = parts::wait(cross_empty, (tiles - 1) & 1, p.status, 94, &abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a = ((base + st * M::stage) >> 4 & 0x3FFF) | lbo, b = ((base + st * M::stage + 4 * kBox) >> 4 & 0x3FFF) | lbo;
        const uint32_t a_lo = a + (2 * kBox >> 4), b_lo = b + (W / 64 * kBox >> 4), cross = tmem + kCross;
        const int slots = min(kBlockK, depth - kb * kBlockK + 15) / 16;  // what is behind the reduction is zeros
        for (int k = 0; k < slots; ++k) {
          parts::mma(cross, a + k * slot_a, desc_hi, b_lo + k * slot_b, desc_hi, idesc, kb > t.k0 || k > 0);
          parts::mma(cross, a_lo + k * slot_a, desc_hi, b + k * slot_b, desc_hi, idesc, 1);
        }
        if (first && chunks > 0) {
          ok = __all_sync(0xffffffffu, parts::wait(acc_empty, (chunks - 1) & 1, p.status, 95, &abort_flag));
          if (!ok) break;
          tc_fence_after();
        }
        for (int k = 0; k < slots; ++k) parts::mma(tmem, a + k * slot_a, desc_hi, b + k * slot_b, desc_hi, idesc, !first || k > 0);
        umma_commit_elect(empty(st));
        if (last) {
          umma_commit_elect(acc_full);
          ++chunks;
        }
      }
      ++tiles;
    }
  } else {
    constexpr int half = W / 2;  // columns of a group of four warps
    const int quad = warp & 3, group = warp >> 2;
    const uint32_t d = tmem + ((uint32_t)(quad * 32) << 16) + group * half;
    uint32_t parity = 0;
    for (int i = blockIdx.x; i < p.items; i += gridDim.x) {  // to the end also if a wait has run out: the warps meet at barriers
      const Tile t = tile_of<PHASE, W>(p, i);
      const Item& q = p.item[t.q];
      const int chunks = (t.k1 - t.k0 + p.chunk - 1) / p.chunk;
      float sum[half];
#pragma unroll
      for (int j = 0; j < half; ++j) sum[j] = 0.f;
      for (int ch = 0; ch < chunks && ok; ++ch) {
        ok = __all_sync(0xffffffffu, parts::wait(acc_full, parity, p.status, 96, &abort_flag));
        if (!ok) break;
        parity ^= 1;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < half; c += 32) {
          float v[32];
          tmem_ld32(d + c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[c + j] += v[j];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty);
      }
      if (ok) {
#pragma unroll
        for (int c = 0; c < half; c += 32) {
          float v[32];
          tmem_ld32(d + kCross + c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[c + j] = (sum[c + j] + v[j] * (1.f / kLow)) * (1.f / (kScale * kScale));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(cross_empty);
      }

      if (q.splits > 1) {
        const int64_t size = (int64_t)W * kTileM;
        float* mine = p.sums + (int64_t)(q.first_part + t.index * q.splits) * size + (int64_t)group * half * kTileM + quad * 32 + lane;
#pragma unroll
        for (int j = 0; j < half; ++j) __stcg(mine + t.split * size + j * kTileM, sum[j]);
        __threadfence();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (threadIdx.x == 0) {
          unsigned* ticket = p.tickets + q.first_ticket + t.index;
          drawn = (int)atomicAdd(ticket, 1u);
          if (drawn == q.splits - 1) *ticket = 0;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const bool mine_to_finish = drawn == q.splits - 1;
        asm volatile("bar.sync 1, 256;" ::: "memory");  // `drawn` has been read
        if (!mine_to_finish) continue;
        __threadfence();
#pragma unroll
        for (int j = 0; j < half; ++j) sum[j] = 0.f;
        for (int o = 0; o < q.splits; ++o)
#pragma unroll
          for (int j = 0; j < half; ++j) sum[j] += __ldcg(mine + o * size + j * kTileM);
      }
      if (!ok) continue;

      const int r = t.row + quad * 32 + lane;
#pragma unroll
      for (int c0 = 0; c0 < half; c0 += 8) {
        const int c = t.col + group * half + c0;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = sum[c0 + j];
        if (PHASE == kGram) {
          if (c < q.m) write_symmetric(q.g, (int64_t)q.m * q.ldm, q.ldm, q.m, r, c, v);
        } else if (PHASE == kSquare) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= kC;
          if (c < q.m && r < q.m) add_parts(v, q.g + (int64_t)r * q.ldm + c, (int64_t)q.m * q.ldm, kB);
          if (c < q.m) write_symmetric(q.s, (int64_t)q.m * q.ldm, q.ldm, q.m, r, c, v);
        } else if (c < q.n && r < q.m) {
          const int64_t plane = (int64_t)q.m * q.ldx, at = (int64_t)r * q.ldx + c;
          add_parts(v, q.x[p.from] + at, plane, kA);
          if (!p.last) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) split2(v[2 * j], v[2 * j + 1], hi[j], lo[j]);
            uint16_t* to = q.x[p.from ^ 1] + at;  // rows are padded to eight values
            *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(to + plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (c + j >= q.n) break;
              float* o = q.out + (q.tall ? (int64_t)(c + j) * q.m + r : (int64_t)r * q.n + c + j);
              *o = q.update ? q.keep * *o - q.step * v[j] : v[j];
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// X as parts: the update divided by its norm, its shorter side first.  Tiles of 64 x 64, turned in shared memory where that is the columns.
struct Parts {
  Update u[kGroup];
  int64_t rows[kGroup], cols[kGroup];
  const double* sums[kGroup];
  uint16_t* x[kGroup];
  int ldx[kGroup];
  unsigned first[kGroup + 1];  // tiles of the matrices before
  int count;
  unsigned *tickets, tickets_end;
};
__device__ __forceinline__ float one_over_norm(const double* __restrict__ sums) {
  double sum = 0.0;
  for (int b = 0; b < kNormBlocks; ++b) sum += __ldg(sums + b);
  return (float)(1.0 / (sqrt(sum) + kEpsilon));
}
__global__ void __launch_bounds__(kThreads) parts_kernel(const __grid_constant__ Parts p) {
  RT_PDL_ENTRY();
  __shared__ float tile[64][65];
  __shared__ float by;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < p.tickets_end; i += gridDim.x * kThreads) p.tickets[i] = 0;
  int q = 0;
  while (blockIdx.x >= p.first[q + 1]) ++q;
  const Update u = p.u[q];
  const int64_t rows = p.rows[q], cols = p.cols[q];
  const unsigned local = blockIdx.x - p.first[q], tiles_c = (unsigned)((cols + 63) / 64);
  const int64_t r0 = (int64_t)(local / tiles_c) * 64, c0 = (int64_t)(local % tiles_c) * 64;
  if (threadIdx.x == 0) by = one_over_norm(p.sums[q]);
  const int lane = threadIdx.x & 63, row = threadIdx.x >> 6;
  float v[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int64_t r = r0 + row + 4 * k, c = c0 + lane;
    v[k] = r < rows && c < cols ? update_at(u, r * cols + c) : 0.f;
  }
  __syncthreads();
  const bool tall = rows > cols;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float w = v[k] * by;
    if (tall) tile[lane][row + 4 * k] = w;
    else tile[row + 4 * k][lane] = w;
  }
  __syncthreads();
  const int64_t m = tall ? cols : rows, n = tall ? rows : cols, y0 = tall ? c0 : r0, x0 = tall ? r0 : c0, ld = p.ldx[q], plane = m * ld;
  const int pair = threadIdx.x & 31, y = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int64_t gy = y0 + y + 8 * k, gx = x0 + 2 * pair;
    if (gy >= m || gx >= ld) continue;  // the padding of a row: zeros
    uint32_t hi, lo;
    split2(tile[y + 8 * k][2 * pair], tile[y + 8 * k][2 * pair + 1], hi, lo);
    uint16_t* o = p.x[q] + gy * ld + gx;
    *reinterpret_cast<uint32_t*>(o) = hi;
    *reinterpret_cast<uint32_t*>(o + plane) = lo;
  }
  (void)n;
}

// [2 planes][rows][cols] halves, rows ld apart, boxes of 64 x 64 of one plane, zeros outside.
bool map_planes(CUtensorMap* map, uint16_t* t, int64_t cols, int64_t rows, int64_t ld) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 2}, strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(ld * rows) * 2};
  const cuuint32_t box[3] = {64, 64, 1}, one[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, t, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a product's tiles are laid out over the SMs: their width, and into how many parts the reduction of each matrix's tiles is split.
struct Plan {
  int width, splits[kGroup];
};
int64_t tiles_of(int phase, int width, int64_t m, int64_t n) {
  const int64_t rows = (m + kTileM - 1) / kTileM;
  if (phase == kApply) return rows * ((n + width - 1) / width);
  return width == kTileM ? rows * (rows + 1) / 2 : (rows / 2) * (rows / 2 + 1) + (rows % 2) * (rows / 2 + 1);
}
// In units of a K-block of a tile of 128 x 128, 0.68 us; one of 128 x 256 takes 1.5 of them, sharing a reduction about 5.
Plan plan_product(const rt_ctx* ctx, int phase, int count, const Item* items) {
  Plan best{};
  double least = 1e300;
  for (int width = 128; width <= 256; width *= 2)
    for (int most = 64; most >= 1; most /= 2) {  // K-blocks of a CTA at most, where that needs several CTAs
      Plan p{};
      p.width = width;
      double work = 0, longest = 0;
      for (int q = 0; q < count; ++q) {
        const int blocks = ((phase == kGram ? items[q].n : items[q].m) + kBlockK - 1) / kBlockK;
        p.splits[q] = most == 64 || width == 256 ? 1 : (blocks + most - 1) / most;
        const double one = (width == 256 ? 1.5 : 1.0) * ((blocks + p.splits[q] - 1) / p.splits[q]) + (p.splits[q] > 1 ? 5 + 0.5 * p.splits[q] : 0);
        work += one * (double)tiles_of(phase, width, items[q].m, items[q].n) * p.splits[q];
        longest = std::max(longest, one);
      }
      const double time = std::max(longest, work / ctx->sm_count) + 0.5 * longest;  // the last tiles do not all end at once
      if (time < least) {
        least = time;
        best = p;
      }
      if (width == 256) break;
    }
  return best;
}
template <int PHASE, int W>
rt_status launch_product(rt_ctx* ctx, const Product& p) {
  static RtDeviceOnce once;
  RT_CUDA(ctx, once([] { return cudaFuncSetAttribute(product_kernel<PHASE, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Smem<W>::bytes); }));
  rt_launch(ctx, product_kernel<PHASE, W>, p.items < ctx->sm_count ? p.items : ctx->sm_count, kProductThreads, Smem<W>::bytes, p);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

// Up to kGroup matrices together.
rt_status orthogonalize_together(rt_ctx* ctx, const Matrix* list, int count, int steps, bool* unavailable) {
  Product p{};
  Parts x{};
  p.count = x.count = count;
  p.status = ctx->device_status;
  size_t halves = 0, at[kGroup];
  for (int q = 0; q < count; ++q) {
    Item& i = p.item[q];
    i.m = (int)std::min(list[q].rows, list[q].cols);
    i.n = (int)std::max(list[q].rows, list[q].cols);
    i.ldx = (i.n + 7) / 8 * 8;
    i.ldm = (i.m + 7) / 8 * 8;
    at[q] = halves;
    halves += ((size_t)4 * i.m * i.ldx + (size_t)4 * i.m * i.ldm + 63) / 64 * 64;
    i.out = list[q].out;
    i.tall = list[q].rows > list[q].cols;
    i.update = list[q].update;
    i.keep = list[q].keep;
    i.step = list[q].step;
  }
  Plan plans[3];
  size_t partials = 0, tickets = 0;
  for (int phase = 0; phase < 3; ++phase) {
    plans[phase] = plan_product(ctx, phase, count, p.item);
    size_t parts_of = 0, tickets_of = 0;
    for (int q = 0; q < count; ++q)
      if (plans[phase].splits[q] > 1) {
        const size_t tiles = (size_t)tiles_of(phase, plans[phase].width, p.item[q].m, p.item[q].n);
        parts_of += tiles * plans[phase].splits[q];
        tickets_of += tiles;
      }
    partials = std::max(partials, parts_of * plans[phase].width * kTileM);
    tickets = std::max(tickets, tickets_of);
  }
  RtScratch work(ctx);
  rt_status st = work.alloc(sizeof(uint16_t) * halves + sizeof(float) * partials + sizeof(double) * kNormBlocks * count + sizeof(unsigned) * tickets);
  if (st != RT_OK) return st;
  p.sums = reinterpret_cast<float*>(work.as<uint16_t>() + halves);
  double* squares = reinterpret_cast<double*>(p.sums + partials);
  p.tickets = reinterpret_cast<unsigned*>(squares + (size_t)kNormBlocks * count);
  unsigned tiles = 0;
  for (int q = 0; q < count; ++q) {
    Item& i = p.item[q];
    const size_t of_x = (size_t)2 * i.m * i.ldx, of_g = (size_t)2 * i.m * i.ldm;
    i.x[0] = work.as<uint16_t>() + at[q];
    i.x[1] = i.x[0] + of_x;
    i.g = i.x[1] + of_x;
    i.s = i.g + of_g;
    if (!map_planes(&p.x[0][q], i.x[0], i.n, i.m, i.ldx) || !map_planes(&p.x[1][q], i.x[1], i.n, i.m, i.ldx) ||
        !map_planes(&p.g[q], i.g, i.m, i.m, i.ldm) || !map_planes(&p.s[q], i.s, i.m, i.m, i.ldm)) {
      *unavailable = true;
      return RT_OK;
    }
    x.u[q] = list[q].u;
    x.rows[q] = list[q].rows;
    x.cols[q] = list[q].cols;
    x.sums[q] = squares + (size_t)kNormBlocks * q;
    x.x[q] = i.x[0];
    x.ldx[q] = i.ldx;
    x.first[q] = tiles;
    tiles += (unsigned)((list[q].rows + 63) / 64 * ((list[q].cols + 63) / 64));
  }
  x.first[count] = tiles;
  x.tickets = p.tickets;
  x.tickets_end = (unsigned)tickets;
  for (int q = 0; q < count; ++q) {
    rt_launch(ctx, squares_kernel, kNormBlocks, kThreads, 0, list[q].u, list[q].rows * list[q].cols, squares + (size_t)kNormBlocks * q);
    RT_LAUNCHED(ctx);
  }
  rt_launch(ctx, parts_kernel, tiles, kThreads, 0, x);
  RT_LAUNCHED(ctx);
  for (int k = 0; k < steps; ++k) {
    p.from = k & 1;
    p.last = k + 1 == steps;
    for (int phase = 0; phase < 3; ++phase) {
      int items = 0, first_part = 0, first_ticket = 0, depth = 0;
      for (int q = 0; q < count; ++q) {
        Item& i = p.item[q];
        const int t = (int)tiles_of(phase, plans[phase].width, i.m, i.n);
        i.splits = plans[phase].splits[q];
        i.first = items;
        i.first_part = first_part;
        i.first_ticket = first_ticket;
        items += t * i.splits;
        if (i.splits > 1) {
          first_part += t * i.splits;
          first_ticket += t;
        }
        depth = std::max(depth, phase == kGram ? i.n : i.m);
      }
      p.items = items;
      p.chunk = depth < 1024 ? 3 : (depth < 2048 ? 4 : 8);
      const bool wide = plans[phase].width == 256;
      if (phase == kGram) st = wide ? launch_product<kGram, 256>(ctx, p) : launch_product<kGram, 128>(ctx, p);
      else if (phase == kSquare) st = wide ? launch_product<kSquare, 256>(ctx, p) : launch_product<kSquare, 128>(ctx, p);
      else st = wide ? launch_product<kApply, 256>(ctx, p) : launch_product<kApply, 128>(ctx, p);
      if (st != RT_OK) return st;
    }
  }
  return RT_OK;
}

// ---- by the framework's other products: without tensor cores, or with no steps ------------------------------------------------------------
rt_status orthogonalize(rt_ctx* ctx, const Matrix& q, int steps) {
  const int64_t m = std::min(q.rows, q.cols), n = std::max(q.rows, q.cols), all = m * n;
  RtScratch work(ctx);
  rt_status st = work.alloc(sizeof(double) * kNormBlocks + sizeof(float) * (size_t)(2 * all + 2 * m * m));
  if (st != RT_OK) return st;
  double* sums = work.as<double>();
  float *x = reinterpret_cast<float*>(sums + kNormBlocks), *y = x + all, *g = y + all, *s = g + m * m;
  rt_launch(ctx, squares_kernel, kNormBlocks, kThreads, 0, q.u, all, sums);
  RT_LAUNCHED(ctx);
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
  rt_launch(ctx, apply_kernel, rt_grid_for(ctx, all, kThreads), kThreads, 0, x, q.rows, q.cols, q.out, q.update, q.keep, q.step);
  RT_LAUNCHED(ctx);
  return RT_OK;
}
rt_status orthogonalize_all(rt_ctx* ctx, const std::vector<Matrix>& list, int steps) {
  rt_status st = RT_OK;
  for (size_t first = 0; first < list.size(); first += kGroup) {
    const int count = (int)std::min<size_t>(kGroup, list.size() - first);
    bool otherwise = steps == 0 || !ctx->use_tensor_cores;
    if (!otherwise && (st = orthogonalize_together(ctx, &list[first], count, steps, &otherwise)) != RT_OK) return st;
    for (int q = 0; otherwise && q < count; ++q)
      if ((st = orthogonalize(ctx, list[first + q], steps)) != RT_OK) return st;
  }
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
  int matrix;    // that it belongs to
  bool written;
};
Block block_of(const float* p, int64_t n, int matrix, bool written) { return {(uintptr_t)p, (uintptr_t)(p + n), matrix, written}; }
// Whether nothing that is written overlaps anything else, `in_place` aside: what is read for a result that takes its very place.
bool apart(std::vector<Block> blocks, bool in_place) {
  std::sort(blocks.begin(), blocks.end(), [](const Block& a, const Block& b) { return a.begin < b.begin; });
  uintptr_t end = 0, written = 0;  // of all blocks so far, of those that are written
  for (size_t i = 0; i < blocks.size(); ++i) {
    const Block& b = blocks[i];
    if (in_place && i > 0) {
      const Block& a = blocks[i - 1];
      if (a.begin == b.begin && a.end == b.end && a.matrix == b.matrix && a.written != b.written) {
        written = std::max(written, b.end);
        continue;
      }
    }
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
      blocks.push_back(block_of(xs[i], rows[i] * cols[i], i, false));
      blocks.push_back(block_of(outs[i], rows[i] * cols[i], i, true));
      Matrix q{};
      q.u.x = xs[i];
      q.rows = rows[i];
      q.cols = cols[i];
      q.out = outs[i];
      list.push_back(q);
    }
    if (!apart(blocks, true)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_orthogonalize_list: a result overlaps another or another's matrix");
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
      blocks.push_back(block_of(params[i], rows[i] * cols[i], i, true));
      blocks.push_back(block_of(grads[i], rows[i] * cols[i], i, false));
      blocks.push_back(block_of(momenta[i], rows[i] * cols[i], i, true));
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
    if (!apart(blocks, false)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_muon_step_multi: a parameter or momentum overlaps another or a gradient");
    RtOnDevice here(ctx);
    if ((st = orthogonalize_all(ctx, list, steps)) != RT_OK) return st;
  } catch (const std::bad_alloc&) {
    RT_FAIL(ctx, RT_ERR_OOM, "rt_muon_step_multi: out of host memory");
  }
  return RT_OK;
}

}  // extern "C"
