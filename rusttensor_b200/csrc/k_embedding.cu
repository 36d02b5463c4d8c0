// Token embeddings: rows of a table by number, and the gradient of the table.
//
//   out[i, :] = scale * table[ids[i], :]          dtable[r, :] (+)= scale * sum over i with ids[i] = r of g[i, :]
//
// A number outside the table is padding: zeros forward, no term backward.  The gradient adds the rows of one token in the order of their
// positions, whatever runs when: the pairs (token, position) are sorted by token first, stably, and no sum is made with atomics.
#include "rt_internal.cuh"

namespace {

constexpr int kThreads = 256;

// ---- forward ----------------------------------------------------------------------------------------------------------------------
// A group of `lanes` lanes has a row, eight pieces of it in flight.  Bound by memory: what is read of the table and the rows written.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const float* __restrict__ table, int64_t rows, int64_t cols, const int32_t* __restrict__ ids,
                                                             int64_t n, float scale, int lanes, float* __restrict__ out) {
  RT_PDL_ENTRY();
  const int per_block = kThreads / lanes, lane = threadIdx.x % lanes;
  const int64_t pieces = VEC ? cols / 4 : cols;
  for (int64_t i = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; i < n; i += (int64_t)gridDim.x * per_block) {
    const int64_t r = __ldg(ids + i);
    const bool there = r >= 0 && r < rows;
    const float* from = table + (there ? r : 0) * cols;
    float* to = out + i * cols;
    for (int64_t c0 = lane; c0 < pieces; c0 += 8 * lanes) {
      if (VEC) {
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t c = c0 + k * lanes;
          v[k] = there && c < pieces ? __ldg(reinterpret_cast<const float4*>(from) + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t c = c0 + k * lanes;
          // padding stays zero, whatever the scale is
          if (c < pieces) reinterpret_cast<float4*>(to)[c] = there ? make_float4(v[k].x * scale, v[k].y * scale, v[k].z * scale, v[k].w * scale) : v[k];
        }
      } else {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t c = c0 + k * lanes;
          v[k] = there && c < pieces ? __ldg(from + c) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t c = c0 + k * lanes;
          if (c < pieces) to[c] = there ? v[k] * scale : 0.f;
        }
      }
    }
  }
}

// Whole numbers held as floats, as the engine holds them; everything else (fractions, NaN, beyond int32) becomes -1.
__global__ void __launch_bounds__(kThreads) token_ids_kernel(const float* __restrict__ x, int64_t n, int32_t* __restrict__ ids) {
  RT_PDL_ENTRY();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const float v = __ldg(x + i);
    ids[i] = v >= 0.f && v < 2147483648.f && v == truncf(v) ? (int32_t)v : -1;
  }
}

// ---- sorting ------------------------------------------------------------------------------------------------------------------------
// Least significant digit first, eight bits a pass, each pass as three launches: how often every digit occurs in each block's items, where
// each block's items of a digit go, the items to their places.  Padding gets the number `rows` and comes last.
constexpr int kDigits = 256, kWarps = kThreads / 32, kRounds = 16, kTile = kThreads * kRounds;
struct Pass {
  const int32_t* ids;             // first pass: the tokens; their positions are their places
  const uint32_t *keys, *places;  // later ones
  uint32_t *keys_out, *places_out;
  int64_t n;
  uint32_t rows;
  int shift, blocks;
  uint32_t* counts;               // [digit][block]
};
__device__ __forceinline__ uint32_t key_at(const Pass& p, int64_t i) {
  if (!p.ids) return __ldg(p.keys + i);
  const int32_t id = __ldg(p.ids + i);
  return id >= 0 && (uint32_t)id < p.rows ? (uint32_t)id : p.rows;
}
__global__ void __launch_bounds__(kThreads) digit_counts_kernel(const Pass p) {
  RT_PDL_ENTRY();
  __shared__ uint32_t count[kDigits];
  count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kTile;
#pragma unroll 4
  for (int k = 0; k < kRounds; ++k) {
    const int64_t i = first + k * kThreads + threadIdx.x;
    if (i < p.n) atomicAdd(&count[key_at(p, i) >> p.shift & (kDigits - 1)], 1u);
  }
  __syncthreads();
  p.counts[(int64_t)threadIdx.x * p.blocks + blockIdx.x] = count[threadIdx.x];
}
// Exclusive sums over [digit][block], one block of 1024 threads.
__global__ void __launch_bounds__(1024) digit_places_kernel(uint32_t* counts, int64_t n) {
  RT_PDL_ENTRY();
  __shared__ uint32_t of_warp[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t before = 0;
  for (int64_t first = 0; first < n; first += 1024) {
    const int64_t i = first + threadIdx.x;
    const uint32_t v = i < n ? counts[i] : 0u;
    uint32_t sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (lane == 31) of_warp[warp] = sum;
    __syncthreads();
    uint32_t all = of_warp[lane], upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    const uint32_t mine = __shfl_sync(0xffffffffu, upto - all, warp);
    if (i < n) counts[i] = before + mine + sum - v;
    before += __shfl_sync(0xffffffffu, upto, 31);
    __syncthreads();
  }
}
// A warp has 512 items one after the other.  An item's place is that of its block's first one of the digit, plus those of the warps before,
// plus those before it in its own warp.
__global__ void __launch_bounds__(kThreads) digit_scatter_kernel(const Pass p) {
  RT_PDL_ENTRY();
  __shared__ uint32_t count[kWarps][kDigits];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) count[w][threadIdx.x] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kTile + warp * 32 * kRounds + lane;
  uint32_t key[kRounds];
  uint16_t rank[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) key[k] = first + k * 32 < p.n ? key_at(p, first + k * 32) : 0xffffffffu;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool in = first + k * 32 < p.n;
    const uint32_t digit = in ? key[k] >> p.shift & (kDigits - 1) : kDigits;
    const uint32_t same = __match_any_sync(0xffffffffu, digit);
    uint32_t before = in ? count[warp][digit] : 0u;
    rank[k] = (uint16_t)(before + __popc(same & ((1u << lane) - 1)));
    __syncwarp();
    if (in && lane == __ffs(same) - 1) count[warp][digit] = before + __popc(same);
    __syncwarp();
  }
  __syncthreads();
  uint32_t at = p.counts[(int64_t)threadIdx.x * p.blocks + blockIdx.x];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t c = count[w][threadIdx.x];
    count[w][threadIdx.x] = at;
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int64_t i = first + k * 32;
    if (i < p.n) {
      const uint32_t to = count[warp][key[k] >> p.shift & (kDigits - 1)] + rank[k];
      p.keys_out[to] = key[k];
      p.places_out[to] = p.ids ? (uint32_t)i : __ldg(p.places + i);
    }
  }
}

// ---- sums ---------------------------------------------------------------------------------------------------------------------------
// The first of the sorted keys that is not below `key`.
__device__ __forceinline__ int64_t first_of(const uint32_t* __restrict__ keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (__ldg(keys + mid) < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
// A block has a row of the table.
__global__ void __launch_bounds__(kThreads) row_sums_kernel(const float* __restrict__ g, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ places,
                                                            int64_t n, int64_t rows, int64_t cols, float scale, float* __restrict__ dtable, int accumulate) {
  RT_PDL_ENTRY();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t begin = first_of(keys, n, (uint32_t)r), end = first_of(keys, n, (uint32_t)r + 1);
    if (begin == end && accumulate) continue;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      float sum = 0.f;
      for (int64_t i = begin; i < end; ++i) sum += __ldg(g + (int64_t)__ldg(places + i) * cols + c);
      float* o = dtable + r * cols + c;
      *o = accumulate ? *o + scale * sum : scale * sum;
    }
  }
}

rt_status check_sizes(rt_ctx* ctx, const char* who, int64_t rows, int64_t cols, int64_t n) {
  if (rows < 0 || cols < 0 || n < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: negative size", who);
  if (rows >= (1ll << 31) || n >= (1ll << 31) || cols >= (1ll << 31) || rows * cols >= (1ll << 40) || n * cols >= (1ll << 40))
    RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: size out of range", who);
  return RT_OK;
}

}  // namespace

extern "C" {

rt_status rt_token_ids(rt_ctx* ctx, const float* x, int64_t n, int32_t* ids) {
  RT_CHECK_CTX(ctx);
  if (n < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_token_ids: negative size");
  if (n == 0) return RT_OK;
  RT_CHECK_PTR(ctx, x);
  RT_CHECK_PTR(ctx, ids);
  RtOnDevice here(ctx);
  rt_launch(ctx, token_ids_kernel, rt_grid_for(ctx, n, kThreads), kThreads, 0, x, n, ids);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

rt_status rt_embedding(rt_ctx* ctx, const float* table, int64_t rows, int64_t cols, const int32_t* ids, int64_t n, float scale, float* out) {
  RT_CHECK_CTX(ctx);
  rt_status st = check_sizes(ctx, "rt_embedding", rows, cols, n);
  if (st != RT_OK) return st;
  if (n == 0 || cols == 0) return RT_OK;
  if (rows > 0) RT_CHECK_PTR(ctx, table);
  RT_CHECK_PTR(ctx, ids);
  RT_CHECK_PTR(ctx, out);
  RtOnDevice here(ctx);
  const bool vec = cols % 4 == 0 && rt_aligned16(table) && rt_aligned16(out);
  const int64_t pieces = vec ? cols / 4 : cols;
  int lanes = 1;
  while (lanes < 32 && lanes < pieces) lanes *= 2;
  rt_launch(ctx, vec ? embedding_kernel<true> : embedding_kernel<false>, rt_grid_for(ctx, n, kThreads / lanes, 16), kThreads, 0, table, rows, cols, ids, n,
            scale, lanes, out);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

rt_status rt_embedding_backward(rt_ctx* ctx, const float* g, const int32_t* ids, int64_t n, int64_t rows, int64_t cols, float scale, float* dtable,
                                int accumulate) {
  RT_CHECK_CTX(ctx);
  rt_status st = check_sizes(ctx, "rt_embedding_backward", rows, cols, n);
  if (st != RT_OK) return st;
  if (rows == 0 || cols == 0) return RT_OK;
  RT_CHECK_PTR(ctx, dtable);
  if (n == 0) return accumulate ? RT_OK : rt_fill(ctx, dtable, 0.f, rows * cols);
  RT_CHECK_PTR(ctx, g);
  RT_CHECK_PTR(ctx, ids);
  RtOnDevice here(ctx);
  const int blocks = (int)((n + kTile - 1) / kTile);
  RtScratch work(ctx);
  if ((st = work.alloc(sizeof(uint32_t) * (4 * (size_t)n + (size_t)kDigits * blocks))) != RT_OK) return st;
  uint32_t *keys = work.as<uint32_t>(), *places = keys + n, *keys2 = places + n, *places2 = keys2 + n;
  Pass p{};
  p.counts = places2 + n;
  p.n = n;
  p.rows = (uint32_t)rows;
  p.blocks = blocks;
  for (p.shift = 0; p.shift < 32 && (p.shift == 0 || (uint64_t)rows >> p.shift); p.shift += 8) {
    p.ids = p.shift == 0 ? ids : nullptr;
    p.keys_out = keys;
    p.places_out = places;
    rt_launch(ctx, digit_counts_kernel, blocks, kThreads, 0, p);
    RT_LAUNCHED(ctx);
    rt_launch(ctx, digit_places_kernel, 1, 1024, 0, p.counts, (int64_t)kDigits * blocks);
    RT_LAUNCHED(ctx);
    rt_launch(ctx, digit_scatter_kernel, blocks, kThreads, 0, p);
    RT_LAUNCHED(ctx);
    p.keys = keys;
    p.places = places;
    uint32_t* t = keys;
    keys = keys2;
    keys2 = t;
    t = places;
    places = places2;
    places2 = t;
  }
  rt_launch(ctx, row_sums_kernel, (unsigned)(rows < 65535 ? rows : 65535), kThreads, 0, g, p.keys, p.places, n, rows, cols, scale, dtable, accumulate);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

}  // extern "C"
