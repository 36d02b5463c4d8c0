// Token embeddings: rows of a table by number, and the gradient of the table.
//
//   out[i, :] = scale * table[ids[i], :]          dtable[r, :] (+)= scale * sum over i with ids[i] = r of g[i, :]
//
// A number outside the table is padding: zeros forward, no term backward.  The gradient adds the rows of one token in the order of their
// positions, whatever runs when: the pairs (token, position) are sorted by token first, stably, and no sum is made with atomics.
//
// rt_gather_rows, the gather of a data set's rows, reads the same but neither scales nor has as many loads in flight: 32768 rows of 1024 of
// 50000 take 33.5 us there and 29.7 here, 64 of 512 1.7 either way (replayed from a graph).
#include <cooperative_groups.h>

#include <utility>

#include "rt_internal.cuh"

namespace {

namespace cg = cooperative_groups;

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

// Whole numbers held as floats, as the engine holds them; everything else (fractions, NaN, beyond int32) becomes -1.  In place, too: no read-only loads.
__global__ void __launch_bounds__(kThreads) token_ids_kernel(const float* x, int64_t n, int32_t* ids) {
  RT_PDL_ENTRY();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const float v = x[i];
    ids[i] = v >= 0.f && v < 2147483648.f && v == truncf(v) ? (int32_t)v : -1;
  }
}

// ---- sorting ------------------------------------------------------------------------------------------------------------------------
// Least significant digit first, eight bits a pass, each pass as three launches: how often every digit occurs in each block's items, where
// each block's items of a digit go, the items to their places.  Padding gets the number `rows` and comes last.
constexpr int kDigits = 256, kWarps = kThreads / 32, kRounds = 16, kTile = kThreads * kRounds;
struct Pass {
  const int32_t* ids;             // first pass: the tokens; their positions are their places
  const uint2* from;              // later ones: pairs of token and place
  uint2* to;
  int64_t n;
  uint32_t rows;
  int shift, blocks;
  uint32_t* counts;               // [digit][block]
  uint32_t* crossing;             // zeroed in the first pass
};
// The lanes that have the same digit, of those that take part; by ballots, because match.any goes through the digits that occur one after the
// other (a pass over 8192 items in one CTA: 16.9 us with it).
__device__ __forceinline__ uint32_t lanes_with(uint32_t digit, bool in) {
  uint32_t same = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const bool set = digit >> b & 1;
    const uint32_t v = __ballot_sync(0xffffffffu, set);
    same &= set ? v : ~v;
  }
  return same;
}
__device__ __forceinline__ uint2 pair_at(const Pass& p, int64_t i) {
  if (!p.ids) return __ldg(p.from + i);
  const int32_t id = __ldg(p.ids + i);
  return make_uint2(id >= 0 && (uint32_t)id < p.rows ? (uint32_t)id : p.rows, (uint32_t)i);
}
__global__ void __launch_bounds__(kThreads) digit_counts_kernel(const Pass p) {
  RT_PDL_ENTRY();
  __shared__ uint32_t count[kDigits];
  if (p.ids && blockIdx.x == 0 && threadIdx.x < 2) p.crossing[threadIdx.x] = 0;
  count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kTile;
#pragma unroll 4
  for (int k = 0; k < kRounds; ++k) {
    const int64_t i = first + k * kThreads + threadIdx.x;
    if (i < p.n) atomicAdd(&count[pair_at(p, i).x >> p.shift & (kDigits - 1)], 1u);
  }
  __syncthreads();
  p.counts[(int64_t)threadIdx.x * p.blocks + blockIdx.x] = count[threadIdx.x];
}
// Exclusive sums over [digit][block], one block of 1024 threads, each with eight of them at a time (a million tokens: with one 56 us a pass).
__global__ void __launch_bounds__(1024) digit_places_kernel(uint32_t* counts, int64_t n) {
  RT_PDL_ENTRY();
  constexpr int kEach = 8;  // n is a multiple of it
  __shared__ uint32_t of_warp[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t before = 0;
  for (int64_t first = 0; first < n; first += 1024 * kEach) {
    const int64_t i = first + threadIdx.x * kEach;
    uint2 v[kEach / 2];
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < kEach / 2; ++k) {
      v[k] = i < n ? *reinterpret_cast<const uint2*>(counts + i + 2 * k) : make_uint2(0u, 0u);
      mine += v[k].x + v[k].y;
    }
    uint32_t sum = mine;
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
    uint32_t at = before + __shfl_sync(0xffffffffu, upto - all, warp) + sum - mine;
    if (i < n) {
#pragma unroll
      for (int k = 0; k < kEach / 2; ++k) {
        *reinterpret_cast<uint2*>(counts + i + 2 * k) = make_uint2(at, at + v[k].x);
        at += v[k].x + v[k].y;
      }
    }
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
  uint2 item[kRounds];
  uint16_t rank[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) item[k] = first + k * 32 < p.n ? pair_at(p, first + k * 32) : make_uint2(0u, 0u);
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool in = first + k * 32 < p.n;
    const uint32_t digit = item[k].x >> p.shift & (kDigits - 1);
    const uint32_t same = lanes_with(digit, in);
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
    if (i < p.n) p.to[count[warp][item[k].x >> p.shift & (kDigits - 1)] + rank[k]] = item[k];
  }
}

// Up to 65536 tokens: a cluster of eight CTAs sorts them in one launch, a CTA up to 8192 of them, which wait in its shared memory from pass to
// pass and go to their places in the CTAs' shared memory.  What the CTAs tell one another per pass is how often every digit occurs among
// their items.  Bound by the scattered stores, one a cycle of an SM, and by the ballots: hence eight CTAs whatever the number of tokens,
// and a pair in one store.
constexpr int kClusterThreads = 1024, kCluster = 8, kMaxItems = 8;
template <int ITEMS>
struct ClusterSmem {
  uint2 pairs[kClusterThreads * ITEMS];
  uint32_t count[kClusterThreads / 32][kDigits];
  uint32_t mine[kDigits], start[kDigits];
  uint32_t of_warp[kDigits / 32];
};
template <int ITEMS>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kClusterThreads)
cluster_sort_kernel(const int32_t* __restrict__ ids, uint32_t n, uint32_t rows, int bits, uint2* __restrict__ out, uint32_t* __restrict__ crossing) {
  RT_PDL_ENTRY();
  extern __shared__ char smem_raw[];
  constexpr uint32_t tile = kClusterThreads * ITEMS;
  ClusterSmem<ITEMS>& s = *reinterpret_cast<ClusterSmem<ITEMS>*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank();
  if (rank == 0 && threadIdx.x < 2) crossing[threadIdx.x] = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // item k of the thread: a warp has 32 * ITEMS of them one after the other
  const uint32_t local = warp * 32 * ITEMS + lane, first = rank * tile + local;
  uint2 item[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t i = first + k * 32;
    const int32_t id = i < n ? __ldg(ids + i) : -1;
    item[k] = make_uint2(id >= 0 && (uint32_t)id < rows ? (uint32_t)id : rows, i);
  }
  for (int shift = 0; shift < bits; shift += 8) {
    if (shift > 0) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) item[k] = s.pairs[local + k * 32];
    }
    for (int i = threadIdx.x; i < kClusterThreads / 32 * kDigits; i += kClusterThreads) (&s.count[0][0])[i] = 0;
    __syncthreads();
    uint32_t before[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const bool in = first + k * 32 < n;
      const uint32_t digit = item[k].x >> shift & (kDigits - 1);
      const uint32_t same = lanes_with(digit, in);
      const uint32_t seen = in ? s.count[warp][digit] : 0u;
      before[k] = seen + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (in && lane == __ffs(same) - 1) s.count[warp][digit] = seen + __popc(same);
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {  // a digit's items of the warps before
      uint32_t sum = 0;
#pragma unroll 8
      for (int w = 0; w < kClusterThreads / 32; ++w) {
        const uint32_t c = s.count[w][threadIdx.x];
        s.count[w][threadIdx.x] = sum;
        sum += c;
      }
      s.mine[threadIdx.x] = sum;
    }
    cluster.sync();
    uint32_t all = 0, lower = 0, upto = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (uint32_t c = 0; c < kCluster; ++c) {
        const uint32_t v = cluster.map_shared_rank(s.mine, c)[threadIdx.x];
        all += v;
        if (c < rank) lower += v;
      }
      upto = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      if (lane == 31) s.of_warp[warp] = upto;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t base = upto - all + lower;
      for (int w = 0; w < warp; ++w) base += s.of_warp[w];
      s.start[threadIdx.x] = base;
    }
    __syncthreads();
    const bool last = shift + 8 >= bits;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      if (first + k * 32 >= n) continue;
      const uint32_t digit = item[k].x >> shift & (kDigits - 1);
      const uint32_t to = s.start[digit] + s.count[warp][digit] + before[k];
      if (last) out[to] = item[k];
      else cluster.map_shared_rank(s.pairs, to / tile)[to % tile] = item[k];
    }
    cluster.sync();  // the items are where they belong; nobody looks at another's counts any more
  }
}

// Up to 2048 tokens: a token's place is the number of smaller keys, plus that of the same ones before it, counted by comparing all with all.  These
// are n^2 comparisons, which all SMs share and of which none waits for another.  A warp has two tokens, its lanes 128 keys a step between them.  The
// gradient of 20011 rows of 333 takes 9.9 us from 200 tokens, 11.9 from 1000 and 13.1 from 2000, sorted by the cluster 14.3, 15.8 and
// 16.3; from 4000 it is 17.8 and 17.4.
constexpr int kRankTokens = 2048, kPerWarp = 2;
__global__ void __launch_bounds__(kThreads) rank_sort_kernel(const int32_t* __restrict__ ids, uint32_t n, uint32_t rows, uint2* __restrict__ out,
                                                             uint32_t* __restrict__ crossing) {
  RT_PDL_ENTRY();
  __shared__ uint4 keys4[kRankTokens / 4];
  uint32_t* keys = reinterpret_cast<uint32_t*>(keys4);
  if (blockIdx.x == 0 && threadIdx.x < 2) crossing[threadIdx.x] = 0;
  const uint32_t steps = (n + 127) / 128, lane = threadIdx.x & 31;
#pragma unroll 8
  for (uint32_t i = threadIdx.x; i < steps * 128; i += kThreads) {
    const int32_t id = i < n ? __ldg(ids + i) : -1;
    keys[i] = i >= n ? ~0u : (id >= 0 && (uint32_t)id < rows ? (uint32_t)id : rows);  // behind the last: before nobody
  }
  __syncthreads();
  const uint32_t first = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * kPerWarp;
  if (first >= n) return;
  uint32_t key[kPerWarp], place[kPerWarp];
#pragma unroll
  for (int t = 0; t < kPerWarp; ++t) {
    key[t] = keys[min(first + t, n - 1)];
    place[t] = 0;
  }
  const uint32_t own = first / 128;  // the step that has these tokens, too: kPerWarp divides 128
  for (uint32_t k = 0; k < steps; ++k) {
    const uint4 q = keys4[k * 32 + lane];
    if (k == own) continue;
    const uint32_t ties = k < own;
#pragma unroll
    for (int t = 0; t < kPerWarp; ++t) {
      const uint32_t limit = key[t] + ties;
      place[t] += (q.x < limit) + (q.y < limit) + (q.z < limit) + (q.w < limit);
    }
  }
  for (uint32_t j = own * 128 + lane; j < own * 128 + 128; j += 32)
#pragma unroll
    for (int t = 0; t < kPerWarp; ++t) place[t] += keys[j] < key[t] + (j < first + t);
#pragma unroll
  for (int t = 0; t < kPerWarp; ++t) {
    const uint32_t to = __reduce_add_sync(0xffffffffu, place[t]);
    if (lane == 0 && first + t < n) out[to] = make_uint2(key[t], first + t);
  }
}

// ---- sums ---------------------------------------------------------------------------------------------------------------------------
// A run is the sorted places of one token.  Its terms are added by tiles of 32 places: a run that lies within a tile is written at once, of
// one that goes over a tile's end every tile leaves its part: slot 0 of the tile if the run began before it, slot 1 if it goes on behind it
// only.  The tile where a run begins is where its parts are then added up, in their order.
struct Runs {
  const float* g;
  const uint2* pairs;       // sorted: token, place
  uint32_t n, rows;
  int64_t cols;
  float scale;
  float* dtable;
  uint32_t tiles, slabs;    // slabs of 32 pieces of the columns
  uint32_t sum_blocks;
  uint32_t fill_rows;       // rows of the table that a block behind those looks through for ones without a token
  float* parts;             // [tile][2][cols]
  // The tiles with a run that begins there and goes on, in no order: how many of those that go on over up to kShort tiles, how many others, and
  // which: the ones from the front, the others from the back.
  uint32_t* crossing;
};
constexpr int kSumThreads = 128, kRun = 32, kShort = 16, kFillRows = 32;
template <bool VEC>
struct Piece;
template <>
struct Piece<true> {
  using T = float4;
  static __device__ __forceinline__ T zero() { return make_float4(0.f, 0.f, 0.f, 0.f); }
  static __device__ __forceinline__ void add(T& a, const T& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }
  static __device__ __forceinline__ T scaled(const T& a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
};
template <>
struct Piece<false> {
  using T = float;
  static __device__ __forceinline__ T zero() { return 0.f; }
  static __device__ __forceinline__ void add(T& a, T b) { a += b; }
  static __device__ __forceinline__ T scaled(T a, float s) { return a * s; }
};
template <bool VEC, bool ACCUMULATE>
__device__ __forceinline__ void write_row(const Runs& r, uint32_t row, int64_t c, typename Piece<VEC>::T sum, const typename Piece<VEC>::T& old) {
  using P = Piece<VEC>;
  sum = P::scaled(sum, r.scale);
  if (ACCUMULATE) P::add(sum, old);
  *(reinterpret_cast<typename P::T*>(r.dtable + (int64_t)row * r.cols) + c) = sum;
}
// The first of the sorted pairs whose key is not below `key`; seven looks at a time, which do not wait for one another.
__device__ __forceinline__ uint32_t first_of(const uint2* __restrict__ pairs, uint32_t n, uint32_t key) {
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t step = (hi - lo + 7) / 8;
    uint32_t seen[7], below = 0;
#pragma unroll
    for (uint32_t j = 0; j < 7; ++j) {
      const uint32_t at = lo + step * (j + 1) - 1;
      seen[j] = at < hi ? __ldg(&pairs[at].x) : ~0u;  // no key is that large
    }
#pragma unroll
    for (uint32_t j = 0; j < 7; ++j) below += seen[j] < key;
    lo += step * below;
    if (below < 7) hi = min(hi, lo + step - 1);
  }
  return lo;
}
// A warp has a tile and 32 pieces of the columns: one load brings the tile's pairs, then eight rows of g at a time, and the rows of the table
// that they are added to.  The blocks behind those of the sums write zeros to the rows without a token.  Bound by memory, which g crosses once:
// 32768 tokens of 1024 columns into 50000 rows take 48 us, 7.0 TB/s.  (The zeros by the SMs that the sort leaves idle, each block finding
// out about its rows from all tokens: 22 us less here and 35 us more there.)
template <bool VEC, bool ACCUMULATE>
__global__ void __launch_bounds__(kSumThreads) run_sums_kernel(const Runs r) {
  RT_PDL_ENTRY();
  using P = Piece<VEC>;
  using T = typename P::T;
  const int64_t pieces = VEC ? r.cols / 4 : r.cols;
  const int lane = threadIdx.x & 31;
  if (blockIdx.x >= r.sum_blocks) {
    __shared__ uint8_t there[kFillRows];
    const uint32_t row0 = (blockIdx.x - r.sum_blocks) * r.fill_rows, rows = min(r.fill_rows, r.rows - row0);
    for (uint32_t k = threadIdx.x; k < rows; k += kSumThreads) {
      const uint32_t i = first_of(r.pairs, r.n, row0 + k);
      there[k] = i < r.n && __ldg(&r.pairs[i].x) == row0 + k;
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x >> 5; k < rows; k += kSumThreads / 32) {
      if (there[k]) continue;
      T* o = reinterpret_cast<T*>(r.dtable + (int64_t)(row0 + k) * r.cols);
      for (int64_t c = lane; c < pieces; c += 32) o[c] = P::zero();
    }
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * (kSumThreads / 32) + (threadIdx.x >> 5);
  const uint32_t t = (uint32_t)(unit / r.slabs);
  if (t >= r.tiles) return;
  const int64_t c = unit % r.slabs * 32 + lane;
  const uint32_t begin = t * kRun, count = min(r.n - begin, (uint32_t)kRun);
  const uint2 mine = lane < count ? __ldg(r.pairs + begin + lane) : make_uint2(r.rows, 0u);
  const uint32_t terms = __popc(__ballot_sync(0xffffffffu, mine.x < r.rows));  // padding comes last
  if (terms == 0) return;
  const uint32_t first = __shfl_sync(0xffffffffu, mine.x, 0), last = __shfl_sync(0xffffffffu, mine.x, count - 1);
  const uint32_t key_before = begin > 0 ? __ldg(&r.pairs[begin - 1].x) : ~0u, key_behind = begin + kRun < r.n ? __ldg(&r.pairs[begin + kRun].x) : ~0u;
  const uint32_t behind = __shfl_down_sync(0xffffffffu, mine.x, 1);
  const uint32_t ends = __ballot_sync(0xffffffffu, lane + 1 == terms || mine.x != behind);  // of runs
  const bool in = c < pieces;
  T* parts = reinterpret_cast<T*>(r.parts + (int64_t)t * 2 * r.cols) + c;
  const T *g = reinterpret_cast<const T*>(r.g) + c, *table = reinterpret_cast<const T*>(r.dtable) + c;
  T sum = P::zero(), v[8], old[8] = {};
  auto load = [&](uint32_t i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t place = __shfl_sync(0xffffffffu, mine.y, i + k);
      v[k] = in && i + k < terms ? __ldg(g + (int64_t)place * pieces) : P::zero();
    }
    if (ACCUMULATE) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t row = __shfl_sync(0xffffffffu, mine.x, i + k);
        old[k] = in && i + k < terms && ends >> (i + k) & 1 ? table[(int64_t)row * pieces] : P::zero();
      }
    }
  };
  load(0);  // before anybody waits for the neighbours' keys
  const bool began = key_before == first;                    // in a tile before
  const bool goes_on = terms == kRun && key_behind == last;  // behind this one
  bool head = began;
  for (uint32_t i = 0; i < terms; i += 8) {
    if (i > 0) load(i);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      P::add(sum, v[k]);
      if (i + k < terms && ends >> (i + k) & 1) {
        const uint32_t row = __shfl_sync(0xffffffffu, mine.x, i + k);
        if (in) {
          if (head) parts[0] = sum;
          else if (goes_on && i + k + 1 == terms) parts[pieces] = sum;
          else write_row<VEC, ACCUMULATE>(r, row, c, sum, old[k]);
        }
        head = false;
        sum = P::zero();
      }
    }
  }
  if (c == 0 && goes_on && !(began && first == last)) {
    const uint32_t far = begin + kRun * (kShort + 1), longer = far < r.n && __ldg(&r.pairs[far].x) == last;
    const uint32_t k = atomicAdd(r.crossing + longer, 1u);
    r.crossing[2 + (longer ? r.tiles - 1 - k : k)] = t;
  }
}
// The parts of the runs that go over the ends of tiles, in the order of the tiles.  Short runs: a warp has 32 pieces of the columns of one.  Long
// ones: a block has them, its warps add up a stretch of the tiles each, then the first adds up the warps' sums.
constexpr int kJoinThreads = 256;
template <bool VEC>
__device__ __forceinline__ typename Piece<VEC>::T add_parts(const typename Piece<VEC>::T* parts, int64_t pieces, uint32_t from, uint32_t to,
                                                            typename Piece<VEC>::T sum) {
  using P = Piece<VEC>;
  for (uint32_t q = from; q < to; q += 8) {
    typename P::T v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = q + k < to ? parts[(int64_t)(q + k) * 2 * pieces] : P::zero();
#pragma unroll
    for (int k = 0; k < 8; ++k) P::add(sum, v[k]);
  }
  return sum;
}
template <bool VEC, bool ACCUMULATE>
__global__ void __launch_bounds__(kJoinThreads) join_runs_kernel(const Runs r) {
  RT_PDL_ENTRY();
  using P = Piece<VEC>;
  using T = typename P::T;
  __shared__ T of_warp[kJoinThreads / 32][32];
  const int64_t pieces = VEC ? r.cols / 4 : r.cols;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kJoinThreads / 32;
  // from the last block on: where there is little work, the first ones have the long runs
  const int64_t w0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * warps + warp;
  const uint32_t t0 = w0 / r.slabs < r.tiles ? __ldg(r.crossing + 2 + w0 / r.slabs) : 0;  // of use if there are so many
  const int64_t shorts = (int64_t)__ldg(r.crossing) * r.slabs, longs = (int64_t)__ldg(r.crossing + 1) * r.slabs;
  const T* table = reinterpret_cast<const T*>(r.dtable);
  for (int64_t w = w0; w < shorts; w += (int64_t)gridDim.x * warps) {
    const uint32_t t = w == w0 ? t0 : __ldg(r.crossing + 2 + w / r.slabs), q = t + 1 + lane;
    const int64_t c = w % r.slabs * 32 + lane;
    const bool in = c < pieces;
    const T* parts = reinterpret_cast<const T*>(r.parts) + (in ? c : 0);
    // the parts of the first tiles are on their way while it is found out how many there are
    T sum = parts[(int64_t)t * 2 * pieces + pieces], v[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) v[k] = t + 1 + k < r.tiles ? parts[(int64_t)(t + 1 + k) * 2 * pieces] : P::zero();
    const uint32_t run = __ldg(&r.pairs[t * kRun + kRun - 1].x);
    // how many tiles behind this one begin with the run
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, q < r.tiles && __ldg(&r.pairs[q * kRun].x) == run));
    if (!in) continue;
    const T old = ACCUMULATE ? table[(int64_t)run * pieces + c] : P::zero();
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (k < count) P::add(sum, v[k]);
    write_row<VEC, ACCUMULATE>(r, run, c, count > 4 ? add_parts<VEC>(parts, pieces, t + 5, t + 1 + count, sum) : sum, old);
  }
  for (int64_t w = blockIdx.x; w < longs; w += gridDim.x) {
    const uint32_t t = __ldg(r.crossing + 2 + r.tiles - 1 - w / r.slabs), run = __ldg(&r.pairs[t * kRun + kRun - 1].x);
    const int64_t c = w % r.slabs * 32 + lane;
    uint32_t count = 0;
    for (int seen = kJoinThreads; seen == kJoinThreads; count += seen) {
      const uint32_t q = t + 1 + count + threadIdx.x;
      seen = __syncthreads_count(q < r.tiles && __ldg(&r.pairs[q * kRun].x) == run);
    }
    const uint32_t each = (count + warps - 1) / warps, from = t + 1 + min(warp * each, count), to = t + 1 + min(warp * each + each, count);
    if (c < pieces) {
      const T* parts = reinterpret_cast<const T*>(r.parts) + c;
      of_warp[warp][lane] = add_parts<VEC>(parts, pieces, from, to, warp == 0 ? parts[(int64_t)t * 2 * pieces + pieces] : P::zero());
    }
    __syncthreads();
    if (warp == 0 && c < pieces) {
      const T old = ACCUMULATE ? table[(int64_t)run * pieces + c] : P::zero();
      T sum = of_warp[0][lane];
#pragma unroll
      for (uint32_t k = 1; k < warps; ++k) P::add(sum, of_warp[k][lane]);
      write_row<VEC, ACCUMULATE>(r, run, c, sum, old);
    }
    __syncthreads();
  }
}
// Few tokens, in one launch: a warp has a row of the table and 32 pieces of the columns, looks through all tokens and adds what is its row's.
// 128 tokens, added to 1000 rows of 1024: 5.6 us, 12.4 sorted.  Tables of more than 65536 such units are left to the sort: 8000 rows of 1024,
// which are 64000, take 6.0 and 12.4 us, 16000 rows 9.8 and 12.4, 50000, of which every warp has 42 units, 25 and 12.8; written instead of added to
// 8.8 and 14.2, 15.5 and 18.6, 44 and 35: they meet at some 20000.  (A unit is 128 columns, 32 where rows are not aligned.)  All tokens the same is what bounds this: one row
// of g after the other.
constexpr int kFew = 128;
constexpr int64_t kFewUnits = 1 << 16;
template <bool VEC, bool ACCUMULATE>
__global__ void __launch_bounds__(kThreads) few_tokens_kernel(const Runs r, const int32_t* __restrict__ ids) {
  RT_PDL_ENTRY();
  using P = Piece<VEC>;
  using T = typename P::T;
  const int64_t pieces = VEC ? r.cols / 4 : r.cols;
  const uint32_t lane = threadIdx.x & 31;
  int32_t id[kFew / 32];
#pragma unroll
  for (int k = 0; k < kFew / 32; ++k) id[k] = k * 32 + lane < r.n ? __ldg(ids + k * 32 + lane) : -1;
  const int64_t units = (int64_t)r.rows * r.slabs;
  for (int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); unit < units; unit += (int64_t)gridDim.x * (kThreads / 32)) {
    const int32_t row = (int32_t)(unit / r.slabs);
    const int64_t c = unit % r.slabs * 32 + lane;
    const bool in = c < pieces;
    uint32_t mine[kFew / 32], any = 0;
#pragma unroll
    for (int k = 0; k < kFew / 32; ++k) any |= mine[k] = __ballot_sync(0xffffffffu, id[k] == row);
    if (ACCUMULATE && !any) continue;
    const T old = ACCUMULATE && in ? reinterpret_cast<const T*>(r.dtable)[(int64_t)row * pieces + c] : P::zero();
    T sum = P::zero();
#pragma unroll
    for (int k = 0; k < kFew / 32; ++k) {
      for (uint32_t left = mine[k]; left;) {
        T v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = k * 32 + __ffs(left) - 1;
          v[j] = left && in ? __ldg(reinterpret_cast<const T*>(r.g) + (int64_t)at * pieces + c) : P::zero();
          left &= left - 1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) P::add(sum, v[j]);
      }
    }
    // no tokens: zeros, whatever the scale is
    if (in && any) write_row<VEC, ACCUMULATE>(r, (uint32_t)row, c, sum, old);
    else if (in) reinterpret_cast<T*>(r.dtable)[(int64_t)row * pieces + c] = P::zero();
  }
}
template <bool VEC, bool ACCUMULATE>
rt_status sum_few(rt_ctx* ctx, Runs r, const int32_t* ids) {
  r.slabs = (uint32_t)(((VEC ? r.cols / 4 : r.cols) + 31) / 32);
  rt_launch(ctx, few_tokens_kernel<VEC, ACCUMULATE>, rt_grid_for(ctx, (int64_t)r.rows * r.slabs, kThreads / 32), kThreads, 0, r, ids);
  RT_LAUNCHED(ctx);
  return RT_OK;
}
template <bool VEC, bool ACCUMULATE>
rt_status sum_runs(rt_ctx* ctx, Runs r) {
  const int64_t pieces = VEC ? r.cols / 4 : r.cols;
  r.slabs = (uint32_t)((pieces + 31) / 32);
  r.tiles = (r.n + kRun - 1) / kRun;
  const int64_t sums = ((int64_t)r.tiles * r.slabs + kSumThreads / 32 - 1) / (kSumThreads / 32);
  const int64_t each = (64 << 10) / (4 * r.cols);  // about 64 KB of the table a block
  r.fill_rows = (uint32_t)(each < 16 ? 16 : (each > kFillRows ? kFillRows : each));
  r.sum_blocks = (uint32_t)sums;
  const int64_t blocks = sums + (ACCUMULATE ? 0 : ((int64_t)r.rows + r.fill_rows - 1) / r.fill_rows);
  rt_launch(ctx, run_sums_kernel<VEC, ACCUMULATE>, (unsigned)blocks, kSumThreads, 0, r);  // below 2^31: n * cols < 2^40
  RT_LAUNCHED(ctx);
  if (r.tiles > 1) {
    rt_launch(ctx, join_runs_kernel<VEC, ACCUMULATE>, rt_grid_for(ctx, (int64_t)(r.tiles - 1) * r.slabs, 1, 4), kJoinThreads, 0, r);
    RT_LAUNCHED(ctx);
  }
  return RT_OK;
}

template <int ITEMS>
rt_status launch_cluster_sort(rt_ctx* ctx, const int32_t* ids, uint32_t n, uint32_t rows, int bits, uint2* out, uint32_t* crossing) {
  static RtDeviceOnce once;
  RT_CUDA(ctx, once([] { return cudaFuncSetAttribute(cluster_sort_kernel<ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ClusterSmem<ITEMS>)); }));
  rt_launch(ctx, cluster_sort_kernel<ITEMS>, kCluster, kClusterThreads, sizeof(ClusterSmem<ITEMS>), ids, n, rows, bits, out, crossing);
  RT_LAUNCHED(ctx);
  return RT_OK;
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
  if ((const void*)x != ids && rt_overlap(x, 4 * n, ids, 4 * n)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_token_ids: ids overlaps x");
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
  if (rt_overlap(out, 4 * n * cols, table, 4 * rows * cols) || rt_overlap(out, 4 * n * cols, ids, 4 * n))
    RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_embedding: out overlaps what is read");
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
  RtOnDevice here(ctx);
  if (n == 0) return accumulate ? RT_OK : rt_fill(ctx, dtable, 0.f, rows * cols);
  RT_CHECK_PTR(ctx, g);
  RT_CHECK_PTR(ctx, ids);
  if (rt_overlap(dtable, 4 * rows * cols, g, 4 * n * cols) || rt_overlap(dtable, 4 * rows * cols, ids, 4 * n))
    RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_embedding_backward: dtable overlaps what is read");
  int bits = 1;  // of the largest key, which is `rows`
  while (bits < 32 && (uint64_t)rows >> bits) ++bits;
  const bool vec = cols % 4 == 0 && rt_aligned16(g) && rt_aligned16(dtable);
  Runs r{};
  r.g = g;
  r.n = (uint32_t)n;
  r.rows = (uint32_t)rows;
  r.cols = cols;
  r.scale = scale;
  r.dtable = dtable;
  const int64_t units = rows * (((vec ? cols / 4 : cols) + 31) / 32);
  if (n <= kFew && units <= kFewUnits) {
    if (accumulate) return vec ? sum_few<true, true>(ctx, r, ids) : sum_few<false, true>(ctx, r, ids);
    return vec ? sum_few<true, false>(ctx, r, ids) : sum_few<false, false>(ctx, r, ids);
  }
  const size_t places = (size_t)(n + 1) / 2 * 2, tiles = (size_t)(n + kRun - 1) / kRun;  // an even number: the parts behind the pairs are aligned
  RtScratch work(ctx), sorting(ctx);
  if ((st = work.alloc(sizeof(uint2) * places + sizeof(float) * 2 * tiles * (size_t)cols + sizeof(uint32_t) * (2 + tiles))) != RT_OK) return st;
  uint2* pairs = work.as<uint2>();
  r.parts = reinterpret_cast<float*>(pairs + places);
  r.crossing = reinterpret_cast<uint32_t*>(r.parts + 2 * tiles * (size_t)cols);
  const uint32_t un = (uint32_t)n, urows = (uint32_t)rows;
  if (n <= kRankTokens) {
    rt_launch(ctx, rank_sort_kernel, (un + kWarps * kPerWarp - 1) / (kWarps * kPerWarp), kThreads, 0, ids, un, urows, pairs, r.crossing);
    RT_LAUNCHED(ctx);
  } else if (n <= kCluster * kClusterThreads) {
    st = launch_cluster_sort<1>(ctx, ids, un, urows, bits, pairs, r.crossing);
  } else if (n <= 2 * kCluster * kClusterThreads) {
    st = launch_cluster_sort<2>(ctx, ids, un, urows, bits, pairs, r.crossing);
  } else if (n <= 4 * kCluster * kClusterThreads) {
    st = launch_cluster_sort<4>(ctx, ids, un, urows, bits, pairs, r.crossing);
  } else if (n <= kMaxItems * kCluster * kClusterThreads) {
    st = launch_cluster_sort<kMaxItems>(ctx, ids, un, urows, bits, pairs, r.crossing);
  } else {
    const int blocks = (int)((n + kTile - 1) / kTile);
    if ((st = sorting.alloc(sizeof(uint2) * (size_t)n + sizeof(uint32_t) * (size_t)kDigits * blocks)) != RT_OK) return st;
    Pass p{};
    p.to = pairs;
    uint2* other = sorting.as<uint2>();
    p.counts = reinterpret_cast<uint32_t*>(other + n);
    p.crossing = r.crossing;
    p.n = n;
    p.rows = urows;
    p.blocks = blocks;
    for (p.shift = 0; p.shift < bits; p.shift += 8) {
      p.ids = p.shift == 0 ? ids : nullptr;
      rt_launch(ctx, digit_counts_kernel, blocks, kThreads, 0, p);
      RT_LAUNCHED(ctx);
      rt_launch(ctx, digit_places_kernel, 1, 1024, 0, p.counts, (int64_t)kDigits * blocks);
      RT_LAUNCHED(ctx);
      rt_launch(ctx, digit_scatter_kernel, blocks, kThreads, 0, p);
      RT_LAUNCHED(ctx);
      p.from = p.to;
      p.to = p.to == pairs ? other : pairs;
    }
    pairs = const_cast<uint2*>(p.from);
  }
  if (st != RT_OK) return st;
  r.pairs = pairs;
  if (accumulate) return vec ? sum_runs<true, true>(ctx, r) : sum_runs<false, true>(ctx, r);
  return vec ? sum_runs<true, false>(ctx, r) : sum_runs<false, false>(ctx, r);
}

}  // extern "C"
