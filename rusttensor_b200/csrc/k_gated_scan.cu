// Gated linear recurrence over a sequence, time-major, and its gradient:
//
//   a_t = sigmoid(f_t)      h_t = a_t h_{t-1} + (1 - a_t) v_t
//   d_t = dh_t + a_{t+1} d_{t+1}      df_t = d_t (h_{t-1} - v_t) a_t (1 - a_t)      dv_t = d_t (1 - a_t)      dh0 = a_0 d_0
//
// No gate depends on the state, so nothing but the state itself goes from timestep to timestep.  f = +inf keeps the state (a padded
// timestep), f = -inf forgets it (the first one of another sequence), both without a gradient.
//
// Timesteps in a row are one timestep: from state h they lead to A h + B, with A the product of the gates.  So the sequence is walked through in
// stretches.  The threads have some columns and timesteps each, units of lanes, warps and the blocks of a cluster one stretch after
// the other; they tell one another their A and B (shuffles, shared memory, the cluster's), after which every thread knows the state
// that it starts from and its timesteps are a multiply-add each.  Everything is read and written once; the loads of the next stretch
// are in flight meanwhile, or those of other blocks.  What is added in which order depends on the sizes alone.
//
// 12 bytes an element forward and 24 backward, in TB/s of those: 128 timesteps of 64 x 512 11.4 us forward (4.4), 19.7 backward (5.1); 1000 of 16 x 1000
// in matrices of their own 38 (5.0); 65536 of 1 x 512 87 - 95 (4.2 - 4.6) and 166 (4.9); 30011 of 3 x 257 backward 136 - 141 (3.9 - 4.1).  Nothing is
// saturated there: long sequences take half of the memory's rate and half of the issue slots (46 and 80 instructions an element, 103 backward with one
// column at a time) with a quarter of the warps, so it is what a warp waits for that counts, its loads and the exchange.  A training batch
// in a row, which the L2 cache holds, takes rounds: 1024 strips for 592 places are two, each with its first loads' latency.  A thread
// per column, which reads ahead eight timesteps, takes 24 us for the first and 9.4 ms for the third; it remains for up to eight timesteps.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "rt_internal.cuh"
#include "tc_common.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 128, kAhead = 8;

struct ScanArgs {
  const float *f, *v;
  int64_t ld;
  const float* h0;
  int64_t steps, batch, hidden;
  float* h;
  const float *states, *dh;
  float *df, *dv;
  int64_t ldd;
  float* dh0;
  int* status;
  uint32_t polls;  // looks at what another block of the cluster has not sent yet
};
// sigmoid(f) and 1 - sigmoid(f), each to the last bits: the smaller one is not the difference of two near ones.  1 + e lies in [1, 2], where the
// approximate reciprocal is within one unit of the last place (a division: half of one).
__device__ __forceinline__ void gate(float f, float& a, float& rest) {
  const float e = expf(-fabsf(f));
  float large;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(large) : "f"(1.f + e));
  const float small = e * large;
  a = f < 0.f ? small : large;
  rest = f < 0.f ? large : small;
}
// A product of gates, of which `least` is the smallest, is not zero unless that is: an infinite state stays infinite, as it does timestep by timestep.
// What that adds is 2^-149 of a state, half of which a product down there is off by anyway.
__device__ __forceinline__ float not_lost(float product, float least) { return fmaxf(product, fminf(least, 0x1p-149f)); }

// A thread has a column and walks through the sequence, the loads of eight timesteps in flight.
__global__ void __launch_bounds__(kThreads) scan_columns_kernel(const ScanArgs s) {
  RT_PDL_ENTRY();
  const int64_t columns = s.batch * s.hidden;
  const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (col >= columns) return;
  const int64_t in = col / s.hidden * s.ld + col % s.hidden, step = s.batch * s.ld;
  const float *f = s.f + in, *v = s.v + in;
  float* h = s.h + col;
  float state = s.h0 ? s.h0[col] : 0.f;
  for (int64_t t = 0; t < s.steps; t += kAhead) {
    float fs[kAhead], vs[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      fs[k] = t + k < s.steps ? f[k * step] : 0.f;  // h may be in the same place: no read-only loads
      vs[k] = t + k < s.steps ? v[k * step] : 0.f;
    }
    f += kAhead * step;
    v += kAhead * step;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float a, rest;
      gate(fs[k], a, rest);
      state = a * state + rest * vs[k];
      if (t + k < s.steps) h[k * columns] = state;
    }
    h += kAhead * columns;
  }
}
__global__ void __launch_bounds__(kThreads) scan_columns_backward_kernel(const ScanArgs s) {
  RT_PDL_ENTRY();
  const int64_t columns = s.batch * s.hidden;
  const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (col >= columns) return;
  const int64_t in = col / s.hidden * s.ld + col % s.hidden, step = s.batch * s.ld;
  const int64_t out = col / s.hidden * s.ldd + col % s.hidden, step_out = s.batch * s.ldd;
  float carry = 0.f;  // a_{t+1} d_{t+1}
  for (int64_t last = s.steps - 1; last >= 0; last -= kAhead) {
    float fs[kAhead], vs[kAhead], hs[kAhead], gs[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t t = last - k;
      fs[k] = t >= 0 ? __ldg(s.f + in + t * step) : 0.f;
      vs[k] = t >= 0 ? __ldg(s.v + in + t * step) : 0.f;
      hs[k] = t > 0 ? __ldg(s.states + col + (t - 1) * columns) : (t == 0 && s.h0 ? __ldg(s.h0 + col) : 0.f);
      gs[k] = t >= 0 ? __ldg(s.dh + col + t * columns) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t t = last - k;
      if (t >= 0) {
        float a, rest;
        gate(fs[k], a, rest);
        const float d = gs[k] + carry;
        carry = a * d;
        s.df[out + t * step_out] = d * (hs[k] - vs[k]) * a * rest;
        s.dv[out + t * step_out] = d * rest;
      }
    }
  }
  if (s.dh0) s.dh0[col] = carry;
}

// ---- stretches ------------------------------------------------------------------------------------------------------------------------
// A block has C = 16 or 32 columns.  A thread has V of them (128-bit accesses where everything is aligned, V = 4) and S timesteps, a warp several
// units of C / V lanes one after the other in time; then come the warps of a block and the blocks of a cluster (backward: against time).
constexpr int kMaxWarps = 16, kMaxCluster = 8, kAloneWarps = 8;  // of a block in a cluster; blocks; of a block by itself
struct Exchange {
  float2 of_warp[2][kMaxWarps][32];             // A and B, turn by turn: a warp may be one ahead of another that still reads
  float2 of_block[2][kMaxCluster][32];          // of the cluster's blocks, turn by turn
  uint64_t arrived[2];                          // barriers that count the bytes of those
  int gave_up[2];                               // whether a wait of such a turn ran out
};
__device__ __forceinline__ int volatile_load(const int* p) { return *const_cast<const volatile int*>(p); }
template <int V>
struct Vec;
template <>
struct Vec<1> {
  static __device__ __forceinline__ void load(float (&v)[1], const float* p) { v[0] = __ldcs(p); }
  static __device__ __forceinline__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
};
template <>
struct Vec<4> {
  static __device__ __forceinline__ void load(float (&v)[4], const float* p) {
    const float4 q = __ldcs(reinterpret_cast<const float4*>(p));
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
};
// What the blocks of a cluster tell one another goes by asynchronous stores, which a barrier in the receiver's shared memory counts: a barrier of
// the whole cluster would wait for the results of the stretch before to be in memory, too (65536 timesteps of 512 columns: 112 us with it).
// Two turns: a block may be one ahead of another that still reads, not two, since it needs what that one sends after reading.
__device__ __forceinline__ void begin_exchange(Exchange& x) {
  if (threadIdx.x == 0) {
    tc::mbar_init(tc::smem_u32(&x.arrived[0]), 1);
    tc::mbar_init(tc::smem_u32(&x.arrived[1]), 1);
    x.gave_up[0] = x.gave_up[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  cg::this_cluster().sync();
}
__device__ __forceinline__ void send(const float2* place, const uint64_t* barrier, uint32_t to, float a, float b) {
  asm volatile(
      "{\n\t.reg .b32 p, q;\n\t.reg .b64 v;\n\t"
      "mapa.shared::cluster.u32 p, %0, %2;\n\t"
      "mapa.shared::cluster.u32 q, %1, %2;\n\t"
      "mov.b64 v, {%3, %4};\n\t"
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [p], v, [q];\n\t}" ::"r"(tc::smem_u32(place)),
      "r"(tc::smem_u32(barrier)), "r"(to), "f"(a), "f"(b)
      : "memory");
}
// Until this turn's bytes are there, which other blocks of the cluster have written; false if they are not after so many looks.
__device__ __forceinline__ bool receive(const uint64_t* barrier, uint32_t parity, uint32_t polls) {
  for (uint32_t i = 0; i < polls; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(tc::smem_u32(barrier)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// Nobody leaves while another block may still send to it.  Where a wait has run out, what was sent may not have landed: that takes microseconds.
__device__ __forceinline__ void end_exchange(const Exchange& x) {
  __syncthreads();
  if (volatile_load(&x.gave_up[0]) | volatile_load(&x.gave_up[1])) {
    const long long from = clock64();
    while (clock64() - from < 2000000) {
    }
  }
  cg::this_cluster().sync();
}
// From the A and B of this thread's timesteps to the state that they start from.  `state`: of column `lane` before the cluster's stretch, afterwards
// before its next one.  False in all of a block if a wait of the turn before ran out: its barrier may be used no more.
template <int C, int V, bool CLUSTER>
__device__ __forceinline__ bool start_of(Exchange& x, const float (&a)[V], const float (&b)[V], int blocks, int rank, int turn, const ScanArgs& s, float& state,
                                         float (&from)[V]) {
  constexpr int kLanes = C / V, kUnits = 32 / kLanes;  // lanes of a unit, units of a warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, unit = lane / kLanes;
  float pa[V], pb[V], ea[V], eb[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {  // over the warp's units: inclusive, then of those before
    pa[j] = a[j];
    pb[j] = b[j];
#pragma unroll
    for (int o = kLanes; o < 32; o *= 2) {
      const float qa = __shfl_up_sync(0xffffffffu, pa[j], o), qb = __shfl_up_sync(0xffffffffu, pb[j], o);
      if (lane >= o) {
        pb[j] = pa[j] * qb + pb[j];
        pa[j] = not_lost(pa[j] * qa, fminf(pa[j], qa));
      }
    }
    ea[j] = 1.f;
    eb[j] = 0.f;
    if (kUnits > 1) {
      const float qa = __shfl_up_sync(0xffffffffu, pa[j], kLanes), qb = __shfl_up_sync(0xffffffffu, pb[j], kLanes);
      if (unit > 0) {
        ea[j] = qa;
        eb[j] = qb;
      }
    }
  }
  if (unit == kUnits - 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) x.of_warp[turn & 1][warp][lane % kLanes * V + j] = make_float2(pa[j], pb[j]);
  }
  __syncthreads();
  if (CLUSTER && volatile_load(&x.gave_up[(turn - 1) & 1])) return false;  // which this turn does not write
  // from here on the lane is the column (lanes beyond C: nobody asks for theirs)
  float wa = 1.f, wb = 0.f, ba = 1.f, bb = 0.f;  // of the warps before this one, of all
  for (int w = 0; w < warps; ++w) {
    if (w == warp) {
      wa = ba;
      wb = bb;
    }
    const float2 q = x.of_warp[turn & 1][w][lane];
    bb = q.x * bb + q.y;
    ba = not_lost(q.x * ba, fminf(q.x, ba));
  }
  float before = state;
  if (CLUSTER) {
    const int slot = turn & 1;
    if (threadIdx.x == 0) tc::mbar_expect_tx(tc::smem_u32(&x.arrived[slot]), blocks * 32 * (uint32_t)sizeof(float2));
    for (int to = warp; to < blocks; to += warps) send(&x.of_block[slot][rank][lane], &x.arrived[slot], to, ba, bb);
    if (!receive(&x.arrived[slot], turn >> 1 & 1, s.polls)) {
      *const_cast<volatile int*>(&x.gave_up[slot]) = 1;
      tc::record_status(s.status, 82);
    }
    for (int r = 0; r < blocks; ++r) {
      if (r == rank) before = state;
      const float2 q = x.of_block[slot][r][lane];
      state = q.x * state + q.y;
    }
  } else {
    state = ba * state + bb;
  }
  before = wa * before + wb;
#pragma unroll
  for (int j = 0; j < V; ++j) from[j] = ea[j] * __shfl_sync(0xffffffffu, before, lane % kLanes * V + j) + eb[j];
  return true;
}

template <int C, int V, int S, bool CLUSTER>
__global__ void __launch_bounds__(32 * (CLUSTER ? kMaxWarps : kAloneWarps), CLUSTER ? 1 : 4) scan_stretches_kernel(const ScanArgs s, int blocks) {
  RT_PDL_ENTRY();
  __shared__ Exchange x;
  constexpr int kLanes = C / V;
  const int rank = CLUSTER ? blockIdx.x % blocks : 0, lane = threadIdx.x & 31;
  const int64_t columns = s.batch * s.hidden, col0 = (int64_t)(CLUSTER ? blockIdx.x / blocks : blockIdx.x) * C, col = col0 + lane % kLanes * V;
  const bool in = col < columns;
  const int64_t step = s.batch * s.ld, at = in ? col / s.hidden * s.ld + col % s.hidden : 0;
  const int units = blockDim.x / kLanes;
  const int64_t all = (int64_t)blocks * units * S;  // timesteps of the cluster
  int64_t t = ((int64_t)rank * units + threadIdx.x / kLanes) * S;
  const float *f = s.f + at + t * step, *v = s.v + at + t * step;
  float* h = s.h + col + t * columns;
  float fs[S][V], vs[S][V];
  int left;
  auto load = [&] {
    left = in ? (int)max((int64_t)0, min((int64_t)S, s.steps - t)) : 0;
    const float *pf = f, *pv = v;
    if (left == S) {
#pragma unroll
      for (int k = 0; k < S; ++k, pf += step, pv += step) {
        Vec<V>::load(fs[k], pf);
        Vec<V>::load(vs[k], pv);
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < S; ++k, pf += step, pv += step) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        fs[k][j] = INFINITY;  // which leaves the state as it is
        vs[k][j] = 0.f;
      }
      if (k < left) {
        Vec<V>::load(fs[k], pf);
        Vec<V>::load(vs[k], pv);
      }
    }
  };
  float state = s.h0 && lane < C && col0 + lane < columns ? __ldg(s.h0 + col0 + lane) : 0.f;
  if (CLUSTER) {  // elsewhere the other blocks of the SM keep the memory busy
    load();
    begin_exchange(x);
  }
  int turn = 0;
  for (int64_t t0 = 0; t0 < s.steps; t0 += all, ++turn) {
    if (!CLUSTER) load();
    float a[S][V], b[S][V], all_a[V], all_b[V], least[V];  // of each timestep; of the thread's together
#pragma unroll
    for (int k = 0; k < S; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float rest;
        gate(fs[k][j], a[k][j], rest);
        b[k][j] = rest * vs[k][j];
        all_b[j] = k > 0 ? a[k][j] * all_b[j] + b[k][j] : b[k][j];
        all_a[j] = k > 0 ? a[k][j] * all_a[j] : a[k][j];
        least[j] = k > 0 ? fminf(a[k][j], least[j]) : a[k][j];
      }
#pragma unroll
    for (int j = 0; j < V; ++j) all_a[j] = not_lost(all_a[j], least[j]);
    const int mine = left;
    t += all;
    f += all * step;
    v += all * step;
    if (CLUSTER && t0 + all < s.steps) load();
    float from[V];
    if (!start_of<C, V, CLUSTER>(x, all_a, all_b, blocks, rank, turn, s, state, from)) break;
    float* ph = h;
#pragma unroll
    for (int k = 0; k < S; ++k, ph += columns) {
#pragma unroll
      for (int j = 0; j < V; ++j) from[j] = a[k][j] * from[j] + b[k][j];
      if (k < mine) Vec<V>::store(ph, from);
    }
    h += all * columns;
  }
  if (CLUSTER) end_exchange(x);
}

// The same against time, for e_t = a_t d_t = a_t e_{t+1} + a_t dh_t, from which d_t = dh_t + e_{t+1}.
template <int C, int V, int S, bool CLUSTER>
__global__ void __launch_bounds__(32 * (CLUSTER ? kMaxWarps : kAloneWarps), CLUSTER ? 1 : 4) scan_stretches_backward_kernel(const ScanArgs s, int blocks) {
  RT_PDL_ENTRY();
  __shared__ Exchange x;
  constexpr int kLanes = C / V;
  const int rank = CLUSTER ? blockIdx.x % blocks : 0, lane = threadIdx.x & 31;
  const int64_t columns = s.batch * s.hidden, col0 = (int64_t)(CLUSTER ? blockIdx.x / blocks : blockIdx.x) * C, col = col0 + lane % kLanes * V;
  const bool in = col < columns;
  const int64_t step = s.batch * s.ld, step_out = s.batch * s.ldd;
  const int64_t at = in ? col / s.hidden * s.ld + col % s.hidden : 0, at_out = in ? col / s.hidden * s.ldd + col % s.hidden : 0;
  const int units = blockDim.x / kLanes;
  const int64_t all = (int64_t)blocks * units * S;
  int64_t t = s.steps - 1 - ((int64_t)rank * units + threadIdx.x / kLanes) * S;  // the thread's last timestep, with which it begins
  const float *f = s.f + at + t * step, *v = s.v + at + t * step, *h = s.states + col + (t - 1) * columns, *g = s.dh + col + t * columns;
  float *df = s.df + at_out + t * step_out, *dv = s.dv + at_out + t * step_out;
  float fs[S][V], vs[S][V], hs[S][V], gs[S][V];
  int left;
  auto load = [&] {
    left = in ? (int)max((int64_t)0, min((int64_t)S, t + 1)) : 0;
    const float *pf = f, *pv = v, *ph = h, *pg = g;
    if (left == S && t >= S) {
#pragma unroll
      for (int k = 0; k < S; ++k, pf -= step, pv -= step, ph -= columns, pg -= columns) {
        Vec<V>::load(fs[k], pf);
        Vec<V>::load(vs[k], pv);
        Vec<V>::load(gs[k], pg);
        Vec<V>::load(hs[k], ph);
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < S; ++k, pf -= step, pv -= step, ph -= columns, pg -= columns) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        fs[k][j] = INFINITY;
        vs[k][j] = hs[k][j] = gs[k][j] = 0.f;
      }
      if (k < left) {
        Vec<V>::load(fs[k], pf);
        Vec<V>::load(vs[k], pv);
        Vec<V>::load(gs[k], pg);
        if (t > k) Vec<V>::load(hs[k], ph);
        else if (s.h0) Vec<V>::load(hs[k], s.h0 + col);
      }
    }
  };
  float state = 0.f;
  if (CLUSTER) {  // elsewhere the other blocks of the SM keep the memory busy
    load();
    begin_exchange(x);
  }
  int turn = 0;
  for (int64_t t0 = 0; t0 < s.steps; t0 += all, ++turn) {
    if (!CLUSTER) load();
    float a[S][V], g_now[S][V], slope[S][V], rest[S][V], all_a[V], all_b[V], least[V];  // of each timestep; of the thread's together: e, from e behind them
#pragma unroll
    for (int k = 0; k < S; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        gate(fs[k][j], a[k][j], rest[k][j]);
        slope[k][j] = (hs[k][j] - vs[k][j]) * a[k][j] * rest[k][j];
        g_now[k][j] = gs[k][j];
        all_b[j] = a[k][j] * (k > 0 ? gs[k][j] + all_b[j] : gs[k][j]);
        all_a[j] = k > 0 ? a[k][j] * all_a[j] : a[k][j];
        least[j] = k > 0 ? fminf(a[k][j], least[j]) : a[k][j];
      }
#pragma unroll
    for (int j = 0; j < V; ++j) all_a[j] = not_lost(all_a[j], least[j]);
    const int mine = left;
    t -= all;
    f -= all * step;
    v -= all * step;
    h -= all * columns;
    g -= all * columns;
    if (CLUSTER && t0 + all < s.steps) load();
    float from[V];
    if (!start_of<C, V, CLUSTER>(x, all_a, all_b, blocks, rank, turn, s, state, from)) break;
    float *pf = df, *pv = dv;
#pragma unroll
    for (int k = 0; k < S; ++k, pf -= step_out, pv -= step_out) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = g_now[k][j] + from[j];
        slope[k][j] *= d;
        rest[k][j] *= d;
        from[j] = a[k][j] * d;
      }
      if (k < mine) {
        Vec<V>::store(pf, slope[k]);
        Vec<V>::store(pv, rest[k]);
      }
    }
    df -= all * step_out;
    dv -= all * step_out;
  }
  if (CLUSTER) end_exchange(x);
  if (s.dh0 && rank == 0 && threadIdx.x < C && col0 + lane < columns) s.dh0[col0 + lane] = state;
}

// How a sequence is cut: columns and warps of a block, blocks of a cluster; a block by itself has no other kind.
struct Cut {
  int columns, warps, blocks;
  int64_t strips;
};
// Clusters that the SMs hold at once, with blocks of 8 warps and of 16.
struct Fits {
  int clusters[2][kMaxCluster + 1];
};
template <class Kernel>
rt_status launch_stretches(rt_ctx* ctx, Kernel kern, const ScanArgs& s, const Cut& c, int* fits = nullptr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(c.strips * c.blocks);
  cfg.blockDim = (unsigned)c.warps * 32;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)c.blocks;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = c.blocks > 1 ? 2 : 1;
  if (fits) {
    RT_CUDA(ctx, cudaOccupancyMaxActiveClusters(fits, kern, &cfg));
    return RT_OK;
  }
  RT_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, s, c.blocks));
  RT_LAUNCHED(ctx);
  return RT_OK;
}
// Asked once a device, of the kernel that needs most: how clusters lie in groups of SMs is the device's (148 SMs hold 15 of 8 blocks if a block takes
// an SM, 26 of 5).
rt_status fits_of(rt_ctx* ctx, Fits* fits) {
  constexpr int kDevices = 64;  // beyond: asked every time
  static std::atomic<int> known[kDevices][2][kMaxCluster + 1];
  for (int k = 0; k < 2; ++k)
    for (int blocks = 2; blocks <= kMaxCluster; ++blocks) {
      int& n = fits->clusters[k][blocks];
      if (ctx->device < kDevices && (n = known[ctx->device][k][blocks].load(std::memory_order_relaxed)) > 0) continue;
      rt_status st = launch_stretches(ctx, scan_stretches_backward_kernel<32, 4, 2, true>, ScanArgs{}, Cut{32, 8 << k, blocks, 1}, &n);
      if (st != RT_OK) return st;
      n = std::max(n, 1);
      if (ctx->device < kDevices) known[ctx->device][k][blocks].store(n, std::memory_order_relaxed);
    }
  return RT_OK;
}
// What takes the fewest rounds of stretches, two more (by itself: one) for a cluster's start, and as often as the clusters do not fit at once.  A
// round takes about 2.7 us if SMs have 16 warps and 0.65 of it with 8; with strips of 16 columns, 64 bytes of a row, a little longer, and a lot
// if rows are not aligned to sectors; without a cluster longer, too, since it waits for its loads.  30011 timesteps of 771 columns, backward:
// five blocks of 16 warps 132 us, eight of 8 164; 65536 of 512: 32 columns and eight of 8 warps 130, 16 columns 85; 40000 of 300, backward:
// six of 16 warps and 16 columns 91, eight of 8 115.
rt_status cut(rt_ctx* ctx, int64_t steps, int64_t columns, int v, int s, Cut* best) {
  Fits fits{};
  rt_status st = fits_of(ctx, &fits);
  if (st != RT_OK) return st;
  double least = 1e300;
  for (int width = 32; width >= 16; width /= 2) {
    const int warp_steps = v * s * 32 / width;
    const int64_t strips = (columns + width - 1) / width, stretches = (steps + warp_steps - 1) / warp_steps;
    for (int k = 0; k < 2; ++k) {
      const int warps = (int)std::min<int64_t>(stretches, 8 << k);
      for (int blocks = 1; blocks <= kMaxCluster && (blocks - 1) * warps < stretches; ++blocks) {
        if (blocks == 1 && (width == 16 || warps > kAloneWarps)) continue;
        const int64_t fit = blocks == 1 ? 4 * (int64_t)ctx->sm_count : fits.clusters[k][blocks];
        const double round = (blocks == 1 ? 1.3 : (width == 32 ? 1.0 : (v == 1 ? 1.4 : 1.02))) * (blocks > 1 && k == 0 && strips <= fits.clusters[1][blocks] ? 0.65 : 1.0);
        const double time = (double)((strips + fit - 1) / fit) * (double)((stretches + blocks * warps - 1) / (blocks * warps) + (blocks > 1 ? 2 : 1)) * round;
        if (time < least) {
          least = time;
          *best = {width, warps, blocks, strips};
        }
      }
    }
  }
  return RT_OK;
}
template <int V, int S>
rt_status launch_forward(rt_ctx* ctx, const ScanArgs& s) {
  Cut c{};
  rt_status st = cut(ctx, s.steps, s.batch * s.hidden, V, S, &c);
  if (st != RT_OK) return st;
  if (c.blocks == 1) return launch_stretches(ctx, scan_stretches_kernel<32, V, S, false>, s, c);
  return c.columns == 16 ? launch_stretches(ctx, scan_stretches_kernel<16, V, S, true>, s, c) : launch_stretches(ctx, scan_stretches_kernel<32, V, S, true>, s, c);
}
template <int V, int S>
rt_status launch_backward(rt_ctx* ctx, const ScanArgs& s) {
  Cut c{};
  rt_status st = cut(ctx, s.steps, s.batch * s.hidden, V, S, &c);
  if (st != RT_OK) return st;
  if (c.blocks == 1) return launch_stretches(ctx, scan_stretches_backward_kernel<32, V, S, false>, s, c);
  return c.columns == 16 ? launch_stretches(ctx, scan_stretches_backward_kernel<16, V, S, true>, s, c)
                         : launch_stretches(ctx, scan_stretches_backward_kernel<32, V, S, true>, s, c);
}
// Whether four columns of every matrix can be had at once.
bool aligned(const ScanArgs& s) {
  bool ok = s.hidden % 4 == 0 && s.ld % 4 == 0 && s.ldd % 4 == 0;
  for (const float* p : {s.f, s.v, s.h0, (const float*)s.h, s.states, s.dh, (const float*)s.df, (const float*)s.dv}) ok = ok && rt_aligned16(p);
  return ok;
}

rt_status check_sizes(rt_ctx* ctx, const char* who, int64_t steps, int64_t batch, int64_t hidden, int64_t ld) {
  if (steps < 0 || batch < 0 || hidden < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: negative size", who);
  if (ld < hidden) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: rows of %lld values, %lld apart", who, (long long)hidden, (long long)ld);
  if (steps >= (1ll << 31) || batch >= (1ll << 31) || hidden >= (1ll << 31) || ld >= (1ll << 31) || batch * hidden >= (1ll << 31) ||
      (double)steps * batch * ld >= (double)(1ll << 40))
    RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: size out of range", who);
  return RT_OK;
}

// `rows` rows of `cols` values, ld apart.
struct Rows {
  const float* p;
  int64_t rows, cols, ld;
};
// Whether they share a value: not if they are different columns of one matrix.
bool meet(const Rows& a, const Rows& b) {
  if (!a.p || !b.p || !rt_overlap(a.p, 4 * ((a.rows - 1) * a.ld + a.cols), b.p, 4 * ((b.rows - 1) * b.ld + b.cols))) return false;
  const int64_t bytes = (int64_t)((intptr_t)b.p - (intptr_t)a.p);
  if (a.ld != b.ld || bytes % 4 != 0) return true;
  const int64_t d = (bytes / 4 % a.ld + a.ld) % a.ld;
  return d < a.cols || a.ld - d < b.cols;
}

}  // namespace

extern "C" {

rt_status rt_gated_scan(rt_ctx* ctx, const float* f, const float* v, int64_t ld, const float* h0, int64_t steps, int64_t batch, int64_t hidden, float* h) {
  RT_CHECK_CTX(ctx);
  rt_status st = check_sizes(ctx, "rt_gated_scan", steps, batch, hidden, ld);
  if (st != RT_OK) return st;
  if (steps == 0 || batch == 0 || hidden == 0) return RT_OK;
  RT_CHECK_PTR(ctx, f);
  RT_CHECK_PTR(ctx, v);
  RT_CHECK_PTR(ctx, h);
  if (h == h0 && steps > 1) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_gated_scan: h may be h0 for a single timestep only");
  const Rows states{h, steps * batch, hidden, hidden};
  const bool in_place = steps == 1 && ld == hidden;
  if ((!(in_place && h == f) && meet(states, {f, steps * batch, hidden, ld})) || (!(in_place && h == v) && meet(states, {v, steps * batch, hidden, ld})) ||
      (h != h0 && meet(states, {h0, batch, hidden, hidden})))
    RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_gated_scan: h overlaps what is read");
  RtOnDevice here(ctx);
  ScanArgs s{};
  s.f = f;
  s.v = v;
  s.ld = ld;
  s.h0 = h0;
  s.steps = steps;
  s.batch = batch;
  s.hidden = hidden;
  s.h = h;
  s.status = ctx->device_status;
  s.polls = ctx->sequence_polls;
  if (steps > kAhead) return aligned(s) ? launch_forward<4, 4>(ctx, s) : launch_forward<1, 16>(ctx, s);
  rt_launch(ctx, scan_columns_kernel, (unsigned)((batch * hidden + kThreads - 1) / kThreads), kThreads, 0, s);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

rt_status rt_gated_scan_backward(rt_ctx* ctx, const float* f, const float* v, int64_t ld, const float* h0, const float* h, const float* dh, int64_t steps,
                                 int64_t batch, int64_t hidden, float* df, float* dv, int64_t ldd, float* dh0) {
  RT_CHECK_CTX(ctx);
  rt_status st = check_sizes(ctx, "rt_gated_scan_backward", steps, batch, hidden, ld < ldd ? ld : ldd);
  if (st == RT_OK) st = check_sizes(ctx, "rt_gated_scan_backward", steps, batch, hidden, ld < ldd ? ldd : ld);
  if (st != RT_OK) return st;
  if (batch == 0 || hidden == 0) return RT_OK;
  RtOnDevice here(ctx);
  if (steps == 0) return dh0 ? rt_fill(ctx, dh0, 0.f, batch * hidden) : RT_OK;
  RT_CHECK_PTR(ctx, f);
  RT_CHECK_PTR(ctx, v);
  RT_CHECK_PTR(ctx, h);
  RT_CHECK_PTR(ctx, dh);
  RT_CHECK_PTR(ctx, df);
  RT_CHECK_PTR(ctx, dv);
  const int64_t all = steps * batch;
  const Rows read[] = {{f, all, hidden, ld}, {v, all, hidden, ld}, {h, all, hidden, hidden}, {dh, all, hidden, hidden}, {h0, batch, hidden, hidden}};
  const Rows written[] = {{df, all, hidden, ldd}, {dv, all, hidden, ldd}, {dh0, batch, hidden, hidden}};
  for (const Rows& w : written)
    for (const Rows& r : read)
      if (meet(w, r)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_gated_scan_backward: a result overlaps what is read");
  if (meet(written[0], written[1]) || meet(written[0], written[2]) || meet(written[1], written[2]))
    RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_gated_scan_backward: results overlap");
  ScanArgs s{};
  s.f = f;
  s.v = v;
  s.ld = ld;
  s.h0 = h0;
  s.steps = steps;
  s.batch = batch;
  s.hidden = hidden;
  s.states = h;
  s.dh = dh;
  s.df = df;
  s.dv = dv;
  s.ldd = ldd;
  s.dh0 = dh0;
  s.status = ctx->device_status;
  s.polls = ctx->sequence_polls;
  if (steps > kAhead) return aligned(s) ? launch_backward<4, 2>(ctx, s) : launch_backward<1, 8>(ctx, s);
  rt_launch(ctx, scan_columns_backward_kernel, (unsigned)((batch * hidden + kThreads - 1) / kThreads), kThreads, 0, s);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

}  // extern "C"
