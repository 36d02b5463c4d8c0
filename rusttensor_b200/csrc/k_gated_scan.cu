// Gated linear recurrence over a sequence, time-major, and its gradient:
//
//   a_t = sigmoid(f_t)      h_t = a_t h_{t-1} + (1 - a_t) v_t
//   d_t = dh_t + a_{t+1} d_{t+1}      df_t = d_t (h_{t-1} - v_t) a_t (1 - a_t)      dv_t = d_t (1 - a_t)      dh0 = a_0 d_0
//
// No gate depends on the state, so nothing but the state itself goes from timestep to timestep.  f = +inf keeps the state (a padded
// timestep), f = -inf forgets it (the first one of another sequence), both without a gradient.
#include "rt_internal.cuh"

namespace {

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
};
// sigmoid(f) and 1 - sigmoid(f), each to the last bits: the smaller one is not the difference of two near ones.
__device__ __forceinline__ void gate(float f, float& a, float& rest) {
  const float e = expf(-fabsf(f)), large = 1.f / (1.f + e), small = e * large;
  a = f < 0.f ? small : large;
  rest = f < 0.f ? large : small;
}

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
      fs[k] = t + k < s.steps ? __ldg(f + k * step) : 0.f;
      vs[k] = t + k < s.steps ? __ldg(v + k * step) : 0.f;
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

rt_status check_sizes(rt_ctx* ctx, const char* who, int64_t steps, int64_t batch, int64_t hidden, int64_t ld) {
  if (steps < 0 || batch < 0 || hidden < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: negative size", who);
  if (ld < hidden) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: rows of %lld values, %lld apart", who, (long long)hidden, (long long)ld);
  if (steps >= (1ll << 31) || batch >= (1ll << 31) || hidden >= (1ll << 31) || ld >= (1ll << 31) || batch * hidden >= (1ll << 31) ||
      (double)steps * batch * ld >= (double)(1ll << 40))
    RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: size out of range", who);
  return RT_OK;
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
  if (steps == 0) return dh0 ? rt_fill(ctx, dh0, 0.f, batch * hidden) : RT_OK;
  RT_CHECK_PTR(ctx, f);
  RT_CHECK_PTR(ctx, v);
  RT_CHECK_PTR(ctx, h);
  RT_CHECK_PTR(ctx, dh);
  RT_CHECK_PTR(ctx, df);
  RT_CHECK_PTR(ctx, dv);
  RtOnDevice here(ctx);
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
  rt_launch(ctx, scan_columns_backward_kernel, (unsigned)((batch * hidden + kThreads - 1) / kThreads), kThreads, 0, s);
  RT_LAUNCHED(ctx);
  return RT_OK;
}

}  // extern "C"
