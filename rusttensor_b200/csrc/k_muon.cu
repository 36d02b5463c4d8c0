// Muon: an optimizer step whose update is the momentum with its singular values brought near one.
//
//   m = mu m + s g      u = m, or s g + mu m (nesterov)      p = (1 - lr wd) p - lr sqrt(max(1, cols / rows)) O(u)
//
// O(u) comes from Newton-Schulz steps on X = u / (|u| + 1e-7): X <- (a I + b G + c G^2) X with G = X X^T, which takes every singular value x to
// a x + b x^3 + c x^5, with the published coefficients 3.4445, -4.7750, 2.0315: five steps bring values between 0.002 and 1 to between 0.7 and
// 1.2.  G is taken on the shorter side; a matrix with more rows than columns is transposed for the steps.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "rt_internal.cuh"

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

rt_status check_sizes(rt_ctx* ctx, const char* who, int count, const int64_t* rows, const int64_t* cols, int steps) {
  if (count < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: %d matrices", who, count);
  if (steps < 0 || steps > 64) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: between 0 and 64 steps, got %d", who, steps);
  if (count == 0) return RT_OK;
  RT_CHECK_PTR(ctx, rows);
  RT_CHECK_PTR(ctx, cols);
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 0 || cols[i] < 0) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: negative size", who);
    if (rows[i] >= (1 << 24) || cols[i] >= (1 << 24) || rows[i] * cols[i] >= (1ll << 40)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "%s: size out of range", who);
  }
  return RT_OK;
}
// Whether no two of the blocks that are written overlap.
bool apart(std::vector<std::pair<uintptr_t, uintptr_t>> blocks) {
  std::sort(blocks.begin(), blocks.end());
  for (size_t i = 1; i < blocks.size(); ++i)
    if (blocks[i].first < blocks[i - 1].second) return false;
  return true;
}
std::pair<uintptr_t, uintptr_t> block_of(const float* p, int64_t n) { return {(uintptr_t)p, (uintptr_t)(p + n)}; }

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
    std::vector<std::pair<uintptr_t, uintptr_t>> written;
    for (int i = 0; i < count; ++i) {
      if (rows[i] == 0 || cols[i] == 0) continue;
      RT_CHECK_PTR(ctx, xs[i]);
      RT_CHECK_PTR(ctx, outs[i]);
      written.push_back(block_of(outs[i], rows[i] * cols[i]));
      Matrix q{};
      q.u.x = xs[i];
      q.rows = rows[i];
      q.cols = cols[i];
      q.out = outs[i];
      list.push_back(q);
    }
    if (!apart(written)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_orthogonalize_list: two results overlap");
    RtOnDevice here(ctx);
    for (const Matrix& q : list)
      if ((st = orthogonalize(ctx, q, steps)) != RT_OK) return st;
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
    std::vector<std::pair<uintptr_t, uintptr_t>> written;
    for (int i = 0; i < n_tensors; ++i) {
      if (rows[i] == 0 || cols[i] == 0) continue;
      RT_CHECK_PTR(ctx, params[i]);
      RT_CHECK_PTR(ctx, grads[i]);
      RT_CHECK_PTR(ctx, momenta[i]);
      written.push_back(block_of(params[i], rows[i] * cols[i]));
      written.push_back(block_of(momenta[i], rows[i] * cols[i]));
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
    if (!apart(written)) RT_FAIL(ctx, RT_ERR_INVALID_OPERATION, "rt_muon_step_multi: two of the parameters and momenta overlap");
    RtOnDevice here(ctx);
    for (const Matrix& q : list)
      if ((st = orthogonalize(ctx, q, steps)) != RT_OK) return st;
  } catch (const std::bad_alloc&) {
    RT_FAIL(ctx, RT_ERR_OOM, "rt_muon_step_multi: out of host memory");
  }
  return RT_OK;
}

}  // extern "C"
