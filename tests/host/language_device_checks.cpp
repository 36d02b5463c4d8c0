// Embeddings and the gated recurrence (k_embedding.cu, k_gated_scan.cu) on a context whose device is not the caller's current one, over stubs of the
// CUDA runtime: whatever a call launches, itself or by another entry point, it launches with the context's device as the current one, and the
// caller's is put back.
#include <cstdio>
#include <cstdlib>

#include "../../rusttensor_b200/csrc/rt_internal.cuh"

static int failures, current, launches, elsewhere;
#define EXPECT(x) ((x) ? (void)0 : (void)(std::printf("line %d: %s\n", __LINE__, #x), ++failures))

static cudaError_t launch() {
  ++launches;
  elsewhere += current != 1;
  return cudaSuccess;
}
extern "C" {
rt_status rt_malloc(rt_ctx*, size_t, void** out) { return *out = std::malloc(64), RT_OK; }
rt_status rt_free(rt_ctx*, void* p) { return std::free(p), RT_OK; }
rt_status rt_fill(rt_ctx*, float*, float, int64_t) { return launch(), RT_OK; }
void** __cudaRegisterFatBinary(void*) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
char __cudaInitModule(void**) { return 1; }
unsigned __cudaPopCallConfiguration(void*, void*, size_t*, void*) { return 0; }
cudaError_t cudaGetDevice(int* d) { return *d = current, cudaSuccess; }
cudaError_t cudaSetDevice(int d) { return current = d, cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaPeekAtLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "stub"; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t*) { return *n = 15, cudaSuccess; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return launch(); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { return launch(); }
}

int main() {
  rt_ctx ctx;
  ctx.device = 1;
  alignas(16) static float x[4096], y[4096], z[4096], w[4096];
  int32_t ids[4] = {};
  auto there = [&](rt_status st, int least) {
    const bool ok = st == RT_OK && launches >= least && elsewhere == 0 && current == 0;
    launches = elsewhere = current = 0;
    return ok;
  };
  EXPECT(there(rt_token_ids(&ctx, x, 4, ids), 1));
  EXPECT(there(rt_embedding(&ctx, x, 4, 4, ids, 4, 1.f, y), 1));
  EXPECT(there(rt_embedding_backward(&ctx, x, ids, 4, 4, 4, 1.f, y, 0), 1));
  EXPECT(there(rt_embedding_backward(&ctx, nullptr, nullptr, 0, 4, 4, 1.f, y, 0), 1));  // no tokens: zeros
  EXPECT(there(rt_gated_scan(&ctx, x, y, 4, nullptr, 3, 1, 4, z), 1));
  EXPECT(there(rt_gated_scan(&ctx, x, y, 4, nullptr, 300, 1, 4, z), 1));
  EXPECT(there(rt_gated_scan_backward(&ctx, x, x, 4, nullptr, x, x, 300, 1, 4, y, z, 4, w), 1));
  EXPECT(there(rt_gated_scan_backward(&ctx, x, x, 4, nullptr, x, x, 0, 1, 4, y, z, 4, w), 1));  // no timesteps: zeros
  return failures ? 1 : 0;
}
