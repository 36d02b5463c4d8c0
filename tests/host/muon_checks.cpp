// Muon's step (k_muon.cu) without a GPU, over stubs of the CUDA runtime that count launches: what can fail is found out before the first launch, which
// changes momenta, and a device that does not hold the products' blocks at once gets them by the framework's other products.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <vector>

#include <cuda.h>
#include "../../rusttensor_b200/csrc/rt_internal.cuh"

static int failures, blocks, mallocs, products, maps_left = -1, mallocs_left = -1, products_left = -1, held = 200;
static unsigned grid;
static std::map<const void*, std::string> names;
static std::vector<std::string> launched;
#define EXPECT(x) ((x) ? (void)0 : (void)(std::printf("line %d: %s\n", __LINE__, #x), ++failures))

static CUresult encode(CUtensorMap* m, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                       CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
  if (maps_left == 0) return CUDA_ERROR_INVALID_VALUE;
  if (maps_left > 0) --maps_left;
  std::memset(m, 0, sizeof(*m));
  return CUDA_SUCCESS;
}
static cudaError_t launch(const void* f, unsigned n) {
  launched.push_back(names[f]);
  if (launched.back().find("newton_schulz") != std::string::npos) grid = n;
  return cudaSuccess;
}
extern "C" {
rt_status rt_malloc(rt_ctx*, size_t bytes, void** out) {
  if (mallocs_left == 0) return RT_ERR_OOM;
  if (mallocs_left > 0) --mallocs_left;
  ++blocks;
  ++mallocs;
  *out = std::malloc(bytes < 64 ? bytes : 64);  // never looked into
  return RT_OK;
}
rt_status rt_free(rt_ctx*, void* p) {
  --blocks;
  std::free(p);
  return RT_OK;
}
rt_status rt_gemm(rt_ctx*, int, int, int64_t, int64_t, int64_t, const float*, int64_t, const float*, int64_t, float*, int64_t, int) {
  if (products_left == 0) return RT_ERR_OOM;
  if (products_left > 0) --products_left;
  ++products;
  return RT_OK;
}
void** __cudaRegisterFatBinary(void*) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char* f, char*, const char* name, int, void*, void*, void*, void*, int*) { names[f] = name; }
char __cudaInitModule(void**) { return 1; }
unsigned __cudaPopCallConfiguration(void*, void*, size_t*, void*) { return 0; }
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaPeekAtLastError() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "stub"; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveClusters(int* n, const void*, const cudaLaunchConfig_t*) { return *n = held / 2, cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int* n, const void*, int, size_t, unsigned) { return *n = held > 0, cudaSuccess; }
cudaError_t cudaLaunchKernel(const void* f, dim3 g, dim3, void**, size_t, cudaStream_t) { return launch(f, g.x); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) { return launch(f, c->gridDim.x); }
cudaError_t cudaGetDriverEntryPoint(const char*, void** f, unsigned long long, cudaDriverEntryPointQueryResult* q) {
  *f = reinterpret_cast<void*>(&encode);
  *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}
}

static int count(const char* name) {
  int n = 0;
  for (const std::string& s : launched) n += s.find(name) != std::string::npos;
  return n;
}

int main() {
  constexpr int kMany = 15;
  char* memory = static_cast<char*>(std::aligned_alloc(256, size_t(1) << 20));  // addresses only
  float *p[kMany], *m[kMany];
  const float* g[kMany];
  int64_t rows[kMany], cols[kMany];
  for (int i = 0; i < kMany; ++i) {
    rows[i] = i == 13 ? 90 : 20;  // one of the second launch's is the largest
    cols[i] = 30;
    p[i] = reinterpret_cast<float*>(memory + 49152 * i);
    m[i] = p[i] + 4096;
    g[i] = p[i] + 8192;
  }
  rt_ctx fresh;
  rt_ctx* ctx = &fresh;
  auto step = [&](int n) {
    launched.clear();
    mallocs = products = 0;
    return rt_muon_step_multi(ctx, n, p, g, m, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f);
  };
  EXPECT(step(1) == RT_OK && launched.size() == 4 && count("newton_schulz") == 1 && mallocs == 1 && products == 0 && blocks == 0);
  EXPECT(step(kMany) == RT_OK && launched.size() == 8 && count("newton_schulz") == 2 && mallocs == 1 && blocks == 0);
  // no room: nothing has been launched, also not the first twelve
  mallocs_left = 0;
  EXPECT(step(kMany) == RT_ERR_OOM && launched.empty() && blocks == 0);
  mallocs_left = -1;
  // a tensor map that cannot be made, of the first matrices or the last ones: all by the other products
  for (int k : {0, 5, 9 * 12, 9 * kMany - 1}) {
    maps_left = k;
    EXPECT(step(kMany) == RT_OK && count("newton_schulz") == 0 && count("apply_kernel") == kMany && products == 15 * kMany && blocks == 0);
    maps_left = k;
    mallocs_left = 1;  // and no room for those
    EXPECT(step(kMany) == RT_ERR_OOM && launched.empty() && blocks == 0);
    mallocs_left = -1;
  }
  maps_left = -1;
  // a product without room: neither its matrix nor those behind it are written
  fresh.use_tensor_cores = false;
  products_left = 15 * 2 + 7;
  EXPECT(step(5) == RT_ERR_OOM && count("apply_kernel") == 2 && count("squares_kernel") == 3 && blocks == 0);
  products_left = -1;
  // a device that does not hold a pair, or a block
  for (held = 1; held >= 0; --held) {
    rt_ctx small;
    ctx = &small;
    EXPECT(step(2) == RT_OK && count("newton_schulz") == (held ? 1 : 0) && products == (held ? 0 : 30));
  }
  // as many blocks as it does hold
  held = 12;
  rt_ctx narrow;
  narrow.sm_count = 10;
  ctx = &narrow;
  rows[0] = cols[0] = 2000;
  p[0] = reinterpret_cast<float*>(std::malloc(3 * 16000000 + 64));
  m[0] = p[0] + 4000000;
  g[0] = m[0] + 4000000;
  EXPECT(step(1) == RT_OK && count("newton_schulz") == 1 && grid > 0 && grid <= 10);
  return failures ? 1 : 0;
}
