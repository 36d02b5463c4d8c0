// Refusals of the entry points for language models, on a context that has no device: each answers with its code and a message, before any
// CUDA call.
#include <cmath>
#include <cstdio>
#include <cstring>

#include "../../rusttensor_b200/csrc/rt_internal.cuh"

static int failures;
#define EXPECT(x) ((x) ? (void)0 : (void)(std::printf("line %d: %s\n", __LINE__, #x), ++failures))
#define REFUSED(call, word) (ctx.last_error.clear(), (call) == RT_ERR_INVALID_OPERATION && ctx.last_error.find(word) != std::string::npos)

int main() {
  rt_ctx ctx;
  float x[64] = {};
  int32_t ids[4] = {};
  const int64_t big = int64_t(1) << 31;
  // embeddings
  EXPECT(rt_embedding(nullptr, x, 1, 1, ids, 1, 1.f, x) == RT_ERR_INVALID_OPERATION);
  EXPECT(REFUSED(rt_embedding(&ctx, x, -1, 1, ids, 1, 1.f, x), "negative"));
  EXPECT(REFUSED(rt_embedding(&ctx, x, 1, -1, ids, 1, 1.f, x), "negative"));
  EXPECT(REFUSED(rt_embedding(&ctx, x, 1, 1, ids, -1, 1.f, x), "negative"));
  EXPECT(REFUSED(rt_embedding(&ctx, x, big, 1, ids, 1, 1.f, x), "out of range"));
  EXPECT(REFUSED(rt_embedding(&ctx, x, big - 1, big - 1, ids, 1, 1.f, x), "out of range"));
  EXPECT(REFUSED(rt_embedding(&ctx, nullptr, 1, 1, ids, 1, 1.f, x), "table"));
  EXPECT(REFUSED(rt_embedding(&ctx, x, 1, 1, nullptr, 1, 1.f, x), "ids"));
  EXPECT(REFUSED(rt_embedding(&ctx, x, 1, 1, ids, 1, 1.f, nullptr), "out"));
  EXPECT(rt_embedding(&ctx, nullptr, 0, 4, nullptr, 0, 1.f, nullptr) == RT_OK);
  EXPECT(REFUSED(rt_embedding_backward(&ctx, x, ids, 1, -1, 1, 1.f, x, 0), "negative"));
  EXPECT(REFUSED(rt_embedding_backward(&ctx, x, ids, big, 1, 1, 1.f, x, 0), "out of range"));
  EXPECT(REFUSED(rt_embedding_backward(&ctx, nullptr, ids, 1, 1, 1, 1.f, x, 0), " g"));
  EXPECT(REFUSED(rt_embedding_backward(&ctx, x, nullptr, 1, 1, 1, 1.f, x, 0), "ids"));
  EXPECT(REFUSED(rt_embedding_backward(&ctx, x, ids, 1, 1, 1, 1.f, nullptr, 0), "dtable"));
  EXPECT(rt_embedding_backward(&ctx, nullptr, nullptr, 0, 3, 4, 1.f, x, 1) == RT_OK);
  EXPECT(rt_embedding_backward(&ctx, nullptr, nullptr, 0, 0, 4, 1.f, nullptr, 0) == RT_OK);
  EXPECT(REFUSED(rt_token_ids(&ctx, x, -1, ids), "negative"));
  EXPECT(REFUSED(rt_token_ids(&ctx, x, 1, nullptr), "ids"));
  EXPECT(rt_token_ids(&ctx, nullptr, 0, nullptr) == RT_OK);
  EXPECT(REFUSED(rt_embedding(&ctx, x, 4, 4, ids, 2, 1.f, x + 15), "overlaps"));
  EXPECT(REFUSED(rt_embedding(&ctx, x, 4, 4, reinterpret_cast<int32_t*>(x + 20), 2, 1.f, x + 16), "overlaps"));
  EXPECT(REFUSED(rt_embedding_backward(&ctx, x, ids, 4, 4, 4, 1.f, x + 15, 1), "overlaps"));
  EXPECT(REFUSED(rt_token_ids(&ctx, x, 4, reinterpret_cast<int32_t*>(x + 1)), "overlaps"));
  // gated scan
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, x, 2, nullptr, -1, 1, 2, x), "negative"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, x, 1, nullptr, 1, 1, 2, x), "apart"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, x, 2, nullptr, big, 1, 2, x), "out of range"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, x, 1 << 20, nullptr, 1, 1 << 20, 1 << 12, x), "out of range"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, nullptr, x, 2, nullptr, 1, 1, 2, x), " f"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, nullptr, 2, nullptr, 1, 1, 2, x), " v"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, x, 2, nullptr, 1, 1, 2, nullptr), " h"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, x, 2, x, 2, 1, 2, x), "h0"));
  EXPECT(rt_gated_scan(&ctx, nullptr, nullptr, 2, nullptr, 0, 1, 2, nullptr) == RT_OK);
  EXPECT(rt_gated_scan(&ctx, nullptr, nullptr, 0, nullptr, 3, 1, 0, nullptr) == RT_OK);
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, x, x, 2, nullptr, x, x, 1, 1, 2, x, x, 1, nullptr), "apart"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, x, x, 2, nullptr, x, x, 1, -1, 2, x, x, 2, nullptr), "negative"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, x, x, 2, nullptr, nullptr, x, 1, 1, 2, x, x, 2, nullptr), " h"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, x, x, 2, nullptr, x, nullptr, 1, 1, 2, x, x, 2, nullptr), "dh"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, x, x, 2, nullptr, x, x, 1, 1, 2, nullptr, x, 2, nullptr), "df"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, x, x, 2, nullptr, x, x, 1, 1, 2, x, nullptr, 2, nullptr), "dv"));
  EXPECT(rt_gated_scan_backward(&ctx, x, x, 2, nullptr, x, x, 0, 1, 2, x, x, 2, nullptr) == RT_OK);
  // 4 rows of 2 columns: h onto f, onto v, onto another part of h0; a gradient onto each thing that is read and onto each other result
  float z[64] = {};
  EXPECT(REFUSED(rt_gated_scan(&ctx, x, z, 4, nullptr, 4, 1, 2, x + 12), "overlaps"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, z, x + 2, 4, nullptr, 4, 1, 2, x), "overlaps"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, z, z, 4, x + 6, 4, 1, 2, x), "overlaps"));
  EXPECT(REFUSED(rt_gated_scan(&ctx, z, z, 4, x + 1, 1, 1, 2, x), "overlaps"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, x, z + 2, 4, nullptr, z + 20, z + 30, 4, 1, 2, x + 1, x + 17, 4, nullptr), "overlaps"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, z, z + 2, 4, nullptr, z + 20, x + 20, 4, 1, 2, x, x + 18, 4, nullptr), "overlaps"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, z, z + 2, 4, x + 40, z + 20, z + 30, 4, 1, 2, x, x + 2, 4, x + 41), "overlaps"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, z, z + 2, 4, nullptr, z + 20, z + 30, 4, 1, 2, x, x + 1, 4, nullptr), "results overlap"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, z, z + 2, 4, nullptr, z + 20, z + 30, 4, 1, 2, x, x + 3, 4, nullptr), "results overlap"));
  EXPECT(REFUSED(rt_gated_scan_backward(&ctx, z, z + 2, 4, nullptr, z + 20, z + 30, 4, 1, 2, x, x + 2, 4, x + 10), "results overlap"));
  // Muon
  float *p[2] = {x, x + 32}, *m[2] = {x + 16, x + 48}, *none[2] = {x, nullptr};
  float y[32] = {};
  const float* g[2] = {y, y};
  const int64_t rows[2] = {4, 2}, cols[2] = {4, 3}, negative[2] = {4, -2}, large[2] = {4, 1 << 24};
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, -1, p, g, m, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "matrices"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, p, g, m, rows, cols, 0.1f, 0.9f, 0, 0.f, -1, 1.f), "steps"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, p, g, m, rows, cols, 0.1f, 0.9f, 0, 0.f, 65, 1.f), "steps"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, p, g, m, rows, negative, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "negative"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, p, g, m, rows, large, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "out of range"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, none, g, m, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "params"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, p, g, none, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "momenta"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, nullptr, g, m, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "params"));
  float *twice[2] = {x, x + 12};
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, twice, g, m, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "overlap"));
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, p, g, p, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "overlap"));
  const float* of_m[2] = {x, x + 40};  // the second within a parameter
  float* q[2] = {x + 20, x + 40};
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, q, of_m, m, rows, cols, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "overlap"));
  const int64_t tall[2] = {4, 65537}, wide[2] = {4, 65537};
  EXPECT(REFUSED(rt_muon_step_multi(&ctx, 2, p, g, m, tall, wide, 0.1f, 0.9f, 0, 0.f, 5, 1.f), "out of range"));
  EXPECT(rt_muon_step_multi(&ctx, 0, nullptr, nullptr, nullptr, nullptr, nullptr, 0.1f, 0.9f, 0, 0.f, 5, 1.f) == RT_OK);
  EXPECT(REFUSED(rt_orthogonalize_list(&ctx, 2, g, rows, cols, 5, twice), "overlap"));
  float* onto[2] = {y + 8, x};  // a result within the other's matrix
  EXPECT(REFUSED(rt_orthogonalize_list(&ctx, 2, g, rows, cols, 5, onto), "overlap"));
  EXPECT(REFUSED(rt_orthogonalize_list(&ctx, 2, g, rows, cols, 5, none), "outs"));
  const float* same[2] = {y, y};  // one of the results in the place that the other is read from, in either order
  float *in_place[2] = {y, x}, *in_place_too[2] = {x, y};
  const int64_t square[2] = {4, 4};
  EXPECT(REFUSED(rt_orthogonalize_list(&ctx, 2, same, square, square, 5, in_place), "overlap"));
  EXPECT(REFUSED(rt_orthogonalize_list(&ctx, 2, same, square, square, 5, in_place_too), "overlap"));
  EXPECT(REFUSED(rt_orthogonalize_list(&ctx, 1, g, nullptr, cols, 5, p), "rows"));
  EXPECT(ctx.launches == 0);
  return failures ? 1 : 0;
}
