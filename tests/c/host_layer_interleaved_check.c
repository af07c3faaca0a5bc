/* host_layer_interleaved_check.c - sums over groups of rows whose results lie row beside row, not matrix behind matrix (include/skl-gfx950.h:
 * skl_gemm_groupedk), through the host layer (skl_amd/csrc/skl_api_grouped.c) on host memory under the sanitizers. The stand-in for the launch writes
 * every element that the interface says is written; what lies between has to come back as it was. Prints "interleaved ok". */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/skl-gfx950.h"
#include "../../skl_amd/csrc/skl_grouped.h"

static int g_failures, g_launches, g_error;
static void expect(int ok, const char *what) {
  if (ok) return;
  ++g_failures;
  printf("FAIL: %s\n", what);
}

void *skl_hip_malloc(size_t bytes) { return malloc(bytes); }
void skl_hip_free(void *p) { free(p); }
int skl_hip_memcpy_h2d(void *d, const void *s, size_t n) {
  memcpy(d, s, n);
  return 0;
}
int skl_hip_memcpy_d2h(void *d, const void *s, size_t n) {
  memcpy(d, s, n);
  return 0;
}
int skl_hip_get_pointer_mode(void) { return 0; }
int skl_hip_pointer_is_device(const void *p) {
  (void)p;
  return 0;
}
int skl_hip_get_beta_zero_mode(void) { return 0; }
void skl_hip_record_error(int code, const char *what) {
  (void)what;
  g_error = code;
}
int skl_hip_launch_group_rows(size_t count, const int32_t *ids, size_t per_row, size_t groups, int32_t *offsets, int32_t *order, int32_t *rows, int32_t *place) {
  (void)count, (void)ids, (void)per_row, (void)groups, (void)offsets, (void)order, (void)rows, (void)place;
  return 0;
}
int skl_hip_launch_gemm_grouped(const skl_grouped_gemm *g) {
  (void)g;
  return 0;
}
int skl_hip_launch_gemm_u4(const skl_grouped_u4 *u) {
  (void)u;
  return 0;
}
static float value(size_t e, size_t i, size_t j) { return (float)(10000 * e + 100 * i + j); }
int skl_hip_launch_gemm_groupedk(const skl_groupedk_gemm *g) {
  ++g_launches;
  for (size_t e = 0; e < g->groups; ++e)
    for (size_t i = 0; i < g->m; ++i)
      for (size_t j = 0; j < g->n; ++j) ((float *)g->c)[e * g->gsc + i * g->rsc + j] = value(e, i, j);
  return 0;
}

/* One call; `taken` says whether the matrices lie apart. */
static void one(size_t groups, size_t m, size_t n, size_t rsc, size_t gsc, int taken) {
  const size_t size = (groups - 1) * gsc + (m - 1) * rsc + n;
  const int32_t offsets[5] = {0, 1, 1, 2, 2};
  float *c = (float *)malloc(size * 4), *want = (float *)malloc(size * 4);
  skl_bf16_t *a = (skl_bf16_t *)calloc(2 * m, 2), *b = (skl_bf16_t *)calloc(2 * n, 2);
  for (size_t i = 0; i < size; ++i) c[i] = want[i] = -1.0f;
  for (size_t e = 0; taken && e < groups; ++e)
    for (size_t i = 0; i < m; ++i)
      for (size_t j = 0; j < n; ++j) want[e * gsc + i * rsc + j] = value(e, i, j);
  g_error = g_launches = 0;
  skl_gemm_groupedk_bf16c_bf16_f32_gfx950(groups, offsets, m, n, 2, 1.0f, a, m, NULL, 0, b, n, NULL, 0, 0.0f, c, rsc, gsc);
  expect(g_launches == taken && g_error == (taken ? 0 : SKL_HIP_ERR_BAD_ARGUMENT), taken ? "a call that is in order" : "a call whose matrices meet");
  expect(memcmp(c, want, size * 4) == 0, "C");
  free(a), free(b), free(c), free(want);
}

int main(void) {
  one(3, 4, 5, 15, 5, 1);  /* [m][groups][n] */
  one(3, 4, 5, 19, 6, 1);  /* ... with something in between */
  one(4, 1, 5, 0, 5, 1);
  one(1, 4, 5, 5, 0, 1);
  one(3, 4, 5, 5, 20, 1);
  one(3, 4, 5, 14, 5, 0);  /* the last group's rows reach into the first one's next */
  one(3, 4, 5, 15, 4, 0);
  one(3, 4, 5, 5, 19, 0);
  one(4, 1, 5, 0, 4, 0);
  if (!g_failures) printf("interleaved ok\n");
  return g_failures != 0;
}
