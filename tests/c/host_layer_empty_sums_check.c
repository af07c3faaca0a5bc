/* host_layer_empty_sums_check.c - what the host layer of the products grouped by expert (skl_amd/csrc/skl_api_grouped.c) hands to the launches where a
 * call's sums are empty: operands that nothing is multiplied of may be anything, a pointer of the other kind among them, so that a kernel must not
 * find them. Linked with stand-ins for all that the host layer calls; prints "empty sums ok". */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/skl-gfx950.h"
#include "../../skl_amd/csrc/skl_grouped.h"

static int g_failures, g_launches, g_error, g_mode;
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
int skl_hip_get_pointer_mode(void) { return g_mode; }
int skl_hip_pointer_is_device(const void *p) { return ((uintptr_t)p & 63) == 32; } /* of the addresses below */
int skl_hip_get_beta_zero_mode(void) { return 0; }
void skl_hip_record_error(int code, const char *what) {
  (void)what;
  g_error = code;
}
int skl_hip_launch_group_rows(size_t count, const int32_t *ids, size_t per_row, size_t groups, int32_t *offsets, int32_t *order, int32_t *rows, int32_t *place) {
  (void)count, (void)ids, (void)per_row, (void)groups, (void)offsets, (void)order, (void)rows, (void)place;
  return 0;
}
static void empty(const skl_grouped_gemm *g) {
  ++g_launches;
  expect(g->k == 0, "no values of k");
  expect(!g->a && !g->b && !g->rows, "operands of which nothing is read");
  expect(g->c && g->m == 3 && g->n == 5, "C as it was given");
}
int skl_hip_launch_gemm_grouped(const skl_grouped_gemm *g) {
  empty(g);
  return 0;
}
int skl_hip_launch_gemm_u4(const skl_grouped_u4 *u) {
  empty(&u->g);
  expect(!u->codes && !u->scales && !u->zeros, "weights of which nothing is read");
  return 0;
}
int skl_hip_launch_gemm_groupedk(const skl_groupedk_gemm *g) {
  ++g_launches;
  expect(g->total == 0, "no rows to sum over");
  expect(!g->a && !g->b && !g->rows_a && !g->rows_b, "operands of no sum");
  return 0;
}

int main(void) {
  /* addresses that nothing follows: C, offsets and, where it is read, the index are of the device, the others of the host */
  float *const c = (float *)(uintptr_t)(4096 + 32);
  const int32_t *const offsets = (const int32_t *)(uintptr_t)(8192 + 32), *const host_rows = (const int32_t *)(uintptr_t)12288;
  const skl_bf16_t *const host = (const skl_bf16_t *)(uintptr_t)16384;
  const skl_f16_t *const host_f16 = (const skl_f16_t *)(uintptr_t)16384;
  const skl_gfx950_u4_t w = {32, (const uint8_t *)host, 32, 32, host, NULL, 1, 1}, w5 = {32, (const uint8_t *)host, 32, 160, host, NULL, 1, 5};
  for (g_mode = 0; g_mode < 2; ++g_mode) {
    /* k == 0: neither A, B nor rows is addressed */
    skl_gemm_grouped_bf16_bf16rc_f32_gfx950(2, offsets, 3, 5, 0, 1.0f, host, 7, host_rows, 4, host, 1, 7, 7, 0.5f, c, 5);
    skl_gemm_grouped_bf16_bf16rc_f32_gfx950(1, NULL, 3, 5, 0, 1.0f, NULL, 7, host_rows, 4, NULL, 1, 7, 7, 0.5f, c, 5);
    skl_gemm_grouped_bf16_u4c_f32_gfx950(2, offsets, 3, 5, 0, 1.0f, host, 7, host_rows, 4, &w, 0.5f, c, 5);
    skl_gemm_grouped_bf16_u4c_f32_gfx950(1, NULL, 3, 5, 0, 1.0f, NULL, 7, host_rows, 4, NULL, 0.5f, c, 5);
    skl_gemm_groupedk_bf16c_bf16_f32_gfx950(2, offsets, 3, 5, 0, 1.0f, host, 3, host_rows, 4, host, 5, host_rows, 4, 0.5f, c, 5, 15);
    expect(g_error == 0, "k == 0: no error");
  }
  expect(g_launches == 10, "every call with k == 0");
  /* operands of no rows: the same */
  g_launches = 0;
  for (g_mode = 0; g_mode < 2; ++g_mode) {
    skl_gemm_grouped_bf16_bf16rc_f32_gfx950(2, offsets, 3, 5, 7, 1.0f, NULL, 7, host_rows, 0, host, 1, 7, 35, 0.5f, c, 5);
    skl_gemm_grouped_f16_u4c_f32_gfx950(2, offsets, 3, 5, 32, 1.0f, NULL, 32, host_rows, 0, &w5, 0.5f, c, 5);
    skl_gemm_groupedk_f16c_f16_f32_gfx950(2, offsets, 3, 5, 9, 1.0f, NULL, 3, host_rows, 0, host_f16, 5, NULL, 0, 0.5f, c, 5, 15);
    skl_gemm_groupedk_f16c_f16_f32_gfx950(2, offsets, 3, 5, 9, 1.0f, host_f16, 3, NULL, 0, NULL, 5, host_rows, 0, 0.5f, c, 5, 15);
    expect(g_error == 0, "operands of no rows: no error");
  }
  expect(g_launches == 8, "every call with an operand of no rows");
  if (!g_failures) printf("empty sums ok\n");
  return g_failures != 0;
}
