/* host_layer_grouped_check.c - the C host layer of the products grouped by expert (skl_amd/csrc/skl_api_grouped.c) under
 * AddressSanitizer and UndefinedBehaviorSanitizer, on the CPU, without a GPU.
 *
 * skl_api_grouped.c is compiled with the sanitizers and linked with the library's real objects; what would reach the GPU is
 * redirected here with the linker's --wrap. Buffers are exactly as long as what the interface says is accessed, so that
 * a stand-in that touches every element of its problem runs into the sanitizer's red zones where a span was staged too
 * short. Stand-ins write a number for each element that the test looks for in the caller's buffers, and the test looks
 * for the old bytes everywhere else. */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "skl-gfx950.h"
#include "../../skl_amd/csrc/skl_grouped.h"

static int g_failures;
static long g_launches, g_refused, g_alive;
static int g_scarce; /* allocations from here on that fail: every g_scarce-th */
static long g_allocations;

static void expect(int ok, const char *what) {
  if (ok) return;
  if (++g_failures < 20) fprintf(stderr, "FAIL: %s\n", what);
}
static uint64_t g_state = 0x9E3779B97F4A7C15ull;
static size_t draw(size_t lo, size_t hi) { /* in [lo, hi] */
  g_state ^= g_state << 13, g_state ^= g_state >> 7, g_state ^= g_state << 17;
  return lo + (size_t)(g_state % (hi - lo + 1));
}

/* ------------------------------------------------------------------ stand-ins */
void *__wrap_skl_hip_malloc(size_t bytes) {
  if (g_scarce && ++g_allocations % g_scarce == 0) return NULL;
  ++g_alive;
  return malloc(bytes);
}
void __wrap_skl_hip_free(void *p) {
  if (p) --g_alive;
  free(p);
}
int __wrap_skl_hip_memcpy_h2d(void *d, const void *s, size_t n) {
  memcpy(d, s, n);
  return 0;
}
int __wrap_skl_hip_memcpy_d2h(void *d, const void *s, size_t n) {
  memcpy(d, s, n);
  return 0;
}
static const void *g_device[16];
int __wrap_skl_hip_pointer_is_device(const void *p) {
  for (int i = 0; i < 16; ++i)
    if (g_device[i] == p && p) return 1;
  return 0;
}

static volatile unsigned g_sink;
static void touch(const void *p, size_t n) {
  const uint8_t *b = (const uint8_t *)p;
  for (size_t i = 0; i < n; ++i) g_sink += b[i];
}
static uint8_t mark(size_t i, size_t j) { return (uint8_t)(31 * i + 7 * j + 1); }

int __wrap_skl_hip_launch_group_rows(size_t count, const int32_t *ids, size_t per_row, size_t groups, int32_t *offsets, int32_t *order, int32_t *rows, int32_t *place) {
  ++g_launches;
  expect(per_row > 0, "picks of a row");
  if (count) touch(ids, count * 4);
  for (size_t e = 0; e <= groups; ++e) memset(&offsets[e], mark(e, 0), 4);
  for (size_t i = 0; i < count; ++i) {
    if (place) memset(&place[i], mark(i, 3), 4);
    if (i + 1 == count) continue; /* as if the last pick belonged to no group */
    if (order) memset(&order[i], mark(i, 1), 4);
    if (rows) memset(&rows[i], mark(i, 2), 4);
  }
  return 0;
}
/* the operands that the products of groups of rows share; every row but the last is in a group */
static void rows_product(const skl_grouped_gemm *g) {
  const size_t es = g->c_single ? 4 : 2;
  expect(g->m > 0 && g->n > 0 && g->groups > 0, "a product of something");
  if (g->offsets) touch(g->offsets, (g->groups + 1) * 4);
  if (g->k) {
    if (g->rows) touch(g->rows, g->m * 4);
    for (size_t i = 0; i < (g->rows ? g->a_rows : g->m); ++i) touch((const uint16_t *)g->a + i * g->rsa, g->k * 2);
  }
  for (size_t i = 0; i + 1 < g->m; ++i)
    for (size_t j = 0; j < g->n; ++j) memset((char *)g->c + (i * g->rsc + j) * es, mark(i, j), es);
}
int __wrap_skl_hip_launch_gemm_grouped(const skl_grouped_gemm *g) {
  ++g_launches;
  rows_product(g);
  for (size_t e = 0; e < g->groups; ++e)
    for (size_t p = 0; p < g->k; ++p)
      for (size_t j = 0; j < g->n; ++j) touch((const uint16_t *)g->b + e * g->gsb + p * g->rsb + j * g->csb, 2);
  return 0;
}
int __wrap_skl_hip_launch_gemm_u4(const skl_grouped_u4 *u) {
  const skl_grouped_gemm *g = &u->g;
  const size_t blocks = g->k ? (g->k + u->group_k - 1) / u->group_k : 0;
  ++g_launches;
  rows_product(g);
  for (size_t e = 0; e < g->groups && g->k; ++e)
    for (size_t j = 0; j < g->n; ++j) {
      touch(u->codes + (e * u->expert + j * u->ld) / 2, (g->k + 1) / 2);
      touch((const uint16_t *)u->scales + e * u->expert_scales + j * u->ld_scales, blocks * 2);
      if (u->zeros) touch(u->zeros + e * u->expert_scales + j * u->ld_scales, blocks);
    }
  return 0;
}
int __wrap_skl_hip_launch_gemm_groupedk(const skl_groupedk_gemm *g) {
  const size_t es = g->c_single ? 4 : 2;
  ++g_launches;
  if (g->offsets) touch(g->offsets, (g->groups + 1) * 4);
  if (g->total) {
    if (g->rows_a) touch(g->rows_a, g->total * 4);
    if (g->rows_b) touch(g->rows_b, g->total * 4);
    for (size_t i = 0; i < (g->rows_a ? g->a_rows : g->total); ++i) touch((const uint16_t *)g->a + i * g->rsa, g->m * 2);
    for (size_t i = 0; i < (g->rows_b ? g->b_rows : g->total); ++i) touch((const uint16_t *)g->b + i * g->rsb, g->n * 2);
  }
  for (size_t e = 0; e < g->groups; ++e)
    for (size_t i = 0; i < g->m; ++i)
      for (size_t j = 0; j < g->n; ++j) memset((char *)g->c + (e * g->gsc + i * g->rsc + j) * es, mark(i + 5 * e, j), es);
  return 0;
}

/* ------------------------------------------------------------------ cases */
static void *filled(size_t bytes) { /* at least a byte, 16-byte aligned */
  void *p = malloc(bytes ? bytes : 1);
  memset(p, 0xA5, bytes ? bytes : 1);
  return p;
}
static size_t span(size_t rows, size_t distance, size_t n) { return rows && n ? (rows - 1) * distance + n : 0; }
/* every byte of `p`: `size` of them, elements of `es` bytes at i * rs + j hold mark(i + i0, j + j0), all others the old byte */
static void expect_marks(const void *p, size_t size, size_t m, size_t n, size_t rs, size_t es, size_t j0, int done, const char *what) {
  uint8_t *want = (uint8_t *)malloc(size ? size : 1);
  memset(want, 0xA5, size);
  for (size_t i = 0; done && i < m; ++i)
    for (size_t j = 0; j < n; ++j) memset(want + (i * rs + j) * es, mark(i, j + j0), es);
  expect(memcmp(p, want, size) == 0, what);
  free(want);
}
static void outcome(long before, int *done) {
  *done = g_launches != before;
  const int code = skl_hip_last_error();
  expect(*done ? code == 0 : g_scarce != 0, "an error, or a call that did nothing");
  g_refused += !*done;
  expect(g_alive == 0, "device memory left");
}

static void one_order(void) {
  const size_t count = draw(0, 40), groups = draw(1, 9), bytes = count * 4;
  void *ids = filled(bytes), *offsets = filled((groups + 1) * 4), *out[3];
  const long before = g_launches;
  int done;
  for (int i = 0; i < 3; ++i) out[i] = draw(0, 2) ? filled(bytes) : NULL;
  skl_group_rows_gfx950(count, ids, draw(1, 4), groups, offsets, out[0], out[1], out[2]);
  outcome(before, &done);
  expect_marks(offsets, (groups + 1) * 4, groups + 1, 1, 1, 4, 0, done, "the offsets");
  for (int i = 0; i < 3; ++i) {
    const size_t filled_in = count == 0 ? 0 : i < 2 ? count - 1 : count;
    uint8_t *want = (uint8_t *)filled(bytes);
    for (size_t j = 0; done && j < filled_in; ++j) memset(want + 4 * j, mark(j, (size_t)i + 1), 4);
    expect(!out[i] || memcmp(out[i], want, bytes) == 0, "order, rows or places");
    free(want), free(out[i]);
  }
  free(ids), free(offsets);
}

static void one_product(int u4) {
  const size_t groups = draw(1, 4), m = draw(1, 9), n = draw(1, 9), k = draw(0, 100), a_rows = draw(0, 7), rsa = k + draw(0, 5), rsc = n + draw(0, 3);
  const int single = (int)draw(0, 1), half = (int)draw(0, 1), indexed = (int)draw(0, 1), transposed = (int)draw(0, 1), listed = groups > 1 || draw(0, 1);
  const size_t es = single ? 4 : 2, nc = span(m, rsc, n) * es, na = span(indexed ? a_rows : m, rsa, k) * 2;
  void *a = filled(na), *c = filled(nc), *rows = indexed ? filled(m * 4) : NULL, *offsets = listed ? filled((groups + 1) * 4) : NULL;
  const long before = g_launches;
  int done;
  if (u4) {
    const size_t group_k = draw(0, 1) ? 32 * draw(1, 3) : k + draw(1, 70), block = group_k % 32 == 0 || group_k >= k ? group_k : 32, blocks = (k + block - 1) / block;
    const size_t ld = 2 * ((k + 1) / 2 + draw(0, 5)), ld_scales = blocks + draw(0, 3), expert = n * ld + 2 * draw(0, 5), expert_scales = n * ld_scales + draw(0, 3);
    const size_t places = k ? span(groups, expert_scales, span(n, ld_scales, blocks)) : 0;
    skl_gfx950_u4_t w;
    void *codes = filled(k ? span(groups, expert / 2, span(n, ld / 2, (k + 1) / 2)) : 0), *scales = filled(places * 2), *zeros = draw(0, 1) ? filled(places) : NULL;
    w.group_k = block, w.codes = codes, w.ld = ld, w.expert = expert, w.scales = scales, w.zeros = zeros, w.ld_scales = ld_scales, w.expert_scales = expert_scales;
    if (half && single) skl_gemm_grouped_f16_u4c_f32_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, &w, 0.0f, c, rsc);
    else if (half) skl_gemm_grouped_f16_u4c_f16_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, &w, 0.0f, c, rsc);
    else if (single) skl_gemm_grouped_bf16_u4c_f32_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, &w, 0.0f, c, rsc);
    else skl_gemm_grouped_bf16_u4c_bf16_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, &w, 0.0f, c, rsc);
    free(codes), free(scales), free(zeros);
  } else {
    const size_t rsb = transposed ? 1 : n + draw(0, 3), csb = transposed ? k + draw(0, 3) : 1, one = k ? (k - 1) * rsb + (n - 1) * csb + 1 : 0, gsb = one + draw(0, 5);
    void *b = filled(span(groups, gsb, one) * 2);
    if (half && single) skl_gemm_grouped_f16_f16rc_f32_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, b, rsb, csb, gsb, 0.0f, c, rsc);
    else if (half) skl_gemm_grouped_f16_f16rc_f16_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, b, rsb, csb, gsb, 0.0f, c, rsc);
    else if (single) skl_gemm_grouped_bf16_bf16rc_f32_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, b, rsb, csb, gsb, 0.0f, c, rsc);
    else skl_gemm_grouped_bf16_bf16rc_bf16_gfx950(groups, offsets, m, n, k, 1.0f, a, rsa, rows, a_rows, b, rsb, csb, gsb, 0.0f, c, rsc);
    free(b);
  }
  outcome(before, &done);
  expect_marks(c, nc, m - 1, n, rsc, es, 0, done, "C");
  free(a), free(c), free(rows), free(offsets);
}

static void one_sum(void) {
  const size_t groups = draw(1, 4), m = draw(1, 9), n = draw(1, 9), total = draw(0, 20), a_rows = draw(0, 7), b_rows = draw(0, 7), rsa = m + draw(0, 5), rsb = n + draw(0, 5), rsc = n + draw(0, 3);
  const int single = (int)draw(0, 1), half = (int)draw(0, 1), by_a = (int)draw(0, 1), by_b = (int)draw(0, 1), listed = groups > 1 || draw(0, 1);
  const size_t es = single ? 4 : 2, gsc = span(m, rsc, n) + draw(0, 3), nc = span(groups, gsc, span(m, rsc, n)) * es;
  void *a = filled(span(by_a ? a_rows : total, rsa, m) * 2), *b = filled(span(by_b ? b_rows : total, rsb, n) * 2), *c = filled(nc);
  void *ra = by_a ? filled(total * 4) : NULL, *rb = by_b ? filled(total * 4) : NULL, *offsets = listed ? filled((groups + 1) * 4) : NULL;
  const long before = g_launches;
  int done;
  if (half && single) skl_gemm_groupedk_f16c_f16_f32_gfx950(groups, offsets, m, n, total, 1.0f, a, rsa, ra, a_rows, b, rsb, rb, b_rows, 0.0f, c, rsc, gsc);
  else if (half) skl_gemm_groupedk_f16c_f16_f16_gfx950(groups, offsets, m, n, total, 1.0f, a, rsa, ra, a_rows, b, rsb, rb, b_rows, 0.0f, c, rsc, gsc);
  else if (single) skl_gemm_groupedk_bf16c_bf16_f32_gfx950(groups, offsets, m, n, total, 1.0f, a, rsa, ra, a_rows, b, rsb, rb, b_rows, 0.0f, c, rsc, gsc);
  else skl_gemm_groupedk_bf16c_bf16_bf16_gfx950(groups, offsets, m, n, total, 1.0f, a, rsa, ra, a_rows, b, rsb, rb, b_rows, 0.0f, c, rsc, gsc);
  outcome(before, &done);
  {
    uint8_t *want = (uint8_t *)filled(nc);
    for (size_t e = 0; done && e < groups; ++e)
      for (size_t i = 0; i < m; ++i)
        for (size_t j = 0; j < n; ++j) memset(want + (e * gsc + i * rsc + j) * es, mark(i + 5 * e, j), es);
    expect(memcmp(c, want, nc) == 0, "C of the groups");
    free(want);
  }
  free(a), free(b), free(c), free(ra), free(rb), free(offsets);
}

static void refusals(void) {
  int32_t i[8] = {0};
  skl_bf16_t h[64];
  float f[64] = {0};
  uint8_t q[64] = {0};
  skl_gfx950_u4_t w = {32, q, 32, 32, h, NULL, 1, 1};
  const long before = g_launches;
  memset(h, 0, sizeof h);
#define REFUSED(call, code) \
  call;                     \
  expect(skl_hip_last_error() == (code) && g_launches == before, #call)
  REFUSED(skl_group_rows_gfx950(2, i, 1, 0, i, NULL, NULL, NULL), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_group_rows_gfx950(2, NULL, 1, 1, i, NULL, NULL, NULL), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_gemm_grouped_bf16_bf16rc_f32_gfx950(2, NULL, 1, 1, 1, 1.0f, h, 1, NULL, 0, h, 1, 1, 1, 0.0f, f, 1), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_gemm_grouped_bf16_bf16rc_f32_gfx950(0, NULL, 1, 1, 1, 1.0f, NULL, 1, NULL, 0, NULL, 1, 1, 1, 0.0f, NULL, 1), 0);
  REFUSED(skl_gemm_groupedk_bf16c_bf16_f32_gfx950(2, i, 2, 2, 1, 1.0f, h, 2, NULL, 0, h, 2, NULL, 0, 0.0f, f, 2, 3), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_gemm_groupedk_bf16c_bf16_f32_gfx950(2, i, 0, 2, 1, 1.0f, NULL, 2, NULL, 0, NULL, 2, NULL, 0, 0.0f, NULL, 2, 3), 0);
  w.group_k = 40; /* not a multiple of 32, and less than k */
  REFUSED(skl_gemm_grouped_bf16_u4c_f32_gfx950(1, NULL, 1, 1, 64, 1.0f, h, 64, NULL, 0, &w, 0.0f, f, 1), SKL_HIP_ERR_BAD_ARGUMENT);
  w.group_k = SIZE_MAX, w.ld = 64, w.ld_scales = 0; /* one scale for all of a column, and two columns that share it */
  REFUSED(skl_gemm_grouped_bf16_u4c_f32_gfx950(1, NULL, 1, 2, 64, 1.0f, h, 64, NULL, 0, &w, 0.0f, f, 2), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_gemm_grouped_bf16_u4c_f32_gfx950(1, NULL, 1, 1, 64, 1.0f, h, 64, NULL, 0, NULL, 0.0f, f, 1), SKL_HIP_ERR_BAD_ARGUMENT);
  g_device[0] = f;
  REFUSED(skl_gemm_grouped_bf16_bf16rc_f32_gfx950(1, NULL, 1, 1, 1, 1.0f, h, 1, NULL, 0, h, 1, 1, 1, 0.0f, f, 1), SKL_HIP_ERR_MIXED_POINTERS);
  g_device[0] = NULL;
#undef REFUSED
}

int main(int argc, char **argv) {
  const int cases = argc > 1 ? atoi(argv[1]) : 300;
  if (argc > 2) g_state = strtoull(argv[2], NULL, 0) | 1u;
  refusals();
  for (int i = 0; i < cases; ++i) {
    g_scarce = i % 4 == 3 ? (int)draw(1, 9) : 0;
    one_order();
    one_product(0);
    one_product(1);
    one_sum();
  }
  expect(g_launches > cases && g_refused > 0, "both outcomes");
  if (g_failures) return 1;
  printf("host layer ok: %ld launches, %ld calls without memory\n", g_launches, g_refused);
  return 0;
}
