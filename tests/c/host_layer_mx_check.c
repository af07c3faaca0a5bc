/* host_layer_mx_check.c - the C host layer of the microscaled 4-bit operators (skl_amd/csrc/skl_api_mx.c) under
 * AddressSanitizer and UndefinedBehaviorSanitizer, on the CPU, without a GPU.
 *
 * skl_api_mx.c is compiled with the sanitizers and linked with the library's real objects; what would reach the GPU is
 * redirected here with the linker's --wrap. Buffers are exactly as long as what the interface says is accessed, so that
 * a stand-in that touches every element of its problem runs into the sanitizer's red zones where a span was staged too
 * short. Stand-ins write a number for each element that the test looks for in the caller's buffers, and the test looks
 * for the old bytes everywhere else. */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "skl-gfx950.h"
#include "../../skl_amd/csrc/skl_mx.h"

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
static void touch_matrix(const skl_mx_operand *o, size_t rows, size_t k) {
  for (size_t i = 0; i < rows; ++i) {
    touch(o->codes + i * (o->ld / 2), (k + 1) / 2);
    touch(o->scales + i * o->lds, (k + 31) / 32);
  }
}
static uint8_t mark(size_t i, size_t j) { return (uint8_t)(31 * i + 7 * j + 1); }

int __wrap_skl_hip_launch_cvt_to_mx(int dt, size_t m, size_t k, const void *src, size_t rs, size_t cs, uint8_t *codes, size_t ld, uint8_t *scales, size_t lds) {
  const size_t es = dt == SKL_DT_F32 ? 4 : 2;
  ++g_launches;
  for (size_t i = 0; i < m; ++i) {
    for (size_t p = 0; p < k; ++p) touch((const char *)src + (i * rs + p * cs) * es, es);
    for (size_t b = 0; b < (k + 1) / 2; ++b) codes[i * (ld / 2) + b] = mark(i, b);
    for (size_t b = 0; b < (k + 31) / 32; ++b) scales[i * lds + b] = mark(i, b + 100);
  }
  return 0;
}
int __wrap_skl_hip_launch_cvt_from_mx(int dt, size_t m, size_t k, const skl_mx_operand *src, void *dst, size_t rs, size_t cs) {
  const size_t es = dt == SKL_DT_F32 ? 4 : 2;
  ++g_launches;
  touch_matrix(src, m, k);
  for (size_t i = 0; i < m; ++i)
    for (size_t p = 0; p < k; ++p) memset((char *)dst + (i * rs + p * cs) * es, mark(i, p), es);
  return 0;
}
int __wrap_skl_hip_launch_gemm_mx(const skl_mx_gemm *g) {
  ++g_launches;
  if (g->k) touch_matrix(&g->a, g->m, g->k), touch_matrix(&g->b, g->n, g->k);
  for (size_t i = 0; i < g->m; ++i)
    for (size_t j = 0; j < g->n; ++j) memset((char *)&g->c[i * g->rsc + j * g->csc], mark(i, j), 4);
  return 0;
}
static size_t g_token; /* of the layer's first chunk on */
int __wrap_skl_hip_launch_moe(const skl_moe_problem *p) {
  ++g_launches;
  expect(p->tokens > 0 && p->tokens <= SKL_MOE_TOKENS, "a chunk of tokens");
  for (size_t e = 0; e < p->experts; ++e) {
    skl_mx_operand o = p->gate;
    o.codes += e * p->expert_in / 2, o.scales += e * p->expert_in_scales;
    touch_matrix(&o, p->inter, p->hidden);
    o = p->up;
    o.codes += e * p->expert_in / 2, o.scales += e * p->expert_in_scales;
    touch_matrix(&o, p->inter, p->hidden);
    o = p->down;
    o.codes += e * p->expert_down / 2, o.scales += e * p->expert_down_scales;
    touch_matrix(&o, p->hidden, p->inter);
    touch(p->router + e * p->ld_router, 2 * p->hidden);
  }
  for (size_t t = 0; t < p->tokens; ++t) {
    touch(p->x + t * p->ldx, 2 * p->hidden);
    if (p->residual) touch(p->residual + t * p->ld_residual, 4 * p->hidden);
    for (size_t j = 0; j < p->hidden; ++j) memset((char *)&p->y[t * p->ldy + j], mark(g_token + t, j), 4);
    for (size_t j = 0; j < p->top_k; ++j) {
      if (p->ids) memset((char *)&p->ids[t * p->top_k + j], mark(g_token + t, j + 50), 4);
      if (p->weights) memset((char *)&p->weights[t * p->top_k + j], mark(g_token + t, j + 60), 4);
    }
  }
  g_token += p->tokens;
  return 0;
}

/* ------------------------------------------------------------------ cases */
static void *filled(size_t bytes) { /* at least a byte, 16-byte aligned */
  void *p = malloc(bytes ? bytes : 1);
  memset(p, 0xA5, bytes ? bytes : 1);
  return p;
}
static size_t span(size_t rows, size_t distance, size_t n) { return (rows - 1) * distance + n; }
/* every byte of `p`: `size` of them, elements of `es` bytes at i * rs + j * cs hold mark(i + i0, j + j0), all others the old byte */
static void expect_marks(const void *p, size_t size, size_t m, size_t n, size_t rs, size_t cs, size_t es, size_t j0, int done, const char *what) {
  uint8_t *want = (uint8_t *)malloc(size);
  memset(want, 0xA5, size);
  for (size_t i = 0; done && i < m; ++i)
    for (size_t j = 0; j < n; ++j) memset(want + (i * rs + j * cs) * es, mark(i, j + j0), es);
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

static void one_conversion(void) {
  const size_t m = draw(1, 9), k = draw(1, 130), row = (k + 1) / 2, blocks = (k + 31) / 32;
  const size_t ld = 2 * (row + draw(0, 5)), lds = blocks + draw(0, 3);
  const int transposed = (int)draw(0, 1), f32 = (int)draw(0, 1), back = (int)draw(0, 1);
  const size_t cs = transposed ? m + draw(0, 3) : draw(1, 2), rs = transposed ? 1 : cs * k + draw(0, 3), es = f32 ? 4 : 2;
  const size_t plain = ((m - 1) * rs + (k - 1) * cs + 1) * es, nc = span(m, ld / 2, row), ns = span(m, lds, blocks);
  void *x = filled(plain), *c = filled(nc), *s = filled(ns);
  const long before = g_launches;
  int done;
  if (back && f32) skl_cvt_mxf4e2m1_f32rc_gfx950(m, k, c, ld, s, lds, x, rs, cs);
  else if (back) skl_cvt_mxf4e2m1_bf16rc_gfx950(m, k, c, ld, s, lds, x, rs, cs);
  else if (f32) skl_cvt_f32rc_mxf4e2m1_gfx950(m, k, x, rs, cs, c, ld, s, lds);
  else skl_cvt_bf16rc_mxf4e2m1_gfx950(m, k, x, rs, cs, c, ld, s, lds);
  outcome(before, &done);
  expect_marks(x, plain, m, k, rs, cs, es, 0, done && back, "the plain matrix");
  expect_marks(c, nc, m, row, ld / 2, 1, 1, 0, done && !back, "the codes");
  expect_marks(s, ns, m, blocks, lds, 1, 1, 100, done && !back, "the scales");
  free(x), free(c), free(s);
}

static void one_product(void) {
  const size_t m = draw(1, 9), n = draw(1, 9), k = draw(0, 100), row = (k + 1) / 2, blocks = (k + 31) / 32;
  const size_t lda = 2 * (row + draw(0, 5)), lsa = blocks + draw(0, 3), ldb = 2 * (row + draw(0, 5)), lsb = blocks + draw(0, 3);
  const size_t csc = draw(0, 1) ? 1 : m + draw(0, 2), rsc = csc == 1 ? n + draw(0, 3) : 1, nc = ((m - 1) * rsc + (n - 1) * csc + 1) * 4;
  void *a = filled(k ? span(m, lda / 2, row) : 0), *sa = filled(k ? span(m, lsa, blocks) : 0), *b = filled(k ? span(n, ldb / 2, row) : 0), *sb = filled(k ? span(n, lsb, blocks) : 0);
  void *c = filled(nc);
  const long before = g_launches;
  int done;
  skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(m, n, k, 1.0f, a, lda, sa, lsa, b, ldb, sb, lsb, 0.0f, c, rsc, csc);
  outcome(before, &done);
  expect_marks(c, nc, m, n, rsc, csc, 4, 0, done, "C");
  free(a), free(sa), free(b), free(sb), free(c);
}

static void one_layer(void) {
  skl_gfx950_moe_t l;
  const size_t tokens = draw(0, 9) == 0 ? draw(65, 140) : draw(1, 5), h = 32 * draw(1, 3), i = 32 * draw(1, 3), e = draw(1, 4);
  const size_t ldx = h + 8 * draw(0, 2), ldy = h + draw(0, 3), ld_residual = h + draw(0, 3);
  const int with_residual = (int)draw(0, 1), with_choice = (int)draw(0, 1);
  memset(&l, 0, sizeof l);
  l.hidden = h, l.inter = i, l.experts = e, l.top_k = draw(1, e), l.activation = 2, l.normalise = 1;
  l.ld_router = h + 8 * draw(0, 2);
  l.ld_in = h + 32 * draw(0, 1), l.ld_in_scales = h / 32 + draw(0, 2), l.ld_down = i + 32 * draw(0, 1), l.ld_down_scales = i / 32 + draw(0, 2);
  l.expert_in = i * l.ld_in + 32 * draw(0, 2), l.expert_in_scales = i * l.ld_in_scales + draw(0, 2);
  l.expert_down = h * l.ld_down + 32 * draw(0, 2), l.expert_down_scales = h * l.ld_down_scales + draw(0, 2);
  const size_t in = span(e, l.expert_in / 2, span(i, l.ld_in / 2, h / 2)), in_s = span(e, l.expert_in_scales, span(i, l.ld_in_scales, h / 32));
  const size_t down = span(e, l.expert_down / 2, span(h, l.ld_down / 2, i / 2)), down_s = span(e, l.expert_down_scales, span(h, l.ld_down_scales, i / 32));
  const size_t ny = span(tokens, ldy, h) * 4, picks = tokens * l.top_k * 4;
  void *router = filled(span(e, l.ld_router, h) * 2), *gate = filled(in), *up = filled(in), *dn = filled(down), *gs = filled(in_s), *us = filled(in_s), *ds = filled(down_s);
  void *x = filled(span(tokens, ldx, h) * 2), *y = filled(ny), *r = with_residual ? filled(span(tokens, ld_residual, h) * 4) : NULL;
  void *ids = filled(picks), *weights = filled(picks);
  const long before = g_launches;
  int done;
  l.router = router, l.gate = gate, l.up = up, l.down = dn, l.gate_scales = gs, l.up_scales = us, l.down_scales = ds;
  if (with_choice) l.ids = ids, l.weights = weights;
  g_token = 0;
  skl_moe_bf16_mxf4e2m1_f32_gfx950(&l, tokens, x, ldx, with_residual ? 1.0f : 0.0f, r, ld_residual, y, ldy);
  outcome(before, &done);
  expect(!done || g_token == tokens, "every token once");
  expect_marks(y, ny, tokens, h, ldy, 1, 4, 0, done, "y");
  expect_marks(ids, picks, tokens, l.top_k, l.top_k, 1, 4, 50, done && with_choice, "the chosen experts");
  expect_marks(weights, picks, tokens, l.top_k, l.top_k, 1, 4, 60, done && with_choice, "their weights");
  free(router), free(gate), free(up), free(dn), free(gs), free(us), free(ds), free(x), free(y), free(r), free(ids), free(weights);
}

static void refusals(void) {
  uint8_t b[64] = {0};
  float f[64] = {0};
  const long before = g_launches;
#define REFUSED(call, code) \
  call;                     \
  expect(skl_hip_last_error() == (code) && g_launches == before, #call)
  REFUSED(skl_cvt_f32rc_mxf4e2m1_gfx950(2, 32, f, 32, 1, b, 33, b, 1), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_cvt_f32rc_mxf4e2m1_gfx950(2, 34, f, 34, 1, b, 32, b, 2), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_cvt_f32rc_mxf4e2m1_gfx950(2, 33, f, 34, 1, b, 34, b, 1), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_cvt_f32rc_mxf4e2m1_gfx950(1, 1, NULL, 1, 1, b, 2, b, 1), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_cvt_f32rc_mxf4e2m1_gfx950(0, 1, NULL, 1, 1, NULL, 2, NULL, 1), 0);
  REFUSED(skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(1, 1, 1, 1.0f, NULL, 2, b, 1, b, 2, b, 1, 0.0f, f, 1, 1), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(0, 1, 1, 1.0f, NULL, 2, NULL, 1, NULL, 2, NULL, 1, 0.0f, NULL, 1, 1), 0);
  g_device[0] = f;
  REFUSED(skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(1, 1, 1, 1.0f, b, 2, b, 1, b, 2, b, 1, 0.0f, f, 1, 1), SKL_HIP_ERR_MIXED_POINTERS);
  g_device[0] = NULL;
  REFUSED(skl_moe_bf16_mxf4e2m1_f32_gfx950(NULL, 1, NULL, 0, 0.0f, NULL, 0, f, 0), SKL_HIP_ERR_BAD_ARGUMENT);
  REFUSED(skl_moe_bf16_mxf4e2m1_f32_gfx950(NULL, 0, NULL, 0, 0.0f, NULL, 0, NULL, 0), 0);
#undef REFUSED
}

int main(int argc, char **argv) {
  const int cases = argc > 1 ? atoi(argv[1]) : 300;
  if (argc > 2) g_state = strtoull(argv[2], NULL, 0) | 1u;
  refusals();
  for (int i = 0; i < cases; ++i) {
    g_scarce = i % 4 == 3 ? (int)draw(1, 9) : 0;
    one_conversion();
    one_product();
    one_layer();
  }
  expect(g_launches > cases && g_refused > 0, "both outcomes");
  if (g_failures) return 1;
  printf("host layer ok: %ld launches, %ld calls without memory\n", g_launches, g_refused);
  return 0;
}
