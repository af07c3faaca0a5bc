/*
 * skl_api_mx.c - the C host layer of the microscaled 4-bit entry points and the mixture-of-experts layer of
 * include/skl-gfx950.h: arguments are checked, ordinary host memory is staged, and the launchers of skl_mx.h do the rest.
 */
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include "../../include/skl-gfx950.h"
#include "skl_host.h"
#include "skl_mx.h"

static size_t blocks_of(size_t k) { return (k + 31) / 32; }
static size_t row_bytes(size_t k) { return (k + 1) / 2; }

/* Bytes from the first to the last of `rows` rows of `bytes`, `distance` apart. */
static size_t span(size_t rows, size_t distance, size_t bytes) { return rows ? (rows - 1) * distance + bytes : 0; }

/* Rows begin on bytes and do not run into each other. */
static int layout_ok(size_t rows, size_t k, size_t ld, size_t lds) {
  return rows <= 1 || ((ld & 1) == 0 && ld >= k && lds >= blocks_of(k));
}

static void bad_argument(const char *who) { skl_hip_record_error(SKL_HIP_ERR_BAD_ARGUMENT, who); }

/* ------------------------------------------------------------------------ */
/* conversions                                                               */
/* ------------------------------------------------------------------------ */

static void to_mx(int dt, size_t m, size_t k, const void *src, size_t rs, size_t cs, uint8_t *dst, size_t ldd, uint8_t *scales, size_t lds,
                  const char *who) {
  const void *given[3] = {src, dst, scales};
  const size_t es = dt == SKL_DT_F32 ? 4 : 2;
  int where;
  if (m == 0 || k == 0) return;
  if (!src || !dst || !scales || !layout_ok(m, k, ldd, lds)) {
    bad_argument(who);
    return;
  }
  where = skl_classify(given, 3, who);
  if (where < 0) return;
  if (where == 1) {
    skl_hip_launch_cvt_to_mx(dt, m, k, src, rs, cs, dst, ldd, scales, lds);
    return;
  }
  {
    const size_t nd = span(m, ldd / 2, row_bytes(k)), ns = span(m, lds, blocks_of(k));
    void *d_src = skl_stage_in(src, ((m - 1) * rs + (k - 1) * cs + 1) * es), *d_dst = skl_stage_in(dst, nd), *d_sc = skl_stage_in(scales, ns);
    /* what lies between the rows travels both ways and comes back unchanged */
    if (d_src && d_dst && d_sc && skl_hip_launch_cvt_to_mx(dt, m, k, d_src, rs, cs, (uint8_t *)d_dst, ldd, (uint8_t *)d_sc, lds) == 0) {
      skl_hip_memcpy_d2h(dst, d_dst, nd);
      skl_hip_memcpy_d2h(scales, d_sc, ns);
    }
    skl_hip_free(d_src);
    skl_hip_free(d_dst);
    skl_hip_free(d_sc);
  }
}

static void from_mx(int dt, size_t m, size_t k, const uint8_t *src, size_t ldsrc, const uint8_t *scales, size_t lds, void *dst, size_t rs,
                    size_t cs, const char *who) {
  const void *given[3] = {src, dst, scales};
  const size_t es = dt == SKL_DT_F32 ? 4 : 2;
  skl_mx_operand op = {src, ldsrc, scales, lds};
  int where;
  if (m == 0 || k == 0) return;
  if (!src || !dst || !scales || !layout_ok(m, k, ldsrc, lds)) {
    bad_argument(who);
    return;
  }
  where = skl_classify(given, 3, who);
  if (where < 0) return;
  if (where == 1) {
    skl_hip_launch_cvt_from_mx(dt, m, k, &op, dst, rs, cs);
    return;
  }
  {
    const size_t nd = ((m - 1) * rs + (k - 1) * cs + 1) * es;
    void *d_src = skl_stage_in(src, span(m, ldsrc / 2, row_bytes(k))), *d_sc = skl_stage_in(scales, span(m, lds, blocks_of(k))), *d_dst = skl_stage_in(dst, nd);
    op.codes = (const uint8_t *)d_src, op.scales = (const uint8_t *)d_sc;
    if (d_src && d_dst && d_sc && skl_hip_launch_cvt_from_mx(dt, m, k, &op, d_dst, rs, cs) == 0) skl_hip_memcpy_d2h(dst, d_dst, nd);
    skl_hip_free(d_src);
    skl_hip_free(d_dst);
    skl_hip_free(d_sc);
  }
}

void skl_cvt_f32rc_mxf4e2m1_gfx950(size_t m, size_t k, const float *src, size_t rs, size_t cs, uint8_t *dst, size_t ldd, uint8_t *scales,
                                   size_t lds) {
  to_mx(SKL_DT_F32, m, k, src, rs, cs, dst, ldd, scales, lds, __func__);
}
void skl_cvt_bf16rc_mxf4e2m1_gfx950(size_t m, size_t k, const skl_bf16_t *src, size_t rs, size_t cs, uint8_t *dst, size_t ldd,
                                    uint8_t *scales, size_t lds) {
  to_mx(SKL_DT_BF16, m, k, src, rs, cs, dst, ldd, scales, lds, __func__);
}
void skl_cvt_mxf4e2m1_f32rc_gfx950(size_t m, size_t k, const uint8_t *src, size_t ldsrc, const uint8_t *scales, size_t lds, float *dst,
                                   size_t rs, size_t cs) {
  from_mx(SKL_DT_F32, m, k, src, ldsrc, scales, lds, dst, rs, cs, __func__);
}
void skl_cvt_mxf4e2m1_bf16rc_gfx950(size_t m, size_t k, const uint8_t *src, size_t ldsrc, const uint8_t *scales, size_t lds,
                                    skl_bf16_t *dst, size_t rs, size_t cs) {
  from_mx(SKL_DT_BF16, m, k, src, ldsrc, scales, lds, dst, rs, cs, __func__);
}

/* ------------------------------------------------------------------------ */
/* product                                                                   */
/* ------------------------------------------------------------------------ */

void skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(size_t m, size_t n, size_t k, float alpha, const uint8_t *a, size_t lda,
                                               const uint8_t *scales_a, size_t lsa, const uint8_t *b, size_t ldb, const uint8_t *scales_b,
                                               size_t lsb, float beta, float *c, size_t rsc, size_t csc) {
  const void *given[5] = {k ? a : NULL, k ? scales_a : NULL, k ? b : NULL, k ? scales_b : NULL, c};
  skl_mx_gemm g;
  int where;
  if (m == 0 || n == 0) return; /* nothing is addressed */
  if (!c || (k && (!a || !scales_a || !b || !scales_b || !layout_ok(m, k, lda, lsa) || !layout_ok(n, k, ldb, lsb)))) {
    bad_argument(__func__);
    return;
  }
  where = skl_classify(given, 5, __func__);
  if (where < 0) return;
  memset(&g, 0, sizeof g);
  g.m = m, g.n = n, g.k = k;
  g.a.codes = a, g.a.ld = lda, g.a.scales = scales_a, g.a.lds = lsa;
  g.b.codes = b, g.b.ld = ldb, g.b.scales = scales_b, g.b.lds = lsb;
  g.c = c, g.rsc = rsc, g.csc = csc;
  g.alpha.f = alpha;
  g.beta.fz.value = beta;
  g.beta.fz.skip_c_read = skl_hip_get_beta_zero_mode() != SKL_HIP_BETA_ZERO_AS_REFERENCE;
  if (where == 1) {
    skl_hip_launch_gemm_mx(&g);
    return;
  }
  {
    const size_t nc = ((m - 1) * rsc + (n - 1) * csc + 1) * sizeof(float);
    const size_t rb = k ? row_bytes(k) : 0, bl = k ? blocks_of(k) : 0;
    void *da = k ? skl_stage_in(a, span(m, lda / 2, rb)) : NULL, *dsa = k ? skl_stage_in(scales_a, span(m, lsa, bl)) : NULL;
    void *db = k ? skl_stage_in(b, span(n, ldb / 2, rb)) : NULL, *dsb = k ? skl_stage_in(scales_b, span(n, lsb, bl)) : NULL;
    void *dc = skl_stage_in(c, nc); /* its whole span travels both ways: the elements in its stride gaps come back unchanged */
    g.a.codes = (const uint8_t *)da, g.a.scales = (const uint8_t *)dsa;
    g.b.codes = (const uint8_t *)db, g.b.scales = (const uint8_t *)dsb;
    g.c = (float *)dc;
    if (dc && (!k || (da && dsa && db && dsb)) && skl_hip_launch_gemm_mx(&g) == 0) skl_hip_memcpy_d2h(c, dc, nc);
    skl_hip_free(da);
    skl_hip_free(dsa);
    skl_hip_free(db);
    skl_hip_free(dsb);
    skl_hip_free(dc);
  }
}

/* ------------------------------------------------------------------------ */
/* mixture of experts                                                        */
/* ------------------------------------------------------------------------ */

static int aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

static int moe_ok(const skl_gfx950_moe_t *l, size_t tokens, const void *x, size_t ldx, float beta, const void *residual, const void *y) {
  const size_t h = l->hidden, i = l->inter;
  if (h == 0 || i == 0 || (h % 32) != 0 || (i % 32) != 0) return 0;
  if (l->experts == 0 || l->experts > 1024 || l->top_k == 0 || l->top_k > l->experts || l->top_k > 64) return 0;
  if (l->activation < SKL_GFX950_ACT_NONE || l->activation > SKL_GFX950_ACT_GELU) return 0;
  if (!x || !y || !l->router || !l->gate || !l->up || !l->down || !l->gate_scales || !l->up_scales || !l->down_scales) return 0;
  if (beta != 0.0f && !residual) return 0;
  if (!aligned16(x) || !aligned16(l->router) || !aligned16(l->gate) || !aligned16(l->up) || !aligned16(l->down)) return 0;
  if ((tokens > 1 && (ldx % 8 != 0 || ldx < h)) || (l->experts > 1 && (l->ld_router % 8 != 0 || l->ld_router < h))) return 0;
  /* 16 bytes of weights are 32 values */
  if (l->ld_in % 32 != 0 || l->ld_in < h || l->expert_in % 32 != 0 || l->ld_down % 32 != 0 || l->ld_down < i || l->expert_down % 32 != 0) return 0;
  if (l->ld_in_scales < h / 32 || l->ld_down_scales < i / 32) return 0;
  /* a workgroup's offsets from its first row are 32-bit numbers */
  if (h > ((size_t)1 << 24) || i > ((size_t)1 << 24) || l->ld_in > ((size_t)1 << 24) || l->ld_down > ((size_t)1 << 24) || (tokens > 1 && ldx > ((size_t)1 << 23))) return 0;
  return 1;
}

/* More than one token: rows do not run into each other, and a residual that is y has its rows where y's are: it is read while other rows of y are written. */
static int rows_of_y_ok(size_t hidden, float beta, const float *residual, size_t ld_residual, const float *y, size_t ldy) {
  if (ldy < hidden) return 0;
  return beta == 0.0f || (ld_residual >= hidden && (residual != y || ld_residual == ldy));
}

static int moe_on_device(const skl_gfx950_moe_t *l, size_t tokens, const void *x, size_t ldx, float beta, const float *residual,
                         size_t ld_residual, float *y, size_t ldy) {
  size_t t;
  for (t = 0; t < tokens; t += SKL_MOE_TOKENS) { /* each chunk writes its own rows of y */
    skl_moe_problem p;
    int rc;
    memset(&p, 0, sizeof p);
    p.tokens = tokens - t < SKL_MOE_TOKENS ? tokens - t : SKL_MOE_TOKENS;
    p.hidden = l->hidden, p.inter = l->inter, p.experts = l->experts, p.top_k = l->top_k;
    p.x = (const uint16_t *)x + t * ldx, p.ldx = ldx;
    p.router = (const uint16_t *)(const void *)l->router, p.ld_router = l->ld_router;
    p.gate.codes = l->gate, p.gate.ld = l->ld_in, p.gate.scales = l->gate_scales, p.gate.lds = l->ld_in_scales;
    p.up.codes = l->up, p.up.ld = l->ld_in, p.up.scales = l->up_scales, p.up.lds = l->ld_in_scales;
    p.down.codes = l->down, p.down.ld = l->ld_down, p.down.scales = l->down_scales, p.down.lds = l->ld_down_scales;
    p.expert_in = l->expert_in, p.expert_in_scales = l->expert_in_scales;
    p.expert_down = l->expert_down, p.expert_down_scales = l->expert_down_scales;
    p.activation = l->activation, p.normalise = l->normalise;
    p.beta = beta;
    p.residual = beta != 0.0f ? residual + t * ld_residual : NULL, p.ld_residual = ld_residual;
    p.y = y + t * ldy, p.ldy = ldy;
    p.ids = l->ids ? l->ids + t * l->top_k : NULL;
    p.weights = l->weights ? l->weights + t * l->top_k : NULL;
    rc = skl_hip_launch_moe(&p);
    if (rc != 0) return rc;
  }
  return 0;
}

void skl_moe_bf16_mxf4e2m1_f32_gfx950(const skl_gfx950_moe_t *layer, size_t tokens, const skl_bf16_t *x, size_t ldx, float beta,
                                      const float *residual, size_t ld_residual, float *y, size_t ldy) {
  const skl_gfx950_moe_t *l = layer;
  int where;
  if (tokens == 0) return;
  if (!l || !moe_ok(l, tokens, x, ldx, beta, residual, y) || (tokens > 1 && !rows_of_y_ok(l->hidden, beta, residual, ld_residual, y, ldy))) {
    bad_argument(__func__);
    return;
  }
  {
    const void *given[12] = {x, y, beta != 0.0f ? residual : NULL, l->router, l->gate, l->up, l->down, l->gate_scales, l->up_scales, l->down_scales, l->ids, l->weights};
    where = skl_classify(given, 12, __func__);
  }
  if (where < 0) return;
  if (where == 1) {
    (void)moe_on_device(l, tokens, x, ldx, beta, residual, ld_residual, y, ldy);
    return;
  }
  {
    const size_t h = l->hidden, i = l->inter, e = l->experts, picks = tokens * l->top_k;
    const size_t in = span(e, l->expert_in / 2, span(i, l->ld_in / 2, h / 2)), in_s = span(e, l->expert_in_scales, span(i, l->ld_in_scales, h / 32));
    const size_t down = span(e, l->expert_down / 2, span(h, l->ld_down / 2, i / 2)), down_s = span(e, l->expert_down_scales, span(h, l->ld_down_scales, i / 32));
    const size_t ny = span(tokens, ldy, h) * sizeof(float);
    const int with_residual = beta != 0.0f;
    skl_gfx950_moe_t d = *l;
    void *dx = skl_stage_in(x, span(tokens, ldx, h) * 2), *dy = skl_stage_in(y, ny);
    void *dr = with_residual ? skl_stage_in(residual, span(tokens, ld_residual, h) * sizeof(float)) : NULL;
    void *router = skl_stage_in(l->router, span(e, l->ld_router, h) * 2);
    void *gate = skl_stage_in(l->gate, in), *up = skl_stage_in(l->up, in), *gate_s = skl_stage_in(l->gate_scales, in_s), *up_s = skl_stage_in(l->up_scales, in_s);
    void *dn = skl_stage_in(l->down, down), *dn_s = skl_stage_in(l->down_scales, down_s);
    void *ids = l->ids ? skl_hip_malloc(picks * sizeof(int32_t)) : NULL, *weights = l->weights ? skl_hip_malloc(picks * sizeof(float)) : NULL;
    d.router = (const skl_bf16_t *)router;
    d.gate = (const uint8_t *)gate, d.up = (const uint8_t *)up, d.down = (const uint8_t *)dn;
    d.gate_scales = (const uint8_t *)gate_s, d.up_scales = (const uint8_t *)up_s, d.down_scales = (const uint8_t *)dn_s;
    d.ids = (int32_t *)ids, d.weights = (float *)weights;
    if (dx && dy && (!with_residual || dr) && router && gate && up && gate_s && up_s && dn && dn_s && (!l->ids || ids) && (!l->weights || weights) &&
        moe_on_device(&d, tokens, dx, ldx, beta, (const float *)dr, ld_residual, (float *)dy, ldy) == 0) {
      skl_hip_memcpy_d2h(y, dy, ny);
      if (ids) skl_hip_memcpy_d2h(l->ids, ids, picks * sizeof(int32_t));
      if (weights) skl_hip_memcpy_d2h(l->weights, weights, picks * sizeof(float));
    }
    skl_hip_free(dx);
    skl_hip_free(dy);
    skl_hip_free(dr);
    skl_hip_free(router);
    skl_hip_free(gate);
    skl_hip_free(up);
    skl_hip_free(gate_s);
    skl_hip_free(up_s);
    skl_hip_free(dn);
    skl_hip_free(dn_s);
    skl_hip_free(ids);
    skl_hip_free(weights);
  }
}
