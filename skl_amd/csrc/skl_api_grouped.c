/*
 * skl_api_grouped.c - the C host layer of the products grouped by expert of include/skl-gfx950.h: arguments are checked,
 * ordinary host memory is staged, and the launchers of skl_grouped.h do the rest.
 */
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include "../../include/skl-gfx950.h"
#include "skl_grouped.h"
#include "skl_host.h"

#define MOST_ROWS ((size_t)1 << 30) /* of anything that 32-bit numbers count */

static void bad_argument(const char *who) { skl_hip_record_error(SKL_HIP_ERR_BAD_ARGUMENT, who); }

/* Elements from the first to the last of `rows` runs of `run` elements, `distance` apart. */
static size_t span(size_t rows, size_t distance, size_t run) { return rows && run ? (rows - 1) * distance + run : 0; }

static skl_scalar beta_of(float beta) {
  skl_scalar s;
  memset(&s, 0, sizeof s);
  s.fz.value = beta;
  /* an old C that is not read counts as +0 */
  s.fz.skip_c_read = skl_hip_get_beta_zero_mode() != SKL_HIP_BETA_ZERO_AS_REFERENCE ? SKL_C_UNTOUCHED : 0;
  return s;
}
static skl_scalar alpha_of(float alpha) {
  skl_scalar s;
  memset(&s, 0, sizeof s);
  s.f = alpha;
  return s;
}

/* A group list: offsets may be missing where there is one group. */
static int groups_ok(size_t groups, const int32_t *offsets) { return groups >= 1 && groups <= SKL_MAX_GROUPS && (offsets || groups == 1); }

/* Copies of host arrays on the device. What was asked for and could not be had leaves `failed`. */
typedef struct {
  void *held[12];
  int count, failed;
} staged;
static void *stage(staged *s, const void *host, size_t bytes) {
  void *d;
  if (!host || bytes == 0) return NULL;
  d = skl_stage_in(host, bytes);
  if (!d) s->failed = 1;
  s->held[s->count++] = d;
  return d;
}
static void unstage(staged *s) {
  int i;
  for (i = 0; i < s->count; ++i) skl_hip_free(s->held[i]);
}

/* ------------------------------------------------------------------------ */
/* the order                                                                 */
/* ------------------------------------------------------------------------ */

void skl_group_rows_gfx950(size_t count, const int32_t *ids, size_t per_row, size_t groups, int32_t *offsets, int32_t *order, int32_t *rows,
                           int32_t *place) {
  const void *given[5] = {count ? ids : NULL, offsets, count ? order : NULL, count ? rows : NULL, count ? place : NULL};
  int where;
  if (groups == 0 || groups > SKL_MAX_GROUPS || count > MOST_ROWS || !offsets || (count && !ids) || (rows && per_row == 0)) {
    bad_argument(__func__);
    return;
  }
  where = skl_classify(given, 5, __func__);
  if (where < 0) return;
  if (where == 1) {
    skl_hip_launch_group_rows(count, ids, per_row, groups, offsets, order, rows, place);
    return;
  }
  {
    const size_t bytes = count * sizeof(int32_t), of_offsets = (groups + 1) * sizeof(int32_t);
    staged s;
    int32_t *d_ids, *d_offsets, *d_order, *d_rows, *d_place;
    memset(&s, 0, sizeof s);
    d_ids = (int32_t *)stage(&s, ids, bytes), d_offsets = (int32_t *)stage(&s, offsets, of_offsets);
    /* the places behind the last group travel both ways and come back unchanged */
    d_order = (int32_t *)stage(&s, order, bytes), d_rows = (int32_t *)stage(&s, rows, bytes), d_place = (int32_t *)stage(&s, place, bytes);
    if (!s.failed && skl_hip_launch_group_rows(count, d_ids, per_row, groups, d_offsets, d_order, d_rows, d_place) == 0) {
      skl_hip_memcpy_d2h(offsets, d_offsets, of_offsets);
      if (d_order) skl_hip_memcpy_d2h(order, d_order, bytes);
      if (d_rows) skl_hip_memcpy_d2h(rows, d_rows, bytes);
      if (d_place) skl_hip_memcpy_d2h(place, d_place, bytes);
    }
    unstage(&s);
  }
}

/* ------------------------------------------------------------------------ */
/* products of groups of rows                                                */
/* ------------------------------------------------------------------------ */

/* What the operands that both kinds of product share have to be. */
static int rows_ok(const skl_grouped_gemm *g) {
  if (!groups_ok(g->groups, g->offsets)) return 0;
  if (g->m > MOST_ROWS || g->n > MOST_ROWS || g->k > MOST_ROWS || g->a_rows > MOST_ROWS) return 0;
  if (!g->c || (g->m > 1 && g->rsc < g->n)) return 0;
  return g->k == 0 || (g->rows && g->a_rows == 0) || g->a != NULL;
}
static size_t rows_of_a(const skl_grouped_gemm *g) { return g->rows ? g->a_rows : g->m; }
static size_t bytes_of_c(const skl_grouped_gemm *g) { return span(g->m, g->rsc, g->n) * (g->c_single ? 4 : 2); }
/* A, its index, the offsets and C of a call in host memory. */
static void stage_rows(staged *s, const skl_grouped_gemm *g, skl_grouped_gemm *d) {
  *d = *g;
  d->offsets = (const int32_t *)stage(s, g->offsets, (g->groups + 1) * sizeof(int32_t));
  d->a = stage(s, g->a, span(rows_of_a(g), g->rsa, g->k) * 2);
  d->rows = (const int32_t *)stage(s, g->rows, g->m * sizeof(int32_t));
  d->c = stage(s, g->c, bytes_of_c(g)); /* its whole span travels both ways: what no group covers comes back unchanged */
}

/* With k == 0, or an A of no rows, sums are empty: nothing is read but the offsets and C. (Kernels look rows up whatever k is.) */
static void no_operands_of_empty_sums(skl_grouped_gemm *g) {
  if (g->rows && g->a_rows == 0) g->k = 0;
  if (g->k == 0) g->a = NULL, g->rows = NULL, g->b = NULL;
}

static void grouped(skl_grouped_gemm g, const char *who) {
  int where;
  if (g.m == 0 || g.n == 0 || g.groups == 0) return; /* nothing is addressed */
  if (!rows_ok(&g) || (g.k && !g.b)) {
    bad_argument(who);
    return;
  }
  no_operands_of_empty_sums(&g);
  {
    const void *given[5] = {g.offsets, g.a, g.rows, g.b, g.c};
    where = skl_classify(given, 5, who);
  }
  if (where < 0) return;
  if (where == 1) {
    skl_hip_launch_gemm_grouped(&g);
    return;
  }
  {
    staged s;
    skl_grouped_gemm d;
    memset(&s, 0, sizeof s);
    stage_rows(&s, &g, &d);
    d.b = g.k ? stage(&s, g.b, ((g.groups - 1) * g.gsb + (g.k - 1) * g.rsb + (g.n - 1) * g.csb + 1) * 2) : NULL;
    if (!s.failed && skl_hip_launch_gemm_grouped(&d) == 0) skl_hip_memcpy_d2h(g.c, d.c, bytes_of_c(&g));
    unstage(&s);
  }
}

static skl_grouped_gemm grouped_problem(int dt, int c_single, size_t groups, const int32_t *offsets, size_t m, size_t n, size_t k, float alpha, const void *a, size_t rsa,
                                        const int32_t *rows, size_t a_rows, float beta, void *c, size_t rsc) {
  skl_grouped_gemm g;
  memset(&g, 0, sizeof g);
  g.dt = dt, g.c_single = c_single, g.groups = groups, g.offsets = offsets, g.m = m, g.n = n, g.k = k;
  g.a = a, g.rsa = rsa, g.rows = rows, g.a_rows = a_rows, g.c = c, g.rsc = rsc;
  g.alpha = alpha_of(alpha), g.beta = beta_of(beta);
  return g;
}

#define SKL_GROUPED(NAME, DT, T, SINGLE, TC)                                                                                                          \
  void NAME(size_t groups, const int32_t *offsets, size_t m, size_t n, size_t k, float alpha, const T *a, size_t rsa, const int32_t *rows,            \
            size_t a_rows, const T *b, size_t rsb, size_t csb, size_t gsb, float beta, TC *c, size_t rsc) {                                           \
    skl_grouped_gemm g = grouped_problem(DT, SINGLE, groups, offsets, m, n, k, alpha, a, rsa, rows, a_rows, beta, c, rsc);                            \
    g.b = b, g.rsb = rsb, g.csb = csb, g.gsb = gsb;                                                                                                   \
    grouped(g, __func__);                                                                                                                             \
  }
SKL_GROUPED(skl_gemm_grouped_bf16_bf16rc_f32_gfx950, SKL_DT_BF16, skl_bf16_t, 1, float)
SKL_GROUPED(skl_gemm_grouped_bf16_bf16rc_bf16_gfx950, SKL_DT_BF16, skl_bf16_t, 0, skl_bf16_t)
SKL_GROUPED(skl_gemm_grouped_f16_f16rc_f32_gfx950, SKL_DT_F16, skl_f16_t, 1, float)
SKL_GROUPED(skl_gemm_grouped_f16_f16rc_f16_gfx950, SKL_DT_F16, skl_f16_t, 0, skl_f16_t)
#undef SKL_GROUPED

/* ------------------------------------------------------------------------ */
/* products summed over groups of rows                                       */
/* ------------------------------------------------------------------------ */

/* The groups' matrices lie one behind the other, or their rows side by side. */
static int results_apart(const skl_groupedk_gemm *g) {
  return g->groups == 1 || g->gsc >= span(g->m, g->rsc, g->n) || (g->gsc >= g->n && g->rsc >= span(g->groups, g->gsc, g->n));
}

static void groupedk(skl_groupedk_gemm g, const char *who) {
  int where;
  if (g.m == 0 || g.n == 0 || g.groups == 0) return; /* nothing is addressed */
  if (!groups_ok(g.groups, g.offsets) || g.m > MOST_ROWS || g.n > MOST_ROWS || g.total > MOST_ROWS || g.a_rows > MOST_ROWS || g.b_rows > MOST_ROWS || !g.c ||
      (g.m > 1 && g.rsc < g.n) || !results_apart(&g) || (g.total && ((!g.a && !(g.rows_a && g.a_rows == 0)) || (!g.b && !(g.rows_b && g.b_rows == 0))))) {
    bad_argument(who);
    return;
  }
  if ((g.rows_a && g.a_rows == 0) || (g.rows_b && g.b_rows == 0)) g.total = 0; /* an operand of no rows: every sum is empty */
  if (g.total == 0) g.a = g.b = NULL, g.rows_a = g.rows_b = NULL;
  {
    const void *given[6] = {g.offsets, g.a, g.b, g.rows_a, g.rows_b, g.c};
    where = skl_classify(given, 6, who);
  }
  if (where < 0) return;
  if (where == 1) {
    skl_hip_launch_gemm_groupedk(&g);
    return;
  }
  {
    const size_t nc = span(g.groups, g.gsc, span(g.m, g.rsc, g.n)) * (g.c_single ? 4 : 2);
    skl_groupedk_gemm d = g;
    staged s;
    memset(&s, 0, sizeof s);
    d.offsets = (const int32_t *)stage(&s, g.offsets, (g.groups + 1) * sizeof(int32_t));
    d.a = stage(&s, g.a, span(g.rows_a ? g.a_rows : g.total, g.rsa, g.m) * 2);
    d.b = stage(&s, g.b, span(g.rows_b ? g.b_rows : g.total, g.rsb, g.n) * 2);
    d.rows_a = (const int32_t *)stage(&s, g.rows_a, g.total * sizeof(int32_t));
    d.rows_b = (const int32_t *)stage(&s, g.rows_b, g.total * sizeof(int32_t));
    d.c = stage(&s, g.c, nc);
    if (!s.failed && skl_hip_launch_gemm_groupedk(&d) == 0) skl_hip_memcpy_d2h(g.c, d.c, nc);
    unstage(&s);
  }
}

#define SKL_GROUPEDK(NAME, DT, T, SINGLE, TC)                                                                                                         \
  void NAME(size_t groups, const int32_t *offsets, size_t m, size_t n, size_t total, float alpha, const T *a, size_t rsa, const int32_t *rows_a,      \
            size_t a_rows, const T *b, size_t rsb, const int32_t *rows_b, size_t b_rows, float beta, TC *c, size_t rsc, size_t gsc) {                 \
    skl_groupedk_gemm g;                                                                                                                              \
    memset(&g, 0, sizeof g);                                                                                                                          \
    g.dt = DT, g.c_single = SINGLE, g.groups = groups, g.offsets = offsets, g.m = m, g.n = n, g.total = total;                                        \
    g.a = a, g.rsa = rsa, g.rows_a = rows_a, g.a_rows = a_rows, g.b = b, g.rsb = rsb, g.rows_b = rows_b, g.b_rows = b_rows;                           \
    g.c = c, g.rsc = rsc, g.gsc = gsc, g.alpha = alpha_of(alpha), g.beta = beta_of(beta);                                                             \
    groupedk(g, __func__);                                                                                                                            \
  }
SKL_GROUPEDK(skl_gemm_groupedk_bf16c_bf16_f32_gfx950, SKL_DT_BF16, skl_bf16_t, 1, float)
SKL_GROUPEDK(skl_gemm_groupedk_bf16c_bf16_bf16_gfx950, SKL_DT_BF16, skl_bf16_t, 0, skl_bf16_t)
SKL_GROUPEDK(skl_gemm_groupedk_f16c_f16_f32_gfx950, SKL_DT_F16, skl_f16_t, 1, float)
SKL_GROUPEDK(skl_gemm_groupedk_f16c_f16_f16_gfx950, SKL_DT_F16, skl_f16_t, 0, skl_f16_t)
#undef SKL_GROUPEDK

/* ------------------------------------------------------------------------ */
/* 4-bit weights                                                             */
/* ------------------------------------------------------------------------ */

static int u4_ok(const skl_gfx950_u4_t *b, size_t groups, size_t n, size_t k) {
  size_t blocks;
  if (!b || b->group_k == 0 || (b->group_k % 32 != 0 && b->group_k < k) || !b->codes || !b->scales) return 0;
  blocks = k / b->group_k + (k % b->group_k != 0);
  if (n > 1 && (b->ld % 2 != 0 || b->ld < k || b->ld_scales < blocks)) return 0;
  return groups <= 1 || b->expert % 2 == 0;
}

static void grouped_u4(skl_grouped_gemm g, const skl_gfx950_u4_t *b, const char *who) {
  skl_grouped_u4 u;
  int where;
  if (g.m == 0 || g.n == 0 || g.groups == 0) return; /* nothing is addressed */
  if (!rows_ok(&g) || (g.k && !u4_ok(b, g.groups, g.n, g.k))) {
    bad_argument(who);
    return;
  }
  no_operands_of_empty_sums(&g);
  memset(&u, 0, sizeof u);
  u.g = g;
  if (g.k) {
    u.group_k = b->group_k < g.k ? b->group_k : g.k;
    u.codes = b->codes, u.ld = b->ld, u.expert = b->expert;
    u.scales = b->scales, u.zeros = b->zeros, u.ld_scales = b->ld_scales, u.expert_scales = b->expert_scales;
  }
  {
    const void *given[7] = {g.offsets, g.a, g.rows, u.codes, u.scales, u.zeros, g.c};
    where = skl_classify(given, 7, who);
  }
  if (where < 0) return;
  if (where == 1) {
    skl_hip_launch_gemm_u4(&u);
    return;
  }
  {
    skl_grouped_u4 d = u;
    staged s;
    memset(&s, 0, sizeof s);
    stage_rows(&s, &g, &d.g);
    if (g.k) {
      const size_t blocks = (g.k + u.group_k - 1) / u.group_k, places = span(g.groups, u.expert_scales, span(g.n, u.ld_scales, blocks));
      d.codes = (const uint8_t *)stage(&s, u.codes, span(g.groups, u.expert / 2, span(g.n, u.ld / 2, (g.k + 1) / 2)));
      d.scales = stage(&s, u.scales, places * 2);
      d.zeros = (const uint8_t *)stage(&s, u.zeros, places);
    }
    if (!s.failed && skl_hip_launch_gemm_u4(&d) == 0) skl_hip_memcpy_d2h(g.c, d.g.c, bytes_of_c(&g));
    unstage(&s);
  }
}

#define SKL_GROUPED_U4(NAME, DT, T, SINGLE, TC)                                                                                                       \
  void NAME(size_t groups, const int32_t *offsets, size_t m, size_t n, size_t k, float alpha, const T *a, size_t rsa, const int32_t *rows,            \
            size_t a_rows, const skl_gfx950_u4_t *b, float beta, TC *c, size_t rsc) {                                                                 \
    grouped_u4(grouped_problem(DT, SINGLE, groups, offsets, m, n, k, alpha, a, rsa, rows, a_rows, beta, c, rsc), b, __func__);                        \
  }
SKL_GROUPED_U4(skl_gemm_grouped_bf16_u4c_f32_gfx950, SKL_DT_BF16, skl_bf16_t, 1, float)
SKL_GROUPED_U4(skl_gemm_grouped_bf16_u4c_bf16_gfx950, SKL_DT_BF16, skl_bf16_t, 0, skl_bf16_t)
SKL_GROUPED_U4(skl_gemm_grouped_f16_u4c_f32_gfx950, SKL_DT_F16, skl_f16_t, 1, float)
SKL_GROUPED_U4(skl_gemm_grouped_f16_u4c_f16_gfx950, SKL_DT_F16, skl_f16_t, 0, skl_f16_t)
#undef SKL_GROUPED_U4
