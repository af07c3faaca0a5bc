/*
 * skl_grouped.h - internal C-ABI of the products grouped by expert, between their host layer (skl_api_grouped.c) and the HIP
 * translation units; what skl_launch.h is for the rest of the library. Every pointer handed to these functions is
 * device-accessible and the arguments have been checked. All return 0 or an error code that has also been recorded.
 */
#ifndef SKL_GROUPED_H
#define SKL_GROUPED_H

#include <stddef.h>
#include <stdint.h>

#include "skl_launch.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SKL_MAX_GROUPS 4096u

/* count > 0 or not; order, rows and place may be NULL. */
int skl_hip_launch_group_rows(size_t count, const int32_t *ids, size_t per_row, size_t groups, int32_t *offsets, int32_t *order, int32_t *rows,
                              int32_t *place);

/* C (m x n, row-major) = alpha * A[rows] * B_e + beta * C, by groups of rows. m, n > 0; k may be 0, with a, rows and b NULL; an A that `rows` points into has a row. */
typedef struct {
  int dt;       /* SKL_DT_BF16 or SKL_DT_F16 */
  int c_single; /* C is fp32, else as A */
  size_t groups;
  const int32_t *offsets; /* NULL: one group of all rows */
  size_t m, n, k;
  const void *a;
  size_t rsa;
  const int32_t *rows; /* NULL: row i */
  size_t a_rows;
  const void *b;
  size_t rsb, csb, gsb;
  void *c;
  size_t rsc;
  skl_scalar alpha, beta; /* beta with fz.skip_c_read */
} skl_grouped_gemm;
int skl_hip_launch_gemm_grouped(const skl_grouped_gemm *g);

/* C_e (m x n) = alpha * A[rows_a]^T B[rows_b] + beta * C_e, the sum over group e's rows. m, n > 0; total may be 0, likewise; operands have rows otherwise. */
typedef struct {
  int dt, c_single;
  size_t groups;
  const int32_t *offsets;
  size_t m, n, total;
  const void *a;
  size_t rsa;
  const int32_t *rows_a;
  size_t a_rows;
  const void *b;
  size_t rsb;
  const int32_t *rows_b;
  size_t b_rows;
  void *c;
  size_t rsc, gsc;
  skl_scalar alpha, beta;
} skl_groupedk_gemm;
int skl_hip_launch_gemm_groupedk(const skl_groupedk_gemm *g);

/* skl_grouped_gemm with 4-bit weights (`b` there is not used). */
typedef struct {
  skl_grouped_gemm g;
  size_t group_k;
  const uint8_t *codes;
  size_t ld, expert;
  const void *scales;
  const uint8_t *zeros;
  size_t ld_scales, expert_scales;
} skl_grouped_u4;
int skl_hip_launch_gemm_u4(const skl_grouped_u4 *g);

#ifdef __cplusplus
}
#endif
#endif /* SKL_GROUPED_H */
