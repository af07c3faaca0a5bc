/*
 * skl_mx.h - internal C-ABI of the microscaled 4-bit kernels and the mixture-of-experts layer, between their host layer
 * (skl_api_mx.c) and the HIP translation units; what skl_launch.h is for the rest of the library. Every pointer handed
 * to these functions is device-accessible and the arguments have been checked. All return 0 or an error code that has
 * also been recorded.
 */
#ifndef SKL_MX_H
#define SKL_MX_H

#include <stddef.h>
#include <stdint.h>

#include "skl_launch.h"

#ifdef __cplusplus
extern "C" {
#endif

/* An MXFP4 matrix: value (i, p) is 4-bit number i * ld + p of `codes` times 2^(scales[i * lds + p / 32] - 127). */
typedef struct {
  const uint8_t *codes;
  size_t ld; /* in values, even */
  const uint8_t *scales;
  size_t lds;
} skl_mx_operand;

/* `dt`: SKL_DT_F32 or SKL_DT_BF16. Element (i, p) of the other matrix at i * rs + p * cs. */
int skl_hip_launch_cvt_to_mx(int dt, size_t m, size_t k, const void *src, size_t rs, size_t cs, uint8_t *codes, size_t ld,
                             uint8_t *scales, size_t lds);
int skl_hip_launch_cvt_from_mx(int dt, size_t m, size_t k, const skl_mx_operand *src, void *dst, size_t rs, size_t cs);

typedef struct {
  size_t m, n, k;
  skl_mx_operand a, b; /* rows of A, columns of B */
  float *c;
  size_t rsc, csc;
  skl_scalar alpha, beta; /* beta with fz.skip_c_read */
} skl_mx_gemm;
int skl_hip_launch_gemm_mx(const skl_mx_gemm *g);

/* One chunk of at most SKL_MOE_TOKENS tokens of a mixture-of-experts layer (include/skl-gfx950.h has the formulas). */
#define SKL_MOE_TOKENS 64u
typedef struct {
  size_t tokens, hidden, inter, experts, top_k;
  const uint16_t *x;
  size_t ldx;
  const uint16_t *router;
  size_t ld_router;
  skl_mx_operand gate, up, down;
  size_t expert_in, expert_in_scales, expert_down, expert_down_scales;
  int activation, normalise;
  float beta;
  const float *residual;
  size_t ld_residual;
  float *y;
  size_t ldy;
  int32_t *ids;   /* NULL: not wanted */
  float *weights;
} skl_moe_problem;
int skl_hip_launch_moe(const skl_moe_problem *p);

#ifdef __cplusplus
}
#endif
#endif /* SKL_MX_H */
