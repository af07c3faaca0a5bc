// skl_gemm_u4.hip - products with integer 4-bit weights that have scales for groups along k (include/skl-gfx950.h: skl_gfx950_u4_t).
#include <hip/hip_runtime.h>

#include "skl_groups.hpp"
#include "../../include/skl-hip.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct U4Args {
  const uint16_t *a;
  size_t rsa;
  const int32_t *offsets, *rows;
  unsigned groups, m, n, k, a_rows, group_k;
  const uint8_t *codes;
  size_t ld, expert;
  const uint16_t *scales;
  const uint8_t *zeros;
  size_t ld_scales, expert_scales;
  void *c;
  size_t rsc;
  skl_scalar alpha, beta;
};

template <typename T>
__device__ __forceinline__ v4f product(T a, T b, v4f c);
template <>
__device__ __forceinline__ v4f product(v8bf a, v8bf b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
template <>
__device__ __forceinline__ v4f product(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Any layout: a wave takes 16 columns, 16 rows at a time, 32 of k per instruction, value by value.
template <typename T, typename TC>
__global__ void __launch_bounds__(256) gemm_u4_any_kernel(U4Args p) {
  typedef T Frag __attribute__((ext_vector_type(8)));
  const unsigned lane = threadIdx.x & 63u, l = lane & 15u, part = lane >> 4, e = blockIdx.y;
  const unsigned col0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
  if (col0 >= p.n) return;
  const SklRange r = skl_group_range(p.offsets, e, p.m);
  const unsigned col = col0 + l < p.n ? col0 + l : p.n - 1;
  const size_t first_code = (size_t)e * p.expert + (size_t)col * p.ld, first_scale = (size_t)e * p.expert_scales + (size_t)col * p.ld_scales;
  const bool read_c = !skl_beta_is_zero<float>(p.beta);
  for (unsigned row0 = 0; row0 < r.rows; row0 += 16) {
    unsigned row = row0 + l < r.rows ? r.first + row0 + l : r.first;
    bool there = row0 + l < r.rows;
    if (p.rows) {
      row = (unsigned)p.rows[row];
      there = there && row < p.a_rows;
    }
    const uint16_t *const a = p.a + (size_t)(there ? row : 0u) * p.rsa;
    v4f sum = {0, 0, 0, 0};
    for (unsigned k0 = 0; k0 < p.k; k0 += 32) {
      const unsigned block = k0 / p.group_k;  // the same for all 32
      Frag x, w;
      const int zero = p.zeros ? (int)p.zeros[first_scale + block] : 8;
#pragma unroll
      for (unsigned i = 0; i < 8; ++i) {
        const unsigned at = k0 + 8 * part + i;
        const bool in = at < p.k;
        const uint16_t v = in && there ? a[at] : (uint16_t)0;
        x[i] = __builtin_bit_cast(T, v);
        const unsigned byte = in ? p.codes[(first_code + at) / 2] : 0u;
        w[i] = (T)(float)(in ? (int)((at & 1) ? byte >> 4 : byte & 15u) - zero : 0);
      }
      const v4f part_sum = product(x, w, v4f{0, 0, 0, 0});
      const float scale = skl_widen(p.scales[first_scale + block], sizeof(T) == 2 && __is_same(T, __bf16));
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(part_sum[i], scale, sum[i]);
    }
    if (col0 + l >= p.n) continue;
    TC *const c = reinterpret_cast<TC *>(p.c) + (size_t)r.first * p.rsc + col;
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
      const unsigned at = row0 + 4 * part + i;
      if (at >= r.rows) continue;
      TC *const to = c + (size_t)at * p.rsc;
      *to = skl_grouped_result(sum[i], to, p.alpha, p.beta, read_c);
    }
  }
}

template <typename T, typename TC>
int launch(const U4Args &p) {
  gemm_u4_any_kernel<T, TC><<<dim3(skl_div_up(p.n, 64), p.groups), dim3(256), 0, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_u4");
}

}  // namespace

int skl_hip_launch_gemm_u4(const skl_grouped_u4 *u) {
  const skl_grouped_gemm *g = &u->g;
  U4Args p{};
  p.a = (const uint16_t *)g->a, p.rsa = g->rsa, p.offsets = g->offsets, p.rows = g->rows;
  p.groups = (unsigned)g->groups, p.m = (unsigned)g->m, p.n = (unsigned)g->n, p.k = (unsigned)g->k, p.a_rows = (unsigned)g->a_rows, p.group_k = (unsigned)u->group_k;
  p.codes = u->codes, p.ld = u->ld, p.expert = u->expert;
  p.scales = (const uint16_t *)u->scales, p.zeros = u->zeros, p.ld_scales = u->ld_scales, p.expert_scales = u->expert_scales;
  p.c = g->c, p.rsc = g->rsc, p.alpha = g->alpha, p.beta = g->beta;
  if (g->dt == SKL_DT_BF16) return g->c_single ? launch<__bf16, float>(p) : launch<__bf16, __bf16>(p);
  return g->c_single ? launch<_Float16, float>(p) : launch<_Float16, _Float16>(p);
}
