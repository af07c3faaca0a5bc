// skl_gemm_u4.hip - products with integer 4-bit weights that have scales for groups along k (include/skl-gfx950.h: skl_gfx950_u4_t).
//
// v_mfma_f32_16x16x32 of 16 rows of A and 16 columns of weights: lane l holds eight k of row (column) l % 16 and, of the sums, rows 4 (l / 16) .. + 3 of
// column l % 16, so that a column's scale is one value of its lanes. A product is a * (q - z), exact: q - z is made in registers as bf16 or f16. The sums of
// at most 128 k of one group are scaled and added to the result in fp32.
#include <hip/hip_runtime.h>

#include <atomic>

#include "skl_groups.hpp"
#include "../../include/skl-hip.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

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
__device__ __forceinline__ v4f product(v4i a, v4i b, v4f c);
template <>
__device__ __forceinline__ v4f product<__bf16>(v4i a, v4i b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0); }
template <>
__device__ __forceinline__ v4f product<_Float16>(v4i a, v4i b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0); }

template <typename T>
constexpr bool is_bf16 = __is_same(T, __bf16);

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
      const v4f part_sum = product<T>(__builtin_bit_cast(v4i, x), __builtin_bit_cast(v4i, w), v4f{0, 0, 0, 0});
      const float scale = skl_widen(p.scales[first_scale + block], is_bf16<T>);
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

// ---------------------------------------------------------------------------
// The stream over the codes: rows of codes and of A on 16-byte boundaries, k a multiple of 32, group_k 32, 64, 128 or a multiple of 256 (one group of all k
// among them).
// A workgroup takes 16 F columns and all of k, its waves units of 256 k - a line of each column's codes - in turn, and up to 16 R rows per pass; the
// waves' sums meet in LDS. What bounds it is the codes' way from memory: two units are under way per wave.
// ---------------------------------------------------------------------------

// Eight values q - z, natural order of k; `z` as prepared by zero_of().
template <typename T>
struct Zero;
template <>
struct Zero<__bf16> {
  float z;
  __device__ __forceinline__ explicit Zero(unsigned v) : z((float)v) {}
};
template <>
struct Zero<_Float16> {
  v2h z;
  __device__ __forceinline__ explicit Zero(unsigned v) : z(__builtin_bit_cast(v2h, (0x6400u + v) * 0x10001u)) {}  // 1024 + v, twice (v < 1024)
};
__device__ __forceinline__ v4i widened(unsigned codes, Zero<__bf16> z) {
  const unsigned even = codes & 0x0F0F0F0Fu, odd = (codes >> 4) & 0x0F0F0F0Fu;
  v8bf w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[2 * i] = (__bf16)((float)((even >> (8 * i)) & 255u) - z.z);
    w[2 * i + 1] = (__bf16)((float)((odd >> (8 * i)) & 255u) - z.z);
  }
  return __builtin_bit_cast(v4i, w);
}
// f16: k0 k4, k1 k5, k2 k6, k3 k7 as the nibbles lie; the fragment of A is put into that order (arranged()). 1024 + q has q for its last bits.
__device__ __forceinline__ v4i widened(unsigned codes, Zero<_Float16> z) {
  v4i w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, ((codes >> (4 * i)) & 0x000F000Fu) | 0x64006400u) - z.z);
  return w;
}
template <typename T>
__device__ __forceinline__ v4i arranged(v4i a) {
  if constexpr (is_bf16<T>) {
    return a;
  } else {
    v4i r;
    r[0] = (int)__builtin_amdgcn_perm((unsigned)a[2], (unsigned)a[0], 0x05040100u);
    r[1] = (int)__builtin_amdgcn_perm((unsigned)a[2], (unsigned)a[0], 0x07060302u);
    r[2] = (int)__builtin_amdgcn_perm((unsigned)a[3], (unsigned)a[1], 0x05040100u);
    r[3] = (int)__builtin_amdgcn_perm((unsigned)a[3], (unsigned)a[1], 0x07060302u);
    return r;
  }
}

// Dword i of the four quarters of a wave, transposed: quarter p's dword j becomes quarter j's dword p.
__device__ __forceinline__ v4i quarters_transposed(v4i v) {
  typedef unsigned v2u __attribute__((ext_vector_type(2)));
  const v2u a = __builtin_amdgcn_permlane32_swap((unsigned)v[0], (unsigned)v[2], false, false), b = __builtin_amdgcn_permlane32_swap((unsigned)v[1], (unsigned)v[3], false, false);
  const v2u c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return v4i{(int)c[0], (int)c[1], (int)d[0], (int)d[1]};
}

constexpr unsigned kUnit = 256;  // of k

// Of a column's unit: its codes as two pieces per lane - piece j of quarter p holds k 128 j + 32 p .. + 31 -, its scales and zero points.
// PER: groups of a unit, 8, 4, 2 or 1.
template <int PER, bool ZEROS>
struct UnitOf {
  v4i piece[2];
  uint16_t scale[PER];
  uint8_t zero[ZEROS ? PER : 1];
  // `tail`: the row's last, partial unit, `left` k of it (a multiple of 32): pieces beyond are zeros, groups beyond the row's last one again.
  __device__ __forceinline__ void load(const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros, unsigned part, unsigned unit, bool tail, unsigned left, unsigned first_group, unsigned last_group) {
    const uint8_t *const at = codes + (size_t)unit * (kUnit / 2) + 16 * part;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool there = !tail || 128u * j + 32u * part < left;
      piece[j] = there ? __builtin_nontemporal_load(reinterpret_cast<const v4i *>(at + 64 * j)) : v4i{0, 0, 0, 0};
    }
#pragma unroll
    for (int g = 0; g < PER; ++g) {
      const unsigned group = first_group + g < last_group ? first_group + g : last_group;
      scale[g] = scales[group];
      if constexpr (ZEROS) zero[g] = zeros[group];
    }
  }
};

template <typename T, int PER, bool ZEROS, int F, int R, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) gemm_u4_stream_kernel(U4Args p, int c_single) {
  constexpr bool kFine = PER > 2;  // groups smaller than the 128 k whose codes the quarters of a wave hold side by side
  __shared__ float sums_lds[WAVES][16 * R][16 * F + 1];
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, l = lane & 15u, part = lane >> 4, e = blockIdx.y;
  const SklRange range = skl_group_range(p.offsets, e, p.m);
  if (range.rows == 0) return;
  const unsigned col0 = blockIdx.x * (16 * F);
  const unsigned units = (p.k + kUnit - 1) / kUnit, last_group = p.k ? (p.k - 1) / p.group_k : 0;
  const unsigned units_per_group = PER == 1 ? p.group_k / kUnit : 1;
  const uint8_t *codes[F], *zeros[F];
  const uint16_t *scales[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const unsigned col = col0 + 16 * f + l < p.n ? col0 + 16 * f + l : p.n - 1;
    codes[f] = p.codes + ((size_t)e * p.expert + (size_t)col * p.ld) / 2;
    scales[f] = p.scales + (size_t)e * p.expert_scales + (size_t)col * p.ld_scales;
    zeros[f] = ZEROS ? p.zeros + (size_t)e * p.expert_scales + (size_t)col * p.ld_scales : nullptr;
  }
  const bool read_c = !skl_beta_is_zero<float>(p.beta);
  const unsigned limit = p.rows ? p.a_rows : p.m;  // an A without rows: nothing to multiply
  for (unsigned row0 = 0; row0 < range.rows; row0 += 16 * R) {
    // Rows that do not exist are the group's first again, those that an index puts outside A its first: computed, and written nowhere or as zeros.
    const uint16_t *a[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      unsigned row = range.first + (row0 + 16 * r + l < range.rows ? row0 + 16 * r + l : 0u);
      if (p.rows) row = (unsigned)p.rows[row];
      a[r] = p.a + (size_t)(row < limit ? row : 0u) * p.rsa;
    }
    v4f sum[R][F];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int f = 0; f < F; ++f) sum[r][f] = v4f{0, 0, 0, 0};
    UnitOf<PER, ZEROS> unit[2][F];
    const auto load = [&](int slot, unsigned u) __attribute__((always_inline)) {
      const bool tail = (u + 1) * kUnit > p.k;
#pragma unroll
      for (int f = 0; f < F; ++f) unit[slot][f].load(codes[f], scales[f], zeros[f], part, u, tail, p.k - u * kUnit, PER == 1 ? u / units_per_group : u * PER, last_group);
    };
    const auto multiply = [&](int slot, unsigned u) __attribute__((always_inline)) {
      const bool tail = (u + 1) * kUnit > p.k;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v4i piece[F];
#pragma unroll
        for (int f = 0; f < F; ++f) piece[f] = kFine ? quarters_transposed(unit[slot][f].piece[j]) : unit[slot][f].piece[j];
        v4f acc[R][F];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          constexpr int kOf = PER >= 2 ? 8 / PER : 8;  // instructions of a group in a unit
          const int at = 4 * j + i, group = at / kOf;
          const bool begins = at % kOf == 0 || i == 0, ends = (at + 1) % kOf == 0 || i == 3;
          const unsigned k = u * kUnit + 128 * j + (kFine ? 32 * i + 8 * part : 32 * part + 8 * i);
          v4i x[R];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            x[r] = !tail || k < p.k ? *reinterpret_cast<const v4i *>(a[r] + k) : v4i{0, 0, 0, 0};
            x[r] = arranged<T>(x[r]);
          }
#pragma unroll
          for (int f = 0; f < F; ++f) {
            const v4i w = widened((unsigned)piece[f][i], Zero<T>(ZEROS ? unit[slot][f].zero[ZEROS ? group : 0] : 8u));
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][f] = product<T>(x[r], w, begins ? v4f{0, 0, 0, 0} : acc[r][f]);
          }
          if (ends) {
#pragma unroll
            for (int f = 0; f < F; ++f) {
              const float scale = skl_widen(unit[slot][f].scale[group], is_bf16<T>);
#pragma unroll
              for (int r = 0; r < R; ++r)
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[r][f][q] = __builtin_fmaf(acc[r][f][q], scale, sum[r][f][q]);
            }
          }
        }
      }
    };
    if (limit != 0) {
      if (wave < units) load(0, wave);
      for (unsigned u = wave; u < units; u += 2 * WAVES) {
        if (u + WAVES < units) load(1, u + WAVES);
        multiply(0, u);
        if (u + WAVES >= units) break;
        if (u + 2 * WAVES < units) load(0, u + 2 * WAVES);
        multiply(1, u + WAVES);
      }
    }
    if (row0) __syncthreads();  // the sums of the pass before have been read
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) sums_lds[wave][16 * r + 4 * part + q][16 * f + l] = sum[r][f][q];
    __syncthreads();
    for (unsigned i = threadIdx.x; i < 256 * R * F; i += WAVES * 64) {
      const unsigned row = i / (16 * F), c = i % (16 * F), col = col0 + c;
      if (row0 + row >= range.rows || col >= p.n) continue;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) v = __fadd_rn(v, sums_lds[w][row][c]);
      const unsigned out = range.first + row0 + row;
      if (p.rows && (unsigned)p.rows[out] >= limit) v = 0.0f;
      const size_t at = (size_t)out * p.rsc + col;
      if (c_single) {
        float *const to = reinterpret_cast<float *>(p.c) + at;
        *to = skl_grouped_result(v, to, p.alpha, p.beta, read_c);
      } else {
        T *const to = reinterpret_cast<T *>(p.c) + at;
        *to = skl_grouped_result(v, to, p.alpha, p.beta, read_c);
      }
    }
  }
}

template <typename T, int PER, int F, int R, int WAVES>
int launch_stream(const U4Args &p, int c_single) {
  const dim3 grid(skl_div_up(p.n, 16 * F), p.groups), block(WAVES * 64);
  if (p.zeros) gemm_u4_stream_kernel<T, PER, true, F, R, WAVES><<<grid, block, 0, skl_current_stream()>>>(p, c_single);
  else gemm_u4_stream_kernel<T, PER, false, F, R, WAVES><<<grid, block, 0, skl_current_stream()>>>(p, c_single);
  return skl_check_launch("gemm_u4");
}

template <typename T, int PER>
int stream_by_size(const U4Args &p, int c_single) {
  if (p.m > 16 * p.groups) return launch_stream<T, PER, 2, 2, 8>(p, c_single);
  const size_t cols = (size_t)p.n * (p.groups < p.m ? p.groups : p.m);
  if (cols >= 16384) return launch_stream<T, PER, 4, 1, 8>(p, c_single);
  return launch_stream<T, PER, 1, 1, 4>(p, c_single);
}

template <typename T>
int launch(U4Args p, int c_single) {
  const auto aligned = [](const void *at) { return ((uintptr_t)at & 15) == 0; };
  const bool one = p.group_k >= p.k;
  if (p.k % 32 == 0 && aligned(p.a) && aligned(p.codes) && p.rsa % 8 == 0 && p.ld % 32 == 0 && p.expert % 32 == 0 &&
      (one || p.group_k == 32 || p.group_k == 64 || p.group_k == 128 || p.group_k % 256 == 0)) {
    if (one || p.group_k % 256 == 0) {
      if (one) p.group_k = (p.k + kUnit - 1) / kUnit * kUnit;
      return stream_by_size<T, 1>(p, c_single);
    }
    if (p.group_k == 32) return stream_by_size<T, 8>(p, c_single);
    return p.group_k == 64 ? stream_by_size<T, 4>(p, c_single) : stream_by_size<T, 2>(p, c_single);
  }
  const dim3 grid(skl_div_up(p.n, 64), p.groups);
  if (c_single) gemm_u4_any_kernel<T, float><<<grid, dim3(256), 0, skl_current_stream()>>>(p);
  else gemm_u4_any_kernel<T, T><<<grid, dim3(256), 0, skl_current_stream()>>>(p);
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
  // Columns of a launch: beyond 2^32 threads the runtime takes what is left of the number in 32 bits.
  const size_t slab = size_t(1) << 26;
  for (size_t col = 0; col < g->n; col += slab) {
    p.n = (unsigned)(g->n - col < slab ? g->n - col : slab);
    p.codes = u->codes + col * (u->ld / 2);
    p.scales = (const uint16_t *)u->scales + col * u->ld_scales;
    p.zeros = u->zeros ? u->zeros + col * u->ld_scales : nullptr;
    p.c = (char *)g->c + col * (g->c_single ? 4 : 2);
    const int rc = g->dt == SKL_DT_BF16 ? launch<__bf16>(p, g->c_single) : launch<_Float16>(p, g->c_single);
    if (rc != 0) return rc;
  }
  return 0;
}
