// skl_gemm_grouped.hip - products grouped by expert (include/skl-gfx950.h): the kernels for any layout.
//
// C = alpha * A[rows] * B_e + beta * C by groups of rows, and C_e = alpha * A[rows]^T * B[rows] + beta * C_e by groups of what is summed over. 128 x 128 tiles
// of four waves, operands through registers into two stages of 64 k in LDS in the orientation they have in memory.
#include "skl_gemm_mfma_impl.hpp"
#include "skl_groups.hpp"
#include "../../include/skl-hip.h"

namespace {

struct GroupedArgs {
  const uint16_t *a, *b;
  const int32_t *offsets, *rows_a, *rows_b;
  void *c;
  size_t rsa, rsb, csb, gsb, rsc, gsc;
  unsigned groups, m, n, k, a_rows, b_rows;  // k: summed over groups, the rows in all
  unsigned tiles_m, tiles_n;                 // tiles_m: of a group, where the sums go over groups
  skl_scalar alpha, beta;
};

enum { kAlongK, kAcross, kStrided };  // an operand's unit stride: along what is summed over, across it, none

typedef v4i v4i_at2 __attribute__((aligned(2)));

constexpr int kEdge = 128, kSliceK = 64;

// 8 elements from p, of which the first `have` exist (at least one): the others are zeros.
__device__ __forceinline__ v4i load_first(const uint16_t *p, size_t step, unsigned have) {
  unsigned v[8];
#pragma unroll
  for (unsigned e = 0; e < 8; ++e) v[e] = p[(e < have ? e : have - 1) * step];
  v4i r;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) r[e] = (int)((2 * e < have ? v[2 * e] : 0u) | (2 * e + 1 < have ? v[2 * e + 1] << 16 : 0u));
  return r;
}

// A tile's operand on its way from memory to LDS, four pieces of eight elements per thread. `line` is what the pieces of a thread lie in: rows of the
// tile (kAlongK, kStrided), which stay, or slices of what is summed over (kAcross), which a slice of 64 k moves on.
template <int MODE>
struct Operand {
  static constexpr bool KC = MODE != kAcross;
  using T = Tile<2, kEdge, KC, 256>;
  const uint16_t *line[4];
  bool there[4];
  v4i piece[4];

  // kAlongK, kStrided: rows first .. first + count - 1 of the operand, through `index` if there is one, of which `limit` exist.
  __device__ __forceinline__ void rows(const uint16_t *base, size_t pitch, const int32_t *index, unsigned limit, unsigned first, unsigned count) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned r = (threadIdx.x >> 3) + 32u * i;
      there[i] = r < count;
      unsigned at = first + (there[i] ? r : 0u);
      if (index) at = (unsigned)index[at];
      there[i] = there[i] && at < limit;
      line[i] = base + (size_t)(there[i] ? at : 0u) * pitch;
    }
  }
  __device__ __forceinline__ void load_along(unsigned k0, unsigned k, size_t step) {
    const unsigned at = k0 + (threadIdx.x & 7u) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (MODE == kAlongK && k0 + kSliceK <= k) {
        piece[i] = there[i] ? *reinterpret_cast<const v4i_at2 *>(line[i] + at) : v4i{0, 0, 0, 0};
      } else {
        piece[i] = there[i] && at < k ? load_first(line[i] + (size_t)at * step, step, k - at < 8 ? k - at : 8) : v4i{0, 0, 0, 0};
      }
    }
  }
  // kAcross: columns col0 .. of `cols`, rows first + k0 .. of `count` in all.
  __device__ __forceinline__ void load_across(const uint16_t *base, size_t pitch, const int32_t *index, unsigned limit, unsigned first, unsigned k0, unsigned count, unsigned col0, unsigned cols) {
    const unsigned col = col0 + (threadIdx.x & 15u) * 8;
    bool in[4];
    unsigned at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned r = k0 + (threadIdx.x >> 4) + 16u * i;
      in[i] = r < count && col < cols;
      at[i] = first + r;
      if (index) at[i] = in[i] ? (unsigned)index[at[i]] : 0u;
      in[i] = in[i] && at[i] < limit;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t *p = base + (size_t)at[i] * pitch + col;
      if (col0 + kEdge <= cols) piece[i] = in[i] ? *reinterpret_cast<const v4i_at2 *>(p) : v4i{0, 0, 0, 0};
      else piece[i] = in[i] ? load_first(p, 1, cols - col < 8 ? cols - col : 8) : v4i{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void store(char *tile) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (KC) *reinterpret_cast<v4i *>(tile + ((threadIdx.x >> 3) + 32 * i) * T::kPitchKC + (threadIdx.x & 7) * 16) = piece[i];
      else *reinterpret_cast<v4i *>(tile + T::mc((int)(threadIdx.x >> 4) + 16 * i, (threadIdx.x & 15) * 16)) = piece[i];
    }
  }
};

template <typename TC>
__device__ __forceinline__ void write_blocks(TC *c, size_t rsc, const v16f (&acc)[2][2], unsigned row0, unsigned col0, unsigned rows, unsigned cols, skl_scalar alpha, skl_scalar beta) {
  const unsigned lane = threadIdx.x & 63u;
  const bool read_c = !skl_beta_is_zero<float>(beta);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const unsigned row = row0 + 32u * i + 8u * (r >> 2) + 4u * (lane >> 5) + (r & 3), col = col0 + 32u * j + (lane & 31u);
        if (row < rows && col < cols) {
          TC *at = c + (size_t)row * rsc + col;
          *at = skl_grouped_result(acc[i][j][r], at, alpha, beta, read_c);
        }
      }
}

// OVER: the sums go over the groups' rows.
template <int DT, typename TC, bool OVER, int AMODE, int BMODE>
__global__ void __launch_bounds__(256) gemm_grouped_kernel(GroupedArgs p) {
  using TA = Operand<AMODE>;
  using TB = Operand<BMODE>;
  constexpr int kBytesA = TA::T::kBytes, kStage = kBytesA + TB::T::kBytes;
  extern __shared__ __attribute__((aligned(128))) char grouped_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned e, first, rows, row0;  // the group, its rows; the tile's first row of C, counted from the group's (OVER: from C_e's)
  const unsigned col0 = blockIdx.x % p.tiles_n * kEdge;
  if constexpr (OVER) {
    const unsigned t = blockIdx.x / p.tiles_n;
    e = t / p.tiles_m, row0 = t % p.tiles_m * kEdge;
    const SklRange r = skl_group_range(p.offsets, e, p.k);
    first = r.first, rows = r.rows;
  } else {
    // Tile t of the groups' tiles, group after group. Lane l counts those of groups l * each .. + each - 1.
    const unsigned lane = threadIdx.x & 63u, each = (p.groups + 63) / 64, t = blockIdx.x / p.tiles_n;
    unsigned mine = 0;
    for (unsigned g = lane * each; g < (lane + 1) * each && g < p.groups; ++g) mine += (skl_group_range(p.offsets, g, p.m).rows + kEdge - 1) / kEdge;
    const unsigned upto = skl_wave_scan(mine);
    const unsigned long long behind = __ballot(t < upto);
    if (behind == 0) return;
    const int owner = (int)__builtin_ctzll(behind);
    unsigned at = (unsigned)__builtin_amdgcn_readlane((int)(upto - mine), owner);
    e = (unsigned)owner * each;
    SklRange r = skl_group_range(p.offsets, e, p.m);
    while (t >= at + (r.rows + kEdge - 1) / kEdge) {
      at += (r.rows + kEdge - 1) / kEdge;
      r = skl_group_range(p.offsets, ++e, p.m);
    }
    first = r.first, rows = r.rows, row0 = (t - at) * kEdge;
  }
  const unsigned k = OVER ? rows : p.k;
  const uint16_t *const b = OVER ? p.b : p.b + (size_t)e * p.gsb;
  TA ta;
  TB tb;
  if constexpr (!OVER) {
    ta.rows(p.a, p.rsa, p.rows_a, p.rows_a ? p.a_rows : p.m, first + row0, rows - row0 < (unsigned)kEdge ? rows - row0 : kEdge);
    if constexpr (BMODE != kAcross) tb.rows(b, p.csb, nullptr, p.n, col0, p.n - col0 < (unsigned)kEdge ? p.n - col0 : kEdge);
  }
  const auto load = [&](unsigned k0) __attribute__((always_inline)) {
    if constexpr (OVER) {
      ta.load_across(p.a, p.rsa, p.rows_a, p.rows_a ? p.a_rows : p.k, first, k0, k, row0, p.m);
      tb.load_across(b, p.rsb, p.rows_b, p.rows_b ? p.b_rows : p.k, first, k0, k, col0, p.n);
    } else {
      ta.load_along(k0, k, 1);
      if constexpr (BMODE == kAcross) tb.load_across(b, p.rsb, nullptr, p.k, 0, k0, k, col0, p.n);
      else tb.load_along(k0, k, p.rsb);
    }
  };
  v16f acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  const int wm = wave / 2 * 64, wn = wave % 2 * 64;
  if (k) load(0);
  for (unsigned k0 = 0, s = 0; k0 < k; k0 += kSliceK, s ^= 1) {
    char *const tile_a = grouped_lds + s * kStage, *const tile_b = tile_a + kBytesA;
    ta.store(tile_a);
    tb.store(tile_b);
    __syncthreads();  // one per slice: who writes this stage again has seen every wave through the slice in between
    if (k0 + kSliceK < k) load(k0 + kSliceK);
#pragma unroll
    for (int kb = 0; kb < kSliceK * 2; kb += 32) {
      v4i x[2], y[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = read_frag<2, kEdge, TA::KC, 16>(tile_a, wm + 32 * i, kb);
#pragma unroll
      for (int j = 0; j < 2; ++j) y[j] = read_frag<2, kEdge, TB::KC, 16>(tile_b, wn + 32 * j, kb);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = Mma<DT, DT>::run(x[i], y[j], acc[i][j]);
    }
  }
  TC *const c = reinterpret_cast<TC *>(p.c) + (OVER ? (size_t)e * p.gsc : (size_t)first * p.rsc);
  write_blocks(c, p.rsc, acc, row0 + wm, col0 + wn, OVER ? p.m : rows, p.n, p.alpha, p.beta);
}

template <int DT, typename TC, bool OVER, int AMODE, int BMODE>
int launch(const GroupedArgs &p, size_t blocks) {
  constexpr int kLds = 2 * (Operand<AMODE>::T::kBytes + Operand<BMODE>::T::kBytes);
  static std::atomic<int> allowed{0};
  if (!allowed.load(std::memory_order_relaxed)) {
    const int rc = skl_check_hip(hipFuncSetAttribute(reinterpret_cast<const void *>(&gemm_grouped_kernel<DT, TC, OVER, AMODE, BMODE>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds), "gemm_grouped: LDS size");
    if (rc != 0) return rc;
    allowed.store(1, std::memory_order_relaxed);
  }
  gemm_grouped_kernel<DT, TC, OVER, AMODE, BMODE><<<dim3((unsigned)blocks), dim3(256), kLds, skl_current_stream()>>>(p);
  return skl_check_launch("gemm_grouped");
}

// Workgroups of a launch: beyond 2^32 threads the runtime takes what is left of the number in 32 bits.
constexpr size_t kMostBlocks = size_t(1) << 23;

template <int DT, typename T>
int grouped(const skl_grouped_gemm &g, GroupedArgs p) {
  const auto by_layout = [&](auto c, size_t blocks) {
    using TC = decltype(c);
    if (g.rsb == 1) return launch<DT, TC, false, kAlongK, kAlongK>(p, blocks);
    if (g.csb == 1) return launch<DT, TC, false, kAlongK, kAcross>(p, blocks);
    return launch<DT, TC, false, kAlongK, kStrided>(p, blocks);
  };
  const size_t tiles = g.m / kEdge + (g.m < g.groups ? g.m : g.groups);  // whole ones, and one more for each group that has a row
  const size_t slab = tiles < kMostBlocks ? kMostBlocks / tiles * kEdge : kEdge;
  for (size_t col = 0; col < g.n; col += slab) {
    p.n = (unsigned)(g.n - col < slab ? g.n - col : slab);
    p.tiles_n = skl_div_up(p.n, kEdge);
    p.b = (const uint16_t *)g.b + col * g.csb;
    p.c = (char *)g.c + col * (g.c_single ? 4 : 2);
    const int rc = g.c_single ? by_layout(float{}, tiles * p.tiles_n) : by_layout(T{}, tiles * p.tiles_n);
    if (rc != 0) return rc;
  }
  return 0;
}

template <int DT, typename T>
int groupedk(const skl_groupedk_gemm &g, GroupedArgs p) {
  p.tiles_m = skl_div_up(g.m, kEdge);
  const size_t all_n = skl_div_up(g.n, kEdge), left = kMostBlocks / p.tiles_m > 0 ? kMostBlocks / p.tiles_m : 1;
  const size_t slab_n = (left < all_n ? left : all_n) * kEdge, slab = left / all_n > 0 ? left / all_n : 1;
  for (size_t e = 0; e < g.groups; e += slab) {
    p.groups = (unsigned)(g.groups - e < slab ? g.groups - e : slab);
    p.offsets = g.offsets ? g.offsets + e : nullptr;
    for (size_t col = 0; col < g.n; col += slab_n) {
      p.n = (unsigned)(g.n - col < slab_n ? g.n - col : slab_n);
      p.tiles_n = skl_div_up(p.n, kEdge);
      p.b = (const uint16_t *)g.b + col;
      p.c = (char *)g.c + (e * g.gsc + col) * (g.c_single ? 4 : 2);
      const size_t blocks = (size_t)p.tiles_m * p.tiles_n * p.groups;
      const int rc = g.c_single ? launch<DT, float, true, kAcross, kAcross>(p, blocks) : launch<DT, T, true, kAcross, kAcross>(p, blocks);
      if (rc != 0) return rc;
    }
  }
  return 0;
}

}  // namespace

int skl_hip_launch_gemm_grouped(const skl_grouped_gemm *g) {
  if (skl_grouped_ring_takes(*g)) return g->dt == SKL_DT_BF16 ? skl_launch_grouped_ring_bf16(*g) : skl_launch_grouped_ring_f16(*g);
  GroupedArgs p{};
  p.a = (const uint16_t *)g->a, p.offsets = g->offsets, p.rows_a = g->rows;
  p.rsa = g->rsa, p.rsb = g->rsb, p.csb = g->csb, p.gsb = g->gsb, p.rsc = g->rsc;
  p.groups = (unsigned)g->groups, p.m = (unsigned)g->m, p.k = (unsigned)g->k, p.a_rows = (unsigned)g->a_rows;
  p.alpha = g->alpha, p.beta = g->beta;
  return g->dt == SKL_DT_BF16 ? grouped<SKL_DT_BF16, __bf16>(*g, p) : grouped<SKL_DT_F16, _Float16>(*g, p);
}

int skl_hip_launch_gemm_groupedk(const skl_groupedk_gemm *g) {
  if (skl_groupedk_ring_takes(*g)) return g->dt == SKL_DT_BF16 ? skl_launch_groupedk_ring_bf16(*g) : skl_launch_groupedk_ring_f16(*g);
  GroupedArgs p{};
  p.a = (const uint16_t *)g->a, p.rows_a = g->rows_a, p.rows_b = g->rows_b;
  p.rsa = g->rsa, p.rsb = g->rsb, p.rsc = g->rsc, p.gsc = g->gsc;
  p.m = (unsigned)g->m, p.k = (unsigned)g->total, p.a_rows = (unsigned)g->a_rows, p.b_rows = (unsigned)g->b_rows;
  p.alpha = g->alpha, p.beta = g->beta;
  return g->dt == SKL_DT_BF16 ? groupedk<SKL_DT_BF16, __bf16>(*g, p) : groupedk<SKL_DT_F16, _Float16>(*g, p);
}
