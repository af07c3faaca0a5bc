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

// An operand's unit stride: along what is summed over, across it, none. kAcrossFew: across, fewer than eight values.
enum { kAlongK, kAcross, kAcrossFew, kStrided };

typedef v4i v4i_at2 __attribute__((aligned(2)));

constexpr int kEdge = 128, kSliceK = 64;

// 8 elements from p, `step` apart, of which the first `have` exist (at least one): the others are zeros.
__device__ __forceinline__ v4i load_first(const uint16_t *p, size_t step, unsigned have) {
  unsigned v[8];
#pragma unroll
  for (unsigned e = 0; e < 8; ++e) v[e] = p[(e < have ? e : have - 1) * step];
  v4i r;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) r[e] = (int)((2 * e < have ? v[2 * e] : 0u) | (2 * e + 1 < have ? v[2 * e + 1] << 16 : 0u));
  return r;
}

// A tile's operand on its way from memory to LDS, two slices of 64 k ahead: four pieces of eight elements per thread and slice. What a thread's pieces lie in is rows of the
// tile (kAlongK, kStrided), which stay, or slices of what is summed over. Whole slices are loaded without a branch, at whose end everything under way is waited for (with one, 1001 tokens
// 3 of 20, 2077 to 1443, took 91 us): a row that does not exist is one that does, with zeros in its place on the way to LDS, and at the edge of the columns a piece is loaded from further down
// and moved into place there. Pieces begin on any element: 16 bytes from between two dwords load as fast as from a dword on to within a tenth (from the dword on that holds the first element, with
// the dword that holds the last, and moved into place, half as fast).
template <int MODE>
struct Operand {
  static constexpr bool KC = MODE == kAlongK || MODE == kStrided;
  using T = Tile<2, kEdge, KC, 256>;
  struct Piece {
    v4i v;
    bool in;
  };
  const uint16_t *line[4];
  bool there[4];
  unsigned shift;  // kAcross: elements that this thread's pieces are loaded further down

  // kAlongK, kStrided: rows first .. first + count - 1 of the operand (count > 0), through `index` if there is one, of which `limit` exist (one at least).
  __device__ __forceinline__ void rows(const uint16_t *base, size_t pitch, const int32_t *index, unsigned limit, unsigned first, unsigned count) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned r = (threadIdx.x >> 3) + 32u * i;
      unsigned at = first + (r < count ? r : 0u);
      if (index) at = (unsigned)index[at];
      there[i] = at < limit;
      line[i] = base + (size_t)(there[i] ? at : 0u) * pitch;
    }
  }
  // TAIL: the last, partial slice.
  template <bool TAIL>
  __device__ __forceinline__ void load_along(Piece (&to)[4], unsigned k0, unsigned k, size_t step) const {
    const unsigned at = k0 + (threadIdx.x & 7u) * 8;
    const bool some = !TAIL || at < k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (MODE == kAlongK && !TAIL) {
        to[i].v = *reinterpret_cast<const v4i_at2 *>(line[i] + at);
      } else {
        to[i].v = load_first(line[i] + (size_t)(some ? at : k - 1) * step, step, !TAIL || (some && k - at >= 8) ? 8 : some ? k - at : 1);
      }
      to[i].in = there[i] && some;
    }
  }
  // kAcross, kAcrossFew: columns col0 .. of `cols`, rows first + k0 .. of `count` in all (count > 0).
  template <bool TAIL>
  __device__ __forceinline__ void load_across(Piece (&to)[4], const uint16_t *base, size_t pitch, const int32_t *index, unsigned limit, unsigned first, unsigned k0, unsigned count, unsigned col0, unsigned cols) {
    const unsigned col = col0 + (threadIdx.x & 15u) * 8;
    shift = MODE == kAcross && col + 8 > cols ? col + 8 - cols : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned r = k0 + (threadIdx.x >> 4) + 16u * i;
      unsigned at = first + (!TAIL || r < count ? r : count - 1);
      if (index) at = (unsigned)index[at];
      to[i].in = (!TAIL || r < count) && at < limit && col < cols;
      const uint16_t *const row = base + (size_t)(at < limit ? at : 0u) * pitch;
      if constexpr (MODE == kAcross) {
        to[i].v = *reinterpret_cast<const v4i_at2 *>(row + (col - shift));
      } else {
        to[i].v = load_first(row + (col < cols ? col : 0u), 1, col < cols ? cols - col : 1);
      }
    }
  }
  __device__ __forceinline__ void store(const Piece (&from)[4], char *tile, bool edge) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4i v = from[i].v;
      if (MODE == kAcross && edge) v = __builtin_bit_cast(v4i, shift < 8 ? __builtin_bit_cast(unsigned __int128, v) >> (16 * shift) : (unsigned __int128)0);
      if (!from[i].in) v = v4i{0, 0, 0, 0};
      if constexpr (KC) *reinterpret_cast<v4i *>(tile + ((threadIdx.x >> 3) + 32 * i) * T::kPitchKC + (threadIdx.x & 7) * 16) = v;
      else *reinterpret_cast<v4i *>(tile + T::mc((int)(threadIdx.x >> 4) + 16 * i, (threadIdx.x & 15) * 16)) = v;
    }
  }
};

// A wave's 128 x 32 values of C: four blocks of 32 x 32.
template <typename TC>
__device__ __forceinline__ void write_blocks(TC *c, size_t rsc, const v16f (&acc)[4], unsigned col, unsigned rows, unsigned cols, skl_scalar alpha, skl_scalar beta) {
  const unsigned lane = threadIdx.x & 63u;
  const bool read_c = !skl_beta_is_zero<float>(beta);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const unsigned row = 32u * i + 8u * (r >> 2) + 4u * (lane >> 5) + (r & 3);
      if (row < rows && col < cols) {
        TC *at = c + (size_t)row * rsc + col;
        *at = skl_grouped_result(acc[i][r], at, alpha, beta, read_c);
      }
    }
}

// OVER: the sums go over the groups' rows.
template <int DT, typename TC, bool OVER, int AMODE, int BMODE>
__global__ void __launch_bounds__(256, 2) gemm_grouped_kernel(GroupedArgs p) {
  using TA = Operand<AMODE>;
  using TB = Operand<BMODE>;
  constexpr int kBytesA = TA::T::kBytes, kStage = kBytesA + TB::T::kBytes;
  extern __shared__ __attribute__((aligned(128))) char grouped_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned e, first, rows, row0 = 0, col0;  // the group, its rows (not OVER: the tile's); the tile's first row of C_e (OVER) and column
  if constexpr (OVER) {
    const unsigned t = blockIdx.x / p.tiles_n;
    e = t / p.tiles_m, row0 = t % p.tiles_m * kEdge, col0 = blockIdx.x % p.tiles_n * kEdge;
    const SklRange r = skl_group_range(p.offsets, e, p.k);
    first = r.first, rows = r.rows;
  } else {
    const GroupedPlace at = grouped_place<kEdge>(p.offsets, p.groups, p.m, p.tiles_n, blockIdx.x);
    if (at.none) return;
    e = at.e, first = at.first, rows = at.rows, col0 = at.tile_n * kEdge;
  }
  const unsigned k = OVER ? rows : p.k;
  const uint16_t *const b = OVER ? p.b : p.b + (size_t)e * p.gsb;
  TA ta;
  TB tb;
  if constexpr (!OVER) {
    ta.rows(p.a, p.rsa, p.rows_a, p.rows_a ? p.a_rows : p.m, first, rows);
    if constexpr (TB::KC) tb.rows(b, p.csb, nullptr, p.n, col0, p.n - col0 < (unsigned)kEdge ? p.n - col0 : kEdge);
  }
  typename TA::Piece pa[2][4];
  typename TB::Piece pb[2][4];
  const auto load = [&](auto tail, typename TA::Piece (&to_a)[4], typename TB::Piece (&to_b)[4], unsigned k0) __attribute__((always_inline)) {
    constexpr bool TAIL = decltype(tail)::value;
    if constexpr (OVER) {
      ta.template load_across<TAIL>(to_a, p.a, p.rsa, p.rows_a, p.rows_a ? p.a_rows : p.k, first, k0, k, row0, p.m);
      tb.template load_across<TAIL>(to_b, b, p.rsb, p.rows_b, p.rows_b ? p.b_rows : p.k, first, k0, k, col0, p.n);
    } else {
      ta.template load_along<TAIL>(to_a, k0, k, 1);
      if constexpr (!TB::KC) tb.template load_across<TAIL>(to_b, b, p.rsb, nullptr, p.k, 0, k0, k, col0, p.n);
      else tb.template load_along<TAIL>(to_b, k0, k, p.rsb);
    }
  };
  v16f acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
  const unsigned c_rows = OVER ? p.m - row0 : rows;  // blocks of rows beyond are not multiplied: a group's last tile costs what it has
  const bool edge_a = row0 + kEdge > p.m, edge_b = col0 + kEdge > p.n;
  // One barrier per slice: who writes a stage again has seen every wave through the slice in between.
  const auto put = [&](int s, const typename TA::Piece (&from_a)[4], const typename TB::Piece (&from_b)[4]) __attribute__((always_inline)) {
    char *const tile_a = grouped_lds + s * kStage;
    ta.store(from_a, tile_a, edge_a);
    tb.store(from_b, tile_a + kBytesA, edge_b);
    __syncthreads();
  };
  // BLOCKS: of 32 rows. A group's last tile, of up to 64 rows, costs two.
  const auto sum = [&](auto blocks) __attribute__((always_inline)) {
    constexpr int BLOCKS = decltype(blocks)::value;
    const auto multiply = [&](int s) __attribute__((always_inline)) {
      const char *const tile_a = grouped_lds + s * kStage, *const tile_b = tile_a + kBytesA;
#pragma unroll
      for (int kb = 0; kb < kSliceK * 2; kb += 32) {
        const v4i y = read_frag<2, kEdge, TB::KC, 16>(tile_b, 32 * wave, kb);
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i) acc[i] = Mma<DT, DT>::run(read_frag<2, kEdge, TA::KC, 16>(tile_a, 32 * i, kb), y, acc[i]);
      }
    };
    const unsigned whole = k / kSliceK;
    if (whole != 0) {
      // Two slices a trip and nothing decided in between; what is loaded behind the last one is that again.
      const auto ahead = [&](unsigned s) { return (s < whole ? s : whole - 1) * kSliceK; };
      load(std::false_type{}, pa[0], pb[0], 0);
      load(std::false_type{}, pa[1], pb[1], ahead(1));
      for (unsigned s0 = 0; s0 + 2 <= whole; s0 += 2) {
        put(0, pa[0], pb[0]);
        load(std::false_type{}, pa[0], pb[0], ahead(s0 + 2));
        __builtin_amdgcn_sched_barrier(0);  // the loads ahead of the products, and the other slice's, still under way, behind them
        multiply(0);
        __builtin_amdgcn_sched_barrier(0);
        put(1, pa[1], pb[1]);
        load(std::false_type{}, pa[1], pb[1], ahead(s0 + 3));
        __builtin_amdgcn_sched_barrier(0);
        multiply(1);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (whole % 2) {
        put(0, pa[0], pb[0]);
        multiply(0);
      }
    }
    if (k % kSliceK != 0) {
      load(std::true_type{}, pa[0], pb[0], whole * kSliceK);
      put(whole % 2, pa[0], pb[0]);
      multiply(whole % 2);
    }
  };
  if (c_rows > 64) sum(std::integral_constant<int, 4>{});
  else sum(std::integral_constant<int, 2>{});
  TC *const c = reinterpret_cast<TC *>(p.c) + (OVER ? (size_t)e * p.gsc + (size_t)row0 * p.rsc : (size_t)first * p.rsc);
  write_blocks(c, p.rsc, acc, col0 + 32 * wave + (threadIdx.x & 31u), c_rows, p.n, p.alpha, p.beta);
}

template <int DT, typename TC, bool OVER, int AMODE, int BMODE>
int launch(const GroupedArgs &p, size_t blocks) {
  constexpr int kLds = 2 * (Operand<AMODE>::T::kBytes + Operand<BMODE>::T::kBytes);
  static std::atomic<unsigned long long> allowed{0};
  const int rc = skl_allow_lds(reinterpret_cast<const void *>(&gemm_grouped_kernel<DT, TC, OVER, AMODE, BMODE>), kLds, allowed);
  if (rc != 0) return rc;
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
    if (g.csb == 1 && p.n >= 8) return launch<DT, TC, false, kAlongK, kAcross>(p, blocks);
    return launch<DT, TC, false, kAlongK, kStrided>(p, blocks);
  };
  const size_t tiles = g.m / kEdge + (g.m < g.groups ? g.m : g.groups);  // whole ones, and one more for each group that has a row
  static_assert(kEdge >= 8);  // a slab of columns but the last has eight
  const size_t slab = tiles + 16 < kMostBlocks ? kMostBlocks / (tiles + 16) * kEdge : kEdge;
  for (size_t col = 0; col < g.n; col += slab) {
    p.n = (unsigned)(g.n - col < slab ? g.n - col : slab);
    p.tiles_n = skl_div_up(p.n, kEdge);
    p.b = (const uint16_t *)g.b + col * g.csb;
    p.c = (char *)g.c + col * (g.c_single ? 4 : 2);
    const size_t blocks = (tiles * p.tiles_n / 8 + 2) * 8;
    const int rc = g.c_single ? by_layout(float{}, blocks) : by_layout(T{}, blocks);
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
      const auto by_layout = [&](auto c) {
        using TC = decltype(c);
        if (g.m < 8 || p.n < 8) return launch<DT, TC, true, kAcrossFew, kAcrossFew>(p, blocks);
        return launch<DT, TC, true, kAcross, kAcross>(p, blocks);
      };
      const int rc = g.c_single ? by_layout(float{}) : by_layout(T{});
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
