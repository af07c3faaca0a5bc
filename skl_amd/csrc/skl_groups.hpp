// skl_groups.hpp - what the kernels of the products grouped by expert share: which tile of which group a workgroup takes, elements of
// 16 bits, and the last step of a result (not installed).
#pragma once

#include <atomic>

#include "skl_device.hpp"
#include "skl_grouped.h"
#include "../../include/skl-hip.h"

// The streaming kernels (skl_grouped_ring.hpp), and what they take: operands and the distances of their lines on 16-byte boundaries, whole 16 bytes of what lies
// side by side along k, offsets in 32 bits. Across k they read whole 16 bytes, too, of which those behind an operand's last column go nowhere.
int skl_launch_grouped_ring_bf16(const skl_grouped_gemm &g);
int skl_launch_grouped_ring_f16(const skl_grouped_gemm &g);
int skl_launch_groupedk_ring_bf16(const skl_groupedk_gemm &g);
int skl_launch_groupedk_ring_f16(const skl_groupedk_gemm &g);
constexpr size_t kGroupedReach = 0xC0000000u;  // bytes that an offset covers
static inline bool skl_grouped_aligned(const void *p, size_t distance) { return ((uintptr_t)p & 15) == 0 && distance % 8 == 0 && distance < kGroupedReach / 1024; }
static inline bool skl_grouped_ring_takes(const skl_grouped_gemm &g) {
  const bool kc = g.rsb == 1;
  return (kc || g.csb == 1) && g.k % 8 == 0 && g.k != 0 && skl_grouped_aligned(g.a, g.rsa) && skl_grouped_aligned(g.b, kc ? g.csb : g.rsb) && (g.groups == 1 || g.gsb % 8 == 0) &&
         (!g.rows || (g.a_rows * g.rsa + g.k) * 2 < kGroupedReach);
}
static inline bool skl_groupedk_ring_takes(const skl_groupedk_gemm &g) {
  return skl_grouped_aligned(g.a, g.rsa) && skl_grouped_aligned(g.b, g.rsb) && (!g.rows_a || (g.a_rows * g.rsa + g.m) * 2 < kGroupedReach) && (!g.rows_b || (g.b_rows * g.rsb + g.n) * 2 < kGroupedReach);
}

namespace {

// Lets `kernel` have `bytes` of LDS on the current device, once on each: `devices` has a bit for those where it may. (Racing threads ask for the same.)
inline int skl_allow_lds(const void *kernel, unsigned bytes, std::atomic<unsigned long long> &devices) {
  int device = 0;
  int rc = skl_check_hip(hipGetDevice(&device), "hipGetDevice");
  const unsigned long long bit = device < 64 ? 1ull << device : 0;
  if (rc != 0 || (devices.load(std::memory_order_relaxed) & bit)) return rc;
  rc = skl_check_hip(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "products grouped by expert: LDS size");
  if (rc == 0) devices.fetch_or(bit, std::memory_order_relaxed);
  return rc;
}

// Inclusive sum over the lanes of a wave up to this one.
__device__ __forceinline__ unsigned skl_wave_scan(unsigned v) {
#define SKL_SCAN_STEP(CTRL, ROWS) v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false)
  SKL_SCAN_STEP(0x111, 0xf);  // from 1, 2, 4 and 8 lanes below in the row of 16
  SKL_SCAN_STEP(0x112, 0xf);
  SKL_SCAN_STEP(0x114, 0xf);
  SKL_SCAN_STEP(0x118, 0xf);
  SKL_SCAN_STEP(0x142, 0xa);  // the row's last lane to the next row
  SKL_SCAN_STEP(0x143, 0xc);  // the lower half's last lane to the upper half
#undef SKL_SCAN_STEP
  return v;
}

// Rows first .. first + rows - 1 of a list of groups: group e's, cut off at 0 and `most`.
struct SklRange {
  unsigned first, rows;
};
__device__ __forceinline__ unsigned skl_cut(int at, unsigned most) { return at < 0 ? 0u : (unsigned)at < most ? (unsigned)at : most; }
__device__ __forceinline__ SklRange skl_group_range(const int32_t *offsets, unsigned e, unsigned most) {
  if (!offsets) return {0, most};
  const unsigned b = skl_cut(offsets[e], most), f = skl_cut(offsets[e + 1], most);
  return {b, f > b ? f - b : 0u};
}

// Which tile of which group a workgroup takes. A group's rows are lines of MOST; the last one, if it is a small tile - for MOST == 256 of up to 128 rows -, comes behind everybody's others, so that
// what ends last ends soon. Both kinds go group after group, up to eight lines of a group column by column so that a column of B serves them together, and are dealt out to the eight dies in runs, so that a die's
// workgroups share operands. (Last lines of more than 128 rows behind the whole ones, too, read B once more: 8 groups of 14336 x 4096 with 8192 rows 926 us against 870, 64 of 2048 x 1408 with 32768
// 270 against 250; all of a group's lines together and the dies' runs cut by cost 869 and 259, of 4096 x 4096 16 groups with 32768 rows 940 against 900.) Lane l counts for groups
// l * each .. + each - 1.
struct GroupedPlace {
  unsigned e, first, rows, tile_n;  // rows first .. first + rows - 1 of A and C
  bool none;
};
template <int MOST>
__device__ __forceinline__ GroupedPlace grouped_place(const int32_t *offsets, unsigned groups, unsigned m, unsigned tiles_n, unsigned id) {
  // Lines of tiles of (nearly) MOST rows, and whether a smaller one is left.
  constexpr unsigned kSmall = MOST == 256 ? 128 : MOST - 1;
  const auto whole_of = [](unsigned rows) { return rows / MOST + (rows % MOST > kSmall); };
  const auto rest_of = [](unsigned rows) { return (unsigned)(rows % MOST != 0 && rows % MOST <= kSmall); };
  const unsigned lane = threadIdx.x & 63u, each = (groups + 63) / 64, g0 = lane * each;
  unsigned whole = 0, rest = 0;
  SklRange mine_last{0, 0};  // with one group to a lane, the lane's
  for (unsigned g = g0; g < g0 + each && g < groups; ++g) {
    mine_last = skl_group_range(offsets, g, m);
    whole += whole_of(mine_last.rows), rest += rest_of(mine_last.rows);
  }
  const unsigned whole_upto = skl_wave_scan(whole), rest_upto = skl_wave_scan(rest);
  const unsigned all_whole = (unsigned)__builtin_amdgcn_readlane((int)whole_upto, 63) * tiles_n, all_rest = (unsigned)__builtin_amdgcn_readlane((int)rest_upto, 63) * tiles_n;
  // This die's share of both, one after the other.
  const unsigned die = id % 8, slot = id / 8;
  const unsigned whole_first = all_whole / 8 * die + (die < all_whole % 8 ? die : all_whole % 8), whole_mine = all_whole / 8 + (die < all_whole % 8);
  const unsigned rest_first = all_rest / 8 * die + (die < all_rest % 8 ? die : all_rest % 8), rest_mine = all_rest / 8 + (die < all_rest % 8);
  GroupedPlace at{0, 0, 0, 0, slot >= whole_mine + rest_mine};
  if (at.none) return at;
  const bool is_whole = slot < whole_mine;
  const unsigned t = is_whole ? whole_first + slot : rest_first + slot - whole_mine, line = t / tiles_n;  // line: row of tiles
  const unsigned upto = is_whole ? whole_upto : rest_upto, mine = is_whole ? whole : rest;
  const unsigned long long behind = __ballot(line < upto);
  at.none = behind == 0;  // (sums beyond 32 bits, of offsets that fall back)
  if (at.none) return at;
  const int owner = (int)__builtin_ctzll(behind);
  unsigned before = (unsigned)__builtin_amdgcn_readlane((int)(upto - mine), owner);  // lines of the groups ahead
  unsigned e = (unsigned)owner * each;
  SklRange r;
  unsigned lines;
  if (each == 1) {  // (what the lane holds: no second trip to memory)
    r = {(unsigned)__builtin_amdgcn_readlane((int)mine_last.first, owner), (unsigned)__builtin_amdgcn_readlane((int)mine_last.rows, owner)};
    lines = is_whole ? whole_of(r.rows) : rest_of(r.rows);
  } else {
    for (;; ++e) {
      r = skl_group_range(offsets, e, m);
      lines = is_whole ? whole_of(r.rows) : rest_of(r.rows);
      if (line < before + lines || e + 1 >= groups) break;
      before += lines;
    }
  }
  at.e = e;
  if (is_whole) {  // up to eight lines of a group column by column
    const unsigned in = t - before * tiles_n, block = in / (8 * tiles_n), in_block = in - block * (8 * tiles_n), deep = lines - 8 * block < 8 ? lines - 8 * block : 8;
    at.tile_n = in_block / deep;
    at.first = r.first + (8 * block + in_block % deep) * MOST;
    at.rows = r.rows - (at.first - r.first) < MOST ? r.rows - (at.first - r.first) : MOST;
  } else {
    at.tile_n = t % tiles_n;
    at.first = r.first + r.rows / MOST * MOST;
    at.rows = r.rows % MOST;
  }
  // uniform, and the compiler is told: branches and descriptors go by them
  at.e = (unsigned)__builtin_amdgcn_readfirstlane((int)at.e), at.first = (unsigned)__builtin_amdgcn_readfirstlane((int)at.first);
  at.rows = (unsigned)__builtin_amdgcn_readfirstlane((int)at.rows), at.tile_n = (unsigned)__builtin_amdgcn_readfirstlane((int)at.tile_n);
  return at;
}

__device__ __forceinline__ float skl_widen(uint16_t v, bool bf16) { return bf16 ? __uint_as_float((unsigned)v << 16) : (float)__builtin_bit_cast(_Float16, v); }

// The result for one element of C: TC is float, __bf16 or _Float16; a 16-bit C is widened, combined in fp32 and rounded once, to the nearest.
template <typename TC>
__device__ __forceinline__ TC skl_grouped_result(float acc, const TC *c, skl_scalar alpha, skl_scalar beta, bool read_c) {
  return (TC)(read_c ? skl_combine(acc, (float)*c, alpha, beta) : skl_initialise_plain(acc, alpha, beta));
}

}  // namespace
