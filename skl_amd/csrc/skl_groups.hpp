// skl_groups.hpp - what the kernels of the products grouped by expert share: which tile of which group a workgroup takes, elements of
// 16 bits, and the last step of a result (not installed).
#pragma once

#include <atomic>

#include "skl_device.hpp"
#include "skl_grouped.h"
#include "../../include/skl-hip.h"

// The streaming kernels (skl_grouped_ring.hpp), and what they take: operands and the distances of their lines on 16-byte boundaries, whole 16 bytes of what lies
// side by side along k, offsets in 32 bits.
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

// Which tile of which group a workgroup takes. `whole` tiles of MOST rows come first, group after group, then one for what is left of each group; both are dealt out to the
// eight dies in runs, so that a die's workgroups share operands. Lane l counts for groups l * each .. + each - 1.
struct GroupedPlace {
  unsigned e, first, rows, tile_n;  // rows first .. first + rows - 1 of A and C
  bool none;
};
template <int MOST>
__device__ __forceinline__ GroupedPlace grouped_place(const int32_t *offsets, unsigned groups, unsigned m, unsigned tiles_n, unsigned id) {
  const unsigned lane = threadIdx.x & 63u, each = (groups + 63) / 64, g0 = lane * each;
  unsigned whole = 0, rest = 0;
  SklRange mine_last{0, 0};  // with one group to a lane, the lane's
  for (unsigned g = g0; g < g0 + each && g < groups; ++g) {
    mine_last = skl_group_range(offsets, g, m);
    whole += mine_last.rows / MOST, rest += mine_last.rows % MOST != 0;
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
    lines = is_whole ? r.rows / MOST : r.rows % MOST != 0;
  } else {
    for (;; ++e) {
      r = skl_group_range(offsets, e, m);
      lines = is_whole ? r.rows / MOST : r.rows % MOST != 0;
      if (line < before + lines || e + 1 >= groups) break;
      before += lines;
    }
  }
  at.e = e;
  if (is_whole) {  // up to eight lines of a group column by column
    const unsigned in = t - before * tiles_n, block = in / (8 * tiles_n), in_block = in - block * (8 * tiles_n), deep = lines - 8 * block < 8 ? lines - 8 * block : 8;
    at.tile_n = in_block / deep;
    at.first = r.first + (8 * block + in_block % deep) * MOST;
    at.rows = MOST;
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

// The other order, of tiles of 256 rows and what is left as smaller ones: a group's tiles together, up to eight lines at a time column by column, so that B comes once for all of them.
// Each die's run is as long by what its tiles cost as the grid's `slots` for a die let it be. Its last tiles may be large ones: for many tiles (grouped_rows_by_size).
__device__ __forceinline__ GroupedPlace grouped_place_by_group(const int32_t *offsets, unsigned groups, unsigned m, unsigned tiles_n, unsigned id, unsigned slots) {
  constexpr unsigned MOST = 256;
  const auto lines_of = [](unsigned rows) { return (rows + MOST - 1) / MOST; };
  const unsigned lane = threadIdx.x & 63u, each = (groups + 63) / 64, g0 = lane * each;
  unsigned count = 0, cost = 0;
  SklRange last{0, 0};  // with one group to a lane, the lane's
  for (unsigned g = g0; g < g0 + each && g < groups; ++g) {
    last = skl_group_range(offsets, g, m);
    count += lines_of(last.rows);
    const unsigned rest = last.rows % MOST;
    cost += last.rows / MOST * 8 + (rest > 128 ? 8 : rest > 64 ? 5 : rest > 0 ? 4 : 0);
  }
  const unsigned upto = skl_wave_scan(count), all = (unsigned)__builtin_amdgcn_readlane((int)upto, 63) * tiles_n;
  const unsigned die = id % 8, slot = id / 8;
  const unsigned cost_upto = skl_wave_scan(cost), whole_cost = (unsigned)__builtin_amdgcn_readlane((int)cost_upto, 63);
  unsigned first = 0, end = 0;  // this die's run
  for (unsigned d = 0; d <= die; ++d) {
    first = end;
    // In the lane where d + 1 eighths of the cost are reached, as far into its tiles as into its cost; the dies behind have to hold the others.
    const float reached = (float)whole_cost * (float)(d + 1) * 0.125f;
    const unsigned long long behind = __ballot((float)cost_upto > reached);
    end = all;
    if (behind && d < 7) {
      const int at = (int)__builtin_ctzll(behind);
      const float ahead = (float)__builtin_amdgcn_readlane((int)(cost_upto - cost), at), mine = (float)__builtin_amdgcn_readlane((int)cost, at);
      const unsigned lines = (unsigned)__builtin_amdgcn_readlane((int)count, at), before = (unsigned)__builtin_amdgcn_readlane((int)(upto - count), at);
      const float part = (reached - ahead) / mine * (float)(lines * tiles_n);
      end = before * tiles_n + (part > 0 ? (unsigned)part : 0u);
    }
    const unsigned behind_hold = (7 - d) * slots;
    end = end < first ? first : end - first > slots ? first + slots : end;
    if (all > behind_hold && end < all - behind_hold) end = all - behind_hold;
  }
  const unsigned t = first + slot, line = t / tiles_n;  // line: row of tiles
  GroupedPlace at{0, 0, 0, 0, t >= end};
  if (at.none) return at;
  const unsigned long long behind = __ballot(line < upto);
  at.none = behind == 0;  // (sums beyond 32 bits, of offsets that fall back)
  if (at.none) return at;
  const int owner = (int)__builtin_ctzll(behind);
  unsigned before = (unsigned)__builtin_amdgcn_readlane((int)(upto - count), owner);  // lines of the groups ahead
  unsigned e = (unsigned)owner * each;
  SklRange r;
  unsigned lines;
  if (each == 1) {  // (what the lane holds: no second trip to memory)
    r = {(unsigned)__builtin_amdgcn_readlane((int)last.first, owner), (unsigned)__builtin_amdgcn_readlane((int)last.rows, owner)};
    lines = lines_of(r.rows);
  } else {
    for (;; ++e) {
      r = skl_group_range(offsets, e, m);
      lines = lines_of(r.rows);
      if (line < before + lines || e + 1 >= groups) break;
      before += lines;
    }
  }
  at.none = line - before >= lines;
  if (at.none) return at;
  const unsigned in = t - before * tiles_n, block = in / (8 * tiles_n), in_block = in - block * (8 * tiles_n), deep = lines - 8 * block < 8 ? lines - 8 * block : 8;
  const unsigned in_group = (8 * block + in_block % deep) * MOST;
  at.e = e, at.tile_n = in_block / deep, at.first = r.first + in_group, at.rows = r.rows - in_group < MOST ? r.rows - in_group : MOST;
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
