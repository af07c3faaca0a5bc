// skl_group_rows.hip - the order of picks by their groups (include/skl-gfx950.h: skl_group_rows).
//
// A counting sort that keeps the order of equals. Every wave owns a run of picks and has a row of counters in LDS; a pick's place is where its group begins, the
// picks of that group in earlier workgroups and waves, those of earlier steps of its own wave - all in the counters - and those in lower lanes of its step, which are the
// lanes that agree with it in every bit of the group's number: a ballot for each bit. No order comes from an atomic: those only count.
// Up to 2048 picks one workgroup does it in a launch; more are counted by a first launch, whose counts each workgroup of the second adds up for itself.
#include <hip/hip_runtime.h>

#include <atomic>

#include "skl_groups.hpp"
#include "../../include/skl-hip.h"

namespace {

struct GroupRowsArgs {
  const int32_t *ids;
  unsigned count, per_row, groups, bits;
  unsigned each;      // picks of a wave
  unsigned *counts;   // [workgroups][groups], from the launch before; NULL: there is one workgroup
  int32_t *offsets, *order, *rows, *place;
};

// The picks of this wave.
__device__ __forceinline__ void run_of(const GroupRowsArgs &p, unsigned wave, unsigned waves, unsigned &first, unsigned &end) {
  first = (blockIdx.x * waves + wave) * p.each;
  end = first < p.count ? (p.count - first < p.each ? p.count : first + p.each) : first;
}

__global__ void __launch_bounds__(1024) group_count_kernel(GroupRowsArgs p) {
  extern __shared__ unsigned count_lds[];
  const unsigned waves = blockDim.x / 64, lane = threadIdx.x & 63u;
  for (unsigned g = threadIdx.x; g < p.groups; g += blockDim.x) count_lds[g] = 0;
  __syncthreads();
  unsigned first, end;
  run_of(p, threadIdx.x >> 6, waves, first, end);
  for (unsigned i = first + lane; i < end; i += 64) {
    const unsigned g = (unsigned)p.ids[i];
    if (g < p.groups) atomicAdd(&count_lds[g], 1u);
  }
  __syncthreads();
  for (unsigned g = threadIdx.x; g < p.groups; g += blockDim.x) p.counts[(size_t)blockIdx.x * p.groups + g] = count_lds[g];
}

__global__ void __launch_bounds__(1024) group_rows_kernel(GroupRowsArgs p) {
  extern __shared__ unsigned rows_lds[];  // [waves][groups] next places; [groups] where a group begins; [groups] its picks in earlier workgroups
  __shared__ unsigned sums[16];
  const unsigned threads = blockDim.x, waves = threads / 64, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, groups = p.groups;
  unsigned *const next = rows_lds, *const begin = next + waves * groups, *const before = begin + groups;
  for (unsigned at = threadIdx.x; at < (waves + 2) * groups; at += threads) next[at] = 0;
  unsigned first, end;
  run_of(p, wave, waves, first, end);
  // The first two steps' picks, looked at again below.
  const unsigned held = first + lane < end ? (unsigned)p.ids[first + lane] : ~0u, held_next = first + 64 + lane < end ? (unsigned)p.ids[first + 64 + lane] : ~0u;
  __syncthreads();
  if (p.counts) {  // a thread per group and part of the workgroups, eight counts under way at a time
    const unsigned parts = threads / groups > 0 ? threads / groups : 1;
    for (unsigned at = threadIdx.x; at < parts * groups; at += threads) {
      const unsigned g = at % groups;
      unsigned all = 0, lower = 0;
#pragma unroll 8
      for (unsigned b = at / groups; b < gridDim.x; b += parts) {
        const unsigned c = p.counts[(size_t)b * groups + g];
        all += c;
        lower += b < blockIdx.x ? c : 0u;
      }
      atomicAdd(&begin[g], all);
      atomicAdd(&before[g], lower);
    }
  }
  unsigned *const mine = next + wave * groups;
  const auto pick = [&](unsigned i0) { return i0 < end && end - i0 > lane ? (unsigned)p.ids[i0 + lane] : ~0u; };
  unsigned chosen = held, chosen_next = held_next;  // two steps ahead
  for (unsigned i0 = first; i0 < end; i0 += 64) {
    const unsigned after = pick(i0 + 128);
    if (chosen < groups) atomicAdd(&mine[chosen], 1u);
    chosen = chosen_next, chosen_next = after;
  }
  __syncthreads();
  // Thread t: groups t * per .. + per - 1.
  const unsigned per = (groups + threads - 1) / threads, g0 = threadIdx.x * per, g1 = g0 + per < groups ? g0 + per : groups;
  unsigned sum = 0;
  for (unsigned g = g0; g < g1; ++g) {
    if (!p.counts) {
      unsigned all = 0;
      for (unsigned w = 0; w < waves; ++w) all += next[w * groups + g];
      begin[g] = all;
    }
    sum += begin[g];
  }
  const unsigned upto = skl_wave_scan(sum);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  unsigned at = upto - sum;
  for (unsigned w = 0; w < wave; ++w) at += sums[w];
  for (unsigned g = g0; g < g1; ++g) {
    const unsigned all = begin[g];
    if (blockIdx.x == 0) p.offsets[g] = (int)at;
    unsigned to = at + before[g];
    for (unsigned w = 0; w < waves; w += 4) {  // (4 or 16 of them: four reads at a time)
      unsigned *const four = next + w * groups + g;
      const unsigned c0 = four[0], c1 = four[groups], c2 = four[2 * groups], c3 = four[3 * groups];
      four[0] = to, four[groups] = to + c0, four[2 * groups] = to + c0 + c1, four[3 * groups] = to + c0 + c1 + c2;
      to += c0 + c1 + c2 + c3;
    }
    at += all;
  }
  if (blockIdx.x == 0 && g1 == groups && g0 < groups) p.offsets[groups] = (int)at;
  __syncthreads();
  chosen = held, chosen_next = held_next;
  for (unsigned i0 = first; i0 < end; i0 += 64) {
    const unsigned i = i0 + lane, after = pick(i0 + 128);
    const bool in = chosen < groups;
    unsigned long long same = __ballot(in);
    for (unsigned b = 0; b < p.bits; ++b) {
      const bool set = (chosen >> b) & 1u;
      const unsigned long long of_bit = __ballot(set);
      same &= set ? of_bit : ~of_bit;
    }
    const unsigned lower = __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0u));
    unsigned to = 0;
    if (in) {
      volatile unsigned *const here = &mine[chosen];  // other lanes write it
      to = *here + lower;
      if (p.order && to < p.count) p.order[to] = (int)i;  // (true unless somebody else writes into this stream's scratch memory meanwhile)
      if (p.rows && to < p.count) p.rows[to] = (int)(i / p.per_row);
      if (lower + 1 == (unsigned)__popcll(same)) *here = to + 1;  // the last of them; a wave's accesses are in order
    }
    if (p.place && i < end) p.place[i] = in ? (int)to : -1;
    chosen = chosen_next, chosen_next = after;
  }
}

}  // namespace

int skl_hip_launch_group_rows(size_t count, const int32_t *ids, size_t per_row, size_t groups, int32_t *offsets, int32_t *order, int32_t *rows,
                              int32_t *place) {
  GroupRowsArgs p{};
  p.ids = ids, p.count = (unsigned)count, p.groups = (unsigned)groups;
  p.per_row = per_row > 0xFFFFFFFFu ? 0xFFFFFFFFu : per_row ? (unsigned)per_row : 1u;  // (more than there are picks: one row)
  p.offsets = offsets, p.order = order, p.rows = rows, p.place = place;
  while ((size_t(1) << p.bits) < groups) ++p.bits;
  const unsigned waves = groups <= 2048 ? 16 : 4;  // their counters fit LDS
  const unsigned lds = (waves + 2) * p.groups * 4;
  // Workgroups: a launch costs about 2 us, one workgroup 1 us for 1000 picks. What each goes through, its picks and everybody's counts, is least with sqrt(8 count / groups) of them (measured: of
  // 131072 picks 128 / 64 / 32 workgroups with 64 groups 8.9 / 8.7 / 10.8 us, with 256 16 / 12.9 / 13.7; 32 / 16 / 8 with 2048 34 / 33 / 43); of fewer than 1024 picks each nothing is won.
  size_t blocks = 1;
  if (count > 2048) {
    while (blocks < 256 && (blocks + 1) * (blocks + 1) * groups <= 8 * count) ++blocks;
    if (blocks > (count + 1023) / 1024) blocks = (count + 1023) / 1024;
  }
  const bool sequence = blocks > 1;
  if (sequence) {
    skl_hip_sequence_begin();
    p.counts = (unsigned *)skl_workspace(blocks * groups * 4, true);
    if (!p.counts) blocks = 1;  // no scratch memory: the same result from one workgroup
  }
  p.each = (skl_div_up(count, blocks * waves) + 63) / 64 * 64;
  int rc = 0;
  if (p.counts) {
    group_count_kernel<<<dim3((unsigned)blocks), dim3(waves * 64), groups * 4, skl_current_stream()>>>(p);
    rc = skl_check_launch("group_rows: counts");
  }
  static std::atomic<unsigned long long> allowed{0};
  if (rc == 0) rc = skl_allow_lds(reinterpret_cast<const void *>(&group_rows_kernel), 18 * 2048 * 4, allowed);
  if (rc == 0) {
    group_rows_kernel<<<dim3((unsigned)blocks), dim3(waves * 64), lds, skl_current_stream()>>>(p);
    rc = skl_check_launch("group_rows");
  }
  if (sequence) skl_hip_sequence_end();
  return rc;
}
