// skl_group_rows.hip - the order of picks by their groups (include/skl-gfx950.h: skl_group_rows).
#include <hip/hip_runtime.h>

#include "skl_groups.hpp"
#include "../../include/skl-hip.h"

namespace {

struct GroupRowsArgs {
  const int32_t *ids;
  unsigned count, per_row, groups;
  int32_t *offsets, *order, *rows, *place;
};

// One workgroup: counts, their sums, then the picks in turn, 1024 at a time, each behind those of its group before it.
__global__ void __launch_bounds__(1024) group_rows_kernel(GroupRowsArgs p) {
  __shared__ unsigned next[SKL_MAX_GROUPS];  // where the next pick of a group goes
  __shared__ unsigned carried, total[16];
  __shared__ int batch[1024];
  const unsigned t = threadIdx.x, lane = t & 63u, wave = t >> 6;
  for (unsigned g = t; g < p.groups; g += 1024) next[g] = 0;
  if (t == 0) carried = 0;
  __syncthreads();
  for (unsigned i = t; i < p.count; i += 1024) {
    const unsigned g = (unsigned)p.ids[i];
    if (g < p.groups) atomicAdd(&next[g], 1u);
  }
  __syncthreads();
  for (unsigned g0 = 0; g0 < p.groups; g0 += 1024) {
    const unsigned g = g0 + t, mine = g < p.groups ? next[g] : 0u, upto = skl_wave_scan(mine);
    if (lane == 63) total[wave] = upto;
    __syncthreads();
    unsigned before = carried;
    for (unsigned w = 0; w < wave; ++w) before += total[w];
    if (g < p.groups) {
      next[g] = before + upto - mine;
      p.offsets[g] = (int)(before + upto - mine);
    }
    __syncthreads();
    if (t == 1023) carried = before + upto;
    __syncthreads();
  }
  if (t == 0) p.offsets[p.groups] = (int)carried;
  for (unsigned i0 = 0; i0 < p.count; i0 += 1024) {
    const unsigned i = i0 + t, g = i < p.count ? (unsigned)p.ids[i] : ~0u;
    batch[t] = (int)g;
    __syncthreads();
    unsigned before = 0, after = 0;
    for (unsigned j = 0; j < 1024; ++j) {
      before += j < t && batch[j] == (int)g;
      after += j > t && batch[j] == (int)g;
    }
    const bool in = g < p.groups;
    const unsigned at = in ? next[g] + before : 0u;
    __syncthreads();
    if (in && after == 0) next[g] = at + 1;
    if (in) {
      if (p.order) p.order[at] = (int)i;
      if (p.rows) p.rows[at] = (int)(i / p.per_row);
    }
    if (p.place && i < p.count) p.place[i] = in ? (int)at : -1;
    __syncthreads();
  }
}

}  // namespace

int skl_hip_launch_group_rows(size_t count, const int32_t *ids, size_t per_row, size_t groups, int32_t *offsets, int32_t *order, int32_t *rows,
                              int32_t *place) {
  GroupRowsArgs p{};
  p.ids = ids, p.count = (unsigned)count, p.groups = (unsigned)groups;
  p.per_row = per_row > 0xFFFFFFFFu ? 0xFFFFFFFFu : (unsigned)per_row;  // (more than there are picks: one row)
  p.offsets = offsets, p.order = order, p.rows = rows, p.place = place;
  group_rows_kernel<<<dim3(1), dim3(1024), 0, skl_current_stream()>>>(p);
  return skl_check_launch("group_rows");
}
