/*
 * skl_host.h - what the C host layers (skl_api.c, skl_api_mx.c) share: where a call's pointers lie, and device copies of
 * host memory.
 */
#ifndef SKL_HOST_H
#define SKL_HOST_H

#include <stddef.h>

#include "../../include/skl-hip.h"
#include "skl_launch.h"

/* Classifies `n` pointers (NULL entries are skipped). Returns 1 all device, 0 all host, -1 mixed (error recorded). */
static inline int skl_classify(const void *const *p, int n, const char *who) {
  int given = 0, dev = 0;
  if (skl_hip_get_pointer_mode() == SKL_HIP_POINTERS_DEVICE) return 1;
  for (int i = 0; i < n; ++i) {
    if (!p[i]) continue;
    ++given;
    dev += skl_hip_pointer_is_device(p[i]) ? 1 : 0;
  }
  if (dev == given) return 1;
  if (dev == 0) return 0;
  skl_hip_record_error(SKL_HIP_ERR_MIXED_POINTERS, who);
  return -1;
}

/* Device copy of a host span (NULL on failure or empty span). */
static inline void *skl_stage_in(const void *host, size_t bytes) {
  void *d;
  if (bytes == 0) return NULL;
  d = skl_hip_malloc(bytes);
  if (d && skl_hip_memcpy_h2d(d, host, bytes) != 0) {
    skl_hip_free(d);
    d = NULL;
  }
  return d;
}

#endif /* SKL_HOST_H */
