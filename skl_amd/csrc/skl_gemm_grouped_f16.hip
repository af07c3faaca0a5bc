// skl_gemm_grouped_f16.hip - the streaming kernels of the products grouped by expert for f16 operands (skl_grouped_ring.hpp).
#include "skl_grouped_ring.hpp"

int skl_launch_grouped_ring_f16(const skl_grouped_gemm &g) { return grouped_ring<SKL_DT_F16>(g); }
int skl_launch_groupedk_ring_f16(const skl_groupedk_gemm &g) { return grouped_over_ring<SKL_DT_F16>(g); }
