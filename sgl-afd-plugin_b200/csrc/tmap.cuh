// Host-side TMA tensor maps (the driver's encoder, resolved at run time), shared by the GEMM translation units.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace asap {

// 2-D map of `outer` rows of `inner` elements, `row_bytes` apart, read in boxes of box_outer x box_inner.
int make_tmap_2d(CUtensorMap* m, CUtensorMapDataType dt, const void* base, uint64_t inner, uint64_t outer,
                 uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer, const char* what,
                 CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B);

}  // namespace asap
