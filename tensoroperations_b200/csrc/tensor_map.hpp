// tensor_map.hpp -- cuTensorMapEncodeTiled through the runtime's driver entry
// point (the library does not link the driver).
#pragma once

#include <cuda.h>

#include "common.hpp"

namespace to_b200 {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Null, with *st set, where the driver lacks it.
EncodeTiled tensor_map_encoder(int* st);

}  // namespace to_b200
