// What the kernels on a paged cache share.
#pragma once

#include "fl_device.h"
#include "fl_paged_map.h"

namespace fl {

// A stored scale's value; finite for a slot never written, which may hold any code.
__device__ __forceinline__ float scale_of(uint32_t code) { return __uint_as_float(min(code, 254u) << 23); }

}  // namespace fl
