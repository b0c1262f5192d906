// What the kernels on a paged cache share.
#pragma once

#include "fl_device.h"
#include "fl_paged_map.h"

namespace fl {

// A stored scale's value (a slot never written may hold 0 or 255: no scale's codes).
__device__ __forceinline__ float scale_of(uint32_t code) { return __uint_as_float(code << 23); }

}  // namespace fl
