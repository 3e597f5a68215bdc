// Sums of per-block partial gradients in a fixed order (parts.hip).  Internal.
#pragma once
#include <hip/hip_runtime.h>

namespace asca {

// Up to three arrays whose partial sums lie one behind the other in a row of
// n[0] + n[1] + n[2] floats; an array with a null pointer is not written.
struct PartsOut {
    float* out[3];
    long n[3];
};

// out = sum over the `parts` rows of `part` (zeros for no rows).
int sum_parts_launch(const float* part, long parts, const PartsOut& o, hipStream_t st);

}  // namespace asca
