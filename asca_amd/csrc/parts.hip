// Sums of per-block partial gradients.  A gradient that many blocks add to (a
// weight's, a bias's) is written by each as a row of partial sums; one wave
// here adds every fourth row of 64 columns, PU loads in flight, and the block's
// four waves' sums are added through LDS: a fixed order, no atomics.
#include "parts.h"

#include "common.h"
#include "runtime.h"

namespace asca {

constexpr int PU = 8;

__global__ __launch_bounds__(256) void sum_parts_k(const float* __restrict__ part, long parts, long row, PartsOut o) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long i = (long)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (i < row)
        for (long k = w; k < parts; k += 4 * PU) {
            float v[PU];
#pragma unroll
            for (int u = 0; u < PU; ++u) v[u] = k + 4 * u < parts ? part[(k + 4 * u) * row + i] : 0.0f;
#pragma unroll
            for (int u = 0; u < PU; ++u) s += v[u];
        }
    red[w][lane] = s;
    __syncthreads();
    if (w || i >= row) return;
    s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    long at = i;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if (at >= 0 && at < o.n[k] && o.out[k]) o.out[k][at] = s;
        at -= o.n[k];
    }
}

int sum_parts_launch(const float* part, long parts, const PartsOut& o, hipStream_t st) {
    const long row = o.n[0] + o.n[1] + o.n[2];
    if (row == 0) return ASCA_OK;
    int rc = pre_launch("sum_parts");
    if (rc) return rc;
    hipLaunchKernelGGL(sum_parts_k, dim3((unsigned)((row + 63) / 64)), dim3(256), 0, st, part, parts, row, o);
    return post_launch("sum_parts");
}

}  // namespace asca
