// Sums of per-block partial gradients.  A gradient that many blocks add to (a
// weight's, a bias's) is written by each as a row of partial sums; one wave
// here adds every PWth row of 64 columns, PU loads in flight, and the block's
// waves' sums are added through LDS: a fixed order, no atomics.  Bound by latency,
// one or two rounds of loads: 3 to 5 us (a convolution's 512 rows of 10240, 21 MB, 6.2).
#include "parts.h"

#include "common.h"
#include "runtime.h"

namespace asca {

constexpr int PU = 8, PW = 16;

__global__ __launch_bounds__(64 * PW) void sum_parts_k(const float* __restrict__ part, long parts, long row, PartsOut o) {
    __shared__ float red[PW][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long i = (long)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (i < row)
        for (long k = w; k < parts; k += PW * PU) {
            float v[PU];
#pragma unroll
            for (int u = 0; u < PU; ++u) v[u] = k + PW * u < parts ? part[(k + PW * u) * row + i] : 0.0f;
#pragma unroll
            for (int u = 0; u < PU; ++u) s += v[u];
        }
    red[w][lane] = s;
    __syncthreads();
    if (w || i >= row) return;
#pragma unroll
    for (int k = 1; k < PW; ++k) s += red[k][lane];
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
    const long blocks = (row + 63) / 64;
    if (!grid_fits(blocks, 64 * PW)) return fail(ASCA_ERR_UNSUPPORTED, "sums of %ld values", row);
    int rc = pre_launch("sum_parts");
    if (rc) return rc;
    hipLaunchKernelGGL(sum_parts_k, dim3((unsigned)blocks), dim3(64 * PW), 0, st, part, parts, row, o);
    return post_launch("sum_parts");
}

}  // namespace asca
