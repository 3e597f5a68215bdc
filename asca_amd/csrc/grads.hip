// The global 2-norm of a list of gradient tensors and their clipping by it:
//   norm = sqrt(sum g^2);  c = min(1, max_norm / (norm + 1e-6));  dst = c src
// The list is cut into chunks of one tensor each (a table in device memory,
// made once); a block has a chunk.  The squares are summed in 64 bits; the chunks'
// sums are added in their order by every block that scales, which costs less than a
// launch between (and than a last block's: a fence in each block before it took the
// norm of 143M gradients from 122 to 310 us).  Bound by memory: 143M f32 gradients
// are read in 113 us (5.1 TB/s; 155 just after a kernel that filled the last-level
// cache with its writes) and read and written in 206 us (5.5 TB/s, the part that the
// cache still holds coming first).  Stores past the caches leave more of the list there,
// which the next call on it sees (321 -> 294 us) but not an update between (890 us both).
// The chunks' sums are added by every block, so the time grows with the square of the
// tensors where these are thousands: 1000 of 256 elements 7 us, 3000 12, 10000 61, 30000 415.
#include <algorithm>
#include <vector>

#include "act.h"

namespace asca {

struct GradChunk {
    const void* src;
    void* dst;
    long n;
};

constexpr int GC_U = 4;                            // accesses of 4 elements a thread has in flight
constexpr long GC_IT = 256 * 4 * GC_U;             // elements a block takes at a time
constexpr long GC_MIN = GC_IT, GC_BLOCKS = 4096;   // elements a chunk at least; about so many chunks (2048: 334 us, 4096: 321)

ASCA_DEV double wave_sum_d(double x) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) x += __shfl_xor(x, s, 64);
    return x;
}

ASCA_DEV double block_sum_d(double x, double* lds) {
    x = wave_sum_d(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// sums[chunk] = the sum of its squares
template <typename E>
__global__ __launch_bounds__(256) void grads_sums_k(const GradChunk* __restrict__ chunks, double* __restrict__ sums) {
    __shared__ double lds[4];
    const GradChunk c = chunks[blockIdx.x];
    const E* src = static_cast<const E*>(c.src);
    double s = 0.0;
    auto add = [&](float x) {
        const double v = x;
        s = fma(v, v, s);
    };
    long i = 0;
    if (reinterpret_cast<uintptr_t>(src) % (4 * sizeof(E)) == 0)
        for (; i + GC_IT <= c.n; i += GC_IT) {
            act_raw<4, E> r[GC_U];
#pragma unroll
            for (int u = 0; u < GC_U; ++u) r[u] = act_load_raw<4>(src + i + (u * 256 + threadIdx.x) * 4);
#pragma unroll
            for (int u = 0; u < GC_U; ++u) {
                float v[4];
                act_values(r[u], v);
#pragma unroll
                for (int k = 0; k < 4; ++k) add(v[k]);
            }
        }
    for (i += threadIdx.x; i < c.n; i += 256) add(act_load(src + i));
    s = block_sum_d(s, lds);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// The norm from the chunks' sums, the same in every block that asks
ASCA_DEV float grads_total(const double* __restrict__ sums, unsigned n, double* lds) {
    double s = 0.0;
    for (unsigned i = threadIdx.x; i < n; i += 256) s += sums[i];
    return (float)sqrt(block_sum_d(s, lds));
}

__global__ __launch_bounds__(256) void grads_norm_k(const double* __restrict__ sums, unsigned n, float* __restrict__ out) {
    __shared__ double lds[4];
    const float norm = grads_total(sums, n, lds);
    if (threadIdx.x == 0) out[0] = norm;
}

template <typename E>
__global__ __launch_bounds__(256) void grads_scale_k(const GradChunk* __restrict__ chunks, const double* __restrict__ sums,
                                                    float max_norm, float* __restrict__ out) {
    __shared__ double lds[4];
    // the chunks that were read last come first: they may still be in a cache
    const GradChunk c = chunks[gridDim.x - 1 - blockIdx.x];
    const float norm = grads_total(sums, gridDim.x, lds), ratio = max_norm / (norm + 1e-6f);
    const float f = ratio >= 1.0f ? 1.0f : ratio;   // NaN stays
    if (blockIdx.x == 0 && threadIdx.x == 0) out[0] = norm, out[1] = f;
    if (f == 1.0f && c.src == c.dst) return;        // nothing changes
    const E* src = static_cast<const E*>(c.src);
    E* dst = static_cast<E*>(c.dst);
    long i = 0;
    if ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) % (4 * sizeof(E)) == 0)
        for (; i + GC_IT <= c.n; i += GC_IT) {
            act_raw<4, E> r[GC_U];
#pragma unroll
            for (int u = 0; u < GC_U; ++u) r[u] = act_load_raw<4>(src + i + (u * 256 + threadIdx.x) * 4);
#pragma unroll
            for (int u = 0; u < GC_U; ++u) {
                float v[4];
                act_values(r[u], v);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] *= f;
                act_store_n<4>(dst + i + (u * 256 + threadIdx.x) * 4, v);
            }
        }
    for (i += threadIdx.x; i < c.n; i += 256) act_store(dst + i, f * act_load(src + i));
}

__global__ void grads_none_k(float* out, int clip) {
    out[0] = 0.0f;
    if (clip) out[1] = 1.0f;
}

struct GradList {
    GradChunk* chunks = nullptr;   // then the sums, one allocation
    double* sums = nullptr;
    unsigned n = 0;
    int dtype = 0;
};

}  // namespace asca

using namespace asca;

static int grads_run(GradList* g, bool clip, float max_norm, float* out, hipStream_t st) {
    int rc;
    if (g->n == 0) {
        if ((rc = pre_launch("grads_none"))) return rc;
        hipLaunchKernelGGL(grads_none_k, dim3(1), dim3(1), 0, st, out, (int)clip);
        return post_launch("grads_none");
    }
    return act_dispatch(g->dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        int r = pre_launch("grads_sums");
        if (r) return r;
        hipLaunchKernelGGL(grads_sums_k<E>, dim3(g->n), dim3(256), 0, st, g->chunks, g->sums);
        if ((r = post_launch("grads_sums"))) return r;
        if (clip) {
            if ((r = pre_launch("grads_scale"))) return r;
            hipLaunchKernelGGL(grads_scale_k<E>, dim3(g->n), dim3(256), 0, st, g->chunks, g->sums, max_norm, out);
            return post_launch("grads_scale");
        }
        if ((r = pre_launch("grads_norm"))) return r;
        hipLaunchKernelGGL(grads_norm_k, dim3(1), dim3(256), 0, st, g->sums, g->n, out);
        return post_launch("grads_norm");
    });
}

extern "C" {

int asca_grads_create(void** src, void** dst, const uint64_t* sizes, int count, int dtype, void** grads) {
    const char* fn = "asca_grads_create";
    if (!grads) return fail(ASCA_ERR_INVALID, "null output pointer");
    *grads = nullptr;
    if (count < 0) return fail(ASCA_ERR_INVALID, "%s: negative count", fn);
    if (count > 0 && (!src || !sizes)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    int rc = act_dispatch(dtype, [](auto*) { return (int)ASCA_OK; });
    if (rc) return rc;
    const size_t size = dtype == ASCA_F32 ? 4 : 2;
    uint64_t total = 0;
    for (int i = 0; i < count; ++i) {
        if (sizes[i] > (uint64_t)1 << 48) return fail(ASCA_ERR_INVALID, "%s: tensor %d has %lu elements", fn, i, (unsigned long)sizes[i]);
        if (sizes[i] && (!src[i] || (dst && !dst[i]))) return fail(ASCA_ERR_INVALID, "%s: tensor %d is NULL", fn, i);
        total += sizes[i];
    }
    if ((rc = ensure_device())) return rc;
    const long per = std::max(GC_MIN, (long)((total / GC_BLOCKS + GC_MIN - 1) / GC_MIN * GC_MIN));
    GradList* g = nullptr;
    try {
        std::vector<GradChunk> t;
        for (int i = 0; i < count; ++i)
            for (uint64_t o = 0; o < sizes[i]; o += per) {
                char* s = static_cast<char*>(src[i]) + o * size;
                t.push_back({s, dst ? static_cast<char*>(dst[i]) + o * size : s, (long)std::min<uint64_t>(per, sizes[i] - o)});
            }
        if (!grid_fits((long)t.size(), 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many tensors", fn);
        g = new GradList;
        g->n = (unsigned)t.size();
        g->dtype = dtype;
        if (g->n) {
            const size_t tab = t.size() * sizeof(GradChunk), sum = t.size() * sizeof(double);
            char* m = nullptr;
            hipError_t e = hipMalloc(reinterpret_cast<void**>(&m), tab + sum);
            if (e != hipSuccess) {
                delete g;
                return fail(ASCA_ERR_OOM, "%s: %zu bytes: %s", fn, tab + sum, hipGetErrorString(e));
            }
            g->chunks = reinterpret_cast<GradChunk*>(m);
            g->sums = reinterpret_cast<double*>(m + tab);
            e = hipMemcpy(m, t.data(), tab, hipMemcpyHostToDevice);
            if (e == hipSuccess) e = hipDeviceSynchronize();   // done before any stream uses it
            if (e != hipSuccess) {
                (void)hipFree(m);
                delete g;
                return fail(ASCA_ERR_HIP, "%s: %s", fn, hipGetErrorString(e));
            }
        }
    } catch (const std::exception& ex) {
        delete g;
        return fail(ASCA_ERR_OOM, "%s: %s", fn, ex.what());
    }
    *grads = g;
    return ASCA_OK;
}

int asca_grads_destroy(void* grads) {
    GradList* g = static_cast<GradList*>(grads);
    if (!g) return ASCA_OK;
    if (g->chunks) {
        (void)hipDeviceSynchronize();
        (void)hipFree(g->chunks);
    }
    delete g;
    return ASCA_OK;
}

int asca_grads_norm(void* grads, float* out, void* stream) {
    if (!grads || !out) return fail(ASCA_ERR_INVALID, "null pointer in asca_grads_norm");
    return grads_run(static_cast<GradList*>(grads), false, 0.0f, out, as_stream(stream));
}

int asca_grads_clip(void* grads, float max_norm, float* out, void* stream) {
    if (!grads || !out) return fail(ASCA_ERR_INVALID, "null pointer in asca_grads_clip");
    if (!(max_norm >= 0.0f)) return fail(ASCA_ERR_INVALID, "asca_grads_clip: max_norm=%g", (double)max_norm);
    return grads_run(static_cast<GradList*>(grads), true, max_norm, out, as_stream(stream));
}

}  // extern "C"
