// The global 2-norm of a list of gradient tensors and their clipping by it:
//   norm = sqrt(sum g^2);  c = min(1, max_norm / (norm + 1e-6));  dst = c src
// The list is cut into chunks of one tensor each (a table in device memory,
// made once); a block has a chunk.  The squares are summed in 64 bits, a
// chunk's sum is stored, and the block that ends last adds the chunks' sums in
// their order: one launch for the norm, deterministic.  Bound by memory.
#include <algorithm>
#include <vector>

#include "act.h"

namespace asca {

struct GradChunk {
    const void* src;
    void* dst;
    long n;
};

constexpr long GC_MIN = 4096, GC_BLOCKS = 4096;   // elements a chunk at least; about so many chunks

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

// sums[chunk]; the last block writes out[0] (and out[1] with `clip`)
template <typename E>
__global__ __launch_bounds__(256) void grads_norm_k(const GradChunk* __restrict__ chunks, double* sums, unsigned* done,
                                                   int clip, float max_norm, float* __restrict__ out) {
    __shared__ double lds[4];
    __shared__ bool last;
    const GradChunk c = chunks[blockIdx.x];
    const E* src = static_cast<const E*>(c.src);
    double s = 0.0;
    for (long i = threadIdx.x; i < c.n; i += 256) {
        const double v = act_load(src + i);
        s = fma(v, v, s);
    }
    s = block_sum_d(s, lds);
    if (threadIdx.x == 0) {
        sums[blockIdx.x] = s;
        __threadfence();
        last = atomicAdd(done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    s = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += 256) s += __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = block_sum_d(s, lds);
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(s);
        out[0] = norm;
        if (clip) {
            const float r = max_norm / (norm + 1e-6f);
            out[1] = r >= 1.0f ? 1.0f : r;   // NaN stays
        }
        *done = 0;
    }
}

template <typename E>
__global__ __launch_bounds__(256) void grads_scale_k(const GradChunk* __restrict__ chunks, const float* __restrict__ out) {
    const GradChunk c = chunks[blockIdx.x];
    const float f = out[1];
    if (f == 1.0f && c.src == c.dst) return;   // nothing changes
    const E* src = static_cast<const E*>(c.src);
    E* dst = static_cast<E*>(c.dst);
    for (long i = threadIdx.x; i < c.n; i += 256) act_store(dst + i, f * act_load(src + i));
}

__global__ void grads_none_k(float* out, int clip) {
    out[0] = 0.0f;
    if (clip) out[1] = 1.0f;
}

struct GradList {
    GradChunk* chunks = nullptr;   // then the sums and the counter, one allocation
    double* sums = nullptr;
    unsigned* done = nullptr;
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
        int r = pre_launch("grads_norm");
        if (r) return r;
        hipLaunchKernelGGL(grads_norm_k<E>, dim3(g->n), dim3(256), 0, st, g->chunks, g->sums, g->done, (int)clip, max_norm,
                           out);
        if ((r = post_launch("grads_norm")) || !clip) return r;
        if ((r = pre_launch("grads_scale"))) return r;
        hipLaunchKernelGGL(grads_scale_k<E>, dim3(g->n), dim3(256), 0, st, g->chunks, out);
        return post_launch("grads_scale");
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
        if (t.size() > 0x7fffffffu) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many tensors", fn);
        g = new GradList;
        g->n = (unsigned)t.size();
        g->dtype = dtype;
        if (g->n) {
            const size_t tab = t.size() * sizeof(GradChunk), sum = t.size() * sizeof(double);
            char* m = nullptr;
            hipError_t e = hipMalloc(reinterpret_cast<void**>(&m), tab + sum + 16);
            if (e != hipSuccess) {
                delete g;
                return fail(ASCA_ERR_OOM, "%s: %zu bytes: %s", fn, tab + sum + 16, hipGetErrorString(e));
            }
            g->chunks = reinterpret_cast<GradChunk*>(m);
            g->sums = reinterpret_cast<double*>(m + tab);
            g->done = reinterpret_cast<unsigned*>(m + tab + sum);
            e = hipMemcpy(m, t.data(), tab, hipMemcpyHostToDevice);
            if (e == hipSuccess) e = hipMemset(g->done, 0, 4);
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
