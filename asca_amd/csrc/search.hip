// The largest logits of rows, and a beam search's steps over them: the choice among a
// group's beams and tokens, and the states' move to their beams' new slots.
//   top    the K largest of a row, ties to the lower id; lse = log sum exp(z / tau)
//   step   the K best of s_b + z_bi - lse_b over b and i, ties to the lower b V + i
//   states slot <- state of parent[slot], in place or into other buffers
#include <algorithm>

#include "logits.h"

namespace asca {

constexpr int TOP_MAX_K = 64;    // listed logits a row
constexpr int BEAM_MAX_K = 32;   // beams a group
constexpr int BEAM_BUFS = 8;     // state buffers a call

struct TopArgs {
    const void* z;
    long ld, rows;
    int V, K;
    float tau;
    float* values;
    int32_t* ids;
    float* lse;
};

// m and log sum exp((z - m) / tau) of a row by a block of 256; the logarithm in 64 bits
template <typename E>
ASCA_DEV void row_lse(const E* z, int V, float itau, float& m, double& ls, float* lds) {
    float mx = -INFINITY;
    for (int c = threadIdx.x; c < V; c += 256) mx = fmaxf(mx, act_load(z + c));
    m = block_max_t<4>(mx, lds);
    const float ref = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
    for (int c = threadIdx.x; c < V; c += 256) s += __builtin_amdgcn_exp2f((act_load(z + c) - ref) * itau * LOG2E);
    ls = log((double)block_sum_t<4>(s, lds));
    m = ref;
}

template <typename E>
__global__ __launch_bounds__(256) void top_k(TopArgs p) {
    __shared__ float lds[4];
    __shared__ uint64_t keys[4];
    const long row = blockIdx.x;
    const E* z = static_cast<const E*>(p.z) + row * p.ld;
    float m;
    double ls;
    row_lse(z, p.V, 1.0f / p.tau, m, ls, lds);
    if (p.lse && threadIdx.x == 0) p.lse[row] = (float)((double)m / (double)p.tau + ls);
    uint64_t last = ~0ull;
    for (int k = 0; k < p.K; ++k) {
        uint64_t best = 0;
        for (int c = threadIdx.x; c < p.V; c += 256) {
            const uint64_t key = logit_key(act_load(z + c), c);
            if (key < last && key > best) best = key;
        }
        last = block_max_t<4>(best, keys);
        if (threadIdx.x == 0) {
            p.values[row * p.K + k] = last ? key_value(last) : -INFINITY;
            p.ids[row * p.K + k] = last ? (int)key_place(last) : -1;
        }
    }
}

struct BeamArgs {
    const void* z;
    long ld;
    const float* scores;
    const int32_t* ended;
    float* new_scores;
    int32_t* new_ended;
    uint32_t* tokens;
    int32_t* parents;
    int K, V, eos, stay;
};

struct BeamPick {
    double score;   // -inf: none
    int parent;
    unsigned token;
};

// Slots for the K picks in the lanes of a wave, best first (parent < 0: none).  `stay`: the
// best child of a beam takes its slot, the others and the empty ones what is left, in order.
ASCA_DEV int beam_slot(int parent, int K, bool stay) {
    const int lane = threadIdx.x & 63;
    if (!stay) return lane;
    bool first = parent >= 0 && lane < K;
    for (int j = 0; j < K; ++j)
        if (j < lane && __builtin_amdgcn_readlane(parent, j) == parent) first = false;
    const uint64_t firsts = __ballot(first);
    unsigned taken = 0;
    for (int j = 0; j < K; ++j)
        if (firsts >> j & 1) taken |= 1u << __builtin_amdgcn_readlane(parent, j);
    const uint64_t rest = ~firsts & ((K < 64 ? 1ull << K : 0) - 1);
    int want = __popcll(rest & ((1ull << lane) - 1)), slot = parent;
    if (!first)
        for (int j = 0; j < K; ++j)
            if (!(taken >> j & 1) && want-- == 0) slot = j;
    return slot;
}

// A group's picks, best first, in the first K lanes of the first wave, to its slots
ASCA_DEV void beam_write(const BeamArgs& p, long group, const BeamPick& pick) {
    const int lane = threadIdx.x & 63;
    const int slot = beam_slot(pick.parent, p.K, p.stay);
    if (lane >= p.K) return;
    const long at = group * p.K + slot;
    const bool some = pick.parent >= 0;
    const bool end = some && p.ended && (p.ended[group * p.K + pick.parent] != 0 || (int)pick.token == p.eos);
    // every lane has read what the caller's buffers held before any writes: new_ended may be ended
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    p.new_scores[at] = some ? (float)pick.score : -INFINITY;
    p.tokens[at] = some ? pick.token : p.eos >= 0 ? (unsigned)p.eos : 0u;
    p.parents[at] = some ? pick.parent : slot;
    if (p.new_ended) p.new_ended[at] = end;
}

// Whether a beam's candidates count: its score and its logits' sum are finite
ASCA_DEV bool beam_finite(double x) { return fabs(x) < INFINITY; }

template <typename E>
__global__ __launch_bounds__(256) void beam_step_k(BeamArgs p) {
    __shared__ float lds[4];
    __shared__ double base[BEAM_MAX_K], best[4];
    __shared__ uint64_t places[4], chosen[BEAM_MAX_K];
    __shared__ double values[BEAM_MAX_K];
    const long group = blockIdx.x;
    const E* z = static_cast<const E*>(p.z) + group * p.K * p.ld;
    for (int b = 0; b < p.K; ++b) {
        const double s = p.scores[group * p.K + b];
        float m;
        double ls = 0.0, x = -INFINITY;
        const bool end = p.ended && p.ended[group * p.K + b] != 0;
        if (!end) row_lse(z + b * p.ld, p.V, 1.0f, m, ls, lds);
        if (end) x = s;
        else x = s - ((double)m + ls);
        if (threadIdx.x == 0) base[b] = beam_finite(s) && beam_finite(x) ? x : (double)-INFINITY;
    }
    __syncthreads();
    double last = INFINITY;
    uint64_t lastp = 0;
    for (int k = 0; k < p.K; ++k) {
        double v = -INFINITY;
        uint64_t vp = ~0ull;
        auto offer = [&](double x, uint64_t at) {
            if (!(x < last || (x == last && at > lastp))) return;
            if (x > v || (x == v && at < vp)) v = x, vp = at;
        };
        for (int b = 0; b < p.K; ++b) {
            if (base[b] == -INFINITY) continue;
            if (p.ended && p.ended[group * p.K + b] != 0) {
                if (threadIdx.x == 0) offer(base[b], (uint64_t)b * p.V + p.eos);
                continue;
            }
            for (int c = threadIdx.x; c < p.V; c += 256) {
                const float t = act_load(z + b * p.ld + c);
                if (t > -INFINITY) offer(base[b] + t, (uint64_t)b * p.V + c);
            }
        }
        const double top = block_max_t<4>(v, best);
        const uint64_t place = ~block_max_t<4>(v == top ? ~vp : (uint64_t)0, places);
        if (threadIdx.x == 0) values[k] = top, chosen[k] = place;
        last = top, lastp = place;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    BeamPick pick{-INFINITY, -1, 0};
    if (threadIdx.x < p.K && values[threadIdx.x] > -INFINITY) {
        pick.score = values[threadIdx.x];
        pick.parent = (int)(chosen[threadIdx.x] / p.V);
        pick.token = (unsigned)(chosen[threadIdx.x] % p.V);
    }
    beam_write(p, group, pick);
}

struct StatesArgs {
    const char* src[BEAM_BUFS];
    char* dst[BEAM_BUFS];
    unsigned long outer[BEAM_BUFS], bytes[BEAM_BUFS];
    unsigned long first[BEAM_BUFS + 1];   // blocks before each buffer's
    const int32_t* parents;
    int count, groups, ks, kd;
};

// A block takes 256 words of the states of one group in one outer row.  A thread reads its
// words of all the slots that change before it writes any, so that a buffer may be its own
// destination; no other thread touches them.
template <typename W>
__global__ __launch_bounds__(256) void beam_states_k(StatesArgs p) {
    int i = 0;
    while (i + 1 < p.count && blockIdx.x >= p.first[i + 1]) ++i;
    const unsigned long words = p.bytes[i] / sizeof(W), per = (words + 255) / 256;
    unsigned long b = blockIdx.x - p.first[i];
    const unsigned long w = b % per * 256 + threadIdx.x;
    b /= per;
    const long group = b % p.groups, outer = b / p.groups;
    if (w >= words) return;
    const W* src = reinterpret_cast<const W*>(p.src[i]) + (outer * p.groups + group) * p.ks * words + w;
    W* dst = reinterpret_cast<W*>(p.dst[i]) + (outer * p.groups + group) * p.kd * words + w;
    W v[BEAM_MAX_K];
    auto from = [&](int j) {
        const int q = p.parents ? p.parents[group * p.kd + j] : 0;
        return q < 0 || q >= p.ks || (src == dst && q == j) ? -1 : q;
    };
#pragma unroll
    for (int j = 0; j < BEAM_MAX_K; ++j)
        if (j < p.kd) {
            const int q = from(j);
            if (q >= 0) v[j] = src[q * words];
        }
#pragma unroll
    for (int j = 0; j < BEAM_MAX_K; ++j)
        if (j < p.kd && from(j) >= 0) dst[j * words] = v[j];
}

}  // namespace asca

using namespace asca;

static int rows_check(const char* fn, long rows, int V, long ld, const void* z, int dtype) {
    if (rows < 0 || V <= 0) return fail(ASCA_ERR_INVALID, "%s: bad shape %ld x %d", fn, rows, V);
    if (ld < V) return fail(ASCA_ERR_INVALID, "%s: row stride %ld below %d columns", fn, ld, V);
    if (reinterpret_cast<uintptr_t>(z) % (dtype == ASCA_F32 ? 4 : 2))
        return fail(ASCA_ERR_INVALID, "%s: logits at an address that is no multiple of an element", fn);
    return ASCA_OK;
}

extern "C" {

int asca_top_logits(const void* logits, long ld, long rows, int V, int K, float temperature, float* values,
                    int32_t* ids, float* lse, int dtype, void* stream) {
    const char* fn = "asca_top_logits";
    int rc = rows_check(fn, rows, V, ld, logits, dtype);
    if (rc) return rc;
    if (K < 1 || K > TOP_MAX_K) return fail(ASCA_ERR_UNSUPPORTED, "%s: K=%d (1 to %d)", fn, K, TOP_MAX_K);
    if (!(temperature > 0.0f) || !(temperature < INFINITY))
        return fail(ASCA_ERR_INVALID, "%s: temperature %g", fn, (double)temperature);
    if (rows > 0 && (!logits || !values || !ids)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (!grid_fits(rows, 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows (%ld)", fn, rows);
    return act_dispatch(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        if (rows == 0) return (int)ASCA_OK;
        int r = pre_launch("top_logits");
        if (r) return r;
        const TopArgs a{logits, ld, rows, V, K, temperature, values, ids, lse};
        hipLaunchKernelGGL(top_k<E>, dim3((unsigned)rows), dim3(256), 0, as_stream(stream), a);
        return post_launch("top_logits");
    });
}

int asca_beam_step(const void* logits, long ld, const float* scores, const int32_t* ended, int eos, int stay,
                   float* new_scores, int32_t* new_ended, uint32_t* tokens, int32_t* parents, int groups, int K,
                   int V, int dtype, void* stream) {
    const char* fn = "asca_beam_step";
    if (groups < 0) return fail(ASCA_ERR_INVALID, "%s: groups=%d", fn, groups);
    if (K < 1 || K > BEAM_MAX_K) return fail(ASCA_ERR_UNSUPPORTED, "%s: K=%d (1 to %d)", fn, K, BEAM_MAX_K);
    int rc = rows_check(fn, (long)groups * K, V, ld, logits, dtype);
    if (rc) return rc;
    if (eos >= V) return fail(ASCA_ERR_INVALID, "%s: eos=%d of %d tokens", fn, eos, V);
    if ((eos >= 0) != (ended != nullptr) || (eos >= 0) != (new_ended != nullptr))
        if (groups > 0) return fail(ASCA_ERR_INVALID, "%s: eos, ended and new_ended go together", fn);
    if (groups > 0 && (!logits || !scores || !new_scores || !tokens || !parents))
        return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (!grid_fits(groups, 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many groups (%d)", fn, groups);
    return act_dispatch(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        if (groups == 0) return (int)ASCA_OK;
        int r = pre_launch("beam_step");
        if (r) return r;
        const BeamArgs a{logits, ld, scores, ended, new_scores, new_ended, tokens, parents, K, V, eos < 0 ? -1 : eos, stay};
        hipLaunchKernelGGL(beam_step_k<E>, dim3((unsigned)groups), dim3(256), 0, as_stream(stream), a);
        return post_launch("beam_step");
    });
}

int asca_beam_states(void** src, void** dst, const uint64_t* outer, const uint64_t* bytes, int count,
                     const int32_t* parents, int groups, int k_src, int k_dst, void* stream) {
    const char* fn = "asca_beam_states";
    if (count < 0 || count > BEAM_BUFS) return fail(ASCA_ERR_INVALID, "%s: %d buffers (0 to %d)", fn, count, BEAM_BUFS);
    if (groups < 0) return fail(ASCA_ERR_INVALID, "%s: groups=%d", fn, groups);
    if (k_src < 1 || k_src > BEAM_MAX_K || k_dst < 1 || k_dst > BEAM_MAX_K)
        return fail(ASCA_ERR_UNSUPPORTED, "%s: %d beams from %d (1 to %d)", fn, k_dst, k_src, BEAM_MAX_K);
    if (count > 0 && (!src || !outer || !bytes)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    StatesArgs a{};
    a.parents = parents;
    a.groups = groups;
    a.ks = k_src;
    a.kd = k_dst;
    unsigned word = 16;
    for (int i = 0; i < count; ++i) {
        if (outer[i] > (uint64_t)1 << 40 || bytes[i] > (uint64_t)1 << 40)
            return fail(ASCA_ERR_INVALID, "%s: buffer %d has %lu rows of %lu bytes", fn, i, (unsigned long)outer[i],
                        (unsigned long)bytes[i]);
        if (!outer[i] || !bytes[i] || !groups) continue;
        void* d = dst && dst[i] ? dst[i] : src[i];
        if (!src[i]) return fail(ASCA_ERR_INVALID, "%s: buffer %d is NULL", fn, i);
        if (d == src[i] && k_src != k_dst)
            return fail(ASCA_ERR_INVALID, "%s: buffer %d goes from %d to %d beams in place", fn, i, k_src, k_dst);
        if (d != src[i]) {
            const auto s0 = reinterpret_cast<uintptr_t>(src[i]), d0 = reinterpret_cast<uintptr_t>(d);
            const __uint128_t n = (__uint128_t)outer[i] * bytes[i] * groups;
            if (s0 < d0 + n * k_dst && d0 < s0 + n * k_src)
                return fail(ASCA_ERR_INVALID, "%s: buffer %d overlaps its destination", fn, i);
        }
        const auto mix = reinterpret_cast<uintptr_t>(src[i]) | reinterpret_cast<uintptr_t>(d) | (uintptr_t)bytes[i];
        while (mix % word) word = word == 16 ? 4 : 1;
        const int n = a.count++;
        a.src[n] = static_cast<const char*>(src[i]);
        a.dst[n] = static_cast<char*>(d);
        a.outer[n] = outer[i];
        a.bytes[n] = bytes[i];
    }
    if (a.count == 0) return ASCA_OK;
    __uint128_t blocks = 0;
    for (int i = 0; i < a.count; ++i) {
        a.first[i] = (unsigned long)blocks;
        blocks += (__uint128_t)((a.bytes[i] / word + 255) / 256) * a.outer[i] * groups;
        if (blocks >= (1ul << 24)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too much to move in one call", fn);
    }
    int rc = pre_launch("beam_states");
    if (rc) return rc;
    const dim3 grid((unsigned)blocks);
    const hipStream_t st = as_stream(stream);
    if (word == 16)
        hipLaunchKernelGGL(beam_states_k<uint4>, grid, dim3(256), 0, st, a);
    else if (word == 4)
        hipLaunchKernelGGL(beam_states_k<uint32_t>, grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(beam_states_k<uint8_t>, grid, dim3(256), 0, st, a);
    return post_launch("beam_states");
}

}  // extern "C"
