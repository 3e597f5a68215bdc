// Distillation from a teacher's largest logits, loss and gradient in one call.  Row of a
// student's logits z, temperature tau, listed ids S with the teacher's logits v:
//   p_k = exp(v_k / tau - tlse), the rest p_r = 1 - sum p one class more; without tlse the
//   softmax of v / tau over the list, and no rest
//   q = softmax(z / tau), q_r = its sum outside S
//   loss = w [(1 - a) (log sum exp z - z_target) + a tau^2 (sum p log(p / q) + p_r log(p_r / q_r))]
//   dz_i / scale = w [(1 - a) (softmax(z)_i - [i = target]) + a tau (q_i - p_i)] for listed i, for
//   the others q_i (1 - p_r / q_r) in the place of q_i - p_i (without tlse q_i)
// Entries of one id are one entry with the sum of their p.
#include "logits.h"
#include "ops.h"

namespace asca {

constexpr int DISTILL_MAX_K = 64;          // entries a row: one for each lane of a wave
constexpr int DISTILL_MAX_V = 1 << 20;     // columns that the bitmap in LDS has bits for

struct DistillArgs {
    const void* z;
    long ld;
    const float* tval;
    const int32_t* tids;
    const float* tlse;
    const uint32_t* targets;
    const float* weights;
    float* losses;
    void* dz;
    long lddz, T;
    int V, K;
    float tau, alpha, scale;
};

// The lists' entries of a row, one a lane of every wave
struct Entry {
    int id;        // below 0: none
    float z;       // the student's logit there
    double lp;     // log p (-inf: p = 0)
    float p;
};

ASCA_DEV double wave_sum_d(double x) { return wave_sum_t(x); }

template <typename E>
__global__ __launch_bounds__(256) void distill_k(DistillArgs p) {
    extern __shared__ unsigned bits[];   // a bit for every column: it is listed
    __shared__ float lds[4];
    const long row = blockIdx.x;
    const E* z = static_cast<const E*>(p.z) + row * p.ld;
    E* dz = p.dz ? static_cast<E*>(p.dz) + row * p.lddz : nullptr;
    const int V = p.V, lane = threadIdx.x & 63;
    const float w = p.weights ? p.weights[row] : 1.0f;
    if (w == 0.0f) {
        if (threadIdx.x == 0) p.losses[row] = 0.0f;
        if (dz)
            for (int c = threadIdx.x; c < V; c += 256) act_store(dz + c, 0.0f);
        return;
    }
    for (int i = threadIdx.x; i < (V + 31) / 32; i += 256) bits[i] = 0;
    __syncthreads();
    const bool soft = p.alpha > 0.0f, hard = p.alpha < 1.0f;
    const unsigned tg = hard ? p.targets[row] : ~0u;
    const bool has_tg = tg < (unsigned)V;
    const float zt = has_tg ? act_load(z + tg) : 0.0f;
    // entries
    Entry en{-1, 0.0f, -INFINITY, 0.0f};
    if (soft && lane < p.K) en.id = p.tids[row * p.K + lane];
    if (en.id >= V) en.id = -1;
    const double itau = 1.0 / (double)p.tau;
    if (en.id >= 0) {
        en.z = act_load(z + en.id);
        en.lp = (double)p.tval[row * p.K + lane] * itau;
        atomicOr(&bits[en.id >> 5], 1u << (en.id & 31));
    }
    if (p.tlse) {
        en.lp -= soft ? (double)p.tlse[row] : 0.0;
    } else {
        const double m = wave_max_t(en.id >= 0 ? en.lp : (double)-INFINITY);
        if (m == -INFINITY) {
            en.lp = -INFINITY;   // no entry, or none above -inf
        } else {
            en.lp -= m;
            en.lp -= log(wave_sum_d(en.id >= 0 ? exp(en.lp) : 0.0));
        }
    }
    double pd = en.id >= 0 ? exp(en.lp) : 0.0;
    const double total = wave_sum_d(pd);
    // entries of one id: the first has their sum, the others are none
    for (int j = 0; j < p.K && soft; ++j) {
        const int id = __builtin_amdgcn_readlane(en.id, j);
        if (id < 0) continue;
        const uint64_t same = __ballot(en.id == id);
        if ((same & (same - 1)) == 0) continue;
        const double sum = wave_sum_d(en.id == id ? pd : 0.0);
        if (lane == j) pd = sum, en.lp = log(sum);
        else if (en.id == id) en.id = -1, pd = 0.0;
    }
    en.p = (float)pd;
    const bool rest = p.tlse != nullptr && soft;
    const float pr = rest ? (float)fmax(0.0, 1.0 - total) : 0.0f;
    __syncthreads();
    // the columns outside the list: their largest, and their sums at both temperatures
    const float ct = (float)(itau * 1.4426950408889634), c1 = LOG2E;
    auto listed = [&](int c) { return bits[c >> 5] >> (c & 31) & 1; };
    float m = -INFINITY, mx = en.id >= 0 ? en.z : -INFINITY;
    for (int c = threadIdx.x; c < V; c += 256)
        if (!listed(c)) m = fmaxf(m, act_load(z + c));
    m = block_max_t<4>(m, lds);
    mx = fmaxf(m, wave_max_t(mx));
    const float mr = m > -INFINITY ? m : mx;   // what the others are measured from
    float st = 0.0f, s1 = 0.0f;
    for (int c = threadIdx.x; c < V; c += 256)
        if (!listed(c)) {
            const float v = act_load(z + c);
            st += __builtin_amdgcn_exp2f((v - mr) * ct);
            s1 += __builtin_amdgcn_exp2f((v - mr) * c1);
        }
    st = block_sum_t<4>(st, lds);
    s1 = block_sum_t<4>(s1, lds);
    const float et = en.id >= 0 ? __builtin_amdgcn_exp2f((en.z - mx) * ct) : 0.0f;
    const float e1 = en.id >= 0 ? __builtin_amdgcn_exp2f((en.z - mx) * c1) : 0.0f;
    const float ft = __builtin_amdgcn_exp2f((mr - mx) * ct), f1 = __builtin_amdgcn_exp2f((mr - mx) * c1);
    const float at = st * ft + wave_sum(et), a1 = s1 * f1 + wave_sum(e1);   // of all columns, from mx
    const bool tail = pr > 0.0f && st > 0.0f;
    // loss
    if (threadIdx.x < 64) {
        const double lse = (double)mx * itau + log((double)at);
        double kl = en.id >= 0 && en.p > 0.0f ? pd * (en.lp - ((double)en.z * itau - lse)) : 0.0;
        kl = wave_sum_d(kl);
        if (tail) kl += (double)pr * (log((double)pr) - (log((double)st) + (double)mr * itau - lse));
        double loss = soft ? (double)p.alpha * p.tau * p.tau * kl : 0.0;
        if (has_tg) loss += (1.0 - (double)p.alpha) * ((double)mx + log((double)a1) - (double)zt);
        if (threadIdx.x == 0) p.losses[row] = (float)(loss * w);
    }
    if (!dz) return;
    const float gs = p.scale * w * p.alpha * p.tau, gh = has_tg ? p.scale * w * (1.0f - p.alpha) : 0.0f;
    // the sum of p that the gradient meets: a rest that the student cannot give is left out
    const float mass = tail ? 1.0f : (float)total;
    const float Qs = gs * mass / at, As = gs * (mass * ft / at - (tail ? pr / st : 0.0f));
    const float Bt = gh * f1 / a1, Bs = gh / a1;
    __syncthreads();   // every wave has read what it needs of the row: dz may be z
    for (int c = threadIdx.x; c < V; c += 256) {
        if (listed(c) || (has_tg && (unsigned)c == tg)) continue;
        const float v = act_load(z + c) - mr;
        float g = As * __builtin_amdgcn_exp2f(v * ct);
        if (gh != 0.0f) g += Bt * __builtin_amdgcn_exp2f(v * c1);
        act_store(dz + c, g);
    }
    if (threadIdx.x < 64 && en.id >= 0)
        act_store(dz + en.id, Qs * et - gs * en.p + Bs * e1 - ((unsigned)en.id == tg ? gh : 0.0f));
    if (threadIdx.x == 0 && has_tg && !listed(tg)) {
        const float v = zt - mr;
        act_store(dz + tg, As * __builtin_amdgcn_exp2f(v * ct) + Bt * __builtin_amdgcn_exp2f(v * c1) - gh);
    }
}

}  // namespace asca

using namespace asca;

int asca::distill_check(const char* fn, const DistillTeacher& t, const uint32_t* targets, long T, int V) {
    if (T < 0 || V <= 0) return fail(ASCA_ERR_INVALID, "%s: bad shape %ld x %d", fn, T, V);
    if (V > DISTILL_MAX_V) return fail(ASCA_ERR_UNSUPPORTED, "%s: V=%d (up to %d)", fn, V, DISTILL_MAX_V);
    if (!(t.alpha >= 0.0f && t.alpha <= 1.0f)) return fail(ASCA_ERR_INVALID, "%s: alpha=%g (0 to 1)", fn, (double)t.alpha);
    if (!(t.temperature > 0.0f) || !(t.temperature < INFINITY))
        return fail(ASCA_ERR_INVALID, "%s: temperature %g", fn, (double)t.temperature);
    if (t.alpha > 0.0f && (t.K < 1 || t.K > DISTILL_MAX_K))
        return fail(ASCA_ERR_UNSUPPORTED, "%s: K=%d (1 to %d)", fn, t.K, DISTILL_MAX_K);
    if (T > 0 && t.alpha > 0.0f && (!t.tval || !t.tids))
        return fail(ASCA_ERR_INVALID, "%s: alpha=%g without a teacher", fn, (double)t.alpha);
    if (T > 0 && t.alpha < 1.0f && !targets) return fail(ASCA_ERR_INVALID, "%s: alpha=%g without targets", fn, (double)t.alpha);
    if (!grid_fits(T, 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows (%ld)", fn, T);
    return ASCA_OK;
}

extern "C" {

int asca_distill(const void* logits, long ld, const float* tval, const int32_t* tids, const float* tlse, int K,
                 const uint32_t* targets, const float* weights, float temperature, float alpha, float scale,
                 float* losses, void* dlogits, long lddl, long T, int V, int dtype, void* stream) {
    const char* fn = "asca_distill";
    int rc = distill_check(fn, {tval, tids, tlse, K, weights, temperature, alpha}, targets, T, V);
    if (rc) return rc;
    if (ld < V || (dlogits && lddl < V)) return fail(ASCA_ERR_INVALID, "%s: a row stride below %d columns", fn, V);
    if (!(scale - scale == 0.0f)) return fail(ASCA_ERR_INVALID, "%s: scale=%g", fn, (double)scale);
    if (T > 0 && (!logits || !losses)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (dlogits == logits && dlogits && lddl != ld) return fail(ASCA_ERR_INVALID, "%s: in place with another row stride", fn);
    const uintptr_t el = dtype == ASCA_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % el || reinterpret_cast<uintptr_t>(dlogits) % el)
        return fail(ASCA_ERR_INVALID, "%s: rows at an address that is no multiple of an element", fn);
    return act_dispatch(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        if (T == 0) return (int)ASCA_OK;
        const size_t lds = ((size_t)V + 31) / 32 * 4;
        int r = allow_lds(reinterpret_cast<const void*>(&distill_k<E>), lds);
        if (r || (r = pre_launch("distill"))) return r;
        const DistillArgs a{logits, ld, tval, tids, tlse, targets, weights, losses, dlogits, lddl, T, V, alpha > 0.0f ? K : 0,
                            temperature, alpha, scale};
        hipLaunchKernelGGL(distill_k<E>, dim3((unsigned)T), dim3(256), lds, as_stream(stream), a);
        return post_launch("distill");
    });
}

}  // extern "C"
