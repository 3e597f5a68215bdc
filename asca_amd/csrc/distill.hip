// Distillation from a teacher's largest logits, loss and gradient in one call.  Row of a
// student's logits z, temperature tau, listed ids S with the teacher's logits v:
//   p_k = exp(v_k / tau - tlse), the rest p_r = 1 - sum p one class more; without tlse the
//   softmax of v / tau over the list, and no rest
//   q = softmax(z / tau), q_r = its sum outside S
//   loss = w [(1 - a) (log sum exp z - z_target) + a tau^2 (sum p log(p / q) + p_r log(p_r / q_r))]
//   dz_i / scale = w [(1 - a) (softmax(z)_i - [i = target]) + a tau (q_i - p_i)] for listed i, for
//   the others q_i (1 - p_r / q_r) in the place of q_i - p_i (without tlse q_i)
// Entries of one id are one entry with the sum of their p.
#include <algorithm>

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
    float tau, ct, alpha, scale;   // ct = log2(e) / tau
};

// An entry of a row's list, one a lane
struct Entry {
    int id;       // below 0: none
    float z;      // the student's logit there
    double lp;    // log p
    float p;
};

// p of a row's entries (id and the teacher's logit in lp), in a wave; `twice`: some id may
// be there more than once.  The first of one id's entries has their sum, the others are none.
ASCA_DEV void entry_probs(const DistillArgs& p, long row, bool twice, Entry& en, float& total, float& rest) {
    const int lane = threadIdx.x & 63;
    const double itau = 1.0 / (double)p.tau;
    const bool on = en.id >= 0;
    if (p.tlse) {
        en.lp = en.lp * itau - (double)p.tlse[row];
        en.p = on ? exp_d(en.lp) : 0.0f;
    } else {
        const float v = on ? (float)en.lp : -INFINITY, m = wave_max(v);   // a NaN is not the largest
        if (m == -INFINITY) {
            en.lp = -INFINITY;   // no entry, or none above -inf
            en.p = on && v != v ? v : 0.0f;
        } else {
            en.lp = (en.lp - (double)m) * itau;
            const float e = on ? exp_d(en.lp) : 0.0f, s = wave_sum(e);
            en.lp -= log_d(s);
            en.p = e / s;
        }
    }
    if (twice)
        for (int j = 0; j < p.K; ++j) {
            const int id = __builtin_amdgcn_readlane(en.id, j);
            const uint64_t same = __ballot(en.id == id);
            if (id < 0 || (same & (same - 1)) == 0) continue;
            const float sum = wave_sum(en.id == id ? en.p : 0.0f);
            if (lane == j) en.p = sum, en.lp = log_d(sum);
            else if (en.id == id) en.id = -1, en.p = 0.0f;
        }
    total = wave_sum(en.p);
    rest = p.tlse ? fmaxf(0.0f, 1.0f - total) : 0.0f;
}

// The sums over the columns outside the list: the largest of them and their exponentials'
// sums from it, at the temperature and at 1
struct Outside {
    float m, st, s1;
};
ASCA_DEV Outside outside_join(Outside a, Outside b, float ct, bool two) {
    const float m = fmaxf(a.m, b.m), ref = m > -INFINITY ? m : 0.0f;   // sums of nothing are 0, or NaN
    auto at = [&](float x, float s, float c) { return x > -INFINITY ? s * __builtin_amdgcn_exp2f((x - ref) * c) : s; };
    return {m, at(a.m, a.st, ct) + at(b.m, b.st, ct), two ? at(a.m, a.s1, LOG2E) + at(b.m, b.s1, LOG2E) : 0.0f};
}

// What a row's loss and gradient are made of
struct Coefs {
    float mr;          // the others' exponentials are measured from it, the entries' from mx
    float As, Bt;      // dz of the others: As exp((z - mr) / tau) + Bt exp(z - mr)
    float Qs, Bs;      // of an entry: Qs exp((z - mx) / tau) + Bs exp(z - mx) - gs p
    float gs, gh, mx;  // gh is taken off at the target
};

// From the others' sums and the entries, in a wave; the loss where it is wanted.
// Where the temperatures are one, or only one counts, `two` is false and one sum serves both.
template <bool TWO>
ASCA_DEV Coefs distill_coefs(const DistillArgs& p, float w, const Entry& en, float total, float rest, Outside o, bool has_tg, float zt,
                             bool want, float& loss) {
    const bool on = en.id >= 0;
    const float mx = fmaxf(o.m, wave_max(on ? en.z : -INFINITY));   // of the row
    Coefs c;
    c.mx = mx;
    c.mr = o.m > -INFINITY ? o.m : mx;
    const float ft = __builtin_amdgcn_exp2f((c.mr - mx) * p.ct), f1 = TWO ? __builtin_amdgcn_exp2f((c.mr - mx) * LOG2E) : ft;
    const float et = on ? __builtin_amdgcn_exp2f((en.z - mx) * p.ct) : 0.0f;
    const float at = o.st * ft + wave_sum(et);
    float a1 = at;
    if (TWO) a1 = o.s1 * f1 + wave_sum(on ? __builtin_amdgcn_exp2f((en.z - mx) * LOG2E) : 0.0f);
    const bool tail = rest > 0.0f && o.st > 0.0f;
    if (want) {
        const double itau = 1.0 / (double)p.tau, lse = (double)mx * itau + log_d(at);
        float kl = wave_sum(on && en.p != 0.0f ? (float)((double)en.p * (en.lp - ((double)en.z * itau - lse))) : 0.0f);
        double l = 0.0;
        if (p.alpha > 0.0f) {
            l = kl;
            if (tail) l += (double)rest * (log_d(rest) - (log_d(o.st) + (double)c.mr * itau - lse));
            l *= (double)p.alpha * p.tau * p.tau;
        }
        if (has_tg) l += (1.0 - (double)p.alpha) * ((double)mx + log_d(a1) - (double)zt);
        loss = (float)(l * (double)w);
    }
    c.gs = p.scale * w * p.alpha * p.tau;
    c.gh = has_tg ? p.scale * w * (1.0f - p.alpha) : 0.0f;
    // the sum of p that the gradient meets: a rest that the student cannot give is left out
    const float mass = tail ? 1.0f : total;
    c.Qs = c.gs * mass / at;
    c.As = c.gs * (mass * ft / at - (tail ? rest / o.st : 0.0f));
    c.Bs = c.gh / a1;
    c.Bt = c.gh * f1 / a1;
    if (!TWO) c.As += c.Bt, c.Qs += c.Bs;
    return c;
}

template <bool TWO>
ASCA_DEV float grad_other(const Coefs& c, float ct, float z) {
    const float x = z - c.mr;
    const float g = c.As * __builtin_amdgcn_exp2f(x * ct);
    return TWO ? g + c.Bt * __builtin_amdgcn_exp2f(x * LOG2E) : g;
}
template <bool TWO>
ASCA_DEV float grad_entry(const Coefs& c, float ct, float z, float prob, bool target) {
    const float x = z - c.mx;
    const float g = c.Qs * __builtin_amdgcn_exp2f(x * ct) + (TWO ? c.Bs * __builtin_amdgcn_exp2f(x * LOG2E) : 0.0f);
    return g - c.gs * prob - (target ? c.gh : 0.0f);
}

template <int NW, int WORDS>
struct DistillLds {
    unsigned bits[WORDS];   // a bit for every column of a piece: it is listed
    unsigned edge;          // and of those outside the pieces, by thread
    Outside part[NW];
    float z[64], p[64];     // the entries
    int id[64];
    float total, rest, zt;  // zt: the student's logit at the target
};

template <int NW>
ASCA_DEV void distill_sync() {
    if constexpr (NW == 1) {   // a wave's own LDS accesses, in order
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        lds_barrier();         // the row's loads stay in flight
    }
}

// V values of a piece to the same place in another row of the same alignment
ASCA_DEV void piece_store(float* d, const float (&v)[4]) { act_store_n<4>(d, v); }
ASCA_DEV void piece_store(bf16_t* d, const float (&v)[8]) {
    unsigned u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        bf16_t b[2];
        act_store(b, v[2 * k]), act_store(b + 1, v[2 * k + 1]);
        u[k] = b[0] | (unsigned)b[1] << 16;
    }
    *reinterpret_cast<uint4*>(d) = make_uint4(u[0], u[1], u[2], u[3]);
}
template <typename E>
ASCA_DEV void row_piece_store(E* d, bool whole, const float (&v)[16 / sizeof(E)]) {
    if (whole) {
        piece_store(d, v);
    } else {   // the gradient's rows lie otherwise
#pragma unroll
        for (int k = 0; k < 16 / (int)sizeof(E); ++k) act_store(d + k, v[k]);
    }
}

// Rows in the registers of a team of NW waves, R pieces a thread: a row is read once and its
// gradient written once.  The list's columns are taken out by a bitmap in LDS, so that the
// others' sum is formed without them (a difference of sums would lose it where the student is
// sure of the list); the list's own terms are added from one wave's lanes.
template <typename E, int NW, int R, bool TWO>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void distill_rows_k(DistillArgs p) {
    constexpr int NT = 64 * NW, W = Pieces<E>::W, WORDS = NT * R * W / 32, TEAMS = NW == 1 ? 4 : 1;
    __shared__ DistillLds<NW, WORDS> lds[TEAMS];
    const int team = NW == 1 ? wave_id() : 0, tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int lane = threadIdx.x & 63, wave = NW == 1 ? 0 : wave_id();
    const long row = (long)blockIdx.x * TEAMS + team;
    if (row >= p.T) return;
    DistillLds<NW, WORDS>& l = lds[team];
    const E* z = static_cast<const E*>(p.z) + row * p.ld;
    E* dz = p.dz ? static_cast<E*>(p.dz) + row * p.lddz : nullptr;
    const float w = p.weights ? p.weights[row] : 1.0f;
    if (w == 0.0f) {
        if (tid == 0) p.losses[row] = 0.0f;
        if (dz)
            for (int c = tid; c < p.V; c += NT) act_store(dz + c, 0.0f);
        return;
    }
    const bool lists = wave == 0 && lane < p.K;
    Entry en{-1, 0.0f, 0.0, 0.0f};
    float tv = 0.0f;
    if (lists) en.id = p.tids[row * p.K + lane], tv = p.tval[row * p.K + lane];
    const unsigned tg = p.alpha < 1.0f ? p.targets[row] : ~0u;
    const Pieces<E> r(z, p.V);
    uint4 raw[R];
    if (r.nb > 0)
#pragma unroll
        for (int j = 0; j < R; ++j) raw[j] = r.piece(min(j * NT + tid, r.nb - 1));
    const int ec = r.edge(tid);
    float ev = -INFINITY;
    if (ec >= 0) ev = act_load(z + ec);
    const bool has_tg = tg < (unsigned)p.V;
#pragma unroll
    for (int i = tid; i < WORDS; i += NT) l.bits[i] = 0;
    if (tid == 0) l.edge = 0;
    distill_sync<NW>();
    if (wave == 0) {
        bool twice = false;
        const float zt = has_tg ? act_load(z + tg) : 0.0f;
        if (en.id >= p.V) en.id = -1;
        en.lp = tv;
        if (en.id >= 0) {
            en.z = act_load(z + en.id);
            const int rel = en.id - r.head;
            const bool in = rel >= 0 && rel < r.nb * W;
            const unsigned bit = 1u << (in ? rel & 31 : r.edge_thread(en.id));
            twice = (atomicOr(in ? &l.bits[rel >> 5] : &l.edge, bit) & bit) != 0;
        }
        float total, rest;
        entry_probs(p, row, __ballot(twice) != 0, en, total, rest);
        l.id[lane] = en.id, l.z[lane] = en.z, l.p[lane] = en.p;
        if (lane == 0) l.total = total, l.rest = rest, l.zt = zt;
    }
    distill_sync<NW>();
    // the list out of the row, and the others' largest and sums, a wave's own first
    float v[W];
    Outside o{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = j * NT + tid;
        const unsigned bits = l.bits[i * W / 32] >> (i * W % 32) & ((1u << W) - 1);
        if (i >= r.nb) raw[j] = piece_of<E>(-INFINITY);
        if (__ballot(bits != 0)) piece_mask(raw[j], bits, E());
        piece_again(raw[j]);
        piece_values(raw[j], v);
#pragma unroll
        for (int k = 0; k < W; ++k) o.m = max_or_nan(o.m, v[k]);
        if (R >= 8) __builtin_amdgcn_sched_barrier(0);   // one piece's values in registers at a time
    }
    if (l.edge >> (tid & 31) & 1 && tid < 2 * W) ev = -INFINITY;
    o.m = wave_max(fmaxf(o.m, ev));
    const float ref = o.m > -INFINITY ? o.m : 0.0f;
    o.st = __builtin_amdgcn_exp2f((ev - ref) * p.ct);
    if (TWO) o.s1 = __builtin_amdgcn_exp2f((ev - ref) * LOG2E);
#pragma unroll
    for (int j = 0; j < R; ++j) {
        piece_again(raw[j]);
        piece_values(raw[j], v);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            o.st += __builtin_amdgcn_exp2f((v[k] - ref) * p.ct);
            if (TWO) o.s1 += __builtin_amdgcn_exp2f((v[k] - ref) * LOG2E);
        }
        if (R >= 8) __builtin_amdgcn_sched_barrier(0);
    }
    o.st = wave_sum(o.st);
    if (TWO) o.s1 = wave_sum(o.s1);
    if constexpr (NW > 1) {
        if (lane == 0) l.part[wave] = o;
        lds_barrier();
        o = l.part[0];
#pragma unroll
        for (int k = 1; k < NW; ++k) o = outside_join(o, l.part[k], p.ct, TWO);
        if (wave != 0) en.id = l.id[lane], en.z = l.z[lane], en.p = l.p[lane];
    }
    float loss = 0.0f;
    const float zt = l.zt;
    const Coefs c = distill_coefs<TWO>(p, w, en, l.total, l.rest, o, has_tg, zt, wave == 0, loss);
    if (tid == 0) p.losses[row] = loss;
    if (!dz) return;
    const bool whole = (reinterpret_cast<uintptr_t>(dz) - reinterpret_cast<uintptr_t>(z)) % 16 == 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = j * NT + tid;
        piece_again(raw[j]);
        piece_values(raw[j], v);
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = grad_other<TWO>(c, p.ct, v[k]);
        if (i < r.nb) row_piece_store<E>(dz + r.col(i), whole, v);
        if (R >= 8) __builtin_amdgcn_sched_barrier(0);
    }
    if (ec >= 0) act_store(dz + ec, grad_other<TWO>(c, p.ct, ev));
    // the list's columns and the target's, over what was written there just now: by the wave that
    // wrote it, whose stores to an address stay in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    auto mine = [&](int col) {
        const int rel = col - r.head;
        return NW == 1 || (rel >= 0 && rel < r.nb * W ? rel / W % NT / 64 : 0) == wave;
    };
    if (en.id >= 0 && mine(en.id)) act_store(dz + en.id, grad_entry<TWO>(c, p.ct, en.z, en.p, (unsigned)en.id == tg));
    const bool tg_listed = __ballot(has_tg && en.id == (int)tg) != 0;
    if (lane == 0 && has_tg && !tg_listed && mine(tg)) act_store(dz + tg, grad_other<TWO>(c, p.ct, zt) - c.gh);
}

// Rows that no team's registers hold: read twice, by 1024 threads, the second time mostly from
// a cache (256 rows of 131072 f32 are half of the last-level one's)
template <typename E, bool TWO>
__global__ __launch_bounds__(1024) void distill_long_k(DistillArgs p) {
    constexpr int NW = 16, NT = 1024, W = Pieces<E>::W, U = 4;
    extern __shared__ unsigned bits[];
    __shared__ DistillLds<NW, 1> l;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const long row = blockIdx.x;
    const E* z = static_cast<const E*>(p.z) + row * p.ld;
    E* dz = p.dz ? static_cast<E*>(p.dz) + row * p.lddz : nullptr;
    const float w = p.weights ? p.weights[row] : 1.0f;
    if (w == 0.0f) {
        if (tid == 0) p.losses[row] = 0.0f;
        if (dz)
            for (int c = tid; c < p.V; c += NT) act_store(dz + c, 0.0f);
        return;
    }
    Entry en{-1, 0.0f, 0.0, 0.0f};
    float tv = 0.0f;
    if (wave == 0 && lane < p.K) en.id = p.tids[row * p.K + lane], tv = p.tval[row * p.K + lane];
    const unsigned tg = p.alpha < 1.0f ? p.targets[row] : ~0u;
    const bool has_tg = tg < (unsigned)p.V;
    const Pieces<E> r(z, p.V);
    const int words = (r.nb * W + 31) / 32;
    for (int i = tid; i < words; i += NT) bits[i] = 0;
    if (tid == 0) l.edge = 0;
    const int ec = r.edge(tid);
    float ev = -INFINITY;
    if (ec >= 0) ev = act_load(z + ec);
    lds_barrier();
    if (wave == 0) {
        bool twice = false;
        const float zt = has_tg ? act_load(z + tg) : 0.0f;
        if (en.id >= p.V) en.id = -1;
        en.lp = tv;
        if (en.id >= 0) {
            en.z = act_load(z + en.id);
            const int rel = en.id - r.head;
            const bool in = rel >= 0 && rel < r.nb * W;
            const unsigned bit = 1u << (in ? rel & 31 : r.edge_thread(en.id));
            twice = (atomicOr(in ? &bits[rel >> 5] : &l.edge, bit) & bit) != 0;
        }
        float total, rest;
        entry_probs(p, row, __ballot(twice) != 0, en, total, rest);
        l.id[lane] = en.id, l.z[lane] = en.z, l.p[lane] = en.p;
        if (lane == 0) l.total = total, l.rest = rest, l.zt = zt;
    }
    lds_barrier();
    if (tid < 2 * W && l.edge >> tid & 1) ev = -INFINITY;
    Outside o{ev, 0.0f, 0.0f};
    {
        const float ref = ev > -INFINITY ? ev : 0.0f;
        o.st = __builtin_amdgcn_exp2f((ev - ref) * p.ct);   // 1, 0 or NaN
        o.s1 = o.st;
    }
    for (int i0 = tid; i0 < r.nb; i0 += U * NT) {
        uint4 raw[U];
        Outside n{-INFINITY, 0.0f, 0.0f};
        float v[W];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = r.piece(min(i0 + u * NT, r.nb - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * NT;
            if (i >= r.nb) raw[u] = piece_of<E>(-INFINITY);
            else piece_mask(raw[u], bits[i * W / 32] >> (i * W % 32) & ((1u << W) - 1), E());
            piece_values(raw[u], v);
#pragma unroll
            for (int k = 0; k < W; ++k) n.m = max_or_nan(n.m, v[k]);
        }
        const float ref = n.m > -INFINITY ? n.m : 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            piece_values(raw[u], v);
#pragma unroll
            for (int k = 0; k < W; ++k) {
                n.st += __builtin_amdgcn_exp2f((v[k] - ref) * p.ct);
                if (TWO) n.s1 += __builtin_amdgcn_exp2f((v[k] - ref) * LOG2E);
            }
        }
        o = outside_join(o, n, p.ct, TWO);
    }
    {
        const float m = wave_max(o.m);
        const Outside n = outside_join(o, {m, 0.0f, 0.0f}, p.ct, TWO);
        o = {m, wave_sum(n.st), TWO ? wave_sum(n.s1) : 0.0f};
    }
    if (lane == 0) l.part[wave] = o;
    lds_barrier();
    o = l.part[0];
    for (int k = 1; k < NW; ++k) o = outside_join(o, l.part[k], p.ct, TWO);
    if (wave != 0) en.id = l.id[lane], en.z = l.z[lane], en.p = l.p[lane];
    float loss = 0.0f;
    const float zt = l.zt;
    const Coefs c = distill_coefs<TWO>(p, w, en, l.total, l.rest, o, has_tg, zt, wave == 0, loss);
    if (tid == 0) p.losses[row] = loss;
    if (!dz) return;
    const bool whole = (reinterpret_cast<uintptr_t>(dz) - reinterpret_cast<uintptr_t>(z)) % 16 == 0;
    // (dz may be z: a thread writes the pieces that it reads, and all have read the entries)
    for (int i0 = tid; i0 < r.nb; i0 += U * NT) {
        uint4 raw[U];
        float v[W];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = r.piece(min(i0 + u * NT, r.nb - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * NT;
            piece_values(raw[u], v);
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = grad_other<TWO>(c, p.ct, v[k]);
            if (i < r.nb) row_piece_store<E>(dz + r.col(i), whole, v);
        }
    }
    if (ec >= 0) act_store(dz + ec, grad_other<TWO>(c, p.ct, ev));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // as in distill_rows_k
    auto mine = [&](int col) {
        const int rel = col - r.head;
        return (rel >= 0 && rel < r.nb * W ? rel / W % NT / 64 : 0) == wave;
    };
    if (en.id >= 0 && mine(en.id)) act_store(dz + en.id, grad_entry<TWO>(c, p.ct, en.z, en.p, (unsigned)en.id == tg));
    const bool tg_listed = __ballot(has_tg && en.id == (int)tg) != 0;
    if (lane == 0 && has_tg && !tg_listed && mine(tg)) act_store(dz + tg, grad_other<TWO>(c, p.ct, zt) - c.gh);
}

template <typename E, bool TWO>
static int distill_launch(const DistillArgs& a, hipStream_t st) {
    constexpr int W = 16 / sizeof(E);
    const long pieces = (a.V + W - 1) / W;
    int r;
    if (pieces > 1024 * 16) {
        const size_t lds = ((size_t)a.V + 31) / 32 * 4;
        if ((r = allow_lds(reinterpret_cast<const void*>(&distill_long_k<E, TWO>), lds))) return r;
        if ((r = pre_launch("distill_long"))) return r;
        hipLaunchKernelGGL((distill_long_k<E, TWO>), dim3((unsigned)a.T), dim3(1024), lds, st, a);
        return post_launch("distill_long");
    }
    if ((r = pre_launch("distill_rows"))) return r;
    const bool many = a.T >= 4l * std::max(cu_count(), 1);
    auto go = [&](auto nw, auto rr) {
        constexpr int NW = decltype(nw)::value, R = decltype(rr)::value;
        hipLaunchKernelGGL((distill_rows_k<E, NW, R, TWO>), dim3((unsigned)(NW == 1 ? (a.T + 3) / 4 : a.T)), dim3(NW == 1 ? 256 : 64 * NW), 0,
                           st, a);
    };
    std::integral_constant<int, 1> n1;
    std::integral_constant<int, 2> n2;
    std::integral_constant<int, 4> n4;
    std::integral_constant<int, 8> n8;
    std::integral_constant<int, 16> n16;
    if (pieces <= 64) go(n1, n1);
    else if (pieces <= 64 * 2 && many) go(n1, n2);
    else if (pieces <= 64 * 4 && many) go(n1, n4);
    else if (pieces <= 64 * 8 && many) go(n1, n8);
    else if (pieces <= 256) go(n4, n1);
    else if (pieces <= 256 * 2) go(n4, n2);
    else if (pieces <= 256 * 4) go(n4, n4);
    else if (pieces <= 256 * 8) go(n4, n8);
    else if (pieces <= 512 * 8) go(n8, n8);
    else if (pieces <= 512 * 16) go(n8, n16);
    else go(n16, n16);
    return post_launch("distill_rows");
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
        // one exponential serves both parts where they have one temperature, or one does not count
        const bool two = alpha > 0.0f && alpha < 1.0f && temperature != 1.0f;
        const float ct = alpha > 0.0f ? (float)(1.4426950408889634 / (double)temperature) : LOG2E;
        const DistillArgs a{logits, ld, tval, tids, tlse, targets, weights, losses, dlogits, lddl, T, V, alpha > 0.0f ? K : 0,
                            alpha > 0.0f ? temperature : 1.0f, ct, alpha, scale};
        const hipStream_t st = as_stream(stream);
        return two ? distill_launch<E, true>(a, st) : distill_launch<E, false>(a, st);
    });
}

}  // extern "C"
