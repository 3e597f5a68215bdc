// Distillation from a teacher's largest logits, loss and gradient in one call.  Row of a
// student's logits z, temperature tau, listed ids S with the teacher's logits v:
//   p_k = exp(v_k / tau - tlse), the rest p_r = 1 - sum p one class more; without tlse the
//   softmax of v / tau over the list, and no rest
//   q = softmax(z / tau), q_r = its sum outside S
//   loss = w [(1 - a) (log sum exp z - z_target) + a tau^2 (sum p log(p / q) + p_r log(p_r / q_r))]
//   dz_i / scale = w [(1 - a) (softmax(z)_i - [i = target]) + a tau (q_i - p_i)] for listed i, for
//   the others q_i (1 - p_r / q_r) in the place of q_i - p_i (without tlse q_i)
// Entries of one id are one entry with the sum of their p.
//
// A row has to be read once and its gradient written once: as fast as a copy (5.1 TB/s) where the
// rows are long and many.  The exponentials bound it else: two a value (the sum and the gradient),
// four where two temperatures count, each with one step of its own.  Time of a call, one
// temperature | two, 64 entries a row:
//   16384 x 256 (16 entries) f32 15 | 16.4 us, 12.5 | 13 of them the lists';   4096 x 8192 f32 45 | 46 us, bf16 30 | 40
//   4096 x 32768 f32 200 | 202 (5.3 TB/s), bf16 104 (5.2) | 128;   4096 x 50000 bf16 164 | 206
//   2048 x 131072 f32 559 (read twice), bf16 259 | 321;   8 x 131072 in two launches 10
#include <algorithm>

#include "logits.h"
#include "ops.h"

namespace asca {

constexpr int DISTILL_MAX_K = 64;          // entries a row: one for each lane of a wave
constexpr int DISTILL_MAX_V = 1 << 20;     // columns that the bitmap in LDS has bits for

struct Expo;
struct SplitRow;
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
    double itau;                   // 1 / tau
    int S, slice;                  // a split row's slices
    Expo* parts;                   // (T, S)
    SplitRow* split;               // (T)
};

// A sum of exponentials of some of a row's logits, at the temperature and at 1, and the largest
// of them, from which they are measured (-inf: none, or only -inf; the sums are zero, or NaN)
struct Expo {
    float m, st, s1;
};
// One exponential serves both where the temperatures are one or only one counts (not TWO).
template <bool TWO>
ASCA_DEV Expo expo_join(Expo a, Expo b, float ct) {
    const float m = fmaxf(a.m, b.m);
    auto at = [&](float x, float s, float c) { return x > -INFINITY ? s * __builtin_amdgcn_exp2f((x - m) * c) : s; };
    return {m, at(a.m, a.st, ct) + at(b.m, b.st, ct), TWO ? at(a.m, a.s1, LOG2E) + at(b.m, b.s1, LOG2E) : 0.0f};
}

// An entry of a row's list, one a lane
struct Entry {
    int id;       // below 0: none
    float z, p;   // the student's logit there, and p
    double lp;    // log p, without tlse log(p norm)
};
// What a row's entries are together
struct List {
    Expo e;       // of their logits
    float total;  // sum of p
    float rest;   // what it leaves of 1, with tlse
    float norm;   // without: the sum that made it 1
    float zt;     // the student's logit at the target
};

// 1 / x to 2^-23
ASCA_DEV float recip(float x) { return __builtin_amdgcn_rcpf(x); }

// A row's list, in a wave: id and z are there, tv is the teacher's logit; `twice`: some id may
// be there more than once.  The first of one id's entries has their sum, the others are none.
template <bool TWO>
ASCA_DEV List list_of(const DistillArgs& p, long row, float tv, bool twice, Entry& en) {
    const int lane = threadIdx.x & 63;
    bool on = en.id >= 0;
    List l;
    en.p = 0.0f, l.norm = 1.0f;
    if (p.tlse) {
        en.lp = (double)tv * p.itau - (double)p.tlse[row];
        if (on) en.p = exp_d(en.lp);
    } else {
        const float m = wave_max(on ? tv : -INFINITY), ref = m == -INFINITY ? 0.0f : m;   // no entry, or none above -inf
        en.lp = ((double)tv - (double)ref) * p.itau;
        const float e = on ? exp_d(en.lp) : 0.0f, s = wave_sum(e), r = recip(s);
        if (m != -INFINITY) en.p = e * fmaf(fmaf(-s, r, 1.0f), r, r);
        l.norm = s;
    }
    if (twice) {
        for (int j = 0; j < p.K; ++j) {
            const int id = __builtin_amdgcn_readlane(en.id, j);
            const uint64_t same = __ballot(en.id == id);
            if (id < 0 || (same & (same - 1)) == 0) continue;
            const float sum = wave_sum(en.id == id ? en.p : 0.0f);
            if (lane == j) en.p = sum, en.lp = log_exact(sum) + log_exact(l.norm);
            else if (en.id == id) en.id = -1, en.p = 0.0f;
        }
        on = en.id >= 0;
    }
    l.e.m = wave_max(on ? en.z : -INFINITY);
    const float x = en.z - (l.e.m > -INFINITY ? l.e.m : 0.0f);
    l.e.st = on ? __builtin_amdgcn_exp2f(x * p.ct) : 0.0f;
    l.e.s1 = TWO && on ? __builtin_amdgcn_exp2f(x * LOG2E) : 0.0f;
    l.total = en.p;
    float none = 0.0f;
    wave_sum4(l.e.st, l.e.s1, l.total, none);
    l.rest = p.tlse ? fmaxf(0.0f, 1.0f - l.total) : 0.0f;
    return l;
}

// What a row's gradient is made of: of the others (not listed) As 2^((z - mr) ct) + Bt 2^((z - mr) log2 e),
// of an entry Qs 2^((z - mx) ct) + Bs 2^((z - mx) log2 e) - gs p; gh is taken off at the target.
struct Coefs {
    float mr, mx, As, Bt, Qs, Bs, gs, gh;
};

// The whole row's sums from the others' (o) and the list's, measured from mx, and the share of
// either in them
struct Whole {
    float mx, mr, ft, f1, at, a1;   // ft, f1: from mr to mx at both temperatures
    float qr, gap;                  // q_r, and q_r - p_r
    bool tail;                      // there is a rest that the student can give
};
template <bool TWO>
ASCA_DEV Whole whole_of(const DistillArgs& p, Expo o, const List& l) {
    Whole h;
    h.mx = fmaxf(o.m, l.e.m);
    h.mr = o.m > -INFINITY ? o.m : h.mx;
    auto from = [&](float m, float x) { return m > -INFINITY ? __builtin_amdgcn_exp2f((m - h.mx) * x) : 1.0f; };
    const float fl = from(l.e.m, p.ct);
    h.ft = from(h.mr, p.ct);
    h.a1 = h.at = o.st * h.ft + l.e.st * fl;
    h.f1 = h.ft;
    if (TWO) h.f1 = from(h.mr, LOG2E), h.a1 = o.s1 * h.f1 + l.e.s1 * from(l.e.m, LOG2E);
    h.tail = l.rest > 0.0f && o.st > 0.0f;
    // q_r - p_r as the lists' difference where they are the smaller part: it cancels where student
    // and teacher are near
    h.qr = o.st * h.ft / h.at;
    h.gap = l.total < 0.5f ? l.total - l.e.st * fl / h.at : h.qr - l.rest;
    return h;
}
template <bool TWO>
ASCA_DEV Coefs distill_coefs(const DistillArgs& p, float w, Expo o, const List& l, bool has_tg) {
    const Whole h = whole_of<TWO>(p, o, l);
    Coefs c;
    c.mx = h.mx, c.mr = h.mr;
    c.gs = p.scale * w * p.alpha * p.tau;
    c.gh = has_tg ? p.scale * w * (1.0f - p.alpha) : 0.0f;
    // the sum of p that the gradient meets: a rest that the student cannot give is left out
    const float qt = (h.tail ? 1.0f : l.total) * recip(h.at), q1 = c.gh * recip(h.a1);
    c.Qs = c.gs * qt;
    c.As = c.gs * (h.tail ? h.gap * recip(o.st) : qt * h.ft);
    c.Bs = q1;
    c.Bt = q1 * h.f1;
    if (!TWO) c.As += c.Bt, c.Qs += c.Bs;
    return c;
}
// The loss, by the wave that has the entries, after the gradient: its doubles would stand beside the
// row's registers (4096 x 50000 bf16 204 -> 288 us).  An entry's p (log p - log q) is formed before the
// sum, as the parts of either are much larger than their difference, and the logarithms are taken to
// 1e-10, as tau^2 comes to them: four of them at once in as many lanes.  Rows of 75 with 59 entries at
// temperature 4: error 2e-6 of a loss of 0.5, 4.3e-6 with sums of either and logarithms to 2^-24, which
// were 8% faster (16384 x 256 15.6 -> 16.9 us).
template <bool TWO>
ASCA_DEV float distill_loss(const DistillArgs& p, float w, Expo o, const List& l, const Entry& en, bool has_tg) {
    const Whole h = whole_of<TWO>(p, o, l);
    const int lane = threadIdx.x & 63;
    // p_r near q_r: log(p_r / q_r) from their difference
    const bool near = h.tail && fabsf(h.gap) < 0.3f * h.qr;
    const double logs = log_exact(lane == 0 ? h.at : lane == 1 ? h.a1 : lane == 2 ? l.rest : p.tlse ? o.st : l.norm, near && lane == 2,
                                  -(double)h.gap, 2.0 * (double)h.qr - (double)h.gap);
    const double lt = lane_value(logs, 0), l1 = TWO ? lane_value(logs, 1) : lt;
    double v = 0.0;
    if (p.alpha > 0.0f) {
        const float ref = l.e.m > -INFINITY ? l.e.m : 0.0f;
        // log sum exp((z - ref) / tau), less log norm
        const double base = ((double)h.mx - (double)ref) * p.itau + lt - (p.tlse ? 0.0 : lane_value(logs, 3));
        v = wave_sum(en.p != 0.0f ? (float)((double)en.p * (en.lp - ((double)en.z - (double)ref) * p.itau + base)) : 0.0f);
        if (h.tail) {   // + p_r log(p_r / q_r)
            double r = lane_value(logs, 2);
            if (!near) r += ((double)h.mx - (double)h.mr) * p.itau + lt - lane_value(logs, 3);
            v += (double)l.rest * r;
        }
        v *= (double)p.alpha * p.tau * p.tau;
    }
    if (has_tg) v += (1.0 - (double)p.alpha) * ((double)h.mx + l1 - (double)l.zt);
    return (float)(v * (double)w);
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
    unsigned bits[WORDS ? WORDS : 1];   // a bit for every column of a piece: it is listed
    unsigned edge;                      // and of those outside the pieces, by thread
    Expo part[NW];
    Entry en[64];
    List list;
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

// The values of a piece to the same columns of another row
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

// Marks a listed column (of the row that r is of) in the bitmap; whether it was marked before
template <typename E>
ASCA_DEV bool mark(const Pieces<E>& r, int col, unsigned* bits, unsigned* edge) {
    const int rel = col - r.head;
    const bool in = rel >= 0 && rel < r.nb * Pieces<E>::W;
    const unsigned bit = 1u << (in ? rel & 31 : r.edge_thread(col));
    return (atomicOr(in ? bits + (rel >> 5) : edge, bit) & bit) != 0;
}
// The wave of NW that holds a column
template <typename E, int NW>
ASCA_DEV int wave_of(const Pieces<E>& r, int col) {
    const int rel = col - r.head;
    return rel >= 0 && rel < r.nb * Pieces<E>::W ? rel / Pieces<E>::W % (64 * NW) / 64 : 0;
}

// R pieces a thread of a row, or of a slice of one, in the registers of NW waves
template <typename E, int NW, int R>
struct RowRegs {
    static constexpr int NT = 64 * NW, W = Pieces<E>::W;
    // The sums' exponentials stay for the gradient in rows of a wave with up to 8 values a lane (two
    // temperatures, 16384 x 256 f32 16.1 us without and 15.6 with, bf16 18.8 and 17.4; 16384 x 500 bf16
    // 19.9 and 18.6).  16 values would too (16384 x 1000 f32 27.2 and 24.9, bf16 26.9 and 23.6), but are
    // not kept; in 4 waves they gain nothing (512 x 4000 f32 6.9 either way, 4096 x 8192 44.6).
    static constexpr bool KEEP = NW == 1 && R * W <= 8;
    uint4 raw[R ? R : 1];
    float kt[KEEP ? R * W + 1 : 1], k1[KEEP ? R * W + 1 : 1];
    float ev;   // the column outside the pieces that is the thread's
    int ec;

    // (A branch around the pieces that no thread has costs more than they do: 4096 x 50000 bf16,
    // where these are 3 of 16, 162 -> 191 us.)
    ASCA_DEV void load(const Pieces<E>& r, int tid) {
#pragma unroll
        for (int j = 0; j < R; ++j) raw[j] = r.piece(min(j * NT + tid, r.nb - 1));   // nb > 0 with R > 0
        ec = r.edge(tid);
        ev = -INFINITY;
        if (ec >= 0) ev = act_load(r.p + ec);
    }
    // -inf in the place of what is listed and of what lies past the end; the thread's largest
    ASCA_DEV float mask(const Pieces<E>& r, int tid, const unsigned* bits, unsigned edge) {
        float m = -INFINITY, v[W];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int i = j * NT + tid;
            const unsigned b = bits[i * W / 32] >> (i * W % 32) & ((1u << W) - 1);
            if (i >= r.nb) raw[j] = piece_none<E>();
            if (__ballot(b != 0)) piece_mask(raw[j], b, E());
            piece_again(raw[j]);
            piece_values(raw[j], v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) m = max_or_nan(m, v[k]);
            if (R >= 8) __builtin_amdgcn_sched_barrier(0);   // one piece's values in registers at a time
        }
        if (tid < 32 && edge >> tid & 1) ev = -INFINITY;
        return max_or_nan(m, ev);
    }
    // f of every value and its number
    template <typename F>
    ASCA_DEV void each(F f) {
        float v[W];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            piece_again(raw[j]);
            piece_values(raw[j], v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) f(v[k], j * W + k);
            if (R >= 8) __builtin_amdgcn_sched_barrier(0);
        }
        f(ev, R * W);
    }
    // The wave's sums, from its largest m.  exp2(v c - rc) is one step and the exponential; what
    // rounding m c to rc does is the same in every term and taken off at the end.
    template <bool TWO>
    ASCA_DEV Expo sums(float m, float ct) {
        const float ref = m > -INFINITY ? m : 0.0f, rt = ref * ct, r1 = ref * LOG2E;
        float st = 0.0f, s1 = 0.0f;
        auto add = [&](float a, float b, int i) {
            st += a;
            if (TWO) s1 += b;
            if constexpr (KEEP) kt[i] = a, k1[i] = b;
        };
        if (fabsf(rt) < 65536.0f && fabsf(r1) < 65536.0f) {
            each([&](float v, int i) {
                add(__builtin_amdgcn_exp2f(fmaf(v, ct, -rt)), TWO ? __builtin_amdgcn_exp2f(fmaf(v, LOG2E, -r1)) : 0.0f, i);
            });
            st *= __builtin_amdgcn_exp2f(-fmaf(ref, ct, -rt));
            if (TWO) s1 *= __builtin_amdgcn_exp2f(-fmaf(ref, LOG2E, -r1));
        } else {   // where that would be more than the terms
            each([&](float v, int i) {
                add(__builtin_amdgcn_exp2f((v - ref) * ct), TWO ? __builtin_amdgcn_exp2f((v - ref) * LOG2E) : 0.0f, i);
            });
        }
        float x = 0.0f, y = 0.0f;
        if (TWO) wave_sum4(st, s1, x, y);
        else st = wave_sum(st);
        return {m, st, s1};
    }
    template <typename F>
    ASCA_DEV void store_each(const Pieces<E>& r, int tid, E* d, bool whole, F f) {
        float v[W];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int i = j * NT + tid;
            piece_again(raw[j]);
            piece_values(raw[j], v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = f(v[k], j * W + k);
            if (i < r.nb) row_piece_store<E>(d + r.col(i), whole, v);
            if (R >= 8) __builtin_amdgcn_sched_barrier(0);
        }
        if (ec >= 0) act_store(d + ec, f(ev, R * W));
    }
    // The gradient of everything as if it were not listed
    template <bool TWO>
    ASCA_DEV void store(const Pieces<E>& r, int tid, E* d, const Coefs& c, float ct) {
        const bool whole = (reinterpret_cast<uintptr_t>(d) - reinterpret_cast<uintptr_t>(r.p)) % 16 == 0;
        const float rt = c.mr * ct, r1 = c.mr * LOG2E;
        if (fabsf(rt) < 65536.0f && fabsf(r1) < 65536.0f) {   // as in the sums
            const float A = c.As * __builtin_amdgcn_exp2f(-fmaf(c.mr, ct, -rt));
            const float B = TWO ? c.Bt * __builtin_amdgcn_exp2f(-fmaf(c.mr, LOG2E, -r1)) : 0.0f;
            store_each(r, tid, d, whole, [&](float v, int i) {
                const float g = A * (KEEP ? kt[KEEP ? i : 0] : __builtin_amdgcn_exp2f(fmaf(v, ct, -rt)));
                return TWO ? fmaf(B, KEEP ? k1[KEEP ? i : 0] : __builtin_amdgcn_exp2f(fmaf(v, LOG2E, -r1)), g) : g;
            });
        } else {
            store_each(r, tid, d, whole, [&](float v, int) { return grad_other<TWO>(c, ct, v); });
        }
    }
};

// The list's columns and the target's, over what was written there just now, by the wave that
// wrote it: its stores to an address stay in order.  r and d are of the row or of the slice from c0.
template <typename E, int NW, bool TWO>
ASCA_DEV void store_listed(const DistillArgs& p, const Pieces<E>& r, int c0, int wave, E* d, const Coefs& c, const Entry& en,
                           unsigned tg, bool has_tg, float zt) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    auto mine = [&](int col) { return col >= 0 && col < r.n && (NW == 1 || wave_of<E, NW>(r, col) == wave); };
    if (en.id >= 0 && mine(en.id - c0)) act_store(d + en.id - c0, grad_entry<TWO>(c, p.ct, en.z, en.p, (unsigned)en.id == tg));
    const bool listed = __ballot(has_tg && en.id == (int)tg) != 0;
    if ((threadIdx.x & 63) == 0 && has_tg && !listed && mine((int)tg - c0))
        act_store(d + (int)tg - c0, grad_other<TWO>(c, p.ct, zt) - c.gh);
}

ASCA_DEV unsigned target_of(const DistillArgs& p, long row) { return p.alpha < 1.0f ? p.targets[row] : ~0u; }

// A row without weight is not read
template <typename E>
ASCA_DEV void no_weight(const DistillArgs& p, long row, int c0, int n, int tid, int threads) {
    if (tid == 0 && c0 == 0) p.losses[row] = 0.0f;
    if (p.dz)
        for (int c = tid; c < n; c += threads) act_store(static_cast<E*>(p.dz) + row * p.lddz + c0 + c, 0.0f);
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
    const float w = p.weights ? p.weights[row] : 1.0f;
    if (w == 0.0f) return no_weight<E>(p, row, 0, p.V, tid, NT);
    Entry en{-1, 0.0f, 0.0f, 0.0};
    float tv = 0.0f;
    if (wave == 0 && p.K) {
        const long at = row * p.K + min(lane, p.K - 1);
        en.id = p.tids[at], tv = p.tval[at];
    }
    const Pieces<E> r(z, p.V, R > 0);
    RowRegs<E, NW, R> x;
    x.load(r, tid);
#pragma unroll
    for (int i = tid; i < WORDS; i += NT) l.bits[i] = 0;
    if (tid == 0) l.edge = 0;
    distill_sync<NW>();
    const unsigned tg = target_of(p, row);
    const bool has_tg = tg < (unsigned)p.V;
    List li;
    if (wave == 0) {
        if (lane >= p.K || en.id >= p.V) en.id = -1;
        const float zt = has_tg ? act_load(z + tg) : 0.0f;
        bool twice = false;
        if (en.id >= 0) {
            en.z = act_load(z + en.id);
            twice = mark<E>(r, en.id, l.bits, &l.edge);
        }
        li = list_of<TWO>(p, row, tv, __ballot(twice) != 0, en);
        li.zt = zt;
        if constexpr (NW > 1) {
            l.en[lane] = en;
            if (lane == 0) l.list = li;
        }
    }
    distill_sync<NW>();
    Expo o = x.template sums<TWO>(wave_max(x.mask(r, tid, l.bits, l.edge)), p.ct);
    if constexpr (NW > 1) {
        if (lane == 0) l.part[wave] = o;
        lds_barrier();
        o = l.part[0];
#pragma unroll
        for (int k = 1; k < NW; ++k) o = expo_join<TWO>(o, l.part[k], p.ct);
        en = l.en[lane], li = l.list;
    }
    if (p.dz) {
        const Coefs c = distill_coefs<TWO>(p, w, o, li, has_tg);
        E* dz = static_cast<E*>(p.dz) + row * p.lddz;
        x.template store<TWO>(r, tid, dz, c, p.ct);
        store_listed<E, NW, TWO>(p, r, 0, wave, dz, c, en, tg, has_tg, li.zt);
    }
    if (wave != 0) return;
    const float loss = distill_loss<TWO>(p, w, o, li, en, has_tg);
    if (tid == 0) p.losses[row] = loss;
}

// A few long rows: S slices each, a block's of 4 waves.  The first launch leaves the slices'
// sums, and from the first slice the list; the second forms the gradient.  Both wait for memory and
// the launch (8 x 131072 bf16: 5.5 and 3.9 us, where 4 MB take 1).
struct SplitRow {
    Entry en[64];
    List list;
};
template <typename E, int R, bool TWO>
__global__ __launch_bounds__(256) void distill_part_k(DistillArgs p) {
    constexpr int WORDS = 256 * R * Pieces<E>::W / 32;
    __shared__ DistillLds<4, WORDS> l;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int slice = blockIdx.x % (unsigned)p.S, c0 = slice * p.slice, n = min(p.slice, p.V - c0);
    const long row = blockIdx.x / (unsigned)p.S;
    const E* z = static_cast<const E*>(p.z) + row * p.ld;
    if (p.weights && p.weights[row] == 0.0f) return;
    Entry en{-1, 0.0f, 0.0f, 0.0};
    float tv = 0.0f;
    if (wave == 0 && p.K) {
        const long at = row * p.K + min(lane, p.K - 1);
        en.id = p.tids[at], tv = p.tval[at];
    }
    const Pieces<E> r(z + c0, n, true);
    RowRegs<E, 4, R> x;
    x.load(r, tid);
#pragma unroll
    for (int i = tid; i < WORDS; i += 256) l.bits[i] = 0;
    if (tid == 0) l.edge = 0;
    lds_barrier();
    if (wave == 0) {
        if (lane >= p.K || en.id >= p.V) en.id = -1;
        if (en.id >= c0 && en.id - c0 < n) mark<E>(r, en.id - c0, l.bits, &l.edge);
        if (slice == 0) {
            const unsigned tg = target_of(p, row);
            const float zt = tg < (unsigned)p.V ? act_load(z + tg) : 0.0f;
            if (en.id >= 0) en.z = act_load(z + en.id);
            bool twice = false;   // (the bitmap is of this slice alone)
            for (int j = 0; j < p.K; ++j) twice |= j < lane && en.id >= 0 && __builtin_amdgcn_readlane(en.id, j) == en.id;
            List li = list_of<TWO>(p, row, tv, __ballot(twice) != 0, en);
            li.zt = zt;
            p.split[row].en[lane] = en;
            if (lane == 0) p.split[row].list = li;
        }
    }
    lds_barrier();
    const Expo o = x.template sums<TWO>(wave_max(x.mask(r, tid, l.bits, l.edge)), p.ct);
    if (lane == 0) l.part[wave] = o;
    lds_barrier();
    if (tid == 0) {
        Expo a = l.part[0];
        for (int k = 1; k < 4; ++k) a = expo_join<TWO>(a, l.part[k], p.ct);
        p.parts[blockIdx.x] = a;
    }
}
template <typename E, int R, bool TWO>
__global__ __launch_bounds__(256) void distill_finish_k(DistillArgs p) {
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int slice = blockIdx.x % (unsigned)p.S, c0 = slice * p.slice, n = min(p.slice, p.V - c0);
    const long row = blockIdx.x / (unsigned)p.S;
    const E* z = static_cast<const E*>(p.z) + row * p.ld + c0;
    const float w = p.weights ? p.weights[row] : 1.0f;
    if (w == 0.0f) return no_weight<E>(p, row, c0, n, tid, 256);
    const Pieces<E> r(z, n, true);
    RowRegs<E, 4, R> x;
    if (p.dz) x.load(r, tid);
    const Entry en = p.split[row].en[lane];
    const List li = p.split[row].list;
    const unsigned tg = target_of(p, row);
    const bool has_tg = tg < (unsigned)p.V;
    // S <= 64: a slice a lane, joined in the same order by every wave
    Expo o{-INFINITY, 0.0f, 0.0f};
    if (lane < p.S) o = p.parts[row * p.S + lane];
    const float m = wave_max(o.m);
    o = expo_join<TWO>(o, {m, 0.0f, 0.0f}, p.ct);
    float u = 0.0f, v = 0.0f;
    wave_sum4(o.st, o.s1, u, v);
    o.m = m;
    if (p.dz) {
        const Coefs c = distill_coefs<TWO>(p, w, o, li, has_tg);
        E* dz = static_cast<E*>(p.dz) + row * p.lddz + c0;
        x.template store<TWO>(r, tid, dz, c, p.ct);
        store_listed<E, 4, TWO>(p, r, c0, wave, dz, c, en, tg, has_tg, li.zt);
    }
    if (wave != 0 || slice != 0) return;
    const float loss = distill_loss<TWO>(p, w, o, li, en, has_tg);
    if (tid == 0) p.losses[row] = loss;
}

// Rows that no team's registers hold: read twice, by 1024 threads, the second time mostly from
// a cache (256 rows of 131072 f32 are half of the last-level one's).  2048 of these 559 us, 3.8 TB/s
// of the two passes that it cannot do without; as two launches over batches of 64 MB 726 us.
template <typename E, bool TWO>
__global__ __launch_bounds__(1024) void distill_long_k(DistillArgs p) {
    constexpr int NW = 16, NT = 1024, W = Pieces<E>::W, U = 4;
    extern __shared__ unsigned bits[];
    __shared__ DistillLds<NW, 0> l;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const long row = blockIdx.x;
    const E* z = static_cast<const E*>(p.z) + row * p.ld;
    const float w = p.weights ? p.weights[row] : 1.0f;
    if (w == 0.0f) return no_weight<E>(p, row, 0, p.V, tid, NT);
    Entry en{-1, 0.0f, 0.0f, 0.0};
    float tv = 0.0f;
    if (wave == 0 && p.K) {
        const long at = row * p.K + min(lane, p.K - 1);
        en.id = p.tids[at], tv = p.tval[at];
    }
    const Pieces<E> r(z, p.V, true);
    const int words = (r.nb * W + 31) / 32;
    for (int i = tid; i < words; i += NT) bits[i] = 0;
    if (tid == 0) l.edge = 0;
    const int ec = r.edge(tid);
    float ev = -INFINITY;
    if (ec >= 0) ev = act_load(z + ec);
    lds_barrier();
    const unsigned tg = target_of(p, row);
    const bool has_tg = tg < (unsigned)p.V;
    if (wave == 0) {
        if (lane >= p.K || en.id >= p.V) en.id = -1;
        const float zt = has_tg ? act_load(z + tg) : 0.0f;
        bool twice = false;
        if (en.id >= 0) {
            en.z = act_load(z + en.id);
            twice = mark<E>(r, en.id, bits, &l.edge);
        }
        List li = list_of<TWO>(p, row, tv, __ballot(twice) != 0, en);
        li.zt = zt;
        l.en[lane] = en;
        if (lane == 0) l.list = li;
    }
    lds_barrier();
    if (tid < 32 && l.edge >> tid & 1) ev = -INFINITY;
    const float e = __builtin_amdgcn_exp2f(ev - (ev > -INFINITY ? ev : 0.0f));   // 1, 0 or NaN
    Expo o{ev, e, e};
    for (int i0 = tid; i0 < r.nb; i0 += U * NT) {
        uint4 raw[U];
        Expo n{-INFINITY, 0.0f, 0.0f};
        float v[W];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = r.piece(min(i0 + u * NT, r.nb - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * NT;
            if (i >= r.nb) raw[u] = piece_none<E>();
            else piece_mask(raw[u], bits[i * W / 32] >> (i * W % 32) & ((1u << W) - 1), E());
            piece_values(raw[u], v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) n.m = max_or_nan(n.m, v[k]);
        }
        const float ref = n.m > -INFINITY ? n.m : 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            piece_values(raw[u], v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) {
                n.st += __builtin_amdgcn_exp2f((v[k] - ref) * p.ct);
                if (TWO) n.s1 += __builtin_amdgcn_exp2f((v[k] - ref) * LOG2E);
            }
        }
        o = expo_join<TWO>(o, n, p.ct);
    }
    {
        const float m = wave_max(o.m);
        o = expo_join<TWO>(o, {m, 0.0f, 0.0f}, p.ct);
        float x = 0.0f, y = 0.0f;
        wave_sum4(o.st, o.s1, x, y);
        o.m = m;
    }
    if (lane == 0) l.part[wave] = o;
    lds_barrier();
    o = l.part[0];
    for (int k = 1; k < NW; ++k) o = expo_join<TWO>(o, l.part[k], p.ct);
    en = l.en[lane];
    const List li = l.list;
    if (wave == 0) {
        const float loss = distill_loss<TWO>(p, w, o, li, en, has_tg);
        if (tid == 0) p.losses[row] = loss;
    }
    if (!p.dz) return;
    const Coefs c = distill_coefs<TWO>(p, w, o, li, has_tg);
    E* dz = static_cast<E*>(p.dz) + row * p.lddz;
    const bool whole = (reinterpret_cast<uintptr_t>(dz) - reinterpret_cast<uintptr_t>(z)) % 16 == 0;
    // (dz may be z: a thread writes the pieces that it reads, and all have read the entries)
    // backwards: what was read last is still in a near cache
    for (int i0 = (r.nb - 1) / (U * NT) * (U * NT) + tid; i0 >= 0; i0 -= U * NT) {
        uint4 raw[U];
        float v[W];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = r.piece(min(i0 + u * NT, r.nb - 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * NT;
            piece_values(raw[u], v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = grad_other<TWO>(c, p.ct, v[k]);
            if (i < r.nb) row_piece_store<E>(dz + r.col(i), whole, v);
        }
    }
    if (ec >= 0) act_store(dz + ec, grad_other<TWO>(c, p.ct, ev));
    store_listed<E, NW, TWO>(p, r, 0, wave, dz, c, en, tg, has_tg, li.zt);
}

template <typename E, bool TWO>
static int distill_launch(DistillArgs a, hipStream_t st, const char* fn) {
    constexpr int W = 16 / sizeof(E);
    if (!grid_fits(a.T, 1024)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows (%ld)", fn, a.T);
    const long pieces = (a.V + W - 1) / W, cus = std::max(cu_count(), 1);
    int r;
    // Long rows that leave CUs idle: slices of up to 256 x 8 pieces, at most 64 a row.  Up to 8192
    // pieces the second launch costs what the spread gains but for the fewest rows (16 x 32768 f32
    // 9.7 us against 10.6, 32 rows 10.8 and 10.6); longer ones gain up to half of the CUs (8 x 131072
    // f32 10.3 us against 33, 128 rows 37 against 41, 192 rows 51 and 53).  What 64 slices do not hold is
    // a block's row, read twice (1 x 524288 f32 9.9 us, 1 x 524293 83, 1 x 2^20 180; bf16 rows all fit).
    if (pieces > 1024 * 4 && a.T * (pieces > 1024 * 8 ? 2 : 16) <= cus) {
        const long most = std::min(64l, (pieces + 255) / 256), least = std::min(most, (pieces + 256 * 8 - 1) / (256 * 8));
        const long s = std::max(least, std::min(most, 2 * cus / a.T));
        a.slice = (int)((pieces + s - 1) / s * W);
        a.S = (a.V + a.slice - 1) / a.slice;
        if (a.V - (a.S - 1) * a.slice < 2 * W) --a.S, a.slice += 2 * W;   // no slice without a whole piece
        const int per = (a.slice / W + 255) / 256;
        if (per <= 8) {
            StreamScratch scratch;
            const size_t parts = ((size_t)a.T * a.S * sizeof(Expo) + 15) / 16 * 16;
            if ((r = scratch.get((parts + (size_t)a.T * sizeof(SplitRow)) / 4, st))) return r;
            a.parts = reinterpret_cast<Expo*>(scratch.ws.p);
            a.split = reinterpret_cast<SplitRow*>(reinterpret_cast<char*>(scratch.ws.p) + parts);
            const dim3 grid((unsigned)(a.T * a.S)), block(256);
            void (*part)(DistillArgs) = per <= 1   ? distill_part_k<E, 1, TWO>
                                        : per <= 2 ? distill_part_k<E, 2, TWO>
                                        : per <= 4 ? distill_part_k<E, 4, TWO>
                                                   : distill_part_k<E, 8, TWO>;
            void (*finish)(DistillArgs) = per <= 1   ? distill_finish_k<E, 1, TWO>
                                          : per <= 2 ? distill_finish_k<E, 2, TWO>
                                          : per <= 4 ? distill_finish_k<E, 4, TWO>
                                                     : distill_finish_k<E, 8, TWO>;
            if ((r = pre_launch("distill_part"))) return r;
            hipLaunchKernelGGL(part, grid, block, 0, st, a);
            if ((r = post_launch("distill_part")) || (r = pre_launch("distill_finish"))) return r;
            hipLaunchKernelGGL(finish, grid, block, 0, st, a);
            return post_launch("distill_finish");
        }
    }
    if (pieces > 1024 * 16) {   // more than 16 pieces a thread, 64 registers, in the largest block
        const size_t lds = ((size_t)a.V + 31) / 32 * 4;
        if ((r = allow_lds(reinterpret_cast<const void*>(&distill_long_k<E, TWO>), lds))) return r;
        if ((r = pre_launch("distill_long"))) return r;
        hipLaunchKernelGGL((distill_long_k<E, TWO>), dim3((unsigned)a.T), dim3(1024), lds, st, a);
        return post_launch("distill_long");
    }
    if ((r = pre_launch("distill_rows"))) return r;
    // A wave a row, up to 8 pieces a lane, where there are four rows a CU (2048 x 1000 f32 6.6 us, 9.5
    // in blocks of four waves; 256 rows 4.9 and 5.1), else the fewest waves that hold a row in 64
    // registers each: 1000 x 32001 f32 54 us in 8 waves, 78 in 16.
    const bool many = a.T >= 4 * cus;
    auto go = [&](auto nw, auto rr) {
        constexpr int NW = decltype(nw)::value, R = decltype(rr)::value;
        hipLaunchKernelGGL((distill_rows_k<E, NW, R, TWO>), dim3((unsigned)(NW == 1 ? (a.T + 3) / 4 : a.T)),
                           dim3(NW == 1 ? 256 : 64 * NW), 0, st, a);
    };
    std::integral_constant<int, 0> n0;
    std::integral_constant<int, 1> n1;
    std::integral_constant<int, 2> n2;
    std::integral_constant<int, 4> n4;
    std::integral_constant<int, 8> n8;
    std::integral_constant<int, 16> n16;
    if (a.V < 2 * W) go(n1, n0);   // maybe no whole piece
    else if (pieces <= 64) go(n1, n1);
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
    if (!logits_temperature(t.temperature))
        return fail(ASCA_ERR_INVALID, "%s: temperature %g", fn, (double)t.temperature);
    if (t.alpha > 0.0f && (t.K < 1 || t.K > DISTILL_MAX_K))
        return fail(ASCA_ERR_UNSUPPORTED, "%s: K=%d (1 to %d)", fn, t.K, DISTILL_MAX_K);
    if (T > 0 && t.alpha > 0.0f && (!t.tval || !t.tids))
        return fail(ASCA_ERR_INVALID, "%s: alpha=%g without a teacher", fn, (double)t.alpha);
    if (T > 0 && t.alpha < 1.0f && !targets) return fail(ASCA_ERR_INVALID, "%s: alpha=%g without targets", fn, (double)t.alpha);
    if (!grid_fits(T, 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows (%ld)", fn, T);
    return ASCA_OK;
}

// Whether rows of two matrices share memory; those of one stride may lie between each other
static bool rows_overlap(const void* x, long ldx, const void* y, long ldy, long T, int V, uintptr_t el) {
    typedef __int128_t i128;
    const i128 x0 = (i128)(reinterpret_cast<uintptr_t>(x) / el), y0 = (i128)(reinterpret_cast<uintptr_t>(y) / el);
    if (x0 >= y0 + (i128)(T - 1) * ldy + V || y0 >= x0 + (i128)(T - 1) * ldx + V) return false;
    if (ldx != ldy) return true;
    const i128 m = (x0 < y0 ? y0 - x0 : x0 - y0) % ldx;
    return m < V || ldx - m < V;
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
    if (T > 0 && dlogits && dlogits != logits && rows_overlap(logits, ld, dlogits, lddl, T, V, el))
        return fail(ASCA_ERR_INVALID, "%s: dlogits overlap the logits", fn);
    return act_dispatch(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        if (T == 0) return (int)ASCA_OK;
        // one exponential serves both parts where they have one temperature, or one does not count
        const bool two = alpha > 0.0f && alpha < 1.0f && temperature != 1.0f;
        const float ct = alpha > 0.0f ? (float)(1.4426950408889634 / (double)temperature) : LOG2E;
        const DistillArgs a{logits, ld, tval, tids, tlse, targets, weights, losses, dlogits, lddl, T, V, alpha > 0.0f ? K : 0,
                            alpha > 0.0f ? temperature : 1.0f, ct, alpha, scale, alpha > 0.0f ? 1.0 / (double)temperature : 1.0, 1, V,
                            nullptr, nullptr};
        const hipStream_t st = as_stream(stream);
        return two ? distill_launch<E, true>(a, st, fn) : distill_launch<E, false>(a, st, fn);
    });
}

}  // extern "C"
