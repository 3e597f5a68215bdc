// The largest logits of rows, and a beam search's steps over them: the choice among a
// group's beams and tokens, and the states' move to their beams' new slots.
//   top    the K largest of a row, ties to the lower id; lse = log sum exp(z / tau)
//   step   the K best of s_b + z_bi - lse_b over b and i, ties to the lower b, in one b to the larger
//          z, then to the lower i
//   states slot <- state of parent[slot], in place or into other buffers
//
// top and step have to read the logits once (a copy's rate is 5.1 TB/s) and rank what may be
// listed; time of a call, 16 of a row: 4096 x 16384 f32 42 us (6.4 TB/s, part of it from the
// last-level cache), bf16 26 (5.2); 2048 x 131072 f32 196 (5.5), bf16 102 (5.3); 16384 x 256 f32 10.8
// us, 1.6 TB/s, where the vector unit is busy for 89% of the time (64 of a row: 25 us); 1 x 256 4.3,
// 1 x 32768 8 us, the launches.  A step: 1 x 4 x 256 6.9 us, 64 x 4 x 131072 f32 31 (4.3 TB/s).
#include <algorithm>

#include "logits.h"

namespace asca {

constexpr int TOP_MAX_K = 64;    // listed logits a row
constexpr int BEAM_MAX_K = 32;   // beams a group
constexpr int BEAM_BUFS = 8;     // state buffers a call
constexpr int ROW_MAX_V = 1 << 30;   // columns: ends of slices and of pieces past them are ints

// ------------------------------------------------------------ selection
// A team of NW waves finds the K largest of what it holds in registers.  The K-th largest of
// its lanes' own maxima (of groups of lanes, in a wide team) is at most the K-th largest of
// all, so what lies below it is none of them.  The pieces with something above it, some more
// than K, go to LDS by a ballot for each piece of the wave; a wave looks through its own and
// keeps what is above, and what all waves kept is ranked by counting the larger ones.  Where
// more is left than LDS has room for (rows of equal values, or of a finite mask that leaves
// fewer than K), or a NaN is among them, K rounds take the largest key below the last one, each a
// read of the row: 4096 x 50001 bf16, 64 of them, 18 ms, 4096 x 16384 f32, 16 of them, 1.6 ms, 1 x
// 32768, 8 of them, 25 us; a mask of -inf costs nothing.

template <int NW>
struct TeamLds {
    static constexpr int PIECES = NW == 1 ? 128 : 64, KEYS = NW == 1 ? 256 : 128;   // a wave
    uint4 piece[NW][PIECES];
    unsigned place[NW][PIECES];   // of the piece's first value
    alignas(16) uint64_t keys[NW][KEYS];
    float lists[NW][64], sums[NW], tops[NW];
    uint64_t best[NW];
    int n[NW];                    // keys; above KEYS: too many
    int rank[NW == 1 ? 1 : NW * KEYS];
};

template <int NW>
ASCA_DEV void team_sync() {
    if constexpr (NW == 1) {   // a wave's own LDS accesses, in order
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}
template <int NW>
ASCA_DEV int team_wave() { return NW == 1 ? 0 : wave_id(); }

// The 64 largest of four sorted lists in LDS, sorted
ASCA_DEV float four_lists(const float (&l)[4][64]) {
    const int lane = threadIdx.x & 63;
    const float ab = lane_merge<64>(fmaxf(l[0][lane], l[1][63 - lane]));
    const float cd = lane_merge<64>(-fmaxf(l[2][lane], l[3][63 - lane]));   // backwards
    return lane_merge<64>(fmaxf(ab, -cd));
}

// A value that at least K of the team's x and y reach, near the K-th largest of all that they
// are maxima of (-inf where fewer are above it).  With G groups some G log(G / (G - K)) values
// reach it: 18 for K = 16 of 64, 89 for 64 of 128, 74 for 64 of 256.  64 groups up to K = 16, for a
// second list costs a fifth there (16384 x 256 f32, 16 of them, 10.6 us, 12.7 with two).  They would still
// be faster at K = 32 of most rows (12.5 and 14.0, but 300 bf16 columns 20.1 and 15.9) and slower from 48
// on (20.5 and 15.9); a block's rows hardly differ (4096 x 50001 bf16, 32 of them, 85.1 and 86.7).
// A wave's second group is nearly empty just past 64 pieces: 64 of 16384 x 520 bf16 take 163 us, of 512
// columns 27, of 640 38; of 260 f32 54, of 256 23.
template <int NW>
ASCA_DEV float team_kth(float x, float y, int K, TeamLds<NW>& l) {
    const int lane = threadIdx.x & 63, w = team_wave<NW>();
    if constexpr (NW == 1) {
        if (K <= 16) return lane_value(lane_sort(fmaxf(x, y)), K - 1);
        x = lane_sort(x);   // the larger of one sorted list and another backwards are the largest of both
        l.lists[0][lane] = lane_sort(y);
        team_sync<1>();
        return lane_value(lane_merge<64>(fmaxf(x, l.lists[0][63 - lane])), K - 1);
    } else {
        x = fmaxf(x, y);
        if (K > 16) x = lane_sort(x);
        l.lists[w][lane] = x;
        __syncthreads();
        if (K <= 16) {   // 64 groups of 4 lanes
            x = fmaxf(fmaxf(l.lists[0][lane], l.lists[1][lane]), fmaxf(l.lists[2][lane], l.lists[3][lane]));
            return lane_value(lane_sort(x), K - 1);
        }
        return lane_value(four_lists(l.lists), K - 1);
    }
}

// Appends the lanes' keys (0: none) to the wave's; n is the same in all lanes
template <int NW>
ASCA_DEV void wave_push(uint64_t key, int& n, TeamLds<NW>& l) {
    const uint64_t some = __ballot(key != 0);
    const int at = n + __builtin_amdgcn_mbcnt_hi((unsigned)(some >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)some, 0));
    if (key && at < TeamLds<NW>::KEYS) l.keys[team_wave<NW>()][at] = key;
    n += __popcll(some);
}

// How many of the wave's own keys are larger than each of the team's n, R of these a lane;
// a wide team's waves add theirs up
template <int NW, int R, typename Out>
ASCA_DEV void team_count(int K, int n, TeamLds<NW>& l, Out out) {
    const int lane = threadIdx.x & 63, w = team_wave<NW>();
    uint64_t key[R];
    int rank[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        int i = lane + 64 * r, v = 0;
        key[r] = 0, rank[r] = 0;
        if (i >= n) continue;
#pragma unroll
        for (int u = 0; u < NW - 1; ++u)   // the i-th of all
            if (i >= l.n[u] && v == u) i -= l.n[u], ++v;
        key[r] = l.keys[v][i];
    }
    for (int j = 0; j < l.n[w]; j += 2) {   // (an odd number of them ends in a 0)
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&l.keys[w][j]);
#pragma unroll
        for (int r = 0; r < R; ++r) rank[r] += (two.x > key[r]) + (two.y > key[r]);
    }
    if constexpr (NW > 1) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (lane + 64 * r < n) atomicAdd(&l.rank[lane + 64 * r], rank[r]);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) rank[r] = l.rank[lane + 64 * r];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r % NW == w && lane + 64 * r < n && rank[r] < K) out(rank[r], key[r]);
}

// The keys' end, for all to see: their number, and one 0 more
template <int NW>
ASCA_DEV void wave_end(int n, TeamLds<NW>& l) {
    if constexpr (NW > 1)
        for (int i = threadIdx.x; i < NW * TeamLds<NW>::KEYS; i += 64 * NW) l.rank[i] = 0;
    if ((threadIdx.x & 63) != 0) return;
    l.n[team_wave<NW>()] = n;
    if (n < TeamLds<NW>::KEYS) l.keys[team_wave<NW>()][n] = 0;
}

// The K largest of the waves' keys, whose numbers n the team has seen, to out(rank, key), 0
// where there are fewer.  each(f) calls f with every key of the thread's, for the rounds.
template <int NW, typename Each, typename Out>
ASCA_DEV void team_rank(int K, TeamLds<NW>& l, Each each, Out out) {
    const int tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x, w = team_wave<NW>();
    int all = 0;
    bool fits = true;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int k = l.n[i];
        all += k;
        fits &= k <= TeamLds<NW>::KEYS;
    }
    if (fits) {
        if (all <= 64) team_count<NW, 1>(K, all, l, out);
        else if (all <= 128) team_count<NW, 2>(K, all, l, out);
        else if (all <= 256) team_count<NW, 4>(K, all, l, out);
        else if constexpr (NW > 1) team_count<NW, 8>(K, all, l, out);
        for (int r = all + tid; r < K; r += 64 * NW) out(r, 0);
        return;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < K; ++k) {
        uint64_t best = 0;
        each([&](uint64_t key) {
            if (key < last && key > best) best = key;
        });
        best = wave_max_t(best);
        if constexpr (NW > 1) {
            team_sync<NW>();
            if ((threadIdx.x & 63) == 0) l.best[w] = best;
            team_sync<NW>();
            for (int i = 0; i < NW; ++i) best = l.best[i] > best ? l.best[i] : best;
        }
        last = best;
        if (tid == 0) out(k, best);
    }
}

struct TopArgs {
    const void* z;
    long ld, rows;
    int V, K, S, slice;   // S slices of `slice` columns a row, each a team's
    double itau;          // 1 / tau
    float ct;             // log2(e) / tau
    float* values;        // with S = 1 and no search
    int32_t* ids;
    float* lse;
    uint64_t* keys;       // else (rows, S, K)
    float2* sums;         // (rows, S): the largest and the sum of exp((z - it) / tau)
    const float* scores;  // a search's: rows of beams that have no candidates are not read
    const int32_t* ended;
};

ASCA_DEV bool beam_reads(const TopArgs& p, long row) {
    return !p.scores || (fabsf(p.scores[row]) < INFINITY && !(p.ended && p.ended[row] != 0));
}

ASCA_DEV void top_write(const TopArgs& p, long row, int rank, uint64_t key) {
    p.values[row * p.K + rank] = key ? key_value(key) : -INFINITY;
    p.ids[row * p.K + rank] = key ? (int)key_place(key) : -1;
}

// A slice of a row in R pieces of B bytes a thread.  `out` takes (rank, key), `sum` the slice's largest
// and its sum from one thread.  `fixed`, for a search: the sum is the same at every address, as beams of the
// same logits have to tie.  Rows that are no multiple of 16 bytes are then loaded at any address (64 x 4 x
// 50001 bf16 14.9 -> 16.3 us a step, 16 x 8 13.8 -> 14.3, f32 19.5 either way).
template <typename E, int NW, int R, int B, typename Out, typename Sum>
ASCA_DEV void top_slice(const E* row, int c0, int n, int K, float ct, bool fixed, TeamLds<NW>& l, Out out, Sum sum) {
    constexpr int NT = 64 * NW, W = Pieces<E, B>::W, PIECES = TeamLds<NW>::PIECES;
    typedef typename Pieces<E, B>::Raw Raw;
    const int tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x, lane = threadIdx.x & 63, wave = team_wave<NW>();
    const Pieces<E, B> r(row + c0, n, true, fixed);
    Raw raw[R];
    float cm[R], ma = -INFINITY, mb = -INFINITY, ev = -INFINITY;   // two groups a lane
    const int ec = r.edge(tid);
#pragma unroll
    for (int j = 0; j < R; ++j)
        if (j * NT < r.nb) raw[j] = r.piece(min(j * NT + tid, r.nb - 1));
    if (ec >= 0) ev = act_load(r.p + ec);
    float v[W];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        cm[j] = -INFINITY;
        if (j * NT >= r.nb) continue;   // the whole team's
        if (j * NT + tid >= r.nb) raw[j] = piece_none<E, B>();
        piece_values(raw[j], v, E());
        float a = v[0], b = v[W / 2];
#pragma unroll
        for (int k = 1; k < W / 2; ++k) a = max_or_nan(a, v[k]), b = max_or_nan(b, v[k + W / 2]);
        cm[j] = max_or_nan(a, b);
        if (R == 1) ma = a, mb = b;
        else if (j % 2 == 0) ma = max_or_nan(ma, cm[j]);
        else mb = max_or_nan(mb, cm[j]);
    }
    ma = max_or_nan(ma, ev);
    const bool nan = __ballot(ma != ma || mb != mb) != 0;   // (a maximum that leaves it out takes twice as long)
    // The wave's sum from its own largest.  exp2(v ct - rc) is one step and the exponential; what
    // rounding ref ct to rc does is the same in every term and taken off at the end.
    const float m = wave_max(fmaxf(ma, mb)), ref = m > -INFINITY ? m : 0.0f, rc = ref * ct;
    float s;
    if (fabsf(rc) < 65536.0f) {
        s = __builtin_amdgcn_exp2f(fmaf(ev, ct, -rc));
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (j * NT >= r.nb) continue;
            piece_again(raw[j]);
            piece_values(raw[j], v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) s += __builtin_amdgcn_exp2f(fmaf(v[k], ct, -rc));
        }
        s *= __builtin_amdgcn_exp2f(-fmaf(ref, ct, -rc));
    } else {   // where it would be more than the terms
        s = __builtin_amdgcn_exp2f((ev - ref) * ct);
        for (int j = 0; j < R; ++j) {
            const int i = j * NT + tid;
            if (i >= r.nb) break;
            piece_values(r.piece(i), v, E());
#pragma unroll
            for (int k = 0; k < W; ++k) s += __builtin_amdgcn_exp2f((v[k] - ref) * ct);
        }
    }
    s = wave_sum(s);
    const float kth = team_kth<NW>(ma, mb, K, l);
    // pieces with something to keep, and what it is
    int np = 0, nk = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        if (j * NT >= r.nb) continue;
        const bool some = cm[j] >= kth && cm[j] > -INFINITY;
        const uint64_t which = __ballot(some);
        const int at = np + __builtin_amdgcn_mbcnt_hi((unsigned)(which >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)which, 0));
        if (some && at < PIECES) reinterpret_cast<Raw*>(l.piece[wave])[at] = raw[j], l.place[wave][at] = c0 + r.col(j * NT + tid);
        np += __popcll(which);
    }
    wave_push<NW>(ev >= kth ? logit_key(ev, c0 + ec) : 0, nk, l);
    team_sync<1>();   // the wave's own
    if (np > PIECES || nan) {
        nk = TeamLds<NW>::KEYS + 1;
    } else {
        const E* in = reinterpret_cast<const E*>(l.piece[wave]);
        for (int i = lane; i - lane < np * W; i += 64) {
            const float x = i < np * W ? act_load(in + i) : -INFINITY;
            wave_push<NW>(x >= kth ? logit_key(x, l.place[wave][i / W] + i % W) : 0, nk, l);
        }
    }
    wave_end<NW>(nk, l);
    if (lane == 0) l.sums[wave] = s, l.tops[wave] = m;
    team_sync<NW>();
    if (tid == 0) {
        float t = l.tops[0], u = l.sums[0];
        if constexpr (NW > 1) {
            for (int w = 1; w < NW; ++w) t = fmaxf(t, l.tops[w]);
            u = 0.0f;
            for (int w = 0; w < NW; ++w)   // a wave of nothing but -inf: a sum of zero, or NaN
                u += l.tops[w] > -INFINITY ? l.sums[w] * __builtin_amdgcn_exp2f((l.tops[w] - t) * ct) : l.sums[w];
        }
        sum(t, u);
    }
    team_rank<NW>(
        K, l,
        [&](auto f) {   // rare: from memory
            for (int c = tid; c < n; c += NT) f(logit_key(act_load(r.p + c), c0 + c));
        },
        out);
}

// Teams of NW waves, four waves a block, a slice each
template <typename E, int NW, int R, int B>
__global__ __launch_bounds__(256) void top_slice_k(TopArgs p) {
    constexpr int TEAMS = 4 / NW;
    __shared__ TeamLds<NW> lds[TEAMS];
    const int team = NW == 1 ? wave_id() : 0, slice = NW == 1 ? 0 : blockIdx.x % (unsigned)p.S;
    const long unit = (long)blockIdx.x * TEAMS + team, row = NW == 1 ? unit : blockIdx.x / (unsigned)p.S;   // NW = 1: S = 1
    if (row >= p.rows || !beam_reads(p, row)) return;   // a whole team's
    const int c0 = slice * p.slice, n = min(p.slice, p.V - c0);
    auto out = [&](int rank, uint64_t key) {
        if (p.values) top_write(p, row, rank, key);
        else p.keys[unit * p.K + rank] = key;
    };
    auto sum = [&](float m, float s) {
        if (!p.values) p.sums[unit] = make_float2(m, s);
        else if (p.lse) p.lse[row] = (float)((double)m * p.itau + log_d(s));
    };
    top_slice<E, NW, R, B>(static_cast<const E*>(p.z) + row * p.ld, c0, n, p.K, p.ct, p.scores != nullptr, lds[team], out, sum);
}

// log sum exp of a row from its slices, by a wave: in every lane
ASCA_DEV double slices_lse(const float2* sums, int S, double itau) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY, s = 0.0f;
    for (int i = lane; i < S; i += 64) m = fmaxf(m, sums[i].x);
    m = wave_max(m);
    for (int i = lane; i < S; i += 64)   // of nothing but -inf: a sum of zero, or NaN
        s += sums[i].x > -INFINITY ? sums[i].y * exp_d(((double)sums[i].x - (double)m) * itau) : sums[i].y;
    return (double)m * itau + log_d(wave_sum(s));
}

// The K largest of a row's S K keys by a team of NW waves, with R keys a thread in registers (R = 0:
// read twice)
template <int NW, int R>
__global__ __launch_bounds__(256) void top_merge_k(TopArgs p) {
    constexpr int TEAMS = 4 / NW, NT = 64 * NW;
    __shared__ TeamLds<NW> lds[TEAMS];
    const int team = NW == 1 ? wave_id() : 0, tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    TeamLds<NW>& l = lds[team];
    const long row = (long)blockIdx.x * TEAMS + team;
    if (row >= p.rows) return;
    const uint64_t* keys = p.keys + row * p.S * p.K;
    const int n = p.S * p.K;
    const float is = 1.0f / (float)p.S;
    auto at = [&](int i) -> uint64_t {   // the slices' largest first, over all lanes
        if (i >= n) return 0;
        const int rank = R ? (int)(((float)i + 0.5f) * is) : (int)((unsigned)i / (unsigned)p.S);   // (exact for few)
        return keys[(i - rank * p.S) * p.K + rank];
    };
    uint64_t mine[R ? R : 1];
#pragma unroll
    for (int j = 0; j < R; ++j) mine[j] = at(tid + j * NT);
    auto each = [&](auto f) {   // every key of the team's, and for all of its threads together
        if constexpr (R > 0) {
#pragma unroll
            for (int j = 0; j < R; ++j) f(mine[j], j);
        } else {
            for (int i = tid, j = 0; i - tid < n; i += NT, ++j) f(at(i), j);
        }
    };
    float ma = -INFINITY, mb = -INFINITY;
    each([&](uint64_t key, int j) {
        const float v = key ? key_value(key) : -INFINITY;
        if (j & 1) mb = fmaxf(mb, v);
        else ma = fmaxf(ma, v);
    });
    const float kth = team_kth<NW>(ma, mb, p.K, l);
    int nk = 0;
    each([&](uint64_t key, int) { wave_push<NW>(key && key_value(key) >= kth ? key : 0, nk, l); });
    wave_end<NW>(nk, l);
    team_sync<NW>();
    team_rank<NW>(
        p.K, l, [&](auto f) { each([&](uint64_t key, int) { f(key); }); },
        [&](int rank, uint64_t key) { top_write(p, row, rank, key); });
    if (p.lse && tid < 64) {
        const double s = slices_lse(p.sums + row * p.S, p.S, p.itau);
        if (tid == 0) p.lse[row] = (float)s;
    }
}

// ------------------------------------------------------------- beam search

struct BeamArgs {
    const float* scores;
    const int32_t* ended;
    float* new_scores;
    int32_t* new_ended;
    uint32_t* tokens;
    int32_t* parents;
    int K, V, S, eos, stay;
    const uint64_t* keys;   // (groups K, S, K)
    const float2* sums;     // (groups K, S)
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
    const uint64_t rest = ~firsts & ((1ull << K) - 1);
    int want = __popcll(rest & ((1ull << lane) - 1)), slot = parent;
    if (!first)
        for (int j = 0; j < K; ++j)
            if (!(taken >> j & 1) && want-- == 0) slot = j;
    return slot;
}

constexpr int BEAM_CAP = 512;   // candidates that are ranked in LDS

struct BeamLds {
    double base[BEAM_MAX_K];     // what a beam's logits are added to (-inf: it has no candidates)
    int ended[BEAM_MAX_K];
    float lists[4][64];
    double score[BEAM_CAP];
    uint64_t key[BEAM_CAP];      // a beam's tokens in their order, by logit and id
    int beam[BEAM_CAP];
    double best[16];
    uint64_t best_key[16];
    BeamPick picks[BEAM_MAX_K];
    int count;
};

// A group's picks, best first, in the first K lanes of a wave, to its slots
ASCA_DEV void beam_write(const BeamArgs& p, long group, const BeamPick& pick, const int* ended) {
    const int lane = threadIdx.x & 63;
    const int slot = beam_slot(pick.parent, p.K, p.stay);
    if (lane >= p.K) return;
    const long at = group * p.K + slot;
    const bool some = pick.parent >= 0;
    p.new_scores[at] = some ? (float)pick.score : -INFINITY;
    p.tokens[at] = some ? pick.token : p.eos >= 0 ? (unsigned)p.eos : 0u;
    p.parents[at] = some ? pick.parent : slot;
    if (p.new_ended) p.new_ended[at] = some && (ended[pick.parent] != 0 || (int)pick.token == p.eos);
}

// Whether candidate x of beam b comes before y of beam c.  In one beam the keys' order is that of
// the scores before they are rounded, which may make them equal.
ASCA_DEV bool beam_before(double x, int b, uint64_t key, double y, int c, uint64_t other) {
    return x > y || (x == y && (b < c || (b == c && key > other)));
}

// The K best of a group's candidates by the first 256 threads of a block of NW waves.  As a
// row's selection, with the scores in 64 bits; the threshold compares them rounded to 32, which
// keeps their order.  keys (K, S, K) and sums (K, S) are the group's own.  It is a chain of waits
// (loads, four barriers, the ranking), 6 us for 16 x 8 beams of 4 slices with the vector unit busy
// for 12% of them; one read of every key for both passes over them gained nothing.
template <int NW, typename Keys, typename Sums>
ASCA_DEV void beam_merge(const BeamArgs& p, long group, BeamLds& l, Keys keys, Sums sums) {
    const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), K = p.K, S = p.S, L = K * S;
    // log sum exp of every beam, by as many lanes as its slices need; all beams' at once
    int width = 1;
    while (width < S && width < 64) width *= 2;
    const bool in = w < 4;
    for (int b = tid / width; in && b < (K + 256 / width - 1) / (256 / width) * (256 / width); b += 256 / width) {
        const bool on = b < K;
        const double s = on ? (double)p.scores[group * K + b] : (double)-INFINITY;
        const bool end = on && p.ended && p.ended[group * K + b] != 0, fin = fabs(s) < INFINITY;
        float m = -INFINITY, t = 0.0f;
        const bool read = fin && !end;
        for (int i = tid % width; i < S && read; i += width) m = fmaxf(m, sums[b * S + i].x);
        for (int x = width / 2; x >= 1; x /= 2) m = fmaxf(m, __shfl_xor(m, x, 64));
        for (int i = tid % width; i < S && read; i += width) {   // of nothing but -inf: a sum of zero, or NaN
            const float2 v = sums[b * S + i];
            t += v.x > -INFINITY ? v.y * exp_d((double)v.x - (double)m) : v.y;
        }
        for (int x = width / 2; x >= 1; x /= 2) t += __shfl_xor(t, x, 64);
        const double x = read ? s - ((double)m + log_exact(t)) : s;
        if (on && tid % width == 0) l.base[b] = fin && fabs(x) < INFINITY ? x : (double)-INFINITY, l.ended[b] = end;
    }
    if (tid < K) l.picks[tid] = BeamPick{-INFINITY, -1, 0};
    if (tid == 0) l.count = 0;
    __syncthreads();
    // every candidate: the slices' largest first, over all threads
    const float is = 1.0f / (float)S;
    const int dr = 256 / L, ds = 256 % L;
    auto each = [&](int ranks, auto f) {
        for (int rank = in ? tid / L : ranks, slice = tid % L; rank < ranks; rank += dr, slice += ds) {
            if (slice >= L) {
                slice -= L;
                if (++rank >= ranks) break;
            }
            const int b = (int)(((float)slice + 0.5f) * is);   // slice / S
            const double base = l.base[b];
            if (base == -INFINITY) continue;
            if (l.ended[b]) {
                if (rank == 0 && slice == b * S) f(base, b, (uint64_t)~(unsigned)p.eos);
                continue;
            }
            const uint64_t key = keys[slice * K + rank];
            if (key) f(base + (double)key_value(key), b, key);
        }
    };
    // the threshold: from each slice's first ones, as many of them as there are lanes
    float mx = -INFINITY;
    each(min(K, (255 + L) / L), [&](double x, int, uint64_t) { mx = fmaxf(mx, (float)x); });
    if (in) l.lists[w][lane] = lane_sort(mx);
    __syncthreads();
    const float kth = in ? lane_value(four_lists(l.lists), K - 1) : 0.0f;
    each(K, [&](double x, int b, uint64_t key) {
        if ((float)x < kth) return;
        const int i = atomicAdd(&l.count, 1);
        if (i < BEAM_CAP) l.score[i] = x, l.key[i] = key, l.beam[i] = b;
    });
    __syncthreads();
    const int n = l.count;
    if (n <= BEAM_CAP) {
        for (int i = tid; i < n; i += 64 * NW) {
            const double x = l.score[i];
            const uint64_t key = l.key[i];
            const int b = l.beam[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += beam_before(l.score[j], l.beam[j], l.key[j], x, b, key);
            if (rank < K) l.picks[rank] = BeamPick{x, b, key_place(key)};
        }
    } else {   // rows of equal values: K rounds, each the best below the last
        double last = INFINITY;
        int lastb = 0;
        uint64_t lastk = 0;
        for (int k = 0; k < K; ++k) {
            double v = -INFINITY;
            int vb = BEAM_MAX_K;
            uint64_t vk = 0;
            each(K, [&](double x, int b, uint64_t key) {
                if (beam_before(last, lastb, lastk, x, b, key) && beam_before(x, b, key, v, vb, vk)) v = x, vb = b, vk = key;
            });
            const double top = block_max_t<NW>(v, l.best);
            if (top == -INFINITY) break;
            const int b = -(int)block_max_t<NW>(v == top ? -(double)vb : -(double)BEAM_MAX_K, l.best);
            const uint64_t key = block_max_t<NW>(v == top && vb == b ? vk : (uint64_t)0, l.best_key);
            if (tid == 0) l.picks[k] = BeamPick{top, b, key_place(key)};
            last = top, lastb = b, lastk = key;
        }
    }
    __syncthreads();
    if (w == 0) beam_write(p, group, lane < K ? l.picks[lane] : BeamPick{-INFINITY, -1, 0}, l.ended);
}

// A block a group
__global__ __launch_bounds__(256) void beam_merge_k(BeamArgs p) {
    __shared__ BeamLds l;
    const long group = blockIdx.x;
    beam_merge<4>(p, group, l, p.keys + group * p.K * p.S * p.K, p.sums + group * p.K * p.S);
}

// Rows of R pieces of B bytes a lane: a block's NW waves select from the group's rows in turn, then it
// merges them, in one launch
template <typename E, int R, int B, int NW>
__global__ __launch_bounds__(64 * NW) void beam_small_k(BeamArgs p, TopArgs t) {
    __shared__ BeamLds l;
    __shared__ TeamLds<1> team[NW];
    __shared__ uint64_t keys[BEAM_MAX_K * BEAM_MAX_K];
    __shared__ float2 sums[BEAM_MAX_K];
    const long group = blockIdx.x;
    const int w = wave_id(), K = p.K;
    for (int b = w; b < K; b += NW) {
        const long row = group * K + b;
        if (!beam_reads(t, row)) continue;
        top_slice<E, 1, R, B>(
            static_cast<const E*>(t.z) + row * t.ld, 0, t.V, K, t.ct, true, team[w], [&](int rank, uint64_t key) { keys[b * K + rank] = key; },
            [&](float m, float s) { sums[b] = make_float2(m, s); });
    }
    __syncthreads();
    beam_merge<NW>(p, group, l, keys, sums);
}

struct StatesArgs {
    const char* src[BEAM_BUFS];
    char* dst[BEAM_BUFS];
    unsigned long bytes[BEAM_BUFS];
    unsigned first[BEAM_BUFS], chunks[BEAM_BUFS];   // blocks before each buffer's; blocks a state
    const int32_t* parents;
    int count, groups, ks, kd;
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Words a thread moves for each of up to KM slots: 64 registers (128 with KM = 32 and 16 bytes a
// word).  Half of them for KM = 4 were as fast where states move and twice as slow where none does
// (19 us of empty blocks for 128 x 4 x 1 MB); a loop over several runs a block cost 7% where they do.
template <typename W, int KM>
constexpr int st_u() {
    constexpr int u = 64 * 4 / (KM * (sizeof(W) < 4 ? 4 : (int)sizeof(W)));
    return u < 1 ? 1 : u > 8 ? 8 : u;
}

// A block takes 256 U words of the states of one group in one outer row.  A thread reads its
// words of the slots that change before it writes any, so that a buffer may be its own
// destination; no other thread touches them.  What several slots take from one parent comes
// from memory once, then from a cache.  Bound by memory: 128 x 4 x 1 MB of which half moves 94 us,
// 5.7 TB/s of reads and writes.  Words are 16, 4 or 1 bytes, as all buffers' sizes and addresses allow: 50 x 15
// x 272 KB takes 43 us, with 4 bytes more 40, with 2 bytes more 88.
template <typename W, int KM>
__global__ __launch_bounds__(256) void beam_states_k(StatesArgs p) {
    constexpr int U = st_u<W, KM>();
    int i = 0;
    while (i + 1 < p.count && blockIdx.x >= p.first[i + 1]) ++i;
    const unsigned b = blockIdx.x - p.first[i], unit = b / p.chunks[i], group = unit % p.groups;
    const unsigned long words = p.bytes[i] / sizeof(W), at = (unsigned long)(b % p.chunks[i]) * (256 * U) + threadIdx.x;
    const W* src = reinterpret_cast<const W*>(p.src[i]) + (unsigned long)unit * p.ks * words;
    W* dst = reinterpret_cast<W*>(p.dst[i]) + (unsigned long)unit * p.kd * words;
    int from[KM];   // the slot that is read, -1 where nothing changes
#pragma unroll
    for (int j = 0; j < KM; ++j) {
        const int q = j < p.kd ? p.parents ? p.parents[(long)group * p.kd + j] : 0 : -1;
        from[j] = q < 0 || q >= p.ks || (src == dst && q == j) ? -1 : q;
    }
    W v[KM][U];
#pragma unroll
    for (int j = 0; j < KM; ++j)
        if (from[j] >= 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (at + u * 256 < words) v[j][u] = src[from[j] * words + at + u * 256];
#pragma unroll
    for (int j = 0; j < KM; ++j)
        if (from[j] >= 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (at + u * 256 < words) dst[j * words + at + u * 256] = v[j][u];
}

template <typename W>
static void beam_states_launch(const StatesArgs& a, dim3 grid, hipStream_t st) {
    if (a.kd <= 4) hipLaunchKernelGGL((beam_states_k<W, 4>), grid, dim3(256), 0, st, a);
    else if (a.kd <= 8) hipLaunchKernelGGL((beam_states_k<W, 8>), grid, dim3(256), 0, st, a);
    else if (a.kd <= 16) hipLaunchKernelGGL((beam_states_k<W, 16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((beam_states_k<W, 32>), grid, dim3(256), 0, st, a);
}

}  // namespace asca

using namespace asca;

static int rows_check(const char* fn, long rows, int V, long ld, const void* z, int dtype) {
    if (rows < 0 || V <= 0) return fail(ASCA_ERR_INVALID, "%s: bad shape %ld x %d", fn, rows, V);
    if (V > ROW_MAX_V) return fail(ASCA_ERR_UNSUPPORTED, "%s: V=%d (up to %d)", fn, V, ROW_MAX_V);
    if (ld < V) return fail(ASCA_ERR_INVALID, "%s: row stride %ld below %d columns", fn, ld, V);
    if (reinterpret_cast<uintptr_t>(z) % (dtype == ASCA_F32 ? 4 : 2))
        return fail(ASCA_ERR_INVALID, "%s: logits at an address that is no multiple of an element", fn);
    return ASCA_OK;
}

// Slices of the rows and the launch over them; with a.scores, or where a row has more than one,
// their keys and sums go to scratch (and a.values is cleared).
//   A wave's rows of up to 64 x 4 pieces, or 64 x 8 where there are enough of them for four waves
//   a CU (2048 x 2000 f32, 16 of them, 6.1 us against 8.1 in blocks; 512 rows 5.5 against 4.7).
//   Else a block's, whole up to 256 x 16 pieces: the second launch costs a few rows 3 us, more than
//   their slices' spread gains (64 x 16384 f32 7.1 us against 8.5 in two slices and more; 1 x 4096
//   4.1), and many rows pay for the merge.  Longer ones, and a search's, which are merged in any
//   case (1 x 4 x 32768 bf16 9.9 us, 13.4 with whole rows), in as many slices as give two blocks a CU
//   (64 x 32768 f32 9.0 us, 9.7 with four; 256 rows 12.1 and 11.6).  Whole rows in blocks of 16
//   waves were slower than these (4096 x 16384 f32 120 us against 44; few rows were not tried).
constexpr int TOP_R = 16;   // pieces a thread at most
template <typename E>
static int top_slices(TopArgs& a, StreamScratch& scratch, hipStream_t st, const char* fn) {
    constexpr int W = 16 / sizeof(E);
    const long cus = std::max(cu_count(), 1);
    const int nw = a.V <= 64 * 4 * W || (a.V <= 64 * 8 * W && a.rows >= 4 * cus) ? 1 : 4;
    if (nw == 1 || (!a.scores && a.V <= 256 * TOP_R * W)) {
        a.S = 1;
        a.slice = a.V;
    } else {
        const long least = (a.V + 256l * TOP_R * W - 1) / (256l * TOP_R * W), most = (a.V + 256l * W - 1) / (256l * W);
        const long s = std::max(least, std::min(most, (2 * cus + a.rows - 1) / a.rows));
        a.slice = (int)(((a.V + s - 1) / s + W - 1) / W * W);
        a.S = (a.V + a.slice - 1) / a.slice;
    }
    a.ct = (float)(1.4426950408889634 * a.itau);
    const long units = a.rows * a.S, blocks = nw == 1 ? (units + 3) / 4 : units;
    if (!grid_fits(blocks, 256) || !grid_fits(a.rows, 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows (%ld)", fn, a.rows);
    if (a.S > 1 || a.scores) {
        int rc = scratch.get(((size_t)units * a.K + units) * 2, st);
        if (rc) return rc;
        a.keys = reinterpret_cast<uint64_t*>(scratch.ws.p);
        a.sums = reinterpret_cast<float2*>(a.keys + units * a.K);
        a.values = nullptr;
    }
    int rc = pre_launch("top_slice");
    if (rc) return rc;
    const dim3 grid((unsigned)blocks);
    const int per = (a.slice / W + 64 * nw - 1) / (64 * nw);   // pieces a thread
    void (*k)(TopArgs);
    if (nw == 1) {
        // pieces of 8 bytes where 32 lanes hold the row in pieces of 16: 64 of 256 bf16 logits are
        // ranked from 89 of them then, else from all (16384 rows 63 -> 25 us)
        k = a.V <= 32 * W ? top_slice_k<E, 1, 1, 8>
            : per <= 1    ? top_slice_k<E, 1, 1, 16>
            : per <= 2    ? top_slice_k<E, 1, 2, 16>
            : per <= 4    ? top_slice_k<E, 1, 4, 16>
                          : top_slice_k<E, 1, 8, 16>;
    } else {
        k = per <= 1   ? top_slice_k<E, 4, 1, 16>
            : per <= 2 ? top_slice_k<E, 4, 2, 16>
            : per <= 4 ? top_slice_k<E, 4, 4, 16>
            : per <= 8 ? top_slice_k<E, 4, 8, 16>
                       : top_slice_k<E, 4, 16, 16>;
    }
    hipLaunchKernelGGL(k, grid, dim3(256), 0, st, a);
    return post_launch("top_slice");
}

extern "C" {

int asca_top_logits(const void* logits, long ld, long rows, int V, int K, float temperature, float* values,
                    int32_t* ids, float* lse, int dtype, void* stream) {
    const char* fn = "asca_top_logits";
    int rc = rows_check(fn, rows, V, ld, logits, dtype);
    if (rc) return rc;
    if (K < 1 || K > TOP_MAX_K) return fail(ASCA_ERR_UNSUPPORTED, "%s: K=%d (1 to %d)", fn, K, TOP_MAX_K);
    if (!logits_temperature(temperature))
        return fail(ASCA_ERR_INVALID, "%s: temperature %g", fn, (double)temperature);
    if (rows > 0 && (!logits || !values || !ids)) return fail(ASCA_ERR_INVALID, "null pointer in %s", fn);
    if (!grid_fits(rows, 256)) return fail(ASCA_ERR_UNSUPPORTED, "%s: too many rows (%ld)", fn, rows);   // a merge's blocks
    TopArgs a{};
    a.z = logits, a.ld = ld, a.rows = rows, a.V = V, a.K = K, a.itau = 1.0 / (double)temperature;
    a.values = values, a.ids = ids, a.lse = lse;
    return act_dispatch(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        if (rows == 0) return (int)ASCA_OK;
        const hipStream_t st = as_stream(stream);
        StreamScratch scratch;
        int r = top_slices<E>(a, scratch, st, fn);
        if (r || a.S == 1) return r;
        a.values = values;
        if ((r = pre_launch("top_merge"))) return r;
        // a wave a row where it holds few keys
        const int n = a.S * K;
        if (n <= 256) {
            hipLaunchKernelGGL((n <= 128 ? top_merge_k<1, 2> : top_merge_k<1, 4>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
        } else {
            hipLaunchKernelGGL((n <= 1024 ? top_merge_k<4, 4> : top_merge_k<4, 0>), dim3((unsigned)rows), dim3(256), 0, st, a);
        }
        return post_launch("top_merge");
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
    TopArgs a{};
    a.z = logits, a.ld = ld, a.rows = (long)groups * K, a.V = V, a.K = K, a.itau = 1.0;
    a.scores = scores, a.ended = ended;
    return act_dispatch(dtype, [&](auto* e) {
        using E = std::remove_pointer_t<decltype(e)>;
        if (groups == 0) return (int)ASCA_OK;
        const hipStream_t st = as_stream(stream);
        BeamArgs b{scores, ended, new_scores, new_ended, tokens, parents, K, V, 1, eos < 0 ? -1 : eos, stay, nullptr, nullptr};
        int r;
        const int pieces = (V + 16 / (int)sizeof(E) - 1) / (16 / (int)sizeof(E));
        // Both halves in one launch where a lane holds a few pieces of a row (1 x 4 x 256: 7 us against 8.2,
        // 1000 x 16 x 256 19.5 against 22), or some where its block has a wave for every beam (2 x 4 x 2000
        // f32 8.5 against 9.7, 512 x 4 x 2000 9.7 against 11.9, but 300 x 16 x 2000 29 against 20).
        if (pieces <= 128 || (pieces <= 512 && (K <= 4 || groups <= cu_count()))) {
            if ((r = pre_launch("beam_small"))) return r;
            a.S = 1, a.slice = V, a.ct = LOG2E;
            // a wave a beam where the blocks are few
            const int nw = K <= 4 || groups > 2 * cu_count() ? 4 : K <= 8 ? 8 : 16;
            auto of = [&](auto w) {
                constexpr int NW = decltype(w)::value;
                return pieces <= 32    ? beam_small_k<E, 1, 8, NW>
                       : pieces <= 64  ? beam_small_k<E, 1, 16, NW>
                       : pieces <= 128 ? beam_small_k<E, 2, 16, NW>
                       : pieces <= 256 ? beam_small_k<E, 4, 16, NW>
                                       : beam_small_k<E, 8, 16, NW>;
            };
            void (*k)(BeamArgs, TopArgs) = nw == 4   ? of(std::integral_constant<int, 4>())
                                           : nw == 8 ? of(std::integral_constant<int, 8>())
                                                     : of(std::integral_constant<int, 16>());
            hipLaunchKernelGGL(k, dim3((unsigned)groups), dim3(64 * nw), 0, st, b, a);
            return post_launch("beam_small");
        }
        StreamScratch scratch;
        if ((r = top_slices<E>(a, scratch, st, fn)) || (r = pre_launch("beam_merge"))) return r;
        b.S = a.S, b.keys = a.keys, b.sums = a.sums;
        hipLaunchKernelGGL(beam_merge_k, dim3((unsigned)groups), dim3(256), 0, st, b);
        return post_launch("beam_merge");
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
    uint64_t rows[BEAM_BUFS];
    int which[BEAM_BUFS];
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
        const auto mix = reinterpret_cast<uintptr_t>(src[i]) | reinterpret_cast<uintptr_t>(d) | (uintptr_t)bytes[i];
        while (mix % word) word = word == 16 ? 4 : 1;
        const int n = a.count++;
        a.src[n] = static_cast<const char*>(src[i]);
        a.dst[n] = static_cast<char*>(d);
        a.bytes[n] = bytes[i];
        rows[n] = outer[i];
        which[n] = i;
    }
    // what is written is no other's, and its own source whole or not at all
    auto overlap = [&](const char* x, int i, int kx, const char* y, int j, int ky) {
        const auto x0 = reinterpret_cast<uintptr_t>(x), y0 = reinterpret_cast<uintptr_t>(y);
        return x0 < y0 + (__uint128_t)rows[j] * a.bytes[j] * groups * ky && y0 < x0 + (__uint128_t)rows[i] * a.bytes[i] * groups * kx;
    };
    for (int i = 0; i < a.count; ++i)
        for (int j = 0; j < a.count; ++j)
            if ((a.dst[i] != a.src[j] || i != j) && (overlap(a.dst[i], i, k_dst, a.src[j], j, k_src) ||
                                                     (i != j && overlap(a.dst[i], i, k_dst, a.dst[j], j, k_dst))))
                return fail(ASCA_ERR_INVALID, "%s: the destination of buffer %d overlaps buffer %d", fn, which[i], which[j]);
    if (a.count == 0) return ASCA_OK;
    auto steps = [&](auto w) {
        using W = decltype(w);
        return k_dst <= 4 ? st_u<W, 4>() : k_dst <= 8 ? st_u<W, 8>() : k_dst <= 16 ? st_u<W, 16>() : st_u<W, 32>();
    };
    const uint64_t step = 256ull * word * (word == 16 ? steps(u32x4()) : word == 4 ? steps(uint32_t()) : steps(uint8_t()));
    uint64_t blocks = 0;
    for (int i = 0; i < a.count; ++i) {
        const uint64_t chunks = (a.bytes[i] + step - 1) / step;
        const __uint128_t n = (__uint128_t)chunks * rows[i] * groups + blocks;
        if (n >= (uint64_t)1 << 40 || !grid_fits((long)n, 256))
            return fail(ASCA_ERR_UNSUPPORTED, "%s: too much to move in one call", fn);
        a.first[i] = (unsigned)blocks;
        a.chunks[i] = (unsigned)chunks;
        blocks = (uint64_t)n;
    }
    int rc = pre_launch("beam_states");
    if (rc) return rc;
    const dim3 grid((unsigned)blocks);
    const hipStream_t st = as_stream(stream);
    if (word == 16) beam_states_launch<u32x4>(a, grid, st);
    else if (word == 4) beam_states_launch<uint32_t>(a, grid, st);
    else beam_states_launch<uint8_t>(a, grid, st);
    return post_launch("beam_states");
}

}  // extern "C"
