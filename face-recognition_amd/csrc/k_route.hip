// Routing of rows to experts: scores, balance bias, group limit, the best k, weights, and the slots sorted by expert.
// Three launches: choose (and count a chunk's slots per expert), scan the chunks' counts, place every slot; one for up to
// 64 rows, a single chunk.
#include "adapter.h"

namespace {

constexpr int RT_ROWS = 64;              // rows of a chunk = rows of a block of route_choose_kernel
constexpr int RT_EMAX = 512, RT_KMAX = 16;

struct RouteArgs {
    const void* logits; const float* bias;
    float* weights; int* experts; int* order; int* offsets;
    int* counts;                         // [E + 1][chunks]: slots of a chunk per expert (E: none), then those of earlier chunks
    int* totals;                         // [E + 1]
    long T;
    int type, E, k, score, groups, top_groups, renormalise, chunks;
    float scale;
};

// ---- sums and maxima over the LPR lanes of a row, in every lane of it (all lanes of the wave take part) -----------------
template <int CTRL> FR_DEV unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
template <int LPR, typename F>
FR_DEV unsigned row_fold(unsigned v, F f) {
    v = f(v, dpp<0xB1>(v));                                  // lane ^ 1, lane ^ 2, the other half of 8, of 16
    v = f(v, dpp<0x4E>(v));
    v = f(v, dpp<0x141>(v));
    if constexpr (LPR >= 16) v = f(v, dpp<0x140>(v));
    if constexpr (LPR >= 32) v = f(v, (unsigned)__shfl_xor((int)v, 16, 64));
    if constexpr (LPR >= 64) v = f(v, (unsigned)__shfl_xor((int)v, 32, 64));
    return v;
}
template <int LPR> FR_DEV unsigned row_maxu(unsigned v) { return row_fold<LPR>(v, [](unsigned x, unsigned y) { return max(x, y); }); }
template <int LPR> FR_DEV unsigned row_addu(unsigned v) { return row_fold<LPR>(v, [](unsigned x, unsigned y) { return x + y; }); }
template <int LPR> FR_DEV float row_max(float v) {
    return __uint_as_float(row_fold<LPR>(__float_as_uint(v), [](unsigned x, unsigned y) { return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y))); }));
}
template <int LPR> FR_DEV float row_sum(float v) {
    return __uint_as_float(row_fold<LPR>(__float_as_uint(v), [](unsigned x, unsigned y) { return __float_as_uint(__uint_as_float(x) + __uint_as_float(y)); }));
}

// N unsigned numbers in descending order (Batcher's odd-even merge sort: 63 exchanges for 16, 19 for 8).
template <int N>
FR_DEV void sort_down(unsigned (&v)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j <= N - 1 - k; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (p * 2) == (i + j + k) / (p * 2)) {
                        const unsigned hi = max(v[i + j], v[i + j + k]), lo = min(v[i + j], v[i + j + k]);
                        v[i + j] = hi; v[i + j + k] = lo;
                    }
}

// The weight of a chosen expert with logit l, `top` the greatest chosen logit, m and z the row's greatest and its sum of
// exp(l - m).  What renormalising divides by comes after.
FR_DEV float raw_weight(const RouteArgs& a, float l, float top, float m, float z) {
    if (a.score == FR_SCORE_SOFTMAX) {
        const float against = a.renormalise ? top : m;
        const float w = l == against ? 1.f : expf(l - against);
        return a.renormalise ? w : w / z;
    }
    if (a.renormalise && top < -20.f) return expf(l - top);  // sigmoid(l) = e^l to 2e-9 there
    return 1.f / (1.f + expf(-l));
}

// A group's key from its best two: of fewer than two eligible experts -inf, also where the one has a bias of +inf (inf - inf would
// be a NaN, which no rank counts).
template <typename T> FR_DEV T group_sum(T best, T second, int per) { return per == 1 ? best : second > -INFINITY ? best + second : (T)-INFINITY; }

FR_DEV double dpp_step(double v, int ctrl) {                // ctrl is a constant at every call
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    unsigned lo, hi;
    switch (ctrl) {
        case 0: lo = dpp<0xB1>((unsigned)u); hi = dpp<0xB1>((unsigned)(u >> 32)); break;
        case 1: lo = dpp<0x4E>((unsigned)u); hi = dpp<0x4E>((unsigned)(u >> 32)); break;
        case 2: lo = dpp<0x141>((unsigned)u); hi = dpp<0x141>((unsigned)(u >> 32)); break;
        default: lo = dpp<0x140>((unsigned)u); hi = dpp<0x140>((unsigned)(u >> 32)); break;
    }
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
FR_DEV double lane_of(double v, int lane) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)u, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(u >> 32), lane);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
FR_DEV double wave_max(double v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v = fmax(v, dpp_step(v, i));
    return fmax(fmax(lane_of(v, 0), lane_of(v, 16)), fmax(lane_of(v, 32), lane_of(v, 48)));
}
FR_DEV double wave_sum(double v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v += dpp_step(v, i);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
FR_DEV unsigned wave_minu(unsigned v) {
    v = row_fold<16>(v, [](unsigned x, unsigned y) { return min(x, y); });
    const unsigned a = (unsigned)__builtin_amdgcn_readlane((int)v, 0), b = (unsigned)__builtin_amdgcn_readlane((int)v, 16),
                   c = (unsigned)__builtin_amdgcn_readlane((int)v, 32), d = (unsigned)__builtin_amdgcn_readlane((int)v, 48);
    return min(min(a, b), min(c, d));
}

// The choices of one row by a whole wave, decided in doubles: lane l holds experts l, l + 64, ...; chosen[j] gets the j-th
// (-1: none).  Few rows come here, but a wave that has one holds up its block, and its time is that of fetching
// code that no wave nearby has run, then of the chain of dependent steps: loops stay rolled, maxima take DPP steps.
// (Unrolled over the experts, or with LDS shuffles for every step of a maximum, a row took 30 to 40 us.)
template <int NE>
FR_DEV void choose_exact(const RouteArgs& a, long row, double* keys, int* chosen) {
    const int lane = threadIdx.x & 63;
    const double NONE = -INFINITY;
    const bool scored = a.bias != nullptr || a.groups > 1, soft = a.score == FR_SCORE_SOFTMAX;
    float m = -INFINITY;
    {
        float l[NE];
#pragma unroll
        for (int q = 0; q < NE; ++q) l[q] = lane + 64 * q < a.E ? load1(a.logits, row * a.E + lane + 64 * q, a.type) : -INFINITY;
#pragma unroll
        for (int q = 0; q < NE; ++q) {
            l[q] = l[q] > -INFINITY ? l[q] : -INFINITY;      // NaN masks too
            m = fmaxf(m, l[q]);
            keys[lane + 64 * q] = l[q];
        }
    }
    m = row_max<64>(m);
    double z = 0.0;
    if (scored || soft) {
#pragma unroll 1
        for (int e = lane; e < 64 * NE; e += 64) {
            const double l = keys[e], x = l == (double)m && soft ? 1.0 : exp(soft ? l - (double)m : -l);
            const double s = !(l > NONE) ? 0.0 : soft ? x : 1.0 / (1.0 + x);
            z += s;
            if (scored) keys[e] = l > NONE ? s : NONE;
        }
        if (soft) z = wave_sum(z);
    }
    if (scored) {
        const double rz = soft ? z : 1.0;
#pragma unroll 1
        for (int e = lane; e < a.E; e += 64) {
            const float b = a.bias ? a.bias[e] : 0.f;
            const double s = keys[e];
            keys[e] = s > NONE && b > -INFINITY ? s / rz + (double)b : NONE;
        }
    }
    wave_lds_fence();
    if (a.groups > 1) {
        // 64 / groups lanes a group, each its part of it; the first of them joins the parts
        const int per = a.E / a.groups, n = 64 / a.groups, g = lane / n;
        double b1 = NONE, b2 = NONE;
        if (g < a.groups) {
#pragma unroll 1
            for (int i = lane - g * n; i < per; i += n) {
                const double v = keys[g * per + i];
                b2 = fmax(b2, fmin(b1, v));
                b1 = fmax(b1, v);
            }
        }
        double g1 = b1, g2 = b2;
#pragma unroll 1
        for (int p = 1; p < n; ++p) {
            const double o1 = __shfl(b1, (lane + p) & 63, 64), o2 = __shfl(b2, (lane + p) & 63, 64);
            g2 = fmax(fmin(g1, o1), fmax(g2, o2));
            g1 = fmax(g1, o1);
        }
        const double sum = group_sum(g1, g2, per);           // right in the first lane of each group
        int rank = 0;
#pragma unroll 1
        for (int o = 0; o < a.groups; ++o) {
            const double v = lane_of(sum, o * n);
            if (v > sum || (v == sum && o < g)) ++rank;
        }
        const bool drop = g < a.groups && __shfl(rank, g * n, 64) >= a.top_groups;
        if (drop) {
#pragma unroll 1
            for (int i = lane - g * n; i < per; i += n) keys[g * per + i] = NONE;
        }
        wave_lds_fence();
    }
    int j = 0;
#pragma unroll 1
    for (; j < a.k; ++j) {
        double own = NONE;
        unsigned at = RT_EMAX;
#pragma unroll
        for (int q = 0; q < NE; ++q) {
            const double v = keys[lane + 64 * q];
            if (v > own) { own = v; at = lane + 64 * q; }
        }
        const double best = wave_max(own);
        if (best == NONE) break;
        at = wave_minu(own == best ? at : RT_EMAX);
        if (lane == (int)(at & 63)) { keys[at] = NONE; chosen[j] = (int)at; }
        wave_lds_fence();
    }
    if (lane >= j && lane < a.k) chosen[lane] = -1;
    wave_lds_fence();
}

// The experts of a chunk's slots, 64 rows * k: k a lane.
struct Slots { int ex[RT_KMAX]; };
FR_DEV Slots load_slots(const int* experts, int n) {
    const int lane = threadIdx.x & 63;
    Slots s;
#pragma unroll
    for (int j = 0; j < RT_KMAX; ++j) s.ex[j] = j * 64 + lane < n ? experts[j * 64 + lane] : 0;
    return s;
}
// Their places, by one wave: next[e] is the place of expert e's first slot here (E: none).  Equal experts among 64 slots find
// each other by the bits of their number.
FR_DEV void place_slots(const RouteArgs& a, int* next, const Slots& s, int n, long slot0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < RT_KMAX; ++j) {
        if (j * 64 >= n) break;
        const bool on = j * 64 + lane < n;
        const int e = s.ex[j] < 0 ? a.E : s.ex[j];
        unsigned long long same = __ballot(on);              // lanes with this lane's expert
        for (int bit = 0; (1 << bit) <= a.E; ++bit) {
            const bool set = (e >> bit) & 1;
            const unsigned long long with = __ballot(set);
            same &= set ? with : ~with;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        int base = 0;
        if (on) base = next[e];
        wave_lds_fence();
        if (on) a.order[base + rank] = (int)(slot0 + j * 64 + lane);
        if (on && rank == 0) next[e] = base + __popcll(same);
        wave_lds_fence();
    }
}
// next[e] = sum of n(0 .. e - 1) + more(e) for e <= E, by one wave; the sums alone also go to a.offsets if `write`.
template <typename F, typename G>
FR_DEV void first_places(const RouteArgs& a, int* next, bool write, F n, G more) {
    const int lane = threadIdx.x & 63;
    int c[RT_EMAX / 64 + 1], m[RT_EMAX / 64 + 1];            // all asked for before the first is used
#pragma unroll
    for (int q = 0; q <= RT_EMAX / 64; ++q) {
        const int e = q * 64 + lane;
        c[q] = e <= a.E ? n(e) : 0;
        m[q] = e <= a.E ? more(e) : 0;
    }
    int before = 0;
#pragma unroll
    for (int q = 0; q <= RT_EMAX / 64; ++q) {
        if (q * 64 > a.E) break;
        const int e = q * 64 + lane;
        const int s = scan_add(c[q]);
        if (e <= a.E) {
            next[e] = before + s - c[q] + m[q];
            if (write) a.offsets[e] = before + s - c[q];
        }
        before += __builtin_amdgcn_readlane(s, 63);
    }
    wave_lds_fence();
}

// A row takes LPR > k lanes, a lane up to V experts of one group, in index order over the lanes.  A lane sorts its keys, and
// the k best (and one more, for the doubt) are maxima over the row of the lanes' heads.  Keys are unique in their lane: f32
// in unsigned order, the low bits replaced by an index (greater for lower ones).
// BY_LOGIT (no bias, one group): the logits themselves, with the expert's number in NB bits: unique in the row, ties need no
// care, and with 16-bit logits nothing is lost.
// BY_LOGIT_IN_GROUPS (no bias, 16 bits): the same key; only the groups are compared by their scores.  By scores, whose equal
// ones made nearly every row a doubtful one, 171 x 204, 8 of 204 in 4 groups, took 59 us, and takes 24.
// BY_SCORE: score and bias, with the place in the lane in NB = 4 bits.
// A row is done again by the whole wave in doubles where f32 cannot vouch for the choice: where two neighbours in the order
// (or the groups on either side of the cut) are no further apart than the bits dropped and the error of their scores, which
// is at most 4 steps of 2^-24 for a sigmoid (exp2's argument and result, the sum, the reciprocal) and 32 for a softmax
// (the row's sum of up to 512 besides).  At 65536 x 256, biased sigmoids, 8 of 256 in 4 of 8 groups, one row in 500 goes
// that way; with the expert's number in the scored keys too it was one in 50, which took more time than all the rest.
// What bounds it: 970 vector and 370 scalar instructions for 4 rows of 256.  At 65536 x 256 (traced by itself 50 us; the read alone
// would take 15) vector instructions hold the SIMDs for two thirds of that, and a wave lives 40 us in the mean: the one round of
// blocks waits for the waves with rows that doubles decide (about 120 rows, 8.5 us each, one after the other).
enum { BY_LOGIT, BY_SCORE, BY_LOGIT_IN_GROUPS };
template <int V, int LPR, int NE, int NB, int ORDER>
__global__ __launch_bounds__(512, 4) void route_choose_kernel(RouteArgs a) {
    constexpr bool SCORED = ORDER != BY_LOGIT, by_logit = ORDER == BY_LOGIT_IN_GROUPS;
    __shared__ int count[RT_EMAX + 1];
    __shared__ int chosen[RT_ROWS * RT_KMAX];
    __shared__ float bias[SCORED ? RT_EMAX + V : 1];
    extern __shared__ double keys[];                         // [waves][NE * 64]
    constexpr unsigned MASK = (1u << NB) - 1;
    constexpr int RPW = 64 / LPR;
    constexpr float L2E = 1.4426950408889634f, DROP = 1.f / (float)(1u << (23 - NB));
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63, rl = lane % LPR, base = lane - rl;
    for (int e = threadIdx.x; e <= a.E; e += blockDim.x) count[e] = 0;
    if constexpr (SCORED)                                    // in LDS: registers are what limits the waves a SIMD holds
        for (int e = threadIdx.x; e < RT_EMAX + V; e += blockDim.x) {
            const float b = a.bias && e < a.E ? a.bias[e] : 0.f;
            bias[e] = b > -INFINITY ? b : -INFINITY;         // NaN masks too; added to a score, -inf masks it
        }
    __syncthreads();
    static_assert(!SCORED || V <= 1 << NB, "a lane's keys are unique");
    const bool need_z = SCORED || !a.renormalise;
    const int per = a.E / a.groups, LG = (per + V - 1) / V, g = rl / LG, part = rl - g * LG;
    const float slack = a.score == FR_SCORE_SOFTMAX ? 0x1p-18f : 0x1p-21f;
    const int e0 = g * per + part * V, cnt = g < a.groups ? min(V, per - part * V) : 0;
#pragma unroll 1
    for (int it = wave; it * RPW < RT_ROWS && (long)blockIdx.x * RT_ROWS + it * RPW < a.T; it += waves) {
        const int r = it * RPW + lane / LPR;
        const long row = (long)blockIdx.x * RT_ROWS + r;
        const int have = row < a.T ? cnt : 0;
        float l[V];
#pragma unroll
        for (int c = 0; c < V; c += 8) {
            Vec8f x;
            if (have - c >= 8) x = raw_to_f(raw_load8<false>(a.logits, row * a.E + e0 + c, a.type), a.type);
            else {
#pragma unroll
                for (int v = 0; v < 8; ++v) x.v[v] = c + v < have ? load1(a.logits, row * a.E + e0 + c + v, a.type) : -INFINITY;
            }
#pragma unroll
            for (int v = 0; v < 8; ++v) l[c + v] = x.v[v] > -INFINITY ? x.v[v] : -INFINITY;      // NaN masks too
        }
        float m = 0.f, z = 1.f;
        if (a.score == FR_SCORE_SOFTMAX && need_z) {
            m = l[0];
#pragma unroll
            for (int v = 1; v < V; ++v) m = fmaxf(m, l[v]);
            m = row_max<LPR>(m);
        }
        float f[V];                                          // keys: logits or scores + bias; -inf: masked
        if (a.score == FR_SCORE_SOFTMAX && need_z) {
            z = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f[v] = l[v] == m ? 1.f : __builtin_amdgcn_exp2f((l[v] - m) * L2E);
                z += l[v] > -INFINITY ? f[v] : 0.f;
            }
            z = row_sum<LPR>(z);
        }
        if constexpr (SCORED) {
            const float rz = __builtin_amdgcn_rcpf(z);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float s = a.score == FR_SCORE_SOFTMAX ? f[v] * rz : __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-l[v] * L2E));
                f[v] = l[v] > -INFINITY ? s + bias[min(e0, RT_EMAX) + v] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) f[v] = l[v] + 0.f;   // -0 is 0
        }
        bool doubt = false;
        unsigned kept = ~0u;                                 // all bits or none
        if (SCORED && a.groups > 1) {
            float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                b2 = __builtin_amdgcn_fmed3f(b1, b2, f[v]);
                b1 = fmaxf(b1, f[v]);
            }
            float g1 = b1, g2 = b2;
            for (int p = 1; p < LG; ++p) {
                const int from = base + g * LG + (part + p >= LG ? part + p - LG : part + p);
                const float o1 = __shfl(b1, from, 64), o2 = __shfl(b2, from, 64);
                g2 = fmaxf(fminf(g1, o1), fmaxf(g2, o2));
                g1 = fmaxf(g1, o1);
            }
            const float sum = group_sum(g1, g2, per);
            int rank = 0;
            for (int o = 0; o < a.groups; ++o) {
                const float v = __shfl(sum, base + o * LG, 64);
                if (v > sum || (v == sum && o < g)) ++rank;
            }
            const bool keep = g < a.groups && rank < a.top_groups;
            kept = keep ? ~0u : 0u;
            if (a.top_groups < a.groups) {
                // Where the sum may lie: a key is off by its score's error and its rounding, relative to its own size (the sum of
                // two large keys of either sign may be small), and both sums and bounds round again: at most 7 (softmax 35) steps
                // of 2^-24 of the keys' sizes, which slack covers.  A sum beyond f32's range is at least its greatest number.
                const float err = slack * (fmaxf(1.f, fabsf(g1)) + (per > 1 ? fmaxf(1.f, fabsf(g2)) : 0.f));
                const float lo = fminf(sum, 0x1.fffffep127f) - err, hi = sum > -INFINITY ? sum + err : -INFINITY;
                const float least = -row_max<LPR>(keep ? -lo : -INFINITY), most = row_max<LPR>(!keep && g < a.groups ? hi : -INFINITY);
                // a row without any eligible expert needs no second look
                doubt = !(least > most) && row_max<LPR>(b1) > -INFINITY;
            }
        }
        constexpr unsigned NUMBER = RT_EMAX - 1;
        unsigned key[V];                                     // up to that of -inf: not to be chosen
#pragma unroll
        for (int v = 0; v < V; ++v) {
            unsigned u = __float_as_uint(by_logit ? l[v] + 0.f : f[v]);
            u ^= (unsigned)((int)u >> 31) | 0x80000000u;
            if (by_logit) key[v] = ((u & ~NUMBER) | (NUMBER - min((unsigned)(e0 + v), NUMBER))) & kept;
            else key[v] = ((u & ~MASK) | (MASK - (unsigned)(SCORED ? v : e0 + v))) & kept;
        }
        constexpr unsigned LEAST = 0x007FFFFFu | MASK;
        sort_down<V>(key);
        unsigned mine = 0, wins = 0;                         // lane j <= k of the row: its j-th key
        if (SCORED && rl < a.k) chosen[r * a.k + rl] = -1;
        wave_lds_fence();
        for (int j = 0; j <= a.k; ++j) {
            const unsigned max0 = row_maxu<LPR>(key[0]), top = max0 > LEAST ? max0 : 0u;
            if (rl == j) mine = top;
            const bool here = key[0] == top && top;
            if constexpr (SCORED) {
                if (here && j < a.k) chosen[r * a.k + j] = by_logit ? (int)(NUMBER - (top & NUMBER)) : e0 + (int)(MASK - (top & MASK));
                wins += here;
            }
            const unsigned pop = here ? ~0u : 0u;            // the winner's next key moves up: one bit select a key
            if (V <= 8 || a.k <= 8) {                        // no more than k + 1 rounds: nothing behind the ninth key becomes a head
#pragma unroll
                for (int v = 0; v < (V <= 8 ? V - 1 : 8); ++v) key[v] = (key[v + 1] & pop) | (key[v] & ~pop);
                if (V <= 8) key[V - 1] &= ~pop;
            } else {
#pragma unroll
                for (int v = 0; v + 1 < V; ++v) key[v] = (key[v + 1] & pop) | (key[v] & ~pop);
                key[V - 1] &= ~pop;
            }
        }
        {
            const unsigned x = (unsigned)__shfl((int)mine, max(lane - 1, base), 64) & ~MASK, y = mine & ~MASK;
            bool close = false;                              // this lane's key to the one before
            if constexpr (!SCORED) close = a.type == FR_TYPE_F32 && x == y;
            else if constexpr (by_logit) {
                // but for logits whose neighbours in their type may have the same score in doubles, which the lower expert wins:
                // sigmoids next to 1 (steps of 2^-6 times e^-30 still show), scores below e^-600, logits below 2^-30
                const unsigned w = mine & ~NUMBER;
                const float t = __uint_as_float(w & 0x80000000u ? w ^ 0x80000000u : ~w);
                close = t > (a.score == FR_SCORE_SOFTMAX ? INFINITY : 30.f) || t - m < -600.f || (t != 0.f && fabsf(t) < 0x1p-30f);
            } else {
                const float fx = __uint_as_float(x & 0x80000000u ? x ^ 0x80000000u : ~x), fy = __uint_as_float(y & 0x80000000u ? y ^ 0x80000000u : ~y);
                close = !(fx - fy > slack * fmaxf(1.f, fabsf(fx)) + 2.f * DROP * fmaxf(fabsf(fx), fabsf(fy)));
            }
            unsigned flag = close && mine && (rl > 0 || by_logit) && rl <= a.k;
            // equal keys of two lanes win the same round: more wins than keys
            if constexpr (SCORED) flag |= row_addu<LPR>(wins) != row_addu<LPR>(mine && rl <= a.k ? 1u : 0u);
            doubt |= row_maxu<LPR>(flag) != 0;
        }
        // lane j < k of the row: its j-th choice
        if (!SCORED && rl < a.k) chosen[r * a.k + rl] = mine ? (int)(MASK - (mine & MASK)) : -1;
        wave_lds_fence();
        unsigned long long again = __ballot(doubt && row < a.T && rl == 0);
        while (again) {
            const int rr = it * RPW + (__ffsll(again) - 1) / LPR;
            again &= again - 1;
            choose_exact<NE>(a, (long)blockIdx.x * RT_ROWS + rr, keys + wave * NE * 64, chosen + rr * a.k);
        }
        const int pick = rl < a.k && row < a.T ? chosen[r * a.k + rl] : -1;
        const float pl = pick >= 0 ? load1(a.logits, row * a.E + pick, a.type) : -INFINITY;
        const float best = row_max<LPR>(pl);
        float w = pick >= 0 ? raw_weight(a, pl, best, m, z) : 0.f;
        if (a.renormalise) {
            const float sum = row_sum<LPR>(w);
            if (sum > 0.f) w /= sum;
        }
        if (rl < a.k && row < a.T) {
            a.weights[row * a.k + rl] = w * a.scale;
            a.experts[row * a.k + rl] = pick;
            atomicAdd(&count[pick >= 0 ? pick : a.E], 1);    // whole numbers: any order gives the same
        }
    }
    __syncthreads();
    if (a.chunks > 1) {
        for (int e = threadIdx.x; e <= a.E; e += blockDim.x) a.counts[(long)e * a.chunks + blockIdx.x] = count[e];
    } else if (wave == 0) {                                  // one chunk is all: order it here, one launch in place of three
        first_places(a, count, true, [&](int e) { return count[e]; }, [](int) { return 0; });
        place_slots(a, count, load_slots(chosen, (int)(a.T * a.k)), (int)(a.T * a.k), 0);
    }
}

// counts[e][c] -> number of e's slots in the chunks before c; totals[e].  One block per expert, four chunks a thread: 3 to 5 us for
// 256 x 1024, launch and latency.
__global__ __launch_bounds__(256) void route_scan_kernel(RouteArgs a) {
    __shared__ int part[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int* row = a.counts + (long)blockIdx.x * a.chunks;
    int before = 0, turn = 0;
    for (int c0 = 0; c0 < a.chunks; c0 += 1024, ++turn) {
        const int c = c0 + threadIdx.x * 4;
        int n[4], t = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { n[j] = c + j < a.chunks ? row[c + j] : 0; t += n[j]; }
        const int s = scan_add(t);
        int* p = part[turn & 1];
        if (lane == 63) p[wave] = s;
        __syncthreads();
        int at = before + s - t;
#pragma unroll
        for (int w = 0; w < 4; ++w) { if (w < wave) at += p[w]; before += p[w]; }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (c + j < a.chunks) row[c + j] = at;
            at += n[j];
        }
    }
    if (threadIdx.x == 0) a.totals[blockIdx.x] = before;
}

// Places of a chunk's slots: first place of the expert + its slots in earlier chunks + earlier in this chunk.  524288 slots of
// 256 experts 8.6 us: 512 slots a wave, 64 at a time, each after the one before.
__global__ __launch_bounds__(64) void route_place_kernel(RouteArgs a) {
    __shared__ int next[RT_EMAX + 1];
    const long s0 = (long)blockIdx.x * RT_ROWS * a.k;
    const int n = (int)min((long)RT_ROWS * a.k, a.T * a.k - s0);
    const Slots slots = load_slots(a.experts + s0, n);       // on their way while the places are found
    first_places(a, next, blockIdx.x == 0, [&](int e) { return a.totals[e]; }, [&](int e) { return a.counts[(long)e * a.chunks + blockIdx.x]; });
    place_slots(a, next, slots, n, s0);
}

// Blocks of 8 waves while 4 would leave places for waves empty (256 CUs hold 1024 blocks of 4), us a call of all three launches:
// 20000 x 512 60 by 8, 73 by 4; 65536 x 256, whose 1024 blocks of 4 are there at once, 61 by 4, 62 by 8 (without groups 40 and 44).
template <int V, int LPR, int NE, int NB>
void launch_choose(const RouteArgs& a, hipStream_t st) {
    const long needed = (a.T * LPR + 63) / 64;                // of a single chunk
    const int waves = a.chunks > 512 ? 4 : (int)std::max(1l, std::min(8l, needed));
    const dim3 grid(a.chunks), block(64 * waves);
    const size_t lds = (size_t)waves * NE * 64 * sizeof(double);
    if (a.groups > 1 && !a.bias && a.type != FR_TYPE_F32) hipLaunchKernelGGL((route_choose_kernel<V, LPR, NE, 4, BY_LOGIT_IN_GROUPS>), grid, block, lds, st, a);
    else if (a.bias || a.groups > 1) hipLaunchKernelGGL((route_choose_kernel<V, LPR, NE, 4, BY_SCORE>), grid, block, lds, st, a);
    else if constexpr (LPR < 64) hipLaunchKernelGGL((route_choose_kernel<V, LPR, NE, NB, BY_LOGIT>), grid, block, lds, st, a);      // 64 lanes: groups
}

}  // namespace

extern "C" int fr_route_workspace_bytes(int64_t T, int E, int k, size_t* out_bytes) {
    if (!out_bytes || T < 0 || E <= 0 || E > RT_EMAX || k <= 0 || k > RT_KMAX || k > E) FR_FAIL(FR_ERR_ARG, "fr_route_workspace_bytes: bad shape (E <= 512, k <= min(16, E))");
    const size_t chunks = (size_t)((T + RT_ROWS - 1) / RT_ROWS);
    *out_bytes = chunks > 1 ? align_up((chunks + 1) * (E + 1) * 4, 16) : 0;
    return FR_OK;
}

extern "C" int fr_route(const void* logits, int logits_type, int64_t T, int E, int k, int score, const float* bias,
                        int groups, int top_groups, int renormalise, float scale,
                        float* weights, int32_t* experts, int32_t* order, int32_t* offsets,
                        void* workspace, size_t workspace_bytes, void* stream) {
    if (T < 0 || E <= 0 || E > RT_EMAX || k <= 0 || k > RT_KMAX || k > E) FR_FAIL(FR_ERR_ARG, "fr_route: bad shape (E <= 512, k <= min(16, E))");
    if (T >= 1ll << 30 || T * k > 0x7FFFFFFFll) FR_FAIL(FR_ERR_UNSUPPORTED, "fr_route: T * k does not fit 31 bits, or T 30");
    if (!type_ok(logits_type)) FR_FAIL(FR_ERR_ARG, "fr_route: unknown element type");
    if (score != FR_SCORE_SOFTMAX && score != FR_SCORE_SIGMOID) FR_FAIL(FR_ERR_ARG, "fr_route: unknown score");
    if (groups < 1 || groups > 64 || E % groups || top_groups < 1 || top_groups > groups) FR_FAIL(FR_ERR_ARG, "fr_route: groups (at most 64) must divide E, 1 <= top_groups <= groups");
    if ((long)top_groups * (E / groups) < k) FR_FAIL(FR_ERR_ARG, "fr_route: the kept groups hold fewer than k experts");
    size_t need = 0;
    const int rc = fr_route_workspace_bytes(T, E, k, &need);
    if (rc) return rc;
    if (!offsets || (T && (!weights || !experts || !order || !logits))) FR_FAIL(FR_ERR_ARG, "fr_route: NULL tensor");
    if (workspace_bytes < need || (need && !workspace)) FR_FAIL(FR_ERR_WORKSPACE, "fr_route: workspace too small");
    RouteArgs a{logits, bias, weights, experts, order, offsets, (int*)workspace + E + 1, (int*)workspace, T,
                logits_type, E, k, score, groups, top_groups, renormalise, (int)((T + RT_ROWS - 1) / RT_ROWS), scale};
    hipStream_t st = (hipStream_t)stream;
    if (a.chunks == 0) a.chunks = 1;                          // no rows: the offsets are written all the same
    // lanes a row takes: every group a whole number of them, and one for each of the k choices and the one behind them
    const int V = E <= 64 && groups == 1 ? 8 : 16, per = E / groups, lanes = std::max(groups * ((per + V - 1) / V), k + 1);
    if (V == 8 && lanes <= 8) launch_choose<8, 8, 1, 6>(a, st);
    else if (lanes <= 8 && E <= 128) launch_choose<16, 8, 2, 8>(a, st);
    else if (lanes <= 16 && E <= 256) launch_choose<16, 16, 4, 8>(a, st);
    else if (lanes <= 32) launch_choose<16, 32, 8, 9>(a, st);
    else launch_choose<16, 64, 8, 9>(a, st);
    FR_LAUNCH_CHECK("route_choose_kernel");
    if (a.chunks > 1) {
        hipLaunchKernelGGL(route_scan_kernel, dim3(E + 1), dim3(256), 0, st, a);
        FR_LAUNCH_CHECK("route_scan_kernel");
        hipLaunchKernelGGL(route_place_kernel, dim3(a.chunks), dim3(64), 0, st, a);
        FR_LAUNCH_CHECK("route_place_kernel");
    }
    return FR_OK;
}
