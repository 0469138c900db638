// Routing of rows to experts: scores, balance bias, group limit, the best k, weights, and the slots sorted by expert.
// Three launches: choose (and count a chunk's slots per expert), scan the chunks' counts, place every slot.
#include "adapter.h"

namespace {

constexpr int RT_ROWS = 64;              // rows of a chunk = rows of a block of route_choose_kernel
constexpr int RT_WAVES = 4;
constexpr int RT_EMAX = 512, RT_KMAX = 16;

struct RouteArgs {
    const void* logits; const float* bias;
    float* weights; int* experts; int* order; int* offsets;
    int* counts;                         // [chunks][E + 1]: slots of a chunk per expert (E: none), then their first places
    int* totals;                         // [E + 1]
    long T;
    int type, E, k, score, groups, top_groups, renormalise, chunks;
    float scale;
};

template <typename V>
FR_DEV void best_of_wave(V& key, int& idx) {                 // greatest key, ties to the lower index, in every lane
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const V k2 = __shfl_xor(key, o, 64);
        const int i2 = __shfl_xor(idx, o, 64);
        if (k2 > key || (k2 == key && i2 < idx)) { key = k2; idx = i2; }
    }
}

FR_DEV float wave_sum_k(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// LDS written by other lanes of this wave is read behind it.
FR_DEV void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// One row per wave at a time; lane l holds experts l, l + 64, ...  Keys are doubles: exact scores differ by less than a
// float's step often enough to matter, and their order is what the choice is.
template <int NE>
__global__ __launch_bounds__(64 * RT_WAVES) void route_choose_kernel(RouteArgs a) {
    __shared__ int count[RT_EMAX + 1];
    __shared__ double keys[RT_WAVES][NE * 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e <= a.E; e += blockDim.x) count[e] = 0;
    __syncthreads();
    const double NONE = -INFINITY;
    const bool scored = a.bias != nullptr || a.groups > 1;
    for (int r = wave; r < RT_ROWS; r += RT_WAVES) {
        const long row = (long)blockIdx.x * RT_ROWS + r;
        if (row >= a.T) break;
        float l[NE];
        double key[NE];
        float m = -INFINITY;
#pragma unroll
        for (int q = 0; q < NE; ++q) {
            const int e = lane + 64 * q;
            l[q] = e < a.E ? load1(a.logits, row * a.E + e, a.type) : -INFINITY;
            if (!(l[q] > -INFINITY)) l[q] = -INFINITY;       // NaN masks too
            m = fmaxf(m, l[q]);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        float z = 0.f;
        double z64 = 0.0;
        if (a.score == FR_SCORE_SOFTMAX) {
#pragma unroll
            for (int q = 0; q < NE; ++q) {
                const double p = l[q] == m ? 1.0 : exp((double)l[q] - (double)m);
                key[q] = l[q] > -INFINITY ? p : 0.0;
                z64 += key[q];
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) z64 += __shfl_xor(z64, o, 64);
            z = (float)z64;
        }
#pragma unroll
        for (int q = 0; q < NE; ++q) {
            const int e = lane + 64 * q;
            if (!scored) key[q] = l[q];
            else {
                const double s = a.score == FR_SCORE_SOFTMAX ? key[q] / z64 : 1.0 / (1.0 + exp(-(double)l[q]));
                const float b = a.bias && e < a.E ? a.bias[e] : 0.f;
                key[q] = l[q] > -INFINITY && b > -INFINITY ? s + (double)b : NONE;
            }
        }
        if (a.groups > 1) {
            const int per = a.E / a.groups;
#pragma unroll
            for (int q = 0; q < NE; ++q) keys[wave][lane + 64 * q] = key[q];
            wave_lds_fence();
            double g = NONE;
            if (lane < a.groups) {
                double b1 = NONE, b2 = NONE;
                for (int i = 0; i < per; ++i) {
                    const double v = keys[wave][lane * per + i];
                    if (v > b1) { b2 = b1; b1 = v; } else if (v > b2) b2 = v;
                }
                g = per > 1 ? b1 + b2 : b1;
            }
            wave_lds_fence();
            int rank = 0;
            for (int o = 0; o < a.groups; ++o) {
                const double v = __shfl(g, o, 64);
                if (v > g || (v == g && o < lane)) ++rank;
            }
            const unsigned long long keep = __ballot(lane < a.groups && rank < a.top_groups);
#pragma unroll
            for (int q = 0; q < NE; ++q) {
                const int e = lane + 64 * q;
                if (e >= a.E || !((keep >> (e / per)) & 1)) key[q] = NONE;
            }
        }
        int mine = -1;                                       // lane j < k: the j-th choice
        float mine_l = -INFINITY;
        for (int j = 0; j < a.k; ++j) {
            double b = NONE;
            int bi = RT_EMAX;
            float bl = -INFINITY;
#pragma unroll
            for (int q = 0; q < NE; ++q)
                if (key[q] > b) { b = key[q]; bi = lane + 64 * q; }
            best_of_wave(b, bi);
            if (b == NONE) break;
#pragma unroll
            for (int q = 0; q < NE; ++q)
                if (lane + 64 * q == bi) { key[q] = NONE; bl = l[q]; }
            bl = __shfl(bl, bi & 63, 64);
            if (lane == j) { mine = bi; mine_l = bl; }
        }
        float top = mine_l;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        float w = 0.f;
        if (mine >= 0) {
            if (a.score == FR_SCORE_SOFTMAX) {
                const float against = a.renormalise ? top : m;
                w = mine_l == against ? 1.f : expf(mine_l - against);
                if (!a.renormalise) w /= z;
            } else if (a.renormalise && top < -20.f) w = expf(mine_l - top);   // sigmoid(l) = e^l to 2e-9 there
            else w = 1.f / (1.f + expf(-mine_l));
        }
        if (a.renormalise) {
            const float sum = wave_sum_k(w);
            if (sum > 0.f) w /= sum;
        }
        if (lane < a.k) {
            a.weights[row * a.k + lane] = w * a.scale;
            a.experts[row * a.k + lane] = mine;
            atomicAdd(&count[mine >= 0 ? mine : a.E], 1);     // whole numbers: any order gives the same
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e <= a.E; e += blockDim.x) a.counts[(long)blockIdx.x * (a.E + 1) + e] = count[e];
}

// counts[c][e] -> number of e's slots in the chunks before c; totals[e].  One wave per expert.
__global__ __launch_bounds__(64) void route_scan_kernel(RouteArgs a) {
    const int e = blockIdx.x, lane = threadIdx.x;
    int before = 0;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
        const int c = c0 + lane;
        const int n = c < a.chunks ? a.counts[(long)c * (a.E + 1) + e] : 0;
        int s = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(s, o, 64); if (lane >= o) s += t; }
        if (c < a.chunks) a.counts[(long)c * (a.E + 1) + e] = before + s - n;
        before += __shfl(s, 63, 64);
    }
    if (lane == 0) a.totals[e] = before;
}

// Places of a chunk's slots: first place of the expert + its slots in earlier chunks + earlier in this chunk.
__global__ __launch_bounds__(64) void route_place_kernel(RouteArgs a) {
    __shared__ int next[RT_EMAX + 1];
    const int lane = threadIdx.x;
    int before = 0;
    for (int e0 = 0; e0 <= a.E; e0 += 64) {
        const int e = e0 + lane;
        const int n = e <= a.E ? a.totals[e] : 0;
        int s = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(s, o, 64); if (lane >= o) s += t; }
        if (e <= a.E) {
            next[e] = before + s - n + (a.chunks ? a.counts[(long)blockIdx.x * (a.E + 1) + e] : 0);
            if (blockIdx.x == 0) a.offsets[e] = before + s - n;
        }
        before += __shfl(s, 63, 64);
    }
    __syncthreads();
    const long s0 = (long)blockIdx.x * RT_ROWS * a.k, s1 = min(s0 + (long)RT_ROWS * a.k, a.T * a.k);
    for (long b = s0; b < s1; b += 64) {
        const long s = b + lane;
        const bool on = s < s1;
        const int ex = on ? a.experts[s] : -1;
        const int e = ex < 0 ? a.E : ex;
        unsigned long long same = __ballot(on);              // lanes with this lane's expert
        for (int bit = 0; (1 << bit) <= a.E; ++bit) {
            const bool set = (e >> bit) & 1;
            const unsigned long long with = __ballot(set);
            same &= set ? with : ~with;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (on) a.order[next[e] + rank] = (int)s;
        __syncthreads();
        if (on && rank == 0) next[e] += __popcll(same);
        __syncthreads();
    }
}

}  // namespace

extern "C" int fr_route_workspace_bytes(int64_t T, int E, int k, size_t* out_bytes) {
    if (!out_bytes || T < 0 || E <= 0 || E > RT_EMAX || k <= 0 || k > RT_KMAX || k > E) FR_FAIL(FR_ERR_ARG, "fr_route_workspace_bytes: bad shape (E <= 512, k <= min(16, E))");
    const size_t chunks = (size_t)((T + RT_ROWS - 1) / RT_ROWS);
    *out_bytes = align_up((chunks + 1) * (E + 1) * 4, 16);
    return FR_OK;
}

extern "C" int fr_route(const void* logits, int logits_type, int64_t T, int E, int k, int score, const float* bias,
                        int groups, int top_groups, int renormalise, float scale,
                        float* weights, int32_t* experts, int32_t* order, int32_t* offsets,
                        void* workspace, size_t workspace_bytes, void* stream) {
    if (T < 0 || E <= 0 || E > RT_EMAX || k <= 0 || k > RT_KMAX || k > E) FR_FAIL(FR_ERR_ARG, "fr_route: bad shape (E <= 512, k <= min(16, E))");
    if (T * k > 0x7FFFFFFFll) FR_FAIL(FR_ERR_UNSUPPORTED, "fr_route: T * k does not fit 31 bits");
    if (!type_ok(logits_type)) FR_FAIL(FR_ERR_ARG, "fr_route: unknown element type");
    if (score != FR_SCORE_SOFTMAX && score != FR_SCORE_SIGMOID) FR_FAIL(FR_ERR_ARG, "fr_route: unknown score");
    if (groups < 1 || groups > 64 || E % groups || top_groups < 1 || top_groups > groups) FR_FAIL(FR_ERR_ARG, "fr_route: groups (at most 64) must divide E, 1 <= top_groups <= groups");
    if ((long)top_groups * (E / groups) < k) FR_FAIL(FR_ERR_ARG, "fr_route: the kept groups hold fewer than k experts");
    size_t need = 0;
    const int rc = fr_route_workspace_bytes(T, E, k, &need);
    if (rc) return rc;
    if (!weights || !experts || !order || !offsets || (T && !logits)) FR_FAIL(FR_ERR_ARG, "fr_route: NULL tensor");
    if (workspace_bytes < need || !workspace) FR_FAIL(FR_ERR_WORKSPACE, "fr_route: workspace too small");
    RouteArgs a{logits, bias, weights, experts, order, offsets, (int*)workspace + E + 1, (int*)workspace, T,
                logits_type, E, k, score, groups, top_groups, renormalise, (int)((T + RT_ROWS - 1) / RT_ROWS), scale};
    hipStream_t st = (hipStream_t)stream;
    if (a.chunks) {
        const dim3 grid(a.chunks), block(64 * RT_WAVES);
        if (E <= 64) hipLaunchKernelGGL((route_choose_kernel<1>), grid, block, 0, st, a);
        else if (E <= 128) hipLaunchKernelGGL((route_choose_kernel<2>), grid, block, 0, st, a);
        else if (E <= 256) hipLaunchKernelGGL((route_choose_kernel<4>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((route_choose_kernel<8>), grid, block, 0, st, a);
        FR_LAUNCH_CHECK("route_choose_kernel");
    }
    hipLaunchKernelGGL(route_scan_kernel, dim3(E + 1), dim3(64), 0, st, a);
    FR_LAUNCH_CHECK("route_scan_kernel");
    hipLaunchKernelGGL(route_place_kernel, dim3(std::max(1, a.chunks)), dim3(64), 0, st, a);
    FR_LAUNCH_CHECK("route_place_kernel");
    return FR_OK;
}
