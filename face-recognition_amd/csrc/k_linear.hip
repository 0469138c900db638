// Dense products with their epilogue, out = act(x W^T + bias) + residual, for one matrix (fr_linear) and for the rows of
// every expert with that expert's matrix (fr_expert_linear).
//
// MFMA 16x16 tiles, the weights as the row operand: accumulator columns are rows of x, so a lane owns consecutive outputs of
// one row and stores vectors.  A "chunk" is 16 bytes of a row: 8 elements of 16 bits, one lane's share of
// v_mfma_f32_16x16x32, or 4 floats, one each for four v_mfma_f32_16x16x4_f32 (the same k order in both operands, so any
// assignment of chunks to lanes gives the product).
#include "adapter.h"

namespace {

struct GemmArgs {
    const void* x; const void* w; const void* bias; const float* slope; const void* res; void* out;
    long M, ldx, ldr;                    // rows of the output (experts: T * k slots); strides in elements
    int N, K;
    int bias_type, res_type, out_type, act;
    // experts: order == NULL for the plain product
    const int* order; const int* offsets;
    int E, k, rows_sorted, out_slots;
    int n_tiles;
};

template <typename T> struct Elem;       // BYTES, mma over one chunk of both operands
template <> struct Elem<bf16> {
    static constexpr int BYTES = 2;
    static FR_DEV void mma(f32x4& acc, const u32x4& a, const u32x4& b) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    }
};
template <> struct Elem<f16> {
    static constexpr int BYTES = 2;
    static FR_DEV void mma(f32x4& acc, const u32x4& a, const u32x4& b) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    }
};
template <> struct Elem<float> {
    static constexpr int BYTES = 4;
    static FR_DEV void mma(f32x4& acc, const u32x4& a, const u32x4& b) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), acc, 0, 0, 0);
    }
};

// The rows [r0, r1) of the order that row tile `tile` covers, and their expert (E: the slots without one).  False: no such
// tile.  Every wave of a block computes it.  Bounds are clamped to [0, M), so a bad table reads and writes nothing outside.
FR_DEV bool expert_tile(const GemmArgs& a, int tile, int bm, int& expert, long& r0, long& r1) {
    const int lane = threadIdx.x & 63, P = (int)a.M;
    int before = 0;
    for (int e0 = 0; e0 <= a.E; e0 += 64) {
        const int e = e0 + lane;
        int lo = 0, hi = 0;
        if (e <= a.E) {
            lo = min(max(a.offsets[e], 0), P);
            hi = e < a.E ? min(max(a.offsets[e + 1], lo), P) : P;
        }
        const int nt = (hi - lo + bm - 1) / bm;
        int s = nt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(s, o, 64); if (lane >= o) s += t; }
        const unsigned long long past = __ballot(before + s > tile);
        if (past) {
            const int f = __ffsll(past) - 1;
            const int first = before + __shfl(s - nt, f, 64);
            lo = __shfl(lo, f, 64); hi = __shfl(hi, f, 64);
            expert = __builtin_amdgcn_readfirstlane(e0 + f);
            r0 = __builtin_amdgcn_readfirstlane(lo + (tile - first) * bm);
            r1 = min(r0 + bm, (long)__builtin_amdgcn_readfirstlane(hi));
            return true;
        }
        before += __shfl(s, 63, 64);
    }
    return false;
}

// Slot of position p of the order, -1 if the table names none.
FR_DEV int slot_at(const GemmArgs& a, long p) {
    const int s = a.order[p];
    return (unsigned)s < (unsigned)a.M ? s : -1;
}
// Row of x that position p of the order multiplies (0 where there is none: its result goes nowhere).
FR_DEV long x_row(const GemmArgs& a, long p) {
    if (!a.order || a.rows_sorted) return p;
    const int s = slot_at(a, p);
    return s < 0 ? 0 : s / a.k;
}
// Row of the output for position p of the order; -1: none.
FR_DEV long out_row(const GemmArgs& a, long p) {
    if (!a.order || !a.out_slots) return p;
    return slot_at(a, p);
}

FR_DEV Vec8f get8n(const void* base, long i, int n, int type) {
    if (n == 8) return raw_to_f(raw_load8<false>(base, i, type), type);
    Vec8f o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = j < n ? load1(base, i + j, type) : 0.f;
    return o;
}
// Eight outputs n0 .. n0+7 (as many as N has) of row `row`.
FR_DEV void finish8(const GemmArgs& a, long row, int n0, long nbase, Vec8f v) {
    const int n = min(8, a.N - n0);
    if (n <= 0) return;
    if (a.bias) {
        const Vec8f b = get8n(a.bias, nbase + n0, n, a.bias_type);
#pragma unroll
        for (int j = 0; j < 8; ++j) v.v[j] += b.v[j];
    }
    if (a.act != FR_ACT_NONE) {
        Vec8f s{};
        if (a.act == FR_ACT_PRELU) s = get8n(a.slope, nbase + n0, n, FR_TYPE_F32);
#pragma unroll
        for (int j = 0; j < 8; ++j) v.v[j] = adapter_act(v.v[j], a.act, s.v[j]);
    }
    if (a.res) {
        const Vec8f r = get8n(a.res, row * a.ldr + n0, n, a.res_type);
#pragma unroll
        for (int j = 0; j < 8; ++j) v.v[j] += r.v[j];
    }
    const long o = row * a.N + n0;
    if (n == 8) store8t<false>(a.out, o, a.out_type, v);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < n) store1(a.out, o + j, a.out_type, v.v[j]);
    }
}

// 16 bytes of a row from byte `at` of its `len`, zeros behind its end; any alignment.
FR_DEV u32x4 chunk_at(const unsigned char* row, long at, long len) {
    if (at + 16 <= len) return *reinterpret_cast<const u32x4_any*>(row + at);
    union { u32x4 v; unsigned short h[8]; } c;
    c.v = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (at + 2 * j < len) c.h[j] = *reinterpret_cast<const unsigned short*>(row + at + 2 * j);
    return c.v;
}

// Any shape, any alignment: 64 x 64 outputs a block, 4 waves of 32 x 32, slices of 128 bytes of K through registers into
// LDS.  Piece p of LDS row r lies at p ^ ((r >> 1) & 7): the 16 rows of a fragment read fall on different banks.
template <typename T>
__global__ __launch_bounds__(256) void gemm_any_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][64 * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nt = blockIdx.x % a.n_tiles, mt = blockIdx.x / a.n_tiles;
    const int n0 = nt * 64;
    long r0 = (long)mt * 64, r1 = min(r0 + 64, a.M);
    int expert = 0;
    if (a.order && !expert_tile(a, mt, 64, expert, r0, r1)) return;
    const bool none = a.order && expert == a.E;
    const long nbase = (long)expert * a.N;
    const long rowb = (long)a.K * Elem<T>::BYTES;
    const int li = lane & 15, lg = lane >> 4, wm = wave & 1, wn = wave >> 1;

    f32x4 acc[2][2];                                         // [16 of n][16 of m]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!none) {
        // this thread's two chunks of a slice of either operand: rows tid / 8 and tid / 8 + 32, piece tid % 8
        const unsigned char* src[2][2];
        int dst[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = (tid >> 3) + 32 * i;
            src[0][i] = reinterpret_cast<const unsigned char*>(a.w) + (nbase + min(n0 + r, a.N - 1)) * rowb;
            src[1][i] = reinterpret_cast<const unsigned char*>(a.x) + x_row(a, min(r0 + r, r1 - 1)) * a.ldx * Elem<T>::BYTES;
            dst[i] = r * 128 + ((tid & 7) ^ ((r >> 1) & 7)) * 16;
        }
        u32x4 c[2][2];
        auto fetch = [&](long at) {
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int i = 0; i < 2; ++i) c[o][i] = chunk_at(src[o][i], at + (tid & 7) * 16, rowb);
        };
        fetch(0);
        for (long at = 0; at < rowb; at += 128) {
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4*>(lds[o] + dst[i]) = c[o][i];
            __syncthreads();
            if (at + 128 < rowb) fetch(at + 128);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 af[2], bf[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    // row i of n-tile t is output (i >> 2) * 8 + 4 t + (i & 3): a lane's two tiles are 8 consecutive outputs
                    const int rn = wn * 32 + (li >> 2) * 8 + 4 * i + (li & 3), rm = wm * 32 + 16 * i + li;
                    af[i] = *reinterpret_cast<const u32x4*>(lds[0] + rn * 128 + ((s * 4 + lg) ^ ((rn >> 1) & 7)) * 16);
                    bf[i] = *reinterpret_cast<const u32x4*>(lds[1] + rm * 128 + ((s * 4 + lg) ^ ((rm >> 1) & 7)) * 16);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) Elem<T>::mma(acc[i][j], af[i], bf[j]);
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const long p = r0 + wm * 32 + 16 * j + li;
        if (p >= r1) continue;
        const long row = out_row(a, p);
        if (row < 0) continue;
        Vec8f v;
#pragma unroll
        for (int r = 0; r < 4; ++r) { v.v[r] = acc[0][j][r]; v.v[4 + r] = acc[1][j][r]; }
        const int n = n0 + wn * 32 + lg * 8;
        if (none) {
            for (int q = 0; q < 8; ++q) if (n + q < a.N) store1(a.out, row * a.N + n + q, a.out_type, 0.f);
        } else finish8(a, row, n, nbase, v);
    }
}

template <typename T>
int launch_gemm(GemmArgs a, hipStream_t st) {
    const long mt = a.order ? a.M / 64 + std::min<long>(a.M, a.E + 1) : (a.M + 63) / 64;
    a.n_tiles = (a.N + 63) / 64;
    if (mt * a.n_tiles > 0x7FFFFFFFll) FR_FAIL(FR_ERR_UNSUPPORTED, "adapter product: more than 2^31 output tiles");
    hipLaunchKernelGGL((gemm_any_kernel<T>), dim3((unsigned)(mt * a.n_tiles)), dim3(256), 0, st, a);
    FR_LAUNCH_CHECK("gemm_any_kernel");
    return FR_OK;
}
int launch_type(int type, const GemmArgs& a, hipStream_t st) {
    if (type == FR_TYPE_BF16) return launch_gemm<bf16>(a, st);
    if (type == FR_TYPE_F16) return launch_gemm<f16>(a, st);
    return launch_gemm<float>(a, st);
}

}  // namespace

extern "C" int fr_linear_workspace_bytes(int64_t M, int N, int K, int type, size_t* out_bytes) {
    if (!out_bytes || M < 0 || N <= 0 || K <= 0 || !type_ok(type)) FR_FAIL(FR_ERR_ARG, "fr_linear_workspace_bytes: bad shape or type");
    *out_bytes = 0;
    return FR_OK;
}

extern "C" int fr_linear(const void* x, int64_t ldx, const void* w, const void* bias, const float* slope,
                         const void* residual, int64_t ldr, void* out, int64_t M, int N, int K,
                         int type, int bias_type, int res_type, int out_type, int act,
                         void* workspace, size_t workspace_bytes, void* stream) {
    if (M < 0 || N <= 0 || K <= 0 || ldx < 0 || (residual && ldr < 0)) FR_FAIL(FR_ERR_ARG, "fr_linear: bad shape");
    if (!type_ok(type) || !type_ok(out_type) || (bias && bias_type != type && bias_type != FR_TYPE_F32) || (residual && !type_ok(res_type)))
        FR_FAIL(FR_ERR_ARG, "fr_linear: unknown element type (bias: the operands' type or fp32)");
    if (act < FR_ACT_NONE || act > FR_ACT_SILU) FR_FAIL(FR_ERR_ARG, "fr_linear: unknown activation");
    if (act == FR_ACT_PRELU && !slope) FR_FAIL(FR_ERR_ARG, "fr_linear: PReLU without slopes");
    if (M == 0) return FR_OK;
    if (!x || !w || !out) FR_FAIL(FR_ERR_ARG, "fr_linear: NULL tensor");
    GemmArgs a{};
    a.x = x; a.w = w; a.bias = bias; a.slope = slope; a.res = residual; a.out = out;
    a.M = M; a.ldx = ldx; a.ldr = ldr; a.N = N; a.K = K;
    a.bias_type = bias_type; a.res_type = res_type; a.out_type = out_type; a.act = act;
    return launch_type(type, a, (hipStream_t)stream);
}

extern "C" int fr_expert_linear(const void* x, int rows_sorted, const void* w, const void* bias, const float* slope,
                                const int32_t* order, const int32_t* offsets, void* out, int out_slots,
                                int64_t T, int k, int E, int N, int K, int type, int bias_type, int out_type, int act, void* stream) {
    if (T < 0 || k <= 0 || E <= 0 || N <= 0 || K <= 0) FR_FAIL(FR_ERR_ARG, "fr_expert_linear: bad shape");
    if (T * k > 0x7FFFFFFFll) FR_FAIL(FR_ERR_UNSUPPORTED, "fr_expert_linear: T * k does not fit 31 bits");
    if (!type_ok(type) || !type_ok(out_type) || (bias && bias_type != type && bias_type != FR_TYPE_F32))
        FR_FAIL(FR_ERR_ARG, "fr_expert_linear: unknown element type (bias: the operands' type or fp32)");
    if (act < FR_ACT_NONE || act > FR_ACT_SILU) FR_FAIL(FR_ERR_ARG, "fr_expert_linear: unknown activation");
    if (act == FR_ACT_PRELU && !slope) FR_FAIL(FR_ERR_ARG, "fr_expert_linear: PReLU without slopes");
    if (T == 0) return FR_OK;
    if (!x || !w || !out || !order || !offsets) FR_FAIL(FR_ERR_ARG, "fr_expert_linear: NULL tensor");
    GemmArgs a{};
    a.x = x; a.w = w; a.bias = bias; a.slope = slope; a.out = out;
    a.M = T * k; a.ldx = K; a.N = N; a.K = K;
    a.bias_type = bias_type; a.out_type = out_type; a.act = act;
    a.order = order; a.offsets = offsets; a.E = E; a.k = k; a.rows_sorted = rows_sorted; a.out_slots = out_slots;
    return launch_type(type, a, (hipStream_t)stream);
}
