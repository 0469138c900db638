// Dense products with their epilogue, out = act(x W^T + bias) + residual, for one matrix (fr_linear) and for the rows of
// every expert with that expert's matrix (fr_expert_linear).
//
// MFMA 16x16 tiles, the weights as the row operand: accumulator columns are rows of x, so a lane owns consecutive outputs of
// one row and stores vectors.  A "chunk" is 16 bytes of a row: 8 elements of 16 bits, one lane's share of
// v_mfma_f32_16x16x32, or 4 floats, one each for four v_mfma_f32_16x16x4_f32 (the same k order in both operands, so any
// assignment of chunks to lanes gives the product).
#include <math.h>

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
    unsigned k_mul; int k_shift;         // s / k = (s k_mul) >> (31 + k_shift) for 0 <= s < 2^31
    int n_tiles;
    int splits, split_slices;            // K in `splits` parts of split_slices slices each, their sums in `partial` [splits][M][N]
    float* partial;
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

// Expert e0 + lane (E: the slots without one): its rows [lo, hi) of the order and the row tiles from expert e0 to its end.
// Bounds are clamped to [0, M), so a bad table reads and writes nothing outside.
struct ExpertScan { int lo, hi, tiles, upto; };
FR_DEV ExpertScan scan_experts(const GemmArgs& a, int e0, int bm) {
    const int e = e0 + (threadIdx.x & 63), P = (int)a.M;
    ExpertScan x{};
    if (e <= a.E) {
        x.lo = min(max(a.offsets[e], 0), P);
        x.hi = e < a.E ? min(max(a.offsets[e + 1], x.lo), P) : P;
    }
    x.tiles = (x.hi - x.lo + bm - 1) / bm;
    x.upto = scan_add(x.tiles);
    return x;
}
// Number of row tiles; `x`: the scan of the first 64.
FR_DEV int expert_tiles(const GemmArgs& a, int bm, const ExpertScan& x) {
    int n = __builtin_amdgcn_readlane(x.upto, 63);
    for (int e0 = 64; e0 <= a.E; e0 += 64) n += __builtin_amdgcn_readlane(scan_experts(a, e0, bm).upto, 63);
    return n;
}
// The rows [r0, r1) of the order that row tile `tile` covers, and their expert.  False: no such tile.  Every wave of a block
// computes it, from the scan of the first 64 on.
FR_DEV bool expert_tile(const GemmArgs& a, int tile, int bm, ExpertScan x, int& expert, long& r0, long& r1) {
    int before = 0;
    for (int e0 = 0;;) {
        const unsigned long long past = __ballot(before + x.upto > tile);
        if (past) {
            const int f = __ffsll(past) - 1;
            const int first = before + __builtin_amdgcn_readlane(x.upto - x.tiles, f);
            const long begin = __builtin_amdgcn_readlane(x.lo, f), end = __builtin_amdgcn_readlane(x.hi, f);
            expert = e0 + f;
            r0 = begin + (long)(tile - first) * bm;
            r1 = min(r0 + bm, end);
            return r0 >= begin && r0 < end;                  // false only where the counts of a table that lies have overflowed
        }
        before += __builtin_amdgcn_readlane(x.upto, 63);
        e0 += 64;
        if (e0 > a.E) return false;
        x = scan_experts(a, e0, bm);
    }
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
    return s < 0 ? 0 : __umulhi(2u * s, a.k_mul) >> a.k_shift;     // s / k
}
// Row of the output for position p of the order; -1: none, as the table names no slot (where neither side goes by slots it is not read).
FR_DEV long out_row(const GemmArgs& a, long p) {
    if (!a.order || (a.rows_sorted && !a.out_slots)) return p;
    const int s = slot_at(a, p);
    return s < 0 || a.out_slots ? s : p;
}

FR_DEV Vec8f get8n(const void* base, long i, int n, int type) {
    if (n == 8) return raw_to_f(raw_load8<false>(base, i, type), type);
    Vec8f o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = j < n ? load1(base, i + j, type) : 0.f;
    return o;
}
template <int ACT>
FR_DEV void act8(Vec8f& v, const Vec8f& slope) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v.v[j] = adapter_act(v.v[j], ACT, slope.v[j]);
}
FR_DEV void put8n(void* base, long i, int n, int type, const Vec8f& v) {
    if (n == 8) { store8t<false>(base, i, type, v); return; }
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) store1(base, i + j, type, v.v[j]);
}
// Bias and slopes of eight output columns, `have` of which exist.
struct Columns { Vec8f bias, slope; };
FR_DEV Columns columns(const GemmArgs& a, int n, int have, long nbase, bool none) {
    Columns c{};
    if (none || have <= 0) return c;
    if (a.bias) c.bias = get8n(a.bias, nbase + n, have, a.bias_type);
    if (a.act == FR_ACT_PRELU) c.slope = get8n(a.slope, nbase + n, have, FR_TYPE_F32);
    return c;
}
FR_DEV void activate(const GemmArgs& a, Vec8f& v, const Columns& c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v.v[j] += c.bias.v[j];
    switch (a.act) {
        case FR_ACT_PRELU: act8<FR_ACT_PRELU>(v, c.slope); break;
        case FR_ACT_HSWISH: act8<FR_ACT_HSWISH>(v, c.slope); break;
        case FR_ACT_RELU: act8<FR_ACT_RELU>(v, c.slope); break;
        case FR_ACT_HSIGMOID: act8<FR_ACT_HSIGMOID>(v, c.slope); break;
        case FR_ACT_GELU: act8<FR_ACT_GELU>(v, c.slope); break;
        case FR_ACT_SILU: act8<FR_ACT_SILU>(v, c.slope); break;
        default: break;
    }
}
FR_DEV void add8n(const GemmArgs& a, Vec8f& v, long row, int n, int have) {       // the residual
    const Vec8f r = get8n(a.res, row * a.ldr + n, have, a.res_type);
#pragma unroll
    for (int j = 0; j < 8; ++j) v.v[j] += r.v[j];
}
// Eight outputs n .. n+7 (as many as N has) of row `row`; `none`: of a slot without an expert, zeros.
FR_DEV void finish8(const GemmArgs& a, long row, int n, const Columns& c, Vec8f v, bool none) {
    const int have = min(8, a.N - n);
    if (have <= 0) return;
    if (!none) {
        activate(a, v, c);
        if (a.res) add8n(a, v, row, n, have);
    }
    put8n(a.out, row * a.N + n, have, a.out_type, v);
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

// One column of a wave's tiles.  fp32 goes through the tiles once per element of the chunk: four products into one
// accumulator in a row would each wait for the one before.
template <typename T, int TN, int TM>
FR_DEV void column(f32x4 (&acc)[TN][TM], int j, const u32x4 (&w)[TN], const u32x4& x) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < TN; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[i][e]), __uint_as_float(x[e]), acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < TN; ++i) Elem<T>::mma(acc[i][j], w[i], x);
    }
}

template <int VALUE> using Is = std::integral_constant<int, VALUE>;

// ---- the staged kernel --------------------------------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* glb_ptr_t;
__device__ const u32x4 g_zero16 = {0, 0, 0, 0};            // source of the pieces behind a row's end

// s_waitcnt as the compiler knows it (its own waits take it into account): at most VM vector loads and LGKM LDS reads open.
template <int VM, int LGKM> FR_DEV void wait_counts() {
    __builtin_amdgcn_s_waitcnt((VM & 15) | (7 << 4) | (LGKM << 8) | ((VM >> 4) << 14));
    asm volatile("" ::: "memory");
}
FR_DEV void block_barrier() {                              // without the waits of __syncthreads
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Block -> output tile.  Blocks go to the 8 XCDs in turn and each XCD has its own L2: a contiguous run of tiles for each,
// walked in groups of 4 row tiles by every n tile, so that the blocks of an XCD that run at the same time share their operands
// (groups of 8: 4 % slower at 16384 x 2048 x 8192, equal at 8192 cubed; of 16: 15 % slower there).
FR_DEV void tile_of_block(int block, int mtiles, int ntiles, int& mt, int& nt) {
    const int total = mtiles * ntiles, xcd = block & 7, q = total >> 3, r = total & 7;
    const int t = xcd * q + min(xcd, r) + (block >> 3);
    const int per = 4 * ntiles, g = t / per, in = t - g * per, rows = min(4, mtiles - g * 4);
    nt = in / rows;
    mt = g * 4 + (in - nt * rows);
}

// BM x BN outputs a block of WM x WN waves; slices of 128 bytes of K through a ring of ST buffers in LDS, brought by LDS-DMA
// (16 bytes a lane, 8 rows an instruction: whole lines of 128 bytes; with rows of 64 bytes the DMA alone was slower, 24
// against 43 bytes a clock and CU).  Rows are 16-byte aligned whole chunks.  A row in LDS keeps its piece p
// at p ^ key, x row r with the key (r >> 1) & 7, weight row r with that of its bits 1, 3 and 4, so that the 16 rows of a
// fragment read fall on 16 different bank groups.
// A slice is two halves of 64 bytes, their fragments in two register sets: while one set is multiplied the other is read.
// The one barrier of a slice stands between its halves: there its last fragments have been read and the next slice has
// landed, and behind it the DMA of slice s + ST goes into its buffer, spread over the second half's products (in one
// burst it held up the waves that issue it).
// What bounds it: a slice of a 256-tile is 2048 clocks of matrix instructions, as much LDS traffic (each wave's 128 x 64 outputs
// read 24 KB of the two halves, 8 waves 192, and 64 KB are written), and takes 2390 to 2550, at the 1.3 to 1.8 GHz the card
// holds under it; launch, first loads and epilogue are 10 us a tile, which a tile alone on its CU does not hide.
// bf16: 8192 cubed 754 us (1459 TFLOP/s; the library 662), 16384 x 2048 x 8192 383 (1435; 348), with bias and residual 401;
// 65536 x 4096 x 1024 520, with silu 540; experts 65536 slots x 4096 x 1024 with silu 614.  fp32 8192 cubed 7.73 ms (142 of
// 154).  Other ways to a 256-tile: 16 x 16 x 32 instructions reach 2145 TFLOP/s from registers alone, 32 x 32 x 16 1868; 4 waves
// of 128 x 128 read less LDS, but their 256 accumulators leave no registers to read ahead.
// WHOLE false: rows of any alignment.  The chunks of slice s + ST go to registers in the second half of slice s and to LDS in
// the first half of the next, where ST = 2 wants them by its barrier.
template <typename T, int BM, int BN, int WM, int WN, int ST, bool WHOLE>
__global__ __launch_bounds__(64 * WM * WN, BM == 128 && BN == 128 && ST == 2 ? 4 : 2) void gemm_tile_kernel(GemmArgs a) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, XB = BM * 128, BUF = (BM + BN) * 128;
    constexpr int XI = BM / 8 / NW, WI = BN / 8 / NW, DMA = XI + WI, DPG = (DMA + TM - 1) / TM;     // DMA instructions a wave and slice, and a group of products
    static_assert(TN <= TM && TN % 2 == 0 && NW % 4 == 0 && (WHOLE || ST == 2), "the interleaving below");
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4, wm = wave / WN, wn = wave % WN;
    int mtiles = (int)((a.M + BM - 1) / BM), mt, nt, expert = 0;
    ExpertScan scan{};
    if (a.order) {
        scan = scan_experts(a, 0, BM);
        mtiles = min(expert_tiles(a, BM, scan), (int)(gridDim.x / a.n_tiles));     // the second: tables that lie
    }
    const int tiles = mtiles * a.n_tiles, split = a.splits > 1 ? blockIdx.x / tiles : 0;
    if ((int)blockIdx.x - split * tiles >= tiles || split >= a.splits) return;     // experts: the grid is an upper bound
    tile_of_block(blockIdx.x - split * tiles, mtiles, a.n_tiles, mt, nt);
    long r0 = (long)mt * BM, r1 = min(r0 + BM, a.M);
    if (a.order && !expert_tile(a, mt, BM, scan, expert, r0, r1)) return;
    const bool none = a.order && expert == a.E;
    const int n0 = nt * BN;
    const long nbase = (long)expert * a.N, pitch = (long)a.K * Elem<T>::BYTES, k0 = (long)split * a.split_slices * 128;
    const long rowb = a.splits > 1 ? min(pitch - k0, (long)a.split_slices * 128) : pitch;     // bytes of a row in this part of K
    const int full = none ? 0 : (int)(rowb / 128), slices = none ? 0 : (int)((rowb + 127) / 128);

    // this lane's sources: row 8 (wave + NW j) + lane / 8, chunk (lane % 8) ^ key of the slice, as 32-bit offsets from the
    // tile's first row (the matrix's where rows are gathered)
    const int kx = ((lane & 7) ^ (((8 * wave + (lane >> 3)) >> 1) & 7)) * 16;    // the same for every j: NW is a multiple of 4
    const int kw = ((lane & 7) ^ (((lane >> 4) & 1) | ((wave & 3) << 1))) * 16;
    const bool gather = a.order && !a.rows_sorted;
    const unsigned char* xbase = reinterpret_cast<const unsigned char*>(a.x) + (gather ? 0 : r0 * a.ldx * Elem<T>::BYTES) + k0;
    const unsigned char* wbase = reinterpret_cast<const unsigned char*>(a.w) + (none ? 0 : (nbase + n0) * pitch) + k0;
    unsigned off[DMA];                                       // x rows, then weight rows
#pragma unroll
    for (int j = 0; j < WI; ++j) off[XI + j] = (unsigned)(min(8 * (wave + NW * j) + (lane >> 3), a.N - 1 - n0) * pitch) + kw;
#pragma unroll
    for (int j = 0; j < XI; ++j) {
        const long p = min(r0 + 8 * (wave + NW * j) + (lane >> 3), r1 - 1);
        off[j] = (unsigned)((gather ? x_row(a, p) : p - r0) * a.ldx * Elem<T>::BYTES) + kx;
    }
    // Gathered rows in the order's positions: every wave looks over the tile's entries while its first loads are on their way, and
    // the epilogue looks them up only where one names no slot (always: experts bulk 2 % slower).
    bool by_slot = a.order && a.out_slots;
    const bool look = gather && !a.out_slots;
    int slots[BM / 64];
    if (look)
#pragma unroll
        for (int q = 0; q < BM / 64; ++q) slots[q] = slot_at(a, min(r0 + 64 * q + lane, r1 - 1));
    auto looked = [&]() __attribute__((always_inline)) {
        if (!look) return;
        bool lies = false;
#pragma unroll
        for (int q = 0; q < BM / 64; ++q) lies |= slots[q] < 0;
        by_slot = __ballot(lies) != 0;
    };
    auto place = [&](int into, int d) __attribute__((always_inline)) {          // of instruction d in LDS
        return smem + into + (d < XI ? wave + NW * d : BM / 8 + wave + NW * (d - XI)) * 1024;
    };
    // instruction d of the slice whose x and w columns start at xs and ws
    u32x4 held[WHOLE ? 1 : DMA];
    auto dma = [&](const unsigned char* xs, const unsigned char* ws, int into, int d) __attribute__((always_inline)) {
        const unsigned char* src = (d < XI ? xs : ws) + off[d];
        if constexpr (WHOLE) __builtin_amdgcn_global_load_lds((glb_ptr_t)src, (lds_ptr_t)place(into, d), 16, 0, 0);
        else held[d] = *reinterpret_cast<const u32x4_any*>(src);
    };
    // instructions [d0, d1) of a slice in which K may end: zeros behind its end
    auto stage = [&](int s, int into, int d0, int d1) __attribute__((always_inline)) {
        const long at = (long)s * 128;
        if constexpr (WHOLE) {
#pragma unroll
            for (int d = d0; d < d1; ++d) {
                const unsigned lo = at + (d < XI ? kx : kw) >= rowb ? 0u : ~0u;
                const unsigned long long m = ((unsigned long long)lo << 32) | lo, zero = (unsigned long long)&g_zero16 & ~m;
                const unsigned long long u = (unsigned long long)((d < XI ? xbase : wbase) + at + off[d]);
                __builtin_amdgcn_global_load_lds((glb_ptr_t)((u & m) | zero), (lds_ptr_t)place(into, d), 16, 0, 0);
            }
        } else {
#pragma unroll
            for (int d = d0; d < d1; ++d)
                *reinterpret_cast<u32x4*>(place(into, d) + lane * 16) = chunk_at((d < XI ? xbase : wbase) + off[d], at, rowb - (d < XI ? kx : kw));
        }
    };

    // fragments, piece (4 h + lg) ^ key: rows 16 t + li of the wave's part of x; of the weights rows 32 (t / 2) + 8 (li / 4) +
    // 4 (t % 2) + li % 4, so that a lane's accumulators of two tiles are 8 consecutive outputs
    const int xo = wm * TM * 2048 + li * 128 + ((lg ^ ((li >> 1) & 7)) << 4);
    const int wo = XB + wn * TN * 2048 + (8 * (li >> 2) + (li & 3)) * 128 + ((lg ^ (((li >> 1) & 1) | ((li >> 2) << 1))) << 4);
    f32x4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 wf[2][TN], xf[2][TM];
    auto fetch = [&](int from, int h, int q) __attribute__((always_inline)) {    // fragment q of half h: weights, then x
        if (q < TN) wf[h][q] = *reinterpret_cast<const u32x4*>(smem + from + (wo ^ (h << 6)) + (q >> 1) * 4096 + (q & 1) * 512);
        else if (q < TN + TM) xf[h][q - TN] = *reinterpret_cast<const u32x4*>(smem + from + (xo ^ (h << 6)) + (q - TN) * 2048);
    };
    constexpr int FPG = TM == 8 ? 2 : TM == 4 ? 3 : 4;       // fragment reads a group of products: done before the last groups
    static_assert(FPG * TM >= TM + TN, "every fragment has its place");
    int cur = 0;                                             // offset of slice s's buffer
    bool holds = false;                                      // WHOLE false: slice s + 1 is still in `held`
    auto slice = [&](int s, bool fast) __attribute__((always_inline)) {
        wait_counts<63, 0>();                                // the first half's fragments
#pragma unroll
        for (int j = 0; j < TM; ++j) {
#pragma unroll
            for (int q = 0; q < FPG; ++q) fetch(cur, 1, j * FPG + q);
            if constexpr (BM == 256) __builtin_amdgcn_s_setprio(1);    // products before the other waves' reads (2 % there; smaller tiles lose by it)
            column<T, TN, TM>(acc, j, wf[0], xf[0][j]);
            if constexpr (!WHOLE)
                if (j == TM / 2 && holds) {
#pragma unroll
                    for (int d = 0; d < DMA; ++d) *reinterpret_cast<u32x4*>(place(BUF - cur, d) + lane * 16) = held[d];
                }
            if constexpr (BM == 256) __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
        }
        // all but the DMA of the last ST - 2 slices asked for has landed (near the end: all of it), fragments are read
        if (fast || s + ST - 1 < slices) wait_counts<DMA * (ST - 2), 0>();
        else wait_counts<0, 0>();
        block_barrier();
        if (!fast && s + ST < slices) stage(s + ST, cur, 0, DMA);
        holds = fast;
        const unsigned char *xs = xbase + (long)(s + ST) * 128, *ws = wbase + (long)(s + ST) * 128;
        asm("" : "+s"(xs), "+s"(ws));                        // scalar bases: the lanes add their 32-bit offsets
        const int free = cur;
        cur = cur + BUF == ST * BUF ? 0 : cur + BUF;
#pragma unroll
        for (int j = 0; j < TM; ++j) {
#pragma unroll
            for (int q = 0; q < FPG; ++q) fetch(cur, 0, j * FPG + q);      // behind the last slice: whatever that buffer holds, unused
            if (fast)
#pragma unroll
                for (int d = j * DPG; d < (j + 1) * DPG && d < DMA; ++d) dma(xs, ws, free, d);
            if constexpr (BM == 256) __builtin_amdgcn_s_setprio(1);
            column<T, TN, TM>(acc, j, wf[1], xf[1][j]);
            if constexpr (BM == 256) __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (slices) {
        // the weights first: the rows of x may still be looked up (rings of 2, whose next wait is for everything; the deeper
        // ones' waits count in the order of the slices)
        if constexpr (ST == 2) {
            for (int s = 0; s < ST && s < slices; ++s) stage(s, s * BUF, XI, DMA);
            for (int s = 0; s < ST && s < slices; ++s) stage(s, s * BUF, 0, XI);
        } else
            for (int s = 0; s < ST && s < slices; ++s) stage(s, s * BUF, 0, DMA);
        looked();
        if constexpr (!WHOLE) wait_counts<0, 0>();
        if (slices >= ST) wait_counts<(ST == 2 ? XI : DMA) * (ST - 1), 15>();
        else wait_counts<0, 15>();
        block_barrier();
#pragma unroll
        for (int q = 0; q < TM + TN; ++q) fetch(0, 0, q);
        int s = 0;
        for (; s + ST < full; ++s) slice(s, true);
        for (; s < slices; ++s) slice(s, false);
    } else looked();

    // epilogue, from the registers: vector q of x row 16 j + li is outputs n + 32 q .. + 7, a store 16 rows of 64 bytes (fp32: two
    // of 64).  Each choice of type or activation is made once for all vectors it concerns; a part's residuals are asked for
    // before the part before it is stored, so that the wait for them is not one for the stores.
    // Through LDS instead, whole lines a store, the epilogue of a 256-tile took 12 400 clocks (without residual or activation).
    constexpr int V = TN / 2, R = 2;                         // a part: R rows
    GemmArgs o = a;
    if (a.splits > 1) {                                      // a part's plain sums; gemm_join_kernel does the rest
        o.bias = o.res = nullptr; o.act = FR_ACT_NONE; o.out_type = FR_TYPE_F32;
        o.out = a.partial + (long)split * a.M * a.N;
    }
    const int n = n0 + wn * TN * 16 + lg * 8;
    const long p0 = r0 + wm * TM * 16 + li;
    long row[R];
    Raw8 ahead[R][V];
    auto rows_of = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < R; ++e) row[e] = p0 + (j0 + e) * 16 >= r1 ? -1 : by_slot ? out_row(o, p0 + (j0 + e) * 16) : p0 + (j0 + e) * 16;
        auto ask = [&](auto type) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < R; ++e)
#pragma unroll
                for (int q = 0; q < V; ++q)
                    if (row[e] >= 0 && n + 32 * q + 8 <= o.N) ahead[e][q] = raw_load8<false>(o.res, row[e] * o.ldr + n + 32 * q, type());
        };
        if (!o.res) return;
        if (o.res_type == FR_TYPE_F32) ask(Is<FR_TYPE_F32>());
        else ask(Is<FR_TYPE_BF16>());
    };
    Columns col[V];
#pragma unroll
    for (int q = 0; q < V; ++q) col[q] = columns(o, n + 32 * q, min(8, a.N - n - 32 * q), nbase, none);
    rows_of(0);
    const bool ragged = n0 + BN > a.N && a.N % 8;            // some lane's vector has N's end inside
    if (ragged) __syncthreads();                             // the ring is read
#pragma unroll
    for (int j0 = 0; j0 < TM; j0 += R) {
        Vec8f v[R][V];
        long to[R];
        auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < R; ++e)
#pragma unroll
                for (int q = 0; q < V; ++q) f(e, q);
        };
        each([&](int e, int q) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; ++r) { v[e][q].v[r] = acc[2 * q][j0 + e][r]; v[e][q].v[4 + r] = acc[2 * q + 1][j0 + e][r]; }
        });
        if (!none) {
            each([&](int e, int q) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[e][q].v[i] += col[q].bias.v[i];
            });
            auto all = [&](auto act) __attribute__((always_inline)) {
                each([&](int e, int q) __attribute__((always_inline)) {
                    act8<act()>(v[e][q], col[q].slope);
                    __builtin_amdgcn_sched_barrier(0);       // vectors mixed with each other take registers that there are not
                });
            };
            switch (o.act) {
                case FR_ACT_PRELU: all(Is<FR_ACT_PRELU>()); break;
                case FR_ACT_HSWISH: all(Is<FR_ACT_HSWISH>()); break;
                case FR_ACT_RELU: all(Is<FR_ACT_RELU>()); break;
                case FR_ACT_HSIGMOID: all(Is<FR_ACT_HSIGMOID>()); break;
                case FR_ACT_GELU: all(Is<FR_ACT_GELU>()); break;
                case FR_ACT_SILU: all(Is<FR_ACT_SILU>()); break;
                default: break;
            }
        }
        if (ragged)
            each([&](int e, int q) __attribute__((always_inline)) {
                if (n + 32 * q < a.N && n + 32 * q + 8 > a.N) *reinterpret_cast<Vec8f*>(smem + ((wave * TM + j0 + e) * 64 + lane) * 32) = v[e][q];
            });
        auto add = [&](auto type) __attribute__((always_inline)) {
            each([&](int e, int q) __attribute__((always_inline)) {
                const Vec8f r = raw_to_f(ahead[e][q], type());
#pragma unroll
                for (int i = 0; i < 8; ++i) v[e][q].v[i] += r.v[i];
            });
        };
        if (o.res) {
            if (o.res_type == FR_TYPE_F32) add(Is<FR_TYPE_F32>());
            else if (o.res_type == FR_TYPE_BF16) add(Is<FR_TYPE_BF16>());
            else add(Is<FR_TYPE_F16>());
        }
#pragma unroll
        for (int e = 0; e < R; ++e) to[e] = row[e];
        if (j0 + R < TM) rows_of(j0 + R);
        auto put = [&](auto type) __attribute__((always_inline)) {
            each([&](int e, int q) __attribute__((always_inline)) {
                if (to[e] >= 0 && n + 32 * q + 8 <= o.N) store8t<false>(o.out, to[e] * o.N + n + 32 * q, type(), v[e][q]);
            });
        };
        if (o.out_type == FR_TYPE_F32) put(Is<FR_TYPE_F32>());
        else if (o.out_type == FR_TYPE_BF16) put(Is<FR_TYPE_BF16>());
        else put(Is<FR_TYPE_F16>());
    }
    if (ragged) {                                            // those vectors, one element at a time
        const int q = a.N > n ? (a.N - n) / 32 : V, at = n + 32 * q, have = a.N - at;
        if (q < V && have > 0 && have < 8)
#pragma unroll 1
            for (int j = 0; j < TM; ++j) {
                const long p = p0 + j * 16, r = p < r1 ? out_row(o, p) : -1;
                Vec8f v = *reinterpret_cast<const Vec8f*>(smem + ((wave * TM + j) * 64 + lane) * 32);
                if (r < 0) continue;
                if (o.res) add8n(o, v, r, at, have);
                put8n(o.out, r * o.N + at, have, o.out_type, v);
            }
    }
}

// The parts of a split K added in their order, then the epilogue: 8 outputs a thread.  Bound by its launch: 128 x 4096 outputs in
// 8 parts, 4.5 us of the product's 17.
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs a) {
    const int vecs = (a.N + 7) / 8;
    const long i = blockIdx.x * 256l + threadIdx.x, row = i / vecs;
    if (row >= a.M) return;
    const int n = (int)(i - row * vecs) * 8, have = min(8, a.N - n);
    Vec8f v{};
    for (int s0 = 0; s0 < a.splits; s0 += 4) {
        Vec8f p[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s0 + s < a.splits) p[s] = get8n(a.partial, ((s0 + s) * a.M + row) * a.N + n, have, FR_TYPE_F32);
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s0 + s < a.splits) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v.v[j] += p[s].v[j];
            }
    }
    finish8(a, row, n, columns(a, n, have, 0, false), v, false);
}

// Few rows, of one matrix or of each expert: the weights are read once and are nearly all there is to read.  A block takes 16 weight rows and up to 16 MT rows
// of x; its NW waves take the slices of K in turn, each with a ring of R slices of its own in LDS, so that nothing waits but
// a wave for its own oldest slice; the waves' sums meet in LDS, in their order, and one launch does it all.
// The ring is filled by LDS-DMA in whole lines of 128 bytes: fragments straight from memory take 64 bytes of 16 rows an
// instruction, which the address path carries at half the rate (16 x 4096 x 4096: 12 us; 24 rows this way 8.6 in f16, 4.0 TB/s
// of weights, with 3.3 us of launch and first loads in it).  Rows that are not whole 16-byte
// chunks (WHOLE false) go through registers instead.
template <typename T, int MT, int NW, int R, bool WHOLE, bool EXPERTS>
__global__ __launch_bounds__(64 * NW) void gemm_rows_kernel(GemmArgs a) {
    constexpr int ROWS = 16 + 16 * MT, DPS = ROWS / 8, SLOT = ROWS * 128;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int nt = blockIdx.x % a.n_tiles, mt = blockIdx.x / a.n_tiles, n0 = nt * 16;
    long r0 = (long)mt * 16 * MT, r1 = min(r0 + 16 * MT, a.M);
    int expert = 0;
    if constexpr (EXPERTS)
        if (!expert_tile(a, mt, 16 * MT, scan_experts(a, 0, 16 * MT), expert, r0, r1)) return;
    const bool none = EXPERTS && expert == a.E;
    const long nbase = (long)expert * a.N, rowb = (long)a.K * Elem<T>::BYTES;
    f32x4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    unsigned char* ring = smem + wave * R * SLOT;
    // this lane's sources: row 8 d + lane / 8 of the 16 weight rows and then those of x, chunk (lane % 8) ^ key
    const unsigned char* src[DPS];
    int kx[2];                                           // the key of row r is that of r + 16
#pragma unroll
    for (int d = 0; d < 2; ++d) kx[d] = ((lane & 7) ^ (((8 * d + (lane >> 3)) >> 1) & 7)) * 16;
#pragma unroll
    for (int d = 0; d < DPS; ++d) {
        const int r = 8 * d + (lane >> 3);
        src[d] = (d < 2 ? reinterpret_cast<const unsigned char*>(a.w) + ((none ? 0 : nbase) + min(n0 + r, a.N - 1)) * rowb
                        : reinterpret_cast<const unsigned char*>(a.x) + (EXPERTS ? x_row(a, min(r0 + r - 16, r1 - 1)) : min(r0 + r - 16, r1 - 1)) * a.ldx * Elem<T>::BYTES) + kx[d & 1];
    }
    const int slices = none ? 0 : (int)((rowb + 127) / 128), mine = (slices - wave + NW - 1) / NW;    // <= 0: more waves than slices
    auto multiply = [&](const unsigned char* slot) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = li * 128 + (((4 * h + lg) ^ ((li >> 1) & 7)) << 4);
            const u32x4 w = *reinterpret_cast<const u32x4*>(slot + at);
            u32x4 x[MT];
#pragma unroll
            for (int j = 0; j < MT; ++j) x[j] = *reinterpret_cast<const u32x4*>(slot + (j + 1) * 2048 + at);
#pragma unroll
            for (int j = 0; j < MT; ++j) Elem<T>::mma(acc[j], w, x[j]);
        }
    };
    if constexpr (WHOLE) {
        auto stage = [&](int i, int slot) __attribute__((always_inline)) {
            const long at = (long)(wave + i * NW) * 128;
#pragma unroll
            for (int d = 0; d < DPS; ++d) {
                const unsigned lo = at + kx[d & 1] >= rowb ? 0u : ~0u;       // K may end inside the slice: zeros behind it
                const unsigned long long m = ((unsigned long long)lo << 32) | lo;
                const unsigned long long u = ((unsigned long long)(src[d] + at) & m) | ((unsigned long long)&g_zero16 & ~m);
                __builtin_amdgcn_global_load_lds((glb_ptr_t)u, (lds_ptr_t)(ring + slot * SLOT + d * 1024), 16, 0, 0);
            }
        };
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i < mine) stage(i, i);
        int slot = 0;
        for (int i = 0; i < mine; ++i) {
            if (i + R <= mine) wait_counts<(R - 1) * DPS, 15>();
            else wait_counts<0, 15>();
            multiply(ring + slot * SLOT);
            wait_counts<63, 0>();
            if (i + R < mine) stage(i + R, slot);
            slot = slot + 1 == R ? 0 : slot + 1;
        }
    } else {
        u32x4 c[DPS];
        auto fetch = [&](int i) __attribute__((always_inline)) {
            const long at = (long)(wave + i * NW) * 128;
#pragma unroll
            for (int d = 0; d < DPS; ++d) c[d] = chunk_at(src[d], at, rowb - kx[d & 1]);
        };
        if (mine > 0) fetch(0);
        for (int i = 0; i < mine; ++i) {
#pragma unroll
            for (int d = 0; d < DPS; ++d) *reinterpret_cast<u32x4*>(ring + d * 1024 + lane * 16) = c[d];
            if (i + 1 < mine) fetch(i + 1);
            wave_lds_fence();
            multiply(ring);
            wave_lds_fence();
        }
    }
    __syncthreads();
    f32x4* red = reinterpret_cast<f32x4*>(smem);             // [NW][MT][64], over the rings
#pragma unroll
    for (int j = 0; j < MT; ++j) red[(wave * MT + j) * 64 + lane] = acc[j];
    __syncthreads();
    if (tid >= MT * 32) return;
    // thread: row j * 16 + i, columns 8 half .. 8 half + 7: the four of lane groups 2 half and 2 half + 1
    const int j = tid >> 5, i = tid & 15, half = (tid >> 4) & 1;
    Vec8f v{};
#pragma unroll
    for (int q = 0; q < NW; ++q) {
        const f32x4 lo = red[(q * MT + j) * 64 + half * 32 + i], hi = red[(q * MT + j) * 64 + half * 32 + 16 + i];
#pragma unroll
        for (int e = 0; e < 4; ++e) { v.v[e] += lo[e]; v.v[4 + e] += hi[e]; }
    }
    const long at = r0 + 16 * j + i, row = at >= r1 ? -1 : EXPERTS ? out_row(a, at) : at;
    const int n = n0 + half * 8;
    if (row >= 0 && n < a.N) finish8(a, row, n, columns(a, n, min(8, a.N - n), nbase, none), v, none);
}

// Any shape, any alignment: 64 x 64 outputs a block, 4 waves of 32 x 32, slices of 128 bytes of K through registers into
// LDS.  Piece p of LDS row r lies at p ^ ((r >> 1) & 7): the 16 rows of a fragment read fall on different banks.  For what the
// staged kernel does not take: gathered rows beyond its 32-bit offsets, rows of 8 MB, few odd rows (300 x 1001 x 1001 bf16 15 us,
// bound by the latency of one slice after the other).
template <typename T>
__global__ __launch_bounds__(256) void gemm_any_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][64 * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int mt = blockIdx.z * 65535 + blockIdx.y, n0 = blockIdx.x * 64;
    if (!a.order && (long)mt * 64 >= a.M) return;
    long r0 = (long)mt * 64, r1 = min(r0 + 64, a.M);
    int expert = 0;
    if (a.order && !expert_tile(a, mt, 64, scan_experts(a, 0, 64), expert, r0, r1)) return;
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
        finish8(a, row, n, columns(a, n, min(8, a.N - n), nbase, none), v, none);
    }
}

template <typename T, int BM, int BN, int WM, int WN, int ST, bool WHOLE = true>
int launch_tile(GemmArgs a, hipStream_t st) {
    const long mt = a.order ? a.M / BM + std::min<long>(a.M, a.E + 1) : (a.M + BM - 1) / BM;
    a.n_tiles = (int)((a.N + (BN - 1l)) / BN);
    if (mt * a.n_tiles * a.splits >= (1l << 32) / (64 * WM * WN)) FR_FAIL(FR_ERR_UNSUPPORTED, "adapter product: more output tiles than a launch takes");
    const int lds = ST * (BM + BN) * 128;
    static_assert(WN * BM <= ST * (BM + BN), "the ring has room for the vectors that N ends in: 32 bytes a lane and row tile");
    FR_BIG_LDS_ONCE((gemm_tile_kernel<T, BM, BN, WM, WN, ST, WHOLE>), lds);
    hipLaunchKernelGGL((gemm_tile_kernel<T, BM, BN, WM, WN, ST, WHOLE>), dim3((unsigned)(mt * a.n_tiles * a.splits)), dim3(64 * WM * WN), lds, st, a);
    FR_LAUNCH_CHECK("gemm_tile_kernel");
    return FR_OK;
}

// Output tiles of bm x bn; of the experts' products an estimate (the counts are on the device): half a tile more for each.
double tile_count(const GemmArgs& a, int bm, int bn) {
    const double some = a.order ? (double)std::min<long>(a.M, a.E) : 0;
    const double rows = a.order ? std::max((double)a.M / bm + 0.5 * some, some) : (double)((a.M + bm - 1) / bm);
    return rows * ((a.N + (bn - 1l)) / bn);
}
// Estimated time in us with tiles of bm x bn: `each` for a slice of 128 bytes of K and `fixed` for the rest of a tile, for every
// tile of the fullest CU.  The constants are least squares over some 90 shapes of 100 to 18 700 rows on one card, which
// profiles/tuning/adapter_tiles.txt lists with every tile's time (rms 3 % in fp32, 13 to 16 % in 16 bits); what the rule picks takes
// 1.4 % more than the best of all tiles there (fp32: 1.8 %), and 0.79 of the time of the library's plain product (fp32: 1.03; 0.82
// and 0.99 where the library's time is not mostly the host's).
template <typename T>
double tile_cost(const GemmArgs& a, int bm, int bn, double each16, double fixed16, double each32, double fixed32) {
    constexpr bool f32 = std::is_same<T, float>::value;
    return ceil(tile_count(a, bm, bn) / 256) * (((long)a.K * Elem<T>::BYTES + 127) / 128 * (f32 ? each32 : each16) + (f32 ? fixed32 : fixed16));
}

template <typename T, int MT, int NW, int R, bool EXPERTS = false>
int launch_rows(GemmArgs a, bool whole, hipStream_t st) {
    const long mt = EXPERTS ? a.M / (16 * MT) + std::min<long>(a.M, a.E + 1) : (a.M + 16 * MT - 1) / (16 * MT);
    a.n_tiles = (int)((a.N + 15l) / 16);
    if (mt * a.n_tiles >= (1l << 32) / (64 * NW)) FR_FAIL(FR_ERR_UNSUPPORTED, "adapter product: more output tiles than a launch takes");
    const int lds = NW * R * (16 + 16 * MT) * 128;
    const dim3 grid((unsigned)(mt * a.n_tiles)), block(64 * NW);
    if (whole) {
        FR_BIG_LDS_ONCE((gemm_rows_kernel<T, MT, NW, R, true, EXPERTS>), lds);
        hipLaunchKernelGGL((gemm_rows_kernel<T, MT, NW, R, true, EXPERTS>), grid, block, lds, st, a);
    } else hipLaunchKernelGGL((gemm_rows_kernel<T, MT, NW, 1, false, EXPERTS>), grid, block, lds / R, st, a);
    FR_LAUNCH_CHECK("gemm_rows_kernel");
    return FR_OK;
}

// K of a product whose 64-tiles leave most of the card idle is split into parts of at least 4 slices, up to two blocks a CU.
// 128 x 4096 x 4096 bf16: 17 us, 20 in one part; K of fewer than 16 slices saves less than the second launch takes.
int split_count(int64_t M, int N, int K, int type) {
    const long slices = ((long)K * type_bytes(type) + 127) / 128, tiles = ((M + 63) / 64) * ((N + 63l) / 64);
    if (M <= 64 || tiles > 160 || slices < 16) return 1;        // up to 64 rows: gemm_rows_kernel
    return (int)std::max(1l, std::min(std::min(slices / 4, 512 / tiles), 16l));
}

template <typename T>
int launch_gemm(GemmArgs a, hipStream_t st) {
    const long rowb = (long)a.K * Elem<T>::BYTES, ldxb = a.ldx * Elem<T>::BYTES;
    const bool gather = a.order && !a.rows_sorted;
    const bool whole = rowb % 16 == 0 && ldxb % 16 == 0 && ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.w & 15) == 0;
    // the staged kernel adds 32-bit offsets to its tile's (gathered rows: the matrix's) first row
    const bool near = std::max(rowb, ldxb) < (1l << 23) && (!gather || a.M / a.k * ldxb < (1l << 32));
    a.splits = 1;
    if (!a.order && a.M <= 64 && (rowb >= 1024 || !whole)) {
        // us at K = N = 4096 (16 bits) / 2048 (fp32), against 64-tiles with K split: 16 rows 10 and 14, 24 rows 10 and 15,
        // 64 rows 13 and 18; fp32 24 rows 9 and 17, 64 rows 14 and 19 (two tiles of 32 rows there: 17 as one of 64)
        constexpr bool f32 = std::is_same<T, float>::value;
        if (a.M <= 16 || (f32 && a.M <= 32)) return launch_rows<T, 1, 8, 4>(a, whole, st);
        if (a.M <= 32 || f32) return launch_rows<T, 2, 8, 3>(a, whole, st);
        return launch_rows<T, 4, 4, 3>(a, whole, st);
    }
    // experts with few rows each, by the few blocks of one round (fp32: two, its tiles walk K at half the pace), us against
    // 64-tiles: 7 rows of 13 experts x 384 x 2432, 168 blocks, bf16 6.9 and 11, fp32 8.9 and 45; 512 blocks 10 % slower in bf16,
    // 10 to 50 % faster in fp32, 1024 half as fast and equal; odd rows, against gemm_any_kernel, 1134 blocks 13 and 42
    const long some = std::min<long>(a.M, a.E);
    const bool few = a.order && a.M <= 32 * some;
    if (few && (rowb >= 1024 || !whole)) {
        const int rows = a.M <= 8 * some ? 16 : 32;
        if (tile_count(a, rows, 16) <= (!whole ? 2048 : Elem<T>::BYTES == 4 ? 512 : 256))
            return rows == 16 ? launch_rows<T, 1, 8, 4, true>(a, whole, st) : launch_rows<T, 2, 8, 3, true>(a, whole, st);
    }
    // rows of any alignment, us against gemm_any_kernel: 16384 x 2048 x 4097 bf16 440 and 723, 3001 x 2047 x 2049 58 and 90;
    // a 64-tile alone on its CU has its chunks sooner there (300 x 1001 x 1001: 18 and 15, in parts of K 16), but for
    // a long K in parts (554 x 242 x 1461 f32 45 and 22, 156 x 1024 x 7874 f16 73 and 21)
    const double tiles64 = tile_count(a, 64, 64);
    const int splits = a.partial ? split_count(a.M, a.N, a.K, Elem<T>::BYTES == 4 ? FR_TYPE_F32 : FR_TYPE_BF16) : 1;
    const bool parts = splits > 1 && (whole || rowb >= 24 * 128);
    if (near && (whole || tiles64 > 256 || parts)) {
        const bool alone = tile_count(a, 128, 128) <= 256;
        const double c256 = tile_cost<T>(a, 256, 256, 1.10, 5.5, 7.29, 9.0), c64 = tile_cost<T>(a, 64, 64, 0.195, 0.3, 0.535, 0.3);
        const double c128 = alone ? tile_cost<T>(a, 128, 128, 0.412, 0.0, 1.85, 0.8) : tile_cost<T>(a, 128, 128, 0.474, 0.9, 1.91, 1.8);
        const double c12864 = tile_cost<T>(a, 128, 64, 0.296, 0.8, 0.99, 1.1);
        if (parts) {
            const long slices = (rowb + 127) / 128;
            a.split_slices = (int)((slices + splits - 1) / splits);
            a.splits = (int)((slices + a.split_slices - 1) / a.split_slices);
            const int rc = whole ? launch_tile<T, 64, 64, 2, 2, 3>(a, st) : launch_tile<T, 64, 64, 2, 2, 2, false>(a, st);
            if (rc) return rc;
            hipLaunchKernelGGL(gemm_join_kernel, dim3((unsigned)((a.M * ((a.N + 7) / 8) + 255) / 256)), dim3(256), 0, st, a);
            FR_LAUNCH_CHECK("gemm_join_kernel");
            return FR_OK;
        }
        if (!whole) return c128 <= c64 ? launch_tile<T, 128, 128, 2, 4, 2, false>(a, st) : launch_tile<T, 64, 64, 2, 2, 2, false>(a, st);
        // an expert's few rows are one tile of any height: 5 rows, 2 of 32 experts, 512 -> 2048: 7.0 us by 64-tiles, 10.8 by 128
        if (!few && c256 <= std::min(c128, std::min(c12864, c64))) return launch_tile<T, 256, 256, 2, 4, 2>(a, st);
        if (!few && c12864 <= std::min(c128, c64)) return launch_tile<T, 128, 64, 4, 2, 3>(a, st);
        // a deeper ring for a tile alone on its CU, more tiles at a time for others: 2048 cubed bf16 (128-tiles) 20 us, 26 with
        // the ring of 2; 200 x 4096 x 4096 (64-tiles) 16 us, 19 with the ring of 3; 32 experts' 64 rows, 4 tiles a CU, 20 and 16
        if (few || c64 <= c128) return tiles64 <= 256 ? launch_tile<T, 64, 64, 2, 2, 5>(a, st) : launch_tile<T, 64, 64, 2, 2, 3>(a, st);
        return alone ? launch_tile<T, 128, 128, 2, 4, 3>(a, st) : launch_tile<T, 128, 128, 2, 4, 2>(a, st);
    }
    const long mt = a.order ? a.M / 64 + std::min<long>(a.M, a.E + 1) : (a.M + 63) / 64;
    a.n_tiles = (int)((a.N + 63l) / 64);
    if (mt >= 1l << 24 || a.n_tiles >= 1 << 24) FR_FAIL(FR_ERR_UNSUPPORTED, "adapter product: more output tiles than a launch takes");
    hipLaunchKernelGGL((gemm_any_kernel<T>), dim3(a.n_tiles, (unsigned)std::min(mt, 65535l), (unsigned)((mt + 65534) / 65535)), dim3(256), 0, st, a);
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
    if (M >= 1ll << 40) FR_FAIL(FR_ERR_UNSUPPORTED, "fr_linear_workspace_bytes: M does not fit 40 bits");
    const int splits = split_count(M, N, K, type);
    *out_bytes = splits > 1 ? (size_t)splits * M * N * 4 : 0;
    return FR_OK;
}

extern "C" int fr_linear(const void* x, int64_t ldx, const void* w, const void* bias, const float* slope,
                         const void* residual, int64_t ldr, void* out, int64_t M, int N, int K,
                         int type, int bias_type, int res_type, int out_type, int act,
                         void* workspace, size_t workspace_bytes, void* stream) {
    if (M < 0 || N <= 0 || K <= 0 || ldx < 0 || (residual && ldr < 0)) FR_FAIL(FR_ERR_ARG, "fr_linear: bad shape");
    if (M >= 1ll << 40) FR_FAIL(FR_ERR_UNSUPPORTED, "fr_linear: M does not fit 40 bits");
    if (!type_ok(type) || !type_ok(out_type) || (bias && bias_type != type && bias_type != FR_TYPE_F32) || (residual && !type_ok(res_type)))
        FR_FAIL(FR_ERR_ARG, "fr_linear: unknown element type (bias: the operands' type or fp32)");
    if (act < FR_ACT_NONE || act > FR_ACT_SILU) FR_FAIL(FR_ERR_ARG, "fr_linear: unknown activation");
    if (act == FR_ACT_PRELU && !slope) FR_FAIL(FR_ERR_ARG, "fr_linear: PReLU without slopes");
    if (M == 0) return FR_OK;
    if (!x || !w || !out) FR_FAIL(FR_ERR_ARG, "fr_linear: NULL tensor");
    const int splits = split_count(M, N, K, type);
    if (splits > 1 && (!workspace || workspace_bytes < (size_t)splits * M * N * 4)) FR_FAIL(FR_ERR_WORKSPACE, "fr_linear: workspace too small");
    GemmArgs a{};
    a.partial = splits > 1 ? (float*)workspace : nullptr;
    a.x = x; a.w = w; a.bias = bias; a.slope = slope; a.res = residual; a.out = out;
    a.M = M; a.ldx = ldx; a.ldr = ldr; a.N = N; a.K = K;
    a.bias_type = bias_type; a.res_type = res_type; a.out_type = out_type; a.act = act;
    return launch_type(type, a, (hipStream_t)stream);
}

extern "C" int fr_expert_linear(const void* x, int rows_sorted, const void* w, const void* bias, const float* slope,
                                const int32_t* order, const int32_t* offsets, void* out, int out_slots,
                                int64_t T, int k, int E, int N, int K, int type, int bias_type, int out_type, int act, void* stream) {
    if (T < 0 || k <= 0 || E <= 0 || N <= 0 || K <= 0) FR_FAIL(FR_ERR_ARG, "fr_expert_linear: bad shape");
    if (T > 0x7FFFFFFFll / k) FR_FAIL(FR_ERR_UNSUPPORTED, "fr_expert_linear: T * k does not fit 31 bits");
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
    // k_mul = (2^(31 + k_shift) + e) / k with e < k <= 2^k_shift: s e / (k 2^(31 + k_shift)) < 1 / k takes no quotient to the next
    while ((1l << a.k_shift) < k) ++a.k_shift;
    a.k_mul = (unsigned)(((1ull << (31 + a.k_shift)) + k - 1) / k);
    return launch_type(type, a, (hipStream_t)stream);
}
