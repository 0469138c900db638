// Norms around an adapter block, fused with the weighted sum of expert rows, the gate, the scale and the residual:
//   y = x  |  sum_j w_j x_j;   out = residual + scale * g(gate) * norm(y);   next = next_norm(out)
#include "adapter.h"

namespace {

struct NormArgs {
    const void* x; const float* slot_w; const float* weight; const float* bias;
    const void* gate; const void* res; void* out;
    const float* next_weight; const float* next_bias; void* next_out;
    long T, gate_ldt, row0;
    int d, slots, gate_ldc;
    int x_type, gate_type, res_type, out_type, next_type;
    int norm, next_norm, gate_act;
    float eps, next_eps, scale;
};

FR_DEV float wave_sum64(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Sum over the threads of a row: a wave (TPR = 64) or the block (TPR = 256; `part` holds one value per wave and is used
// in turn by successive sums, `turn` counts them, so that one barrier a sum is enough).
template <int TPR>
FR_DEV float row_sum(float v, float (*part)[4], int& turn) {
    v = wave_sum64(v);
    if constexpr (TPR > 64) {
        float* p = part[turn & 1];
        ++turn;
        if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (p[0] + p[1]) + (p[2] + p[3]);
    }
    return v;
}

template <bool VEC>
FR_DEV Vec8f get8(const void* base, long i, int n, int type) {      // n: elements that exist (8 where VEC)
    if (VEC || n == 8) return raw_to_f(raw_load8<VEC>(base, i, type), type);
    Vec8f o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = j < n ? load1(base, i + j, type) : 0.f;
    return o;
}
template <bool VEC>
FR_DEV void put8(void* base, long i, int n, int type, const Vec8f& v) {
    if (VEC || n == 8) { store8t<VEC>(base, i, type, v); return; }
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) store1(base, i + j, type, v.v[j]);
}

// The norm of a row held as NV vectors of 8 a thread; elements behind d are 0 on entry and stay out of the variance.
template <int TPR, int NV, bool VEC>
FR_DEV void norm_row(Vec8f (&v)[NV], int norm, const float* weight, const float* bias, float eps, int d, int col0,
                     float (*part)[4], int& turn) {
    if (norm == FR_NORM_NONE) return;
    float mean = 0.f;
    if (norm == FR_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[q].v[j];
        mean = row_sum<TPR>(s, part, turn) / (float)d;
    }
    float ss = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int n = min(8, d - (col0 + q * TPR * 8));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[q].v[j] = j < n ? v[q].v[j] - mean : 0.f;
            ss = fmaf(v[q].v[j], v[q].v[j], ss);
        }
    }
    ss = row_sum<TPR>(ss, part, turn);
    float inv;
    if (norm == FR_NORM_L2) {
        const float nrm = sqrtf(ss);
        inv = nrm == 0.f ? 0.f : 1.f / nrm;
    } else {
        inv = 1.f / sqrtf(ss / (float)d + eps);
    }
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int c = col0 + q * TPR * 8, n = min(8, d - c);
        if (n <= 0) continue;
        Vec8f w, b;
        if (weight) w = get8<VEC>(weight, c, n, FR_TYPE_F32);
        if (bias) b = get8<VEC>(bias, c, n, FR_TYPE_F32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float t = v[q].v[j] * inv;
            if (weight) t *= w.v[j];
            if (bias) t += b.v[j];
            v[q].v[j] = t;
        }
    }
}

// One row, held in registers from its one read to its writes.
template <int TPR, int NV, bool VEC>
FR_DEV void one_row(const NormArgs& a, long row, int col0, float (*part)[4], int& turn) {
    Vec8f v[NV];
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[q].v[j] = 0.f;
    if (a.slots == 0) {
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int c = col0 + q * TPR * 8, n = min(8, a.d - c);
            if (n > 0) v[q] = get8<VEC>(a.x, row * a.d + c, n, a.x_type);
        }
    } else {
        for (int s = 0; s < a.slots; ++s) {
            const float w = a.slot_w[row * a.slots + s];
            if (w == 0.f) continue;
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                const int c = col0 + q * TPR * 8, n = min(8, a.d - c);
                if (n <= 0) continue;
                const Vec8f x = get8<VEC>(a.x, (row * a.slots + s) * a.d + c, n, a.x_type);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[q].v[j] = fmaf(w, x.v[j], v[q].v[j]);
            }
        }
    }
    norm_row<TPR, NV, VEC>(v, a.norm, a.weight, a.bias, a.eps, a.d, col0, part, turn);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int c = col0 + q * TPR * 8, n = min(8, a.d - c);
        if (n <= 0) continue;
        if (a.gate) {
            Vec8f g;
            if (a.gate_ldc) g = get8<VEC>(a.gate, row * a.gate_ldt + c, n, a.gate_type);
            else {
                const float g1 = load1(a.gate, row * a.gate_ldt, a.gate_type);
#pragma unroll
                for (int j = 0; j < 8; ++j) g.v[j] = g1;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float t = g.v[j];
                if (a.gate_act == FR_GATE_SIGMOID) t = 1.f / (1.f + expf(-t));
                else if (a.gate_act == FR_GATE_TANH) t = tanhf(t);
                v[q].v[j] *= t;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[q].v[j] *= a.scale;
        if (a.res) {
            const Vec8f r = get8<VEC>(a.res, row * a.d + c, n, a.res_type);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[q].v[j] += r.v[j];
        }
        if (a.out) put8<VEC>(a.out, row * a.d + c, n, a.out_type, v[q]);
    }
    if (!a.next_out) return;
    norm_row<TPR, NV, VEC>(v, a.next_norm, a.next_weight, a.next_bias, a.next_eps, a.d, col0, part, turn);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int c = col0 + q * TPR * 8, n = min(8, a.d - c);
        if (n > 0) put8<VEC>(a.next_out, row * a.d + c, n, a.next_type, v[q]);
    }
}

// One row per wave (TPR = 64, 4 rows a block) or per block (TPR = 256).
// VEC: d is a multiple of 8 and every tensor starts at a 16-byte address.
// Bound by memory: 65536 x 512 bf16, gate, residual and unit rows out, moves its 268 MB in 58 us a call over three inputs in turn,
// 4.6 TB/s (a copy of 4 GiB: 4.8); 49 to 54 on one input, part of which stays in the cache.
// Asking for the residual with the row changed nothing, a loop over rows inside the kernel cost a third.
template <int TPR, int NV, bool VEC>
__global__ __launch_bounds__(256) void block_norm_kernel(NormArgs a) {
    __shared__ float part[2][4];
    constexpr int RPB = 256 / TPR;
    const int col0 = (threadIdx.x % TPR) * 8;
    int turn = 0;
    const long row = a.row0 + (long)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row < a.T) one_row<TPR, NV, VEC>(a, row, col0, part, turn);      // TPR = 256: the whole block or none of it
}

// A launch takes 2^22 rows; more take several.
template <int TPR, int NV>
void launch(NormArgs a, bool vec, hipStream_t st) {
    for (a.row0 = 0; a.row0 < a.T; a.row0 += 1l << 22) {
        const dim3 grid((unsigned)((std::min(a.T - a.row0, 1l << 22) + 256 / TPR - 1) / (256 / TPR)));
        if (vec) hipLaunchKernelGGL((block_norm_kernel<TPR, NV, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((block_norm_kernel<TPR, NV, false>), grid, dim3(256), 0, st, a);
    }
}

bool at16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int fr_block_norm(const void* x, int x_type, int slots, const float* slot_weights, int64_t T, int d,
                             int norm, const float* weight, const float* bias, float eps,
                             const void* gate, int gate_type, int64_t gate_ldt, int gate_ldc, int gate_act, float scale,
                             const void* residual, int res_type, void* out, int out_type,
                             int next_norm, const float* next_weight, const float* next_bias, float next_eps,
                             void* next_out, int next_type, void* stream) {
    if (T < 0 || d <= 0 || d > 16384 || slots < 0) FR_FAIL(FR_ERR_ARG, "fr_block_norm: bad shape (1 <= d <= 16384)");
    if (T >= 1ll << 40) FR_FAIL(FR_ERR_UNSUPPORTED, "fr_block_norm: T does not fit 40 bits");
    if (norm < 0 || norm > FR_NORM_L2 || next_norm < 0 || next_norm > FR_NORM_L2) FR_FAIL(FR_ERR_ARG, "fr_block_norm: unknown norm");
    if (gate_act < 0 || gate_act > FR_GATE_TANH) FR_FAIL(FR_ERR_ARG, "fr_block_norm: unknown gate activation");
    if (!type_ok(x_type) || (gate && !type_ok(gate_type)) || (residual && !type_ok(res_type)) || (out && !type_ok(out_type)) ||
        (next_out && !type_ok(next_type))) FR_FAIL(FR_ERR_ARG, "fr_block_norm: unknown element type");
    if (gate && ((gate_ldc != 0 && gate_ldc != 1) || gate_ldt < 0)) FR_FAIL(FR_ERR_ARG, "fr_block_norm: gate strides");
    if (slots > 0 && !slot_weights) FR_FAIL(FR_ERR_ARG, "fr_block_norm: slots without slot_weights");
    if ((norm == FR_NORM_NONE || norm == FR_NORM_L2) && (weight || bias)) FR_FAIL(FR_ERR_ARG, "fr_block_norm: weight / bias belong to the rms and layer norms");
    if ((next_norm == FR_NORM_NONE || next_norm == FR_NORM_L2) && (next_weight || next_bias)) FR_FAIL(FR_ERR_ARG, "fr_block_norm: next_weight / next_bias belong to the rms and layer norms");
    if ((next_norm != FR_NORM_NONE) != (next_out != nullptr)) FR_FAIL(FR_ERR_ARG, "fr_block_norm: next_norm and next_out go together");
    if (!out && !next_out) FR_FAIL(FR_ERR_ARG, "fr_block_norm: no output");
    if (T == 0) return FR_OK;
    if (!x) FR_FAIL(FR_ERR_ARG, "fr_block_norm: x is NULL");
    NormArgs a{x, slot_weights, weight, bias, gate, residual, out, next_weight, next_bias, next_out, T, gate_ldt, 0,
               d, slots, gate_ldc, x_type, gate_type, res_type, out_type, next_type, norm, next_norm, gate_act, eps, next_eps, scale};
    const bool vec = d % 8 == 0 && at16(x) && at16(weight) && at16(bias) && (!gate || !gate_ldc || (at16(gate) && gate_ldt % 8 == 0)) &&
                     at16(residual) && at16(out) && at16(next_weight) && at16(next_bias) && at16(next_out);
    hipStream_t st = (hipStream_t)stream;
    if (d <= 512) launch<64, 1>(a, vec, st);
    else if (d <= 1024) launch<64, 2>(a, vec, st);
    else if (d <= 2048) launch<256, 1>(a, vec, st);
    else if (d <= 4096) launch<256, 2>(a, vec, st);
    else if (d <= 8192) launch<256, 4>(a, vec, st);
    else launch<256, 8>(a, vec, st);
    FR_LAUNCH_CHECK("block_norm_kernel");
    return FR_OK;
}
