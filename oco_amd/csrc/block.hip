// The step between two blocks of a layer in one pass over its rows: the norm
// after a block, its gate, its scale, the residual add, the norm before the
// next block, and that block's input rows in 8-bit floating point.  With v
// the block's output row y, post-normed where there is a weight for it,
//
//     v  = y / sqrt(mean(y^2) + epsilon) * (post_w + offset)
//     x' = x + scale * g * v,  g = 1, gate, sigmoid(gate) or tanh(gate)
//     out = x' / sqrt(mean(x'^2) + epsilon) * (pre_w + offset)
//
// x' is rounded to the residual's type and the second norm reads the rounded
// values, as oco_add_norm does.  Everything between is f32; with 8-bit rows
// the squares, their sums and the values between are 64-bit (the gate's value
// f32), since one value in a million lies within the f32 roundings of a border
// between two codes (512 x 2880 with a gate per row: 10.3 us, 9.3 in f32; 8192
// x 4096 bf16: 95 us, 91 with f32 squares).
//
// Bound by memory: x, y and the gate are read once, x' and out written once.
// A row stays in its threads' registers (runs of eight columns per thread,
// 16-byte accesses for 16-bit types) from its only read to its last write:
// 8192 x 4096 bf16 in 57 to 59 us (268 MB, 4.5 to 4.7 TB/s: the rate of a large
// copy); one row of 4096 in 3.7 us, two memory latencies and two sums over the row.
#include "fp8.h"
#include "rows.h"

namespace oco {

struct BlockArgs {
    const void *x, *y, *gate;
    const float *post_w, *pre_w;
    void *x_out, *out;
    uint8_t *codes;
    float *scales;
    uint32_t rows, n, kind, gate_rows;
    uint64_t x_stride, y_stride, gate_stride, out_stride;
    float scale, epsilon, offset;
};

// 1 / sqrt(mean + epsilon) from the T threads' sums of squares of a row, in every one of them (fixed order).
template <int T, class V>
__device__ __forceinline__ V row_inverse(const BlockArgs &a, V mine, V *part) {
    // one lane's of it: the order of the additions differs between lanes
    V s;
    if constexpr (sizeof(V) == 8)
        s = wave_sum_f64(mine);
    else
        s = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_sum(mine))));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        s = part[0];
#pragma unroll
        for (int w = 1; w < T / 64; w++) s += part[w];
    }
    if constexpr (sizeof(V) == 8)
        return rsqrt_f64(__builtin_fma(s, recip_f64((double)a.n), (double)a.epsilon));
    else
        return 1.0f / sqrtf(s / (float)a.n + a.epsilon);
}

// 1 / d for d >= 1 (0 for Inf).
__device__ __forceinline__ float recip_f32(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return d < INFINITY ? fmaf(fmaf(-d, r, 1.f), r, r) : r;
}
// tanh: its Taylor series to g^21 up to 0.625 (relative remainder 0.16^11), 1 - 2 / (exp(2 |g|) + 1) beyond, within
// 3 x 2^-24.  A gate row that all rows share is formed again for each row, so its instructions count: 8192 x 4096
// bf16 70.5 us with tanh and 67.3 with the sigmoid, 73.1 and 72.1 by tanhf and a division, 54 without a gate.
__device__ __forceinline__ float gate_value(float g, uint32_t kind) {
    if (kind == OCO_GATE_SIGMOID) return recip_f32(1.0f + expf(-g));
    if (kind == OCO_GATE_TANH) {
        constexpr float C[10] = {9.69153796e-05f, -0.000239129114f, 0.000590027441f, -0.00145583439f, 0.00359212804f, -0.00886323553f, 0.0218694885f, -0.053968254f, 0.133333333f, -0.333333333f};
        const float s = g * g, t = fabsf(g);
        float p = C[0];
#pragma unroll
        for (int i = 1; i < 10; i++) p = fmaf(p, s, C[i]);
        const float far = fmaf(-2.f, recip_f32(1.f + __builtin_amdgcn_exp2f(t * 2.88539008f)), 1.f);
        return t < 0.625f ? fmaf(g * s, p, g) : copysignf(far, g);
    }
    return g;
}

// A run of weights and gate values, as the formulas use them.
struct BlockRun {
    float post[8], gate[8], pre[8];
};
template <class YT>
__device__ __forceinline__ void block_load_add(const BlockArgs &a, const YT *gate, uint32_t c0, BlockRun &w) {
    if (a.post_w) load_run(a.post_w, c0, a.n, w.post);
    if (a.kind != OCO_GATE_NONE) load_run(gate, c0, a.n, w.gate);
}
__device__ __forceinline__ void block_load_out(const BlockArgs &a, uint32_t c0, BlockRun &w) {
    if (a.pre_w) load_run(a.pre_w, c0, a.n, w.pre);
}

// x' of one run of columns (rounded), from the run's v; V: the type between.
template <class XT, class V>
__device__ __forceinline__ void block_add(const BlockArgs &a, const float *xv, float *v, const BlockRun &w, V inv) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        V d = (V)v[j];
        if (a.post_w) d = d * inv * ((V)w.post[j] + (V)a.offset);
        if (a.kind != OCO_GATE_NONE) d *= (V)gate_value(w.gate[j], a.kind);
        v[j] = RowIO<XT>::round((float)__builtin_elementwise_fma((V)a.scale, d, (V)xv[j]));
    }
}

// out of one run of columns of x', and its 8-bit form where V is 64-bit.
template <class YT, class V>
__device__ __forceinline__ void block_out(const BlockArgs &a, const float *v, const BlockRun &w, uint64_t row, uint32_t c0, V inv) {
    V d[8];
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        d[j] = c0 + j < a.n ? (V)v[j] * (sizeof(V) == 8 ? (V)1 : inv) * ((V)w.pre[j] + (V)a.offset) : (V)0;
        o[j] = sizeof(V) == 8 ? c0 + j < a.n ? (float)(d[j] * inv) : 0.f : (float)d[j];
    }
    if (a.out) store_run((YT *)a.out + row * a.out_stride, c0, a.n, o);
    if constexpr (sizeof(V) == 8) {  // 16 consecutive threads hold a block of 128 columns
        float scale;
        const uint2 q = fp8_block(d, inv, o, scale);
        if (c0 < a.n) {
            *reinterpret_cast<uint2 *>(a.codes + row * a.n + c0) = q;
            if (c0 % FP8_BLOCK == 0) a.scales[(uint64_t)(c0 / FP8_BLOCK) * a.rows + row] = scale;
        }
    }
}

// s + v^2 (64-bit: the square is exact).
template <class V>
__device__ __forceinline__ V block_square(float v, V s) {
    return __builtin_elementwise_fma((V)v, (V)v, s);
}

// T threads per row (64: four rows per workgroup), P runs of eight columns
// per thread; P == 0: any n, a row read again for each of its three passes.
// A thread of one run requests its weights and gate with the rows, so that
// one memory latency stands before the first sum and none behind it (calls on
// 4096 columns with one run of 512 threads and with two of 256: one row 5.2 and
// 5.6 us, 256 rows 5.2 and 6.3, 1024 rows 11.4 and 11.0, 8192 rows 59 both);
// with two runs the registers cost more than that gives (66 us).
template <class XT, class YT, class V, int T, int P>
__global__ __launch_bounds__(T < 256 ? 256 : T) void block_kernel(BlockArgs a) {
    __shared__ V part[2][T / 64];
    const uint32_t t = T == 64 ? threadIdx.x & 63 : threadIdx.x;
    const uint64_t row = T == 64 ? blockIdx.x * 4ull + (threadIdx.x >> 6) : blockIdx.x;
    if (T == 64 && row >= a.rows) return;
    const XT *x = (const XT *)a.x + row * a.x_stride;
    const YT *y = (const YT *)a.y + row * a.y_stride;
    const YT *gate = (const YT *)a.gate + (uint64_t)(a.gate_rows ? (uint32_t)row / a.gate_rows : 0) * a.gate_stride;
    XT *x_out = (XT *)a.x_out + row * a.x_stride;
    if constexpr (P > 0) {
        constexpr bool EARLY = P == 1;
        float xv[P][8], v[P][8];
        V s = 0, inv = 1;
        BlockRun w[EARLY ? P : 1];
#pragma unroll
        for (int p = 0; p < P; p++) load_run(y, 8 * (t + T * p), a.n, v[p]);
#pragma unroll
        for (int p = 0; p < P; p++) load_run(x, 8 * (t + T * p), a.n, xv[p]);
        if constexpr (EARLY) {
#pragma unroll
            for (int p = 0; p < P; p++) block_load_add(a, gate, 8 * (t + T * p), w[p]);
#pragma unroll
            for (int p = 0; p < P; p++) block_load_out(a, 8 * (t + T * p), w[p]);
        }
        if (a.post_w) {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int j = 0; j < 8; j++) s = block_square<V>(v[p][j], s);
            inv = row_inverse<T, V>(a, s, part[0]);
        }
        s = 0;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const uint32_t c0 = 8 * (t + T * p);
            if constexpr (!EARLY) block_load_add(a, gate, c0, w[0]);
            block_add<XT, V>(a, xv[p], v[p], w[EARLY ? p : 0], inv);
            store_run(x_out, c0, a.n, v[p]);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c0 + j < a.n) s = block_square<V>(v[p][j], s);
        }
        if (!a.pre_w) return;
        inv = row_inverse<T, V>(a, s, part[1]);
#pragma unroll
        for (int p = 0; p < P; p++) {
            if constexpr (!EARLY) block_load_out(a, 8 * (t + T * p), w[0]);
            block_out<YT, V>(a, v[p], w[EARLY ? p : 0], row, 8 * (t + T * p), inv);
        }
    } else {
        float xv[8], v[8];
        V s = 0, inv = 1;
        BlockRun w;
        if (a.post_w) {
            for (uint32_t c0 = 8 * t; c0 < a.n; c0 += 8 * T) {
                load_run(y, c0, a.n, v);
#pragma unroll
                for (int j = 0; j < 8; j++) s = block_square<V>(v[j], s);
            }
            inv = row_inverse<T, V>(a, s, part[0]);
        }
        s = 0;
        for (uint32_t c0 = 8 * t; c0 < a.n; c0 += 8 * T) {
            load_run(y, c0, a.n, v);
            load_run(x, c0, a.n, xv);
            block_load_add(a, gate, c0, w);
            block_add<XT, V>(a, xv, v, w, inv);
            store_run(x_out, c0, a.n, v);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c0 + j < a.n) s = block_square<V>(v[j], s);
        }
        if (!a.pre_w) return;
        inv = row_inverse<T, V>(a, s, part[1]);
        // every thread of a block of 128 columns takes part in its maximum
        for (uint32_t c0 = 8 * t; c0 - c0 % FP8_BLOCK < a.n; c0 += 8 * T) {
            load_run((const XT *)x_out, c0, a.n, v);  // this thread's own columns
            block_load_out(a, c0, w);
            block_out<YT, V>(a, v, w, row, c0, inv);
        }
    }
}

typedef void (*BlockFn)(BlockArgs);

// Threads per row and runs per thread: one run up to 8192 columns, the row in
// registers up to 32768.  The threads are the least of the steps that hold
// the row, as those without columns take places on the compute unit (5339 x
// 2502 bf16: 45 us with 320, 53.5 with 512; 3855 x 4352: 51 with 640, 56 with
// 1024).  Rows of up to 1024 columns, many of them: a wavefront per row with
// two runs and no barrier (1024 bf16 columns, 4096 rows: 11.0 us, 13.0 with a
// workgroup per row; 512 rows: 5.9 against 5.1).
template <class XT, class YT, class V>
static BlockFn block_pick(uint32_t n, uint32_t rows, int &threads) {
#define PICK(T, P) (threads = T, block_kernel<XT, YT, V, T, P>)
    if (n <= 512) return PICK(64, 1);
    if (n <= 1024 && rows > 1024) return PICK(64, 2);
    const uint32_t runs = (n + 7) / 8;
    if (runs <= 256) return PICK(256, 1);
    if (runs <= 320) return PICK(320, 1);
    if (runs <= 448) return PICK(448, 1);
    if (runs <= 512) return PICK(512, 1);
    if (runs <= 640) return PICK(640, 1);
    if (runs <= 768) return PICK(768, 1);
    if (runs <= 1024) return PICK(1024, 1);
    if (n <= 16384) return PICK(1024, 2);
    if (n <= 32768) return PICK(1024, 4);
    return PICK(1024, 0);
#undef PICK
}

}  // namespace oco

using namespace oco;

extern "C" int oco_block_norm(const void *x, const void *y, void *x_out, const void *gate, const float *post_w,
                              const float *pre_w, void *out, uint8_t *codes, float *scales, const oco_block *p,
                              oco_stream stream) {
    if (!p) return fail(OCO_ERR_INVALID, "oco_block_norm: null description");
    if (p->gate > OCO_GATE_TANH) return fail(OCO_ERR_INVALID, "oco_block_norm: gate %u", p->gate);
    if (p->rows == 0 || p->n == 0) return OCO_OK;
    if (!x || !y || !x_out) return fail(OCO_ERR_INVALID, "oco_block_norm: null pointer");
    if (p->gate != OCO_GATE_NONE && !gate) return fail(OCO_ERR_INVALID, "oco_block_norm: a gate kind without gate rows");
    if (p->rows > 0x7fffffffu || p->n > 0x7fffff00u)
        return fail(OCO_ERR_INVALID, "oco_block_norm: %u rows of %u", p->rows, p->n);
    if (!codes != !scales) return fail(OCO_ERR_INVALID, "oco_block_norm: codes and scales come together");
    if (!pre_w != !(out || codes)) return fail(OCO_ERR_INVALID, "oco_block_norm: the second norm needs its weight and an output");
    if (codes && (p->n % 16 || ((uintptr_t)codes & 15u)))
        return fail(OCO_ERR_INVALID, "oco_block_norm: 8-bit rows need n %% 16 == 0 and 16-byte aligned codes (n = %u)", p->n);
    const uint32_t strides[4] = {p->x_stride, p->y_stride, p->gate_stride, p->out_stride};
    for (uint32_t s : strides)
        if (s && s < p->n) return fail(OCO_ERR_INVALID, "oco_block_norm: a row stride of %u under n = %u", s, p->n);
    BlockArgs a;
    a.x = x; a.y = y; a.gate = gate;
    a.post_w = post_w; a.pre_w = pre_w;
    a.x_out = x_out; a.out = out;
    a.codes = codes; a.scales = scales;
    a.rows = p->rows; a.n = p->n;
    a.kind = p->gate; a.gate_rows = p->gate_rows;
    a.x_stride = p->x_stride ? p->x_stride : p->n;
    a.y_stride = p->y_stride ? p->y_stride : p->n;
    a.gate_stride = p->gate_stride ? p->gate_stride : p->n;
    a.out_stride = p->out_stride ? p->out_stride : p->n;
    a.scale = p->scale; a.epsilon = p->epsilon; a.offset = p->weight_offset;
    int threads = 0;
    BlockFn fn = nullptr;
    if (p->x_dtype == OCO_DT_F32 && p->dtype == OCO_DT_F32) fn = codes ? block_pick<float, float, double>(p->n, p->rows, threads) : block_pick<float, float, float>(p->n, p->rows, threads);
    else if (p->x_dtype == OCO_DT_F32 && p->dtype == OCO_DT_BF16) fn = codes ? block_pick<float, bf16_t, double>(p->n, p->rows, threads) : block_pick<float, bf16_t, float>(p->n, p->rows, threads);
    else if (p->x_dtype == OCO_DT_F32 && p->dtype == OCO_DT_F16) fn = codes ? block_pick<float, f16_t, double>(p->n, p->rows, threads) : block_pick<float, f16_t, float>(p->n, p->rows, threads);
    else if (p->x_dtype == OCO_DT_BF16 && p->dtype == OCO_DT_BF16) fn = codes ? block_pick<bf16_t, bf16_t, double>(p->n, p->rows, threads) : block_pick<bf16_t, bf16_t, float>(p->n, p->rows, threads);
    else if (p->x_dtype == OCO_DT_F16 && p->dtype == OCO_DT_F16) fn = codes ? block_pick<f16_t, f16_t, double>(p->n, p->rows, threads) : block_pick<f16_t, f16_t, float>(p->n, p->rows, threads);
    else
        return fail(OCO_ERR_UNSUPPORTED, "oco_block_norm: residual type %u with rows of type %u (an f32 residual, or both alike)",
                    p->x_dtype, p->dtype);
    const uint32_t grid = threads == 64 ? (p->rows + 3) / 4 : p->rows;
    hipLaunchKernelGGL(fn, dim3(grid), dim3(threads < 256 ? 256 : threads), 0, (hipStream_t)stream, a);
    return launch_check("oco_block_norm");
}
