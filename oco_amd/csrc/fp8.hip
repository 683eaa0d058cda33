// Products of rows in 8-bit floating point with weights in 8-bit floating
// point: e4m3 codes with an f32 scale per 128 columns of a row and per 128 x
// 128 block of the weights.  Beside the GGUF formats of matmul.hip: here both
// operands enter the matrix cores as they are stored.
//
//     y[r][c] = sum over blocks b of K: xs[b][r] ws[c / 128][b] (sum in b of x[r][k] w[c][k]) + bf16(bias[c])
//
// The sums of a block start from zero on the matrix core and enter the f32
// accumulators by an FMA with the product of the block's two scales.
//
// Which matrix instruction: the 8-bit one (v_mfma_f32_16x16x128_f8f6f4, one
// block of K) aligns the eight products of each group of eight consecutive k
// to the largest of them and drops what lies under 2^-13 of its binade
// (measured: bits down to 2^3 beside a product of 2^16 stay, 2^2 is lost;
// across groups the sums are f32).  On normal data that is 1.5e-5 relative.
// The f16 instruction on the codes as f16 (exact: v_cvt_scalef32_pk_f16_fp8)
// keeps every bit of the products and 1e-8, at half the rate.
//
// Operands: the weights are the A matrix (16 of their rows, lane l holds row
// l % 16), the activations the B matrix (16 of their rows as its columns), so
// a lane's four results are four consecutive outputs of activation row l % 16.
// Both hold 32 bytes of a block of K per lane; as only pairs of equal k have
// to meet, lane group q = l / 16 takes bytes 16 q .. + 15 and 64 + 16 q .. + 15
// of the block: each load instruction then covers 64 consecutive bytes of a row.
#include "fp8.h"
#include "rows.h"
#include "stream.h"

namespace oco {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- rows to e4m3 --------------------------------------------------------------------

struct QuantArgs {
    const void *x;
    uint8_t *codes;
    float *scales;
    uint32_t rows, k, blocks;
    uint64_t stride;
};

// 16 threads per block of 128 columns, four consecutive blocks of a row per wavefront.
template <class T>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(QuantArgs a) {
    const uint64_t unit = (uint64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const uint64_t row = unit / a.blocks;
    const uint32_t b = (uint32_t)(unit % a.blocks), c0 = FP8_BLOCK * b + 8 * (threadIdx.x & 15);
    const bool live = row < a.rows;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, scale;
    if (live) load_run((const T *)a.x + row * a.stride, c0, a.k, v);
    const uint2 q = fp8_block(v, scale);
    if (live && c0 < a.k) {
        *reinterpret_cast<uint2 *>(a.codes + row * a.k + c0) = q;
        if ((threadIdx.x & 15) == 0) a.scales[(uint64_t)b * a.rows + row] = scale;
    }
}

// ---- products ------------------------------------------------------------------------

struct Fp8Args {
    const uint8_t *w, *x;
    const float *ws, *xs;
    void *y;
    const float *bias;
    uint32_t m, n, k, blocks, y_dtype;
};

__device__ __forceinline__ void fp8_put4(void *y, uint32_t dtype, uint64_t at, const float *v, uint32_t live) {
    if (dtype == OCO_DT_F32) {
        float *p = (float *)y + at;
        for (uint32_t j = 0; j < 4; j++)
            if (j < live) p[j] = v[j];
    } else {
        uint16_t *p = (uint16_t *)y + at;
        for (uint32_t j = 0; j < 4; j++)
            if (j < live) p[j] = dtype == OCO_DT_BF16 ? f32_to_bf16_bits(v[j]) : (uint16_t)RowIO<f16_t>::bits(v[j]);
    }
}

// A lane's 32 codes of a block as f16: four operands of eight.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
struct HalfBlock {
    f16x8 v[4];
    __device__ __forceinline__ HalfBlock(i32x8 c) {
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[2 * s], 1.0f, false);
            const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[2 * s], 1.0f, true);
            const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[2 * s + 1], 1.0f, false);
            const f16x2 e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[2 * s + 1], 1.0f, true);
            v[s] = f16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
        }
    }
};
__device__ __forceinline__ f32x4 half_block_sum(const HalfBlock &w, const HalfBlock &x) {
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; s++) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[s], x.v[s], p, 0, 0, 0);
    return p;
}

// Few rows: bound by the weight stream.  A workgroup's four wavefronts take
// every fourth block of K of 16 NT weight rows straight into the registers
// that the products read, and meet in LDS at the end.  The conversions to f16
// hide behind the stream.
constexpr int FP8_WAVES = 4;
constexpr uint32_t FP8_OFF = 0x80000000u;  // past every range: reads zero without touching memory

template <int MT, int NT>
__global__ __launch_bounds__(64 * FP8_WAVES) void fp8_rows_kernel(Fp8Args a) {
    __shared__ f32x4 part[FP8_WAVES * MT * NT * 64];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const uint32_t n0 = blockIdx.x * 16 * NT, rows = min(a.n - n0, 16u * NT);
    const uint32_t m0 = blockIdx.y * 16 * MT, xrows = min(a.m - m0, 16u * MT);
    const __amdgpu_buffer_rsrc_t wr = uniform_rsrc(a.w + (uint64_t)n0 * a.k, rows * a.k);
    const __amdgpu_buffer_rsrc_t xr = uniform_rsrc(a.x + (uint64_t)m0 * a.k, xrows * a.k);
    auto load = [&](const __amdgpu_buffer_rsrc_t &rs, uint32_t row, bool live, uint32_t b) {
        const uint32_t k0 = FP8_BLOCK * b + 16 * q, at = row * a.k + k0;
        const u32x4 lo = __builtin_amdgcn_raw_buffer_load_b128(rs, live && k0 < a.k ? at : FP8_OFF, 0, 0);
        const u32x4 hi = __builtin_amdgcn_raw_buffer_load_b128(rs, live && k0 + 64 < a.k ? at + 64 : FP8_OFF, 0, 0);
        return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t b = wave; b < a.blocks; b += FP8_WAVES) {
        i32x8 w[NT], x[MT];
        float ws[NT], xs[MT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            w[t] = load(wr, 16 * t + r, 16 * t + r < rows, b);
            ws[t] = a.ws[(uint64_t)(min(n0 + 16 * t, a.n - 1) / FP8_BLOCK) * a.blocks + b];
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
            x[i] = load(xr, 16 * i + r, 16 * i + r < xrows, b);
            xs[i] = a.xs[(uint64_t)b * a.m + min(m0 + 16 * i + r, a.m - 1)];
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const HalfBlock wh(w[t]);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const f32x4 p = half_block_sum(wh, HalfBlock(x[i]));
                const float s = ws[t] * xs[i];
#pragma unroll
                for (int v = 0; v < 4; v++) acc[i][t][v] = fmaf(p[v], s, acc[i][t][v]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) part[(wave * MT * NT + i * NT + t) * 64 + lane] = acc[i][t];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < MT * NT * 64; o += 64 * FP8_WAVES) {
        f32x4 s = part[o];
#pragma unroll
        for (int w = 1; w < FP8_WAVES; w++) s += part[w * MT * NT * 64 + o];
        const uint32_t tile = o / 64, l = o % 64, row = m0 + 16 * (tile / NT) + (l & 15), col = n0 + 16 * (tile % NT) + 4 * (l >> 4);
        if (row >= a.m || col >= a.n) continue;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = s[j] + (a.bias ? round_bf16(a.bias[min(col + j, a.n - 1)]) : 0.f);
        fp8_put4(a.y, a.y_dtype, (uint64_t)row * a.n + col, v, a.n - col);
    }
}

}  // namespace oco

using namespace oco;

extern "C" int oco_fp8_quantize(const void *x, oco_dtype x_dtype, uint32_t rows, uint32_t k, uint64_t x_stride, uint8_t *codes,
                                float *scales, oco_stream stream) {
    if (rows == 0 || k == 0) return OCO_OK;
    if (!x || !codes || !scales) return fail(OCO_ERR_INVALID, "oco_fp8_quantize: null pointer");
    if (k % 16 || ((uintptr_t)codes & 15u))
        return fail(OCO_ERR_INVALID, "oco_fp8_quantize: 8-bit rows need k %% 16 == 0 and 16-byte aligned codes (k = %u)", k);
    if (x_stride && x_stride < k) return fail(OCO_ERR_INVALID, "oco_fp8_quantize: a row stride under k = %u", k);
    QuantArgs a;
    a.x = x;
    a.codes = codes;
    a.scales = scales;
    a.rows = rows;
    a.k = k;
    a.blocks = (k + FP8_BLOCK - 1) / FP8_BLOCK;
    a.stride = x_stride ? x_stride : k;
    const uint64_t groups = ((uint64_t)rows * a.blocks + 15) / 16;
    if (groups > 0x7fffffffull) return fail(OCO_ERR_INVALID, "oco_fp8_quantize: %u rows of %u", rows, k);
    void (*fn)(QuantArgs);
    switch (x_dtype) {
    case OCO_DT_F32: fn = fp8_quantize_kernel<float>; break;
    case OCO_DT_BF16: fn = fp8_quantize_kernel<bf16_t>; break;
    case OCO_DT_F16: fn = fp8_quantize_kernel<f16_t>; break;
    default: return fail(OCO_ERR_UNSUPPORTED, "oco_fp8_quantize: rows of type %d", (int)x_dtype);
    }
    hipLaunchKernelGGL(fn, dim3((uint32_t)groups), dim3(256), 0, (hipStream_t)stream, a);
    return launch_check("oco_fp8_quantize");
}

extern "C" uint64_t oco_fp8_matmul_workspace(const oco_matrix *p) {
    (void)p;
    return 0;
}

extern "C" int oco_fp8_matmul(const uint8_t *w, const float *w_scales, const uint8_t *codes, const float *scales, void *y,
                              oco_dtype y_dtype, const float *bias, const oco_matrix *p, void *workspace,
                              uint64_t workspace_bytes, oco_stream stream) {
    if (!p) return fail(OCO_ERR_INVALID, "oco_fp8_matmul: null matrix");
    if (p->experts > 1) return fail(OCO_ERR_UNSUPPORTED, "oco_fp8_matmul: dense matrices only");
    if (p->has_bias > 1) return fail(OCO_ERR_UNSUPPORTED, "oco_fp8_matmul: has_bias %u", p->has_bias);
    if ((uint32_t)y_dtype > OCO_DT_F16) return fail(OCO_ERR_UNSUPPORTED, "oco_fp8_matmul: outputs of type %d", (int)y_dtype);
    if (p->m == 0 || p->n == 0) return OCO_OK;
    if (p->k == 0 || p->k % 16) return fail(OCO_ERR_INVALID, "oco_fp8_matmul: k = %u is not whole groups of 16", p->k);
    if (!w || !w_scales || !codes || !scales || !y || (p->has_bias && !bias))
        return fail(OCO_ERR_INVALID, "oco_fp8_matmul: null pointer");
    if (((uintptr_t)w | (uintptr_t)codes) & 15u) return fail(OCO_ERR_INVALID, "oco_fp8_matmul: weights and codes are 16-byte aligned");
    // 32-bit offsets inside a workgroup's rows
    if (p->k > 0x1000000u || p->n > 0x7fffff00u || p->m > 0x7fffff00u)
        return fail(OCO_ERR_INVALID, "oco_fp8_matmul: %u x %u x %u", p->m, p->n, p->k);
    (void)workspace;
    (void)workspace_bytes;
    Fp8Args a;
    a.w = w;
    a.x = codes;
    a.ws = w_scales;
    a.xs = scales;
    a.y = y;
    a.bias = p->has_bias ? bias : nullptr;
    a.m = p->m;
    a.n = p->n;
    a.k = p->k;
    a.blocks = (p->k + FP8_BLOCK - 1) / FP8_BLOCK;
    a.y_dtype = y_dtype;
    const dim3 grid((p->n + 31) / 32, (p->m + 31) / 32);
    if (grid.y > 65535) return fail(OCO_ERR_INVALID, "oco_fp8_matmul: %u rows", p->m);
    if (p->m <= 16)
        hipLaunchKernelGGL((fp8_rows_kernel<1, 2>), dim3(grid.x, 1), dim3(64 * FP8_WAVES), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL((fp8_rows_kernel<2, 2>), grid, dim3(64 * FP8_WAVES), 0, (hipStream_t)stream, a);
    return launch_check("oco_fp8_matmul");
}
