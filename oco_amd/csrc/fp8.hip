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

// 16 threads per block of 128 columns, four consecutive blocks of a row per
// wavefront.  Bound by memory: 2048 x 4096 bf16 in 6.6 us (25 MB, 3.8 TB/s);
// two or four such sets per wavefront with their loads ahead take 7.7 and 8.5.
template <class T>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(QuantArgs a) {
    const uint32_t unit = blockIdx.x * 16 + (threadIdx.x >> 4), row = unit / a.blocks, b = unit - row * a.blocks;
    const uint32_t c0 = FP8_BLOCK * b + 8 * (threadIdx.x & 15);
    const bool live = row < a.rows;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, scale;
    if (live) load_run((const T *)a.x + row * a.stride, c0, a.k, v);
    const uint2 q = fp8_block(v, scale);
    if (live && c0 < a.k) {
        *reinterpret_cast<uint2 *>(a.codes + (uint64_t)row * a.k + c0) = q;
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
        if (live >= 4)
            *reinterpret_cast<u32x4_u *>(p) = u32x4_u{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        else
#pragma unroll
            for (uint32_t j = 0; j < 3; j++)
                if (j < live) p[j] = v[j];
    } else {
        uint16_t *p = (uint16_t *)y + at;
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; j++) h[j] = dtype == OCO_DT_BF16 ? f32_to_bf16_bits(v[j]) : RowIO<f16_t>::bits(v[j]);
        if (live >= 4)
            *reinterpret_cast<u32x2_u *>(p) = u32x2_u{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
        else
#pragma unroll
            for (uint32_t j = 0; j < 3; j++)
                if (j < live) p[j] = (uint16_t)h[j];
    }
}

// A lane's 32 codes of a block as f16: four operands of eight.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
struct HalfBlock {
    f16x8 v[4];
    HalfBlock() = default;
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

// Few rows: bound by the weight stream.  A workgroup's WAVES wavefronts share
// the blocks of K of 16 NT weight rows among them, take them straight into
// the registers that the products read, two blocks ahead, and meet in LDS at
// the end.  The conversions to f16 hide behind the stream.  Loads keep their
// lines in the caches: a load instruction takes half a line of each row, and
// the next one the other half (151936 x 4096, 8 rows: 118 us, 129 with the
// nontemporal hint).
constexpr uint32_t FP8_OFF = 0x80000000u;  // past every range: reads zero without touching memory

template <int MT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void fp8_rows_kernel(Fp8Args a) {
    __shared__ f32x4 part[WAVES * MT * NT * 64];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const uint32_t n0 = blockIdx.x * 16 * NT, rows = min(a.n - n0, 16u * NT);
    const __amdgpu_buffer_rsrc_t wr = uniform_rsrc(a.w + (uint64_t)n0 * a.k, rows * a.k);
    const __amdgpu_buffer_rsrc_t xr = uniform_rsrc(a.x, a.m * a.k);
    uint32_t wrow[NT], xrow[MT];
#pragma unroll
    for (int t = 0; t < NT; t++) wrow[t] = 16 * t + r < rows ? (16 * t + r) * a.k + 16 * q : FP8_OFF;
#pragma unroll
    for (int i = 0; i < MT; i++) xrow[i] = 16 * i + r < a.m ? (16 * i + r) * a.k + 16 * q : FP8_OFF;
    static_assert(FP8_BLOCK % (16 * NT) == 0, "one weight scale per block of K");
    const float *const wsrc = a.ws + (uint64_t)(n0 / FP8_BLOCK) * a.blocks;
    struct Buf {
        i32x8 w[NT], x[MT];
        float ws, xs[MT];
    };
    auto load = [&](Buf &f, uint32_t b) {  // blocks past the last, and chunks past k, read zero
        const uint32_t k0 = FP8_BLOCK * b;
        const uint32_t lo = k0 + 16 * q < a.k ? k0 : FP8_OFF, hi = k0 + 64 + 16 * q < a.k ? k0 + 64 : FP8_OFF;
        auto both = [&](const __amdgpu_buffer_rsrc_t &rs, uint32_t row) {
            const u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(rs, (row | lo) & FP8_OFF ? FP8_OFF : row + lo, 0, 0);
            const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, (row | hi) & FP8_OFF ? FP8_OFF : row + hi, 0, 0);
            return i32x8{(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)v.x, (int)v.y, (int)v.z, (int)v.w};
        };
#pragma unroll
        for (int t = 0; t < NT; t++) f.w[t] = both(wr, wrow[t]);
#pragma unroll
        for (int i = 0; i < MT; i++) f.x[i] = both(xr, xrow[i]);
        const uint32_t at = min(b, a.blocks - 1);
        f.ws = wsrc[at];
#pragma unroll
        for (int i = 0; i < MT; i++) f.xs[i] = a.xs[(uint64_t)at * a.m + min(16 * i + r, a.m - 1)];
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](const Buf &f) {
        HalfBlock x[MT];
        float s[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) {
            x[i] = HalfBlock(f.x[i]);
            s[i] = f.ws * f.xs[i];
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const HalfBlock w(f.w[t]);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const f32x4 p = half_block_sum(w, x[i]);
#pragma unroll
                for (int v = 0; v < 4; v++) acc[i][t][v] = fmaf(p[v], s[i], acc[i][t][v]);
            }
        }
    };
    Buf f0, f1;
    load(f0, wave);
    load(f1, wave + WAVES);
    for (uint32_t b = wave; b < a.blocks; b += 2 * WAVES) {
        compute(f0);
        load(f0, b + 2 * WAVES);
        if (b + WAVES < a.blocks) compute(f1);
        load(f1, b + 3 * WAVES);
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int t = 0; t < NT; t++) part[(wave * MT * NT + i * NT + t) * 64 + lane] = acc[i][t];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < MT * NT * 64; o += 64 * WAVES) {
        f32x4 s = part[o];
#pragma unroll
        for (int w = 1; w < WAVES; w++) s += part[w * MT * NT * 64 + o];
        const uint32_t tile = o / 64, l = o % 64, row = 16 * (tile / NT) + (l & 15), col = n0 + 16 * (tile % NT) + 4 * (l >> 4);
        if (row >= a.m || col >= a.n) continue;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = s[j] + (a.bias ? round_bf16(a.bias[min(col + j, a.n - 1)]) : 0.f);
        fp8_put4(a.y, a.y_dtype, (uint64_t)row * a.n + col, v, a.n - col);
    }
}

typedef void (*Fp8RowsFn)(Fp8Args);
// Up to 512 tiles of 16 weight rows, eight wavefronts on one tile, so that the
// loads in flight fill the card (2880 x 4096, one row: 5.6 us; two tiles and
// four wavefronts 8.2); beyond, four wavefronts on two tiles, which read the
// activations half as often (12288 x 4096, 32 rows: 18.6 us against 21.8).
static Fp8RowsFn fp8_rows_pick(uint32_t m, uint32_t n, uint32_t &cols, uint32_t &waves) {
    const bool small = n <= 512 * 16;
    cols = small ? 16 : 32;
    waves = small ? 8 : 4;
    if (m <= 16) return small ? fp8_rows_kernel<1, 1, 8> : fp8_rows_kernel<1, 2, 4>;
    if (m <= 32) return small ? fp8_rows_kernel<2, 1, 8> : fp8_rows_kernel<2, 2, 4>;
    return small ? fp8_rows_kernel<4, 1, 8> : fp8_rows_kernel<4, 2, 4>;
}

// ---- many rows: tiles through LDS ------------------------------------------------------
//
// BM activation rows x BN weight rows per workgroup of WM x WN wavefronts.  A
// stage is one block of K: both operands' 128 bytes per row go from global
// memory straight to LDS (16 bytes per lane), two stages deep, one barrier
// per stage.  HALF: the f16 matrix instruction on converted codes (f32 and f16
// outputs), else the 8-bit one, for bf16 outputs alone: of the largest of eight
// products it drops at most 7 * 2^-13, less than half a bf16 step (2^-9 to 2^-8)
// but more than half an f16 one (2^-12 to 2^-11).  Where a bf16 output is small
// because its products cancel, what is dropped can pass its rounding, as the
// rounding of f32 sums does at 2^-24 of the products.  4096 x 12288 x 4096 to
// f16: 382 us, where the 8-bit instruction would take 209.
//
// Which weight row meets which row of the matrix instruction is free: row j
// of tile t is weight row 4 TN (j / 4) + 4 t + j % 4 of the wavefront's, so
// that a lane's results are 4 TN consecutive outputs and its four lane groups
// write whole lines.
//
// LDS: a row's 16-byte chunk c lies in slot c ^ swizzle(row), with a swizzle
// that takes eight values over the rows that lanes r = 0 .. 7 read (r % 8 for
// the activations; for the weights' order 4 (row / (4 TN) % 2) + row % 4), so
// that fragment reads run at 256 bytes a clock.
//
// Workgroups stay and take tile after tile: the next tile's first stage is
// requested before this one's results are written.
//
// 4096 x 12288 x 4096 to bf16 on 256-tiles: 200 us, 2.1 PFLOP/s; the matrix
// cores are busy for 46% of the clocks, the four FMAs behind each product and
// the waits at the barrier take the rest.  1999 x 4096 x 12288 to f32 on
// 128-tiles: 190 us, 1.06 PFLOP/s, with the conversions to f16 beside the products.

// 16 (4) bytes per lane from a buffer to LDS at `to` + 16 (4) lane (`to` is uniform).
__device__ __forceinline__ void to_lds16(__amdgpu_buffer_rsrc_t rs, void *to, uint32_t at, uint32_t base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)to, 16, at, base, 0, 0);
}
__device__ __forceinline__ void to_lds4(__amdgpu_buffer_rsrc_t rs, void *to, uint32_t at) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)to, 4, at, 0, 0, 0);
}

struct Fp8TileArgs {
    Fp8Args p;
    uint32_t mt, nt, parts;
    float *sums;  // parts > 1: f32 [part][m][n]
};

// N consecutive outputs (N a multiple of 4), `live` of them inside the row.
template <int N>
__device__ __forceinline__ void fp8_put(void *y, uint32_t dtype, uint64_t at, const float *v, uint32_t live) {
    if (live >= N && dtype != OCO_DT_F32) {
        uint32_t h[N / 2];
        if (dtype == OCO_DT_BF16)
#pragma unroll
            for (int j = 0; j < N / 2; j++) h[j] = f32_to_bf16_bits(v[2 * j]) | ((uint32_t)f32_to_bf16_bits(v[2 * j + 1]) << 16);
        else
#pragma unroll
            for (int j = 0; j < N / 2; j++) h[j] = RowIO<f16_t>::bits(v[2 * j]) | (RowIO<f16_t>::bits(v[2 * j + 1]) << 16);
        uint16_t *p = (uint16_t *)y + at;
        if constexpr (N % 8 == 0) {
#pragma unroll
            for (int j = 0; j < N / 8; j++)
                *reinterpret_cast<u32x4_u *>(p + 8 * j) = u32x4_u{h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]};
        } else {
#pragma unroll
            for (int j = 0; j < N / 4; j++) *reinterpret_cast<u32x2_u *>(p + 4 * j) = u32x2_u{h[2 * j], h[2 * j + 1]};
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; j += 4)
        if (j < (int)live) fp8_put4(y, dtype, at + j, v + j, live - j);
}

template <int BM, int BN, int WM, int WN, bool HALF>
__global__ __launch_bounds__(64 * WM * WN, 2) void fp8_tile_kernel(Fp8TileArgs ta) {
    const Fp8Args &a = ta.p;
    constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, OUT = 4 * TN;
    constexpr int XL = BM / 8 / WAVES, WL = BN / 8 / WAVES;  // 1 KB loads per wavefront and stage
    constexpr uint32_t XB = BM * FP8_BLOCK, STAGE = (BM + BN) * FP8_BLOCK;
    static_assert(XL * 8 * WAVES == BM && WL * 8 * WAVES == BN && FP8_BLOCK % (BN / WN) == 0 && BM <= 64 * WAVES, "whole loads, one weight scale per wavefront");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float *const xs_lds = reinterpret_cast<float *>(lds + 2 * STAGE);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const uint32_t wm = wave / WN * TM * 16, wn = wave % WN * TN * 16;
    const uint32_t tiles = ta.mt * ta.nt, part = blockIdx.y;
    const uint32_t b0 = (uint32_t)((uint64_t)a.blocks * part / ta.parts), b1 = (uint32_t)((uint64_t)a.blocks * (part + 1) / ta.parts);
    // the chunk that lane l fetches into slot l % 8 of row l / 8 of eight (the weights': ^ 4 where row / OUT is odd)
    const uint32_t xchunk = ((lane & 7) ^ (lane >> 3)) * 16, wchunk = ((lane & 7) ^ (lane >> 3 & 3)) * 16;

    uint32_t m0, n0;
    __amdgpu_buffer_rsrc_t xr, wr;
    uint32_t xo[XL], wo[WL];
    const float *wsrc;
    // tiles in groups of four columns, rows within: neighbours share operands in one L2
    auto enter = [&](uint32_t id) {
        const uint32_t lin = xcd_order(id, tiles), per = 4 * ta.mt, g = lin / per, wide = min(4u, ta.nt - 4 * g), in = lin - g * per;
        m0 = in / wide * BM;
        n0 = (4 * g + in % wide) * BN;
        const uint32_t xrows = min(a.m - m0, (uint32_t)BM), wrows = min(a.n - n0, (uint32_t)BN);
        xr = uniform_rsrc(a.x + (uint64_t)m0 * a.k, xrows * a.k);
        wr = uniform_rsrc(a.w + (uint64_t)n0 * a.k, wrows * a.k);
        // rows past the last read the last one (their results are not written)
#pragma unroll
        for (int i = 0; i < XL; i++) xo[i] = min((wave * XL + i) * 8 + (lane >> 3), xrows - 1) * a.k;
#pragma unroll
        for (int i = 0; i < WL; i++) wo[i] = min((wave * WL + i) * 8 + (lane >> 3), wrows - 1) * a.k;
        wsrc = a.ws + (uint64_t)(min(n0 + wn, a.n - 1) / FP8_BLOCK) * a.blocks;
    };
    // One of the LOADS requests of a stage.  Columns past k: the row's first chunk, cleared before it is read.
    constexpr int LOADS = XL + WL + 1;
    auto fetch_one = [&](uint32_t b, uint32_t s, int i) {
        const uint32_t base = FP8_BLOCK * b;
        if (i < XL) {
            to_lds16(xr, lds + s * STAGE + (wave * XL + i) * 1024, xo[i < XL ? i : 0] + (base + xchunk < a.k ? xchunk : 0), base);
        } else if (i < XL + WL) {
            const int j = i < XL + WL ? i - XL : 0;
            const uint32_t c = wchunk ^ ((wave * WL + j) * 8 / OUT & 1 ? 64 : 0);
            to_lds16(wr, lds + s * STAGE + XB + (wave * WL + j) * 1024, wo[j] + (base + c < a.k ? c : 0), base);
        } else if (wave < BM / 64) {
            const uint32_t rows = min(a.m - m0, (uint32_t)BM);
            to_lds4(uniform_rsrc(a.xs + (uint64_t)b * a.m + m0, rows * 4), xs_lds + s * BM + wave * 64, min(wave * 64 + lane, rows - 1) * 4);
        }
    };
    auto fetch = [&](uint32_t b, uint32_t s) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) fetch_one(b, s, i);
    };
    // Requests between the products, where registers allow: ahead of them they hold the wavefront up before its
    // first LDS read.  Gains where workgroups take several tiles (1999 x 4096 x 12288 to f32 191 us against 196, to
    // bf16 114 against 117) and costs where the card holds all of them (1024 x 4096 x 12288 to bf16 79 against 73,
    // 300 x 4096 x 4096 24.7 against 23.6).
    constexpr bool BETWEEN = BM * BN <= 128 * 128;
    // fragment addresses: chunks q and 4 + q of the lane's rows
    const uint32_t xlo = (wm + r) * FP8_BLOCK + (q ^ (r & 7)) * 16, wrow = wn + OUT * (r >> 2) + (r & 3);
    const uint32_t wlo = XB + wrow * FP8_BLOCK + (q ^ ((r & 3) | (wrow / OUT % 2 * 4))) * 16;
    auto frag = [&](uint32_t at) {
        const u32x4 u = *reinterpret_cast<const u32x4 *>(lds + at), v = *reinterpret_cast<const u32x4 *>(lds + (at ^ 64));
        return i32x8{(int)u.x, (int)u.y, (int)u.z, (int)u.w, (int)v.x, (int)v.y, (int)v.z, (int)v.w};
    };

    enter(blockIdx.x);
    if (b0 < b1) fetch(b0, 0);
    float ws_next = wsrc[min(b0, a.blocks - 1)];
    for (uint32_t id = blockIdx.x;;) {
        f32x4 acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int t = 0; t < TN; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        f32x4 sum[TN];  // the last step's sums and their scale
        float fs = 0.f;
#pragma unroll
        for (int t = 0; t < TN; t++) sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (uint32_t b = b0; b < b1; b++) {
            const uint32_t s = (b - b0) & 1;
            const float ws = ws_next;
            __syncthreads();  // this stage has arrived; the other buffer is read no more
            if (FP8_BLOCK * (b + 1) > a.k) {
                const uint32_t left = (a.k - FP8_BLOCK * b) / 16;
                for (uint32_t c = threadIdx.x; c < (BM + BN) * 8; c += 64 * WAVES) {
                    const uint32_t row = c >> 3, f = row < BM ? row & 7 : (row & 3) | ((row - BM) / OUT % 2 * 4);
                    if (((c & 7) ^ f) >= left) *reinterpret_cast<u32x4 *>(lds + s * STAGE + c * 16) = u32x4{0, 0, 0, 0};
                }
                __syncthreads();
            }
            // behind the last stage, that one again: its place is free until the next tile
            const uint32_t bn = min(b + 1, b1 - 1);
            if constexpr (!BETWEEN)
                if (b + 1 < b1) fetch(b + 1, s ^ 1);
            ws_next = wsrc[bn];
            const uint32_t xt = s * STAGE + xlo, wt = s * STAGE + wlo;
            const float *const xsb = xs_lds + s * BM + wm + r;
            // Fragments of x are read one step of 16 rows ahead, and a step's sums are added while the next
            // step is on the matrix core.
            f16x8 wh[HALF ? TN : 1][4];
            i32x8 w[HALF ? 1 : TN];
#pragma unroll
            for (int t = 0; t < TN; t++) {
                const i32x8 c = frag(wt + t * 4 * FP8_BLOCK);
                if constexpr (HALF) {
                    const HalfBlock h(c);
#pragma unroll
                    for (int u = 0; u < 4; u++) wh[t][u] = h.v[u];
                } else {
                    w[t] = c;
                }
            }
            i32x8 x = frag(xt);
            float f = ws * xsb[0];
#pragma unroll
            for (int i = 0; i < TM; i++) {
                constexpr int LAST = TM - 1;
                const int before = i ? i - 1 : LAST;
                i32x8 xn = x;
                float fn = f;
                if (i < LAST) {
                    xn = frag(xt + (i + 1) * 16 * FP8_BLOCK);
                    fn = ws * xsb[16 * (i + 1)];
                }
                if constexpr (BETWEEN)
#pragma unroll
                    for (int l = i * LOADS / TM; l < (i + 1) * LOADS / TM; l++) fetch_one(bn, s ^ 1, l);
                f32x4 p[TN];
                if constexpr (HALF) {
                    const HalfBlock h(x);
#pragma unroll
                    for (int t = 0; t < TN; t++) p[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int t = 0; t < TN; t++) {
                            p[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[t][u], h.v[u], p[t], 0, 0, 0);
                            acc[before][t][u] = fmaf(sum[t][u], fs, acc[before][t][u]);
                        }
                } else {
#pragma unroll
                    for (int t = 0; t < TN; t++) {
                        p[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[t], x, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
                        for (int v = 0; v < 4; v++) acc[before][t][v] = fmaf(sum[t][v], fs, acc[before][t][v]);
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // a product, four FMAs
                        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
                    }
                }
#pragma unroll
                for (int t = 0; t < TN; t++) sum[t] = p[t];
                fs = f;
                x = xn;
                f = fn;
            }
        }
#pragma unroll
        for (int t = 0; t < TN; t++)
#pragma unroll
            for (int v = 0; v < 4; v++) acc[TM - 1][t][v] = fmaf(sum[t][v], fs, acc[TM - 1][t][v]);
        // the next tile's first stage, then this one's results
        const uint32_t row0 = m0 + wm + r, col = n0 + wn + OUT * q;
        id += gridDim.x;
        __syncthreads();  // nothing is on its way to LDS any more
        if (id < tiles) {
            enter(id);
            if (b0 < b1) fetch(b0, 0);
            ws_next = wsrc[min(b0, a.blocks - 1)];
        }
        if (col < a.n) {
            float bias[OUT];
#pragma unroll
            for (int j = 0; j < OUT; j++) bias[j] = 0.f;
            if (a.bias && ta.parts == 1)
#pragma unroll
                for (int j = 0; j < OUT; j++) bias[j] = round_bf16(a.bias[min(col + j, a.n - 1)]);
            void *const y = ta.parts > 1 ? (void *)(ta.sums + (uint64_t)part * a.m * a.n) : a.y;
            const uint32_t dtype = ta.parts > 1 ? (uint32_t)OCO_DT_F32 : a.y_dtype;
#pragma unroll
            for (int i = 0; i < TM; i++) {
                if (row0 + 16 * i >= a.m) break;
                float v[OUT];
#pragma unroll
                for (int j = 0; j < OUT; j++) v[j] = acc[i][j / 4][j % 4] + bias[j];
                fp8_put<OUT>(y, dtype, (uint64_t)(row0 + 16 * i) * a.n + col, v, a.n - col);
            }
        }
        if (id >= tiles) break;
    }
}

// The K parts' sums, in order.
__global__ __launch_bounds__(256) void fp8_join_kernel(Fp8TileArgs ta) {
    const Fp8Args &a = ta.p;
    const uint64_t size = (uint64_t)a.m * a.n;
    for (uint64_t at = 4 * ((uint64_t)blockIdx.x * 256 + threadIdx.x); at < size; at += 1024ull * gridDim.x) {
        float v[4];
        const uint32_t live = (uint32_t)min(size - at, (uint64_t)4);
        uint32_t col = a.bias ? (uint32_t)(at % a.n) : 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = 0.f;
            if (j < (int)live) {
                for (uint32_t p = 0; p < ta.parts; p++) v[j] += ta.sums[p * size + at + j];
                if (a.bias) v[j] += round_bf16(a.bias[col]);
                col = col + 1 == a.n ? 0 : col + 1;
            }
        }
        fp8_put4(a.y, a.y_dtype, at, v, live);
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
    const uint64_t units = (uint64_t)rows * a.blocks;
    if (units > 0xfffff000ull) return fail(OCO_ERR_INVALID, "oco_fp8_quantize: %u rows of %u", rows, k);
    void (*fn)(QuantArgs);
    switch (x_dtype) {
    case OCO_DT_F32: fn = fp8_quantize_kernel<float>; break;
    case OCO_DT_BF16: fn = fp8_quantize_kernel<bf16_t>; break;
    case OCO_DT_F16: fn = fp8_quantize_kernel<f16_t>; break;
    default: return fail(OCO_ERR_UNSUPPORTED, "oco_fp8_quantize: rows of type %d", (int)x_dtype);
    }
    hipLaunchKernelGGL(fn, dim3((uint32_t)((units + 15) / 16)), dim3(256), 0, (hipStream_t)stream, a);
    return launch_check("oco_fp8_quantize");
}

namespace oco {

// How a product runs: the few-row kernel, or tiles with K in parts.
struct Fp8Plan {
    uint32_t bm, bn, mt, nt, parts;  // bm 0: few rows
};
constexpr uint32_t FP8_FEW = 64;  // the few-row kernel's limit
// The least of the estimated times, in us, each term fitted to measured calls
// (n, k of 512 x 2880, 2880 x 4096, 4096 x 4096, 4096 x 12288 and 12288 x
// 4096, 1 to 1024 rows; the estimates are within about 15% of them):
//  * few rows: the weight stream at 5.3 TB/s, and 0.2 ns for each product of
//    16 x 16 x 128 past the first 16 rows' (those hide behind the stream);
//  * 128-tiles: a block of K takes 0.82 us (f32 and f16 outputs, on the f16
//    instruction: 1.17) with a workgroup per compute unit, 1.08 (1.45) with two;
//  * 256-tiles (bf16 outputs): 2.15 us, one workgroup per compute unit;
//  * K parts: a launch, 0.4 us each, and their sums written and read at 3 TB/s.
static Fp8Plan fp8_plan(uint32_t m, uint32_t n, uint32_t k, bool half) {
    const uint32_t blocks = (k + FP8_BLOCK - 1) / FP8_BLOCK;
    int32_t knob[4] = {-1, 0, 0, 0};
    const int set = plan_override(OCO_KNOB_FP8, knob);
    Fp8Plan best = {0, 0, 0, 0, 1};
    double least = 1e30;
    if (m <= FP8_FEW && (!set || knob[0] == 0)) {
        const double more = m <= 16 ? 0 : m <= 32 ? 1 : 3;
        least = 4.0 + (double)n * k / 5.3e6 + (more > 0 ? 1.2 + more * ((n + 15) / 16) * blocks * 0.2e-3 : 0.0);
        if (set) return best;
    }
    for (uint32_t tile = 128; tile <= (half ? 128u : 256u); tile *= 2) {
        if (set && knob[0] == 256 && !half && tile != 256) continue;
        if (set && knob[0] != 256 && tile != 128) continue;
        Fp8Plan p = {tile, tile, (m + tile - 1) / tile, (n + tile - 1) / tile, 1};
        const uint64_t tiles = (uint64_t)p.mt * p.nt;
        for (p.parts = 1; p.parts <= 16; p.parts++) {  // by the rule: up to 8, powers of two
            if (set > 1 && p.parts != std::min((uint32_t)std::max(knob[1], 1), std::min(blocks, 16u))) continue;
            if (!(set > 1) && (p.parts > 8 || p.parts & (p.parts - 1) || (p.parts > 1 && blocks / p.parts < 2))) continue;
            const uint64_t work = tiles * p.parts;
            const double stages = (double)((blocks + p.parts - 1) / p.parts);
            double t = 3.0;
            if (tile == 256)
                t += (double)((work + 255) / 256) * stages * 2.15;
            else
                t += work <= 256 ? stages * (half ? 1.17 : 0.82) : (double)((work + 511) / 512) * stages * (half ? 1.45 : 1.08);
            if (p.parts > 1) t += 5.5 + 0.4 * p.parts + (double)p.parts * m * n * 8.0 / 3e6;
            if (t < least) {
                least = t;
                best = p;
            }
        }
    }
    return best;
}

template <int BM, int BN, int WM, int WN, bool HALF>
static int fp8_tiles(const Fp8TileArgs &a, hipStream_t stream) {
    const size_t lds = 2 * ((BM + BN) * FP8_BLOCK + BM * 4);
    auto fn = fp8_tile_kernel<BM, BN, WM, WN, HALF>;
    if (lds > 64 * 1024)
        OCO_TRY(hip_check(hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "hipFuncSetAttribute"));
    // workgroups that fill the card once (256 compute units, one or two each by their LDS), the same number for each XCD
    const uint32_t tiles = a.mt * a.nt, most = lds > 80 * 1024 ? 256 : 512;
    hipLaunchKernelGGL(fn, dim3(tiles < most ? tiles : most, a.parts), dim3(64 * WM * WN), lds, stream, a);
    return launch_check("oco_fp8_matmul (tiles)");
}

}  // namespace oco

static uint64_t fp8_need(const Fp8Plan &plan, const oco_matrix *p) {
    return plan.parts > 1 ? (uint64_t)plan.parts * p->m * p->n * 4 : 0;
}

// For outputs of either kind.
extern "C" uint64_t oco_fp8_matmul_workspace(const oco_matrix *p) {
    if (!p || p->m == 0 || p->n == 0 || p->k == 0) return 0;
    return std::max(fp8_need(fp8_plan(p->m, p->n, p->k, true), p), fp8_need(fp8_plan(p->m, p->n, p->k, false), p));
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
    // 31-bit offsets inside a workgroup's rows
    if (p->k > 0x400000u || p->n > 0x7fffff00u || p->m > 0x7fffff00u)
        return fail(OCO_ERR_INVALID, "oco_fp8_matmul: %u x %u x %u", p->m, p->n, p->k);
    const bool half = y_dtype != OCO_DT_BF16;
    const Fp8Plan plan = fp8_plan(p->m, p->n, p->k, half);
    const uint64_t need = fp8_need(plan, p);
    if (need && (!workspace || ((uintptr_t)workspace & 15u) || workspace_bytes < need))
        return fail(OCO_ERR_INVALID, "oco_fp8_matmul: workspace of %llu bytes, need %llu, 16-byte aligned",
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    if ((uint64_t)plan.mt * plan.nt > 0x7fffffffull) return fail(OCO_ERR_INVALID, "oco_fp8_matmul: %u x %u outputs", p->m, p->n);
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
    hipStream_t st = (hipStream_t)stream;
    if (!plan.bm) {
        uint32_t cols = 0, waves = 0;
        const Fp8RowsFn fn = fp8_rows_pick(p->m, p->n, cols, waves);
        hipLaunchKernelGGL(fn, dim3((p->n + cols - 1) / cols), dim3(64 * waves), 0, st, a);
        return launch_check("oco_fp8_matmul");
    }
    Fp8TileArgs t;
    t.p = a;
    t.mt = plan.mt;
    t.nt = plan.nt;
    t.parts = plan.parts;
    t.sums = (float *)workspace;
    if (plan.bm == 256)
        OCO_TRY((fp8_tiles<256, 256, 2, 4, false>(t, st)));
    else
        OCO_TRY(half ? (fp8_tiles<128, 128, 2, 2, true>(t, st)) : (fp8_tiles<128, 128, 2, 2, false>(t, st)));
    if (plan.parts > 1) {
        const uint64_t groups = ((uint64_t)p->m * p->n + 1023) / 1024;
        hipLaunchKernelGGL(fp8_join_kernel, dim3((uint32_t)(groups < 8192 ? groups : 8192)), dim3(256), 0, st, t);
        return launch_check("oco_fp8_matmul (join)");
    }
    return OCO_OK;
}
