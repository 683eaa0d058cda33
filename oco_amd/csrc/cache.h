// The paged cache in 4 bits: where a token's codes and scales lie, the rows of
// a batch, and E2M1 blocks.
#pragma once
#include "rows.h"

namespace oco {

// A batch of rows on a cache (oco_cache), in the form that kernels take.
struct CacheBatch {
    const uint32_t *table, *starts, *lengths;
    uint32_t sequences, rows, max_rows, max_length, table_stride, page_size, pages, kv_heads;
};
struct CacheSpan {  // a sequence's rows and tokens
    uint32_t first, rows, length;
};

__device__ __forceinline__ CacheSpan cache_span(const CacheBatch &b, uint32_t s) {
    CacheSpan r;
    if (b.starts) {
        r.first = min(b.starts[s], b.rows);
        r.rows = min(max(b.starts[s + 1], r.first), b.rows) - r.first;
    } else {
        r.rows = b.rows / b.sequences;
        r.first = s * r.rows;
    }
    r.rows = min(r.rows, b.max_rows);
    r.length = min(b.lengths[s], b.max_length);
    return r;
}

// The sequence of a row, by one wavefront, uniform: the last one that starts
// at the row or before, 64 starts compared at once.  b.sequences: none does.
__device__ __forceinline__ uint32_t cache_sequence(const CacheBatch &b, uint32_t row) {
    if (!b.starts) return row / (b.rows / b.sequences);
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0, n = b.sequences;
    for (;;) {
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const uint32_t c = __builtin_popcountll(__ballot(i < n && b.starts[min(base + i, b.sequences - 1)] <= row));
        if (c == 0) return b.sequences;
        base += (c - 1) * step;
        if (step == 1) return base;
        n = min(step, n - (c - 1) * step);
    }
}

// A row's sequence (b.sequences: none), rows and tokens, by one wavefront, uniform: of up to 64 sequences a lane's starts and
// length are read at once, for every load that waits for another is a microsecond of a small call.
struct CacheRow {
    uint32_t sequence;
    CacheSpan span;
};
__device__ __forceinline__ CacheRow cache_row(const CacheBatch &b, uint32_t row) {
    CacheRow r;
    if (b.starts && b.sequences <= 64) {
        const uint32_t lane = threadIdx.x & 63, start = b.starts[min(lane, b.sequences - 1)], length = b.lengths[min(lane, b.sequences - 1)];
        const uint32_t last = b.starts[b.sequences];
        const uint32_t c = __builtin_popcountll(__ballot(lane < b.sequences && start <= row));
        r.sequence = c ? c - 1 : b.sequences;
        const uint32_t s = c ? c - 1 : 0;
        r.span.first = min((uint32_t)__builtin_amdgcn_readlane((int)start, s), b.rows);
        const uint32_t next = c == b.sequences ? last : (uint32_t)__builtin_amdgcn_readlane((int)start, c);
        r.span.rows = min(min(max(next, r.span.first), b.rows) - r.span.first, b.max_rows);
        r.span.length = min((uint32_t)__builtin_amdgcn_readlane((int)length, s), b.max_length);
    } else {
        r.sequence = cache_sequence(b, row);
        r.span = cache_span(b, min(r.sequence, b.sequences - 1));
    }
    return r;
}

// A head's bytes in a page, and where a token's parts are in them.  D: head_dim.
__host__ __device__ constexpr uint32_t cache_head_bytes(uint32_t page_size, uint32_t d) { return page_size * d + page_size * d / 16; }
__device__ __forceinline__ uint32_t cache_key_at(uint32_t t, uint32_t word, uint32_t d) { return t * (d / 2) + 4 * word; }
// Bytes of 2 * (d / 64) .. : word w holds values 8w .. 8w + 7; a piece of d / 16 values is d / 32 bytes.
__device__ __forceinline__ uint32_t cache_value_at(uint32_t page_size, uint32_t t, uint32_t byte, uint32_t d) {
    const uint32_t piece = d / 32;
    return page_size * (d / 2) + (t / 4) * (2 * d) + byte / piece * (4 * piece) + (t % 4) * piece + byte % piece;
}
__device__ __forceinline__ uint32_t cache_key_scale_at(uint32_t page_size, uint32_t t, uint32_t block, uint32_t d) {
    return page_size * d + t * (d / 32) + block;
}
__device__ __forceinline__ uint32_t cache_value_scale_at(uint32_t page_size, uint32_t t, uint32_t block, uint32_t d) {
    return page_size * d + page_size * (d / 32) + (t / 4) * (d / 8) + 4 * block + t % 4;
}

// An E8M0 scale of a cached block as f32; 255 is NaN (append writes 1 .. 252 and 255).
__device__ __forceinline__ float cache_scale(uint32_t e) { return __uint_as_float(e == 255 ? 0x7fc00000u : e << 23); }

// Eight values of a block whose 32 are held by four adjacent lanes: their
// codes, and the block's scale byte.  The hardware's conversion rounds to
// nearest, ties to the even code, and takes what is beyond 6 to 6.
__device__ __forceinline__ uint32_t cache_quantize(const float *v, uint32_t &scale) {
    uint32_t top = 0;  // as integers, NaN above infinity above the rest
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, true));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, true));
    const uint32_t e = top >> 23;
    scale = e == 255 ? 255 : max(e, 3u) - 2;
    const float s = __uint_as_float(scale << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
    return scale == 255 ? 0 : w;
}
__device__ __forceinline__ void cache_dequantize(uint32_t w, uint32_t scale, float *v) {
    const float s = cache_scale(scale);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    const float u[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = u[j] * s;
}

// The checks that the cache's entry points share; nullptr: fine.
const char *cache_problem(const oco_cache *p);
CacheBatch cache_batch(const oco_cache *p, const uint32_t *table, const uint32_t *starts, const uint32_t *lengths);

}  // namespace oco
