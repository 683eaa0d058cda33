// Attention over the paged cache: what its kernels share.
#pragma once
#include "cache.h"
#include "eight.h"

namespace oco {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct AttentionArgs {
    CacheBatch b;
    const uint8_t *cache;
    const void *q;
    void *out;
    const float *sinks;
    float *parts;  // [rows][heads][chunks][D], then m and l [rows][heads][chunks][2], then a chunk's tokens (u32)
    uint64_t q_stride, out_stride;
    uint32_t heads, group, window;
    uint32_t tile_rows;      // rows of a tile
    uint32_t chunks, chunk;  // parts of a tile's tokens, at most, and the tokens of each, at least (attention_chunk)
    uint32_t seen;           // the most tokens that a tile sees
    uint32_t works;          // 0: chunks have `chunk` tokens; else attention_chunk's: what is more goes into
    uint32_t pieces[2];      // pieces[1] chunks, what is less into pieces[0]
    float inverse[2], relaxed[2];  // of pieces, and of as many less half a piece per sequence
    float c;                 // scale * log2(e)
};

template <bool BF>
struct Half;  // the 16-bit type of the rows
template <>
struct Half<true> {
    template <int I>
    static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
    }
    // c + the pair's two values
    static __device__ __forceinline__ float add(uint32_t pair, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{(__bf16)1.f, (__bf16)1.f}, c, false);
    }
    static __device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 product32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static constexpr uint32_t ONE = 0x3f80, LIMIT = 252;  // LIMIT: the last scale whose 6 is a number of the type
};
template <>
struct Half<false> {
    template <int I>
    static __device__ __forceinline__ uint32_t pair(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, I));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
    }
    static __device__ __forceinline__ float add(uint32_t pair, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), f16x2{(_Float16)1.f, (_Float16)1.f}, c, false);
    }
    static __device__ __forceinline__ f32x4 product(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 product32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static constexpr uint32_t ONE = 0x3c00, LIMIT = 140;
};
// A block's scale, NaN past the limit; and 0x80 in the bytes of a word of
// scales that are past it (of at least 128).
template <uint32_t LIMIT>
__device__ __forceinline__ float block_scale(uint32_t e) {
    return __uint_as_float(e > LIMIT ? 0x7fc00000u : e << 23);
}
template <uint32_t LIMIT>
__device__ __forceinline__ uint32_t bytes_past(uint32_t x) {
    return ((x & 0x7f7f7f7fu) + (255 - LIMIT) * 0x01010101u) & x & 0x80808080u;
}

// Four tokens' pairs of columns -> the two columns' four tokens.
__device__ __forceinline__ u32x2 low_halves(const uint32_t *c) {
    return u32x2{__builtin_amdgcn_perm(c[1], c[0], 0x05040100), __builtin_amdgcn_perm(c[3], c[2], 0x05040100)};
}
__device__ __forceinline__ u32x2 high_halves(const uint32_t *c) {
    return u32x2{__builtin_amdgcn_perm(c[1], c[0], 0x07060302), __builtin_amdgcn_perm(c[3], c[2], 0x07060302)};
}

// Maximum and sum over the lanes l, l ^ 16, l ^ 32, l ^ 48, which hold one row.
__device__ __forceinline__ float row_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    v = fmaxf(v, dpp_f32<0x124>(v));
    v = fmaxf(v, dpp_f32<0x128>(v));
    return row_max(v);
}
__device__ __forceinline__ float row_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float half_sum(float v) {  // over l and l ^ 32
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Over the wavefront, uniform.
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true);
    return (uint32_t)(__builtin_amdgcn_readlane((int)v, 0) + __builtin_amdgcn_readlane((int)v, 16) + __builtin_amdgcn_readlane((int)v, 32) +
                      __builtin_amdgcn_readlane((int)v, 48));
}

// Up to this lane.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

// A workgroup's sequence and tile where there is one size of chunks: tiles with most to do first, and of 2 to 64 sequences
// with rows of their own those that there are one after the other.  us, with the gaps / so: 4 sequences of up to 1000 rows of
// 32 heads after 3000 tokens 205 / 155, 256 wide after 1000 259 / 180, 16 of up to 300 after 3000 183 / 171; not for few
// tiles, where the search costs as much (8 of up to 5 rows of 64 heads 20.8 / 21.1).
struct AttentionPlace {
    uint32_t sequence, tile;  // sequence past the last one: there is none
    CacheSpan span;
};
__host__ __device__ __forceinline__ bool attention_counts(uint32_t sequences, bool starts, uint32_t tiles) {
    return starts && sequences > 1 && sequences <= 64 && tiles > 4;
}
template <uint32_t TILE>
__device__ __forceinline__ AttentionPlace attention_place(const AttentionArgs &a, uint32_t id, uint32_t tiles) {
    AttentionPlace p;
    if (!attention_counts(a.b.sequences, a.b.starts, tiles)) {
        p.sequence = id % a.b.sequences;
        p.tile = tiles - 1 - id / a.b.sequences;
        p.span = cache_span(a.b, p.sequence);
        return p;
    }
    const uint32_t lane = threadIdx.x & 63;
    const CacheSpan own = cache_span(a.b, min(lane, a.b.sequences - 1));
    const uint32_t mine = lane < a.b.sequences ? (own.rows * a.group + TILE - 1) / TILE : 0;
    p.sequence = a.b.sequences;
    p.tile = 0;
    p.span = CacheSpan{0, 0, 0};
    // the last tile from which on there are more than `id`, 64 compared at once
    for (uint32_t range = tiles;;) {
        const uint32_t step = (range + 63) / 64, t = p.tile + lane * step;
        uint32_t n = 0;
        for (uint32_t i = 0; i < a.b.sequences; i++) n += max((uint32_t)__builtin_amdgcn_readlane((int)mine, i), t) - t;
        const uint32_t c = __builtin_popcountll(__ballot(n > id));
        if (c == 0) return p;
        p.tile += (c - 1) * step;
        if (step == 1) {
            id -= (uint32_t)__builtin_amdgcn_readlane((int)n, c - 1) - (uint32_t)__builtin_popcountll(__ballot(mine > p.tile));  // its place among those of this tile
            break;
        }
        range = step;
    }
    const uint64_t have = __ballot(mine > p.tile);
    const uint32_t rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
    p.sequence = __builtin_ctzll(__ballot(mine > p.tile && rank == id));
    p.span = CacheSpan{(uint32_t)__builtin_amdgcn_readlane((int)own.first, p.sequence), (uint32_t)__builtin_amdgcn_readlane((int)own.rows, p.sequence),
                       (uint32_t)__builtin_amdgcn_readlane((int)own.length, p.sequence)};
    return p;
}

// A workgroup's sequence, tile and chunk where chunks are sized by the lengths as they are (of at most 64 M sequences, a
// lane's M each) and numbered one after the other: the least of a few sizes that leave no more chunks than wanted.
struct AttentionPart {
    uint32_t sequence, tile, chunk, size;  // sequence past the last one: there is none
    CacheSpan span;
};
template <uint32_t TILE, int M>
__device__ __forceinline__ AttentionPart attention_part(const AttentionArgs &a, uint32_t id) {
    const uint32_t lane = threadIdx.x & 63;
    CacheSpan own[M];
    uint32_t units[M], tiles[M], parts[M], of_lane = 0;
#pragma unroll
    for (int i = 0; i < M; i++) {
        const uint32_t s = lane * M + i;
        own[i] = cache_span(a.b, min(s, a.b.sequences - 1));
        units[i] = (min(own[i].length, a.seen) + 127) / 128;
        tiles[i] = s < a.b.sequences ? (own[i].rows * a.group + TILE - 1) / TILE : 0;
        of_lane += units[i] * tiles[i];
    }
    const uint32_t all = wave_total(of_lane), k = all < a.works ? 0 : 1;
    const float least = fmaxf(ceilf((float)all * a.inverse[k]), 1.f);
    float size = fmaxf(least, ceilf((float)all * a.relaxed[k]));
#pragma unroll
    for (int j = 0; j < 3; j++) {
        const float c = ceilf(least * (1.f + 0.125f * j)), by = __builtin_amdgcn_rcpf(c) * 0.9999998f;
        of_lane = 0;
#pragma unroll
        for (int i = 0; i < M; i++) of_lane += (uint32_t)ceilf((float)units[i] * by) * tiles[i];
        if (wave_total(of_lane) <= a.pieces[k]) {
            size = c;
            break;
        }
    }
    AttentionPart p;
    p.size = max(a.chunk, (uint32_t)fminf(size, 8388608.f) * 128);
    of_lane = 0;
#pragma unroll
    for (int i = 0; i < M; i++) {
        parts[i] = max((min(own[i].length, a.seen) + p.size - 1) / p.size, 1u) * tiles[i];
        of_lane += parts[i];
    }
    const uint32_t to = wave_scan(of_lane), c = __builtin_popcountll(__ballot(to <= id)), s = min(c, 63u);
    uint32_t rest = id - (uint32_t)(__builtin_amdgcn_readlane((int)to, s) - __builtin_amdgcn_readlane((int)of_lane, s)), of = 1;
    p.sequence = a.b.sequences;
    p.span = CacheSpan{0, 0, 0};
    bool found = c == 64;
#pragma unroll
    for (int i = 0; i < M; i++) {
        const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)parts[i], s);
        if (!found && rest < n) {
            found = true;
            p.sequence = s * M + i;
            of = (uint32_t)__builtin_amdgcn_readlane((int)tiles[i], s);
            p.span = CacheSpan{(uint32_t)__builtin_amdgcn_readlane((int)own[i].first, s), (uint32_t)__builtin_amdgcn_readlane((int)own[i].rows, s),
                               (uint32_t)__builtin_amdgcn_readlane((int)own[i].length, s)};
        }
        rest -= found ? 0 : n;
    }
    p.tile = rest % of;
    p.chunk = rest / of;
    return p;
}

// A tile of a sequence's rows (a token's query heads of one key-value head
// after the other): its rows, their first and last positions and the tokens
// that any of them sees, from a multiple of 32 on.
struct AttentionTile {
    uint32_t first_row, rows;  // rows: of the sequence
    int32_t least, most;
    uint32_t first, end;
};
__device__ __forceinline__ AttentionTile attention_tile(const CacheSpan &s, uint32_t tile, uint32_t tile_rows, uint32_t group, uint32_t window) {
    AttentionTile t;
    t.first_row = tile * tile_rows;
    t.rows = s.rows * group;
    const int32_t before = (int32_t)s.length - (int32_t)s.rows;
    t.least = before + (int32_t)(t.first_row / group);
    t.most = before + (int32_t)((min(t.first_row + tile_rows, max(t.rows, 1u)) - 1) / group);
    t.first = window && t.least >= (int32_t)window ? ((uint32_t)t.least + 1 - window) / 32 * 32 : 0;
    t.end = t.most < 0 ? 0 : (uint32_t)t.most + 1;
    return t;
}

// exp2 of m - to, 0 for m = -Inf whatever `to` is (NaN for a sink that is NaN).
__device__ __forceinline__ float carry(float m, float to) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to); }

// part / total. A total of 0 is a row that sees nothing (0), or whose scores are all -Inf and have no softmax (NaN): a finite
// one makes it 1 or nearly so at least.
__device__ __forceinline__ float part_of(float part, float total, bool sees) {
    return total > 0.f || total != total ? part / total : sees ? __uint_as_float(0x7fc00000u) : 0.f;
}

// Prompts (attention_prompt.hip; heads of 64 and 128), in tiles of 128 rows, or of 256 where heads are 128 wide.
int attention_prompt_launch(const AttentionArgs &a, uint32_t head_dim, bool bf, uint32_t tiles, uint32_t grid, hipStream_t stream);

}  // namespace oco
