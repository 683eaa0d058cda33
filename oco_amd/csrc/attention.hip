// Causal attention over the paged cache in 4 bits.
//
// out = sum_t p_t v_t with p = softmax(c q . k_t), one pass over the tokens
// with a running maximum m and sum l per row: a step of 32 tokens adds
// exp2(s - m) and its products, and rescales what is there when a row's maximum
// rises.  Rows are the query heads of one key-value head and their tokens, so
// the cache is read once for all of them.
//
// Everything is computed transposed, S^T = K Q^T and O^T = V^T P^T: a row is
// then a lane (of four) from the scores to the output, its statistics need no
// broadcast, and the scores leave the first product in the very lanes that
// feed the second.  The matrix instruction takes its 32 inner indexes in any
// order that both operands share, so a lane's probabilities of tokens 4g ..
// 4g + 3 of two halves stay where they are, and the values' pages hold four
// tokens together to match.
//
// E2M1 times a power of two is exact in bf16 and f16 (an f16 model's cache
// stays in range), so codes go to the matrix instruction through the hardware's
// conversion, two values per instruction, with their scale.
//
// Bound by memory for single tokens of many long sequences (32 of up to 16384,
// 8 heads of 128: 338 MB in 75 us, 4.5 TB/s), by two launches and three loads
// that wait for each other for one (4101 tokens 8.5 to 9).  A few drafted rows
// wait half of the time (8 sequences of up to 5 rows of 64 heads of 64 20 us,
// the join 4.7 of it): a wavefront has four or five steps behind lengths, chunk,
// table and page, 39% of its time goes by for loads and 31% for its turn to
// issue, and vector instructions take 18,000 of 37,000 clocks, a quarter of them
// in the loop conversions and transposes.  Many rows of wide heads are bound by
// the conversions that each tile makes for itself: per step of 32 rows 290
// vector instructions beside 64 products (1700 rows 256 wide 56 us).
#include "attention.h"

namespace oco {

// ---- a workgroup's four wavefronts hold the same 16 R rows and take steps of 32 tokens in turn ----

// One half-step's 16 tokens as a lane holds them: lane m + 16 g has a quarter
// of token m's key, and of tokens 4g .. 4g + 3 one sixteenth of the value.
template <uint32_t D>
struct Keys {
    uint32_t w[D / 32], scale;  // one or two scale bytes
};
template <uint32_t D>
struct Values {
    uint32_t w[D / 32], scale;  // the scale bytes of four tokens
};

template <uint32_t D>
__device__ __forceinline__ void load_words(uint32_t *w, gbytes p, uint32_t at) {
    if constexpr (D == 64) {
        const u32x2 a = *(const GLOBAL u32x2 *)(p + at);
        w[0] = a[0];
        w[1] = a[1];
    } else {
#pragma unroll
        for (int i = 0; i < (int)D / 128; i++) {
            const u32x4 a = *(const GLOBAL u32x4 *)(p + at + 16 * i);
#pragma unroll
            for (int j = 0; j < 4; j++) w[4 * i + j] = a[j];
        }
    }
}
// A half-step's tokens and a lane's places among them: the head's bytes and
// the slot are the same for all lanes, the places the same for all steps.
template <uint32_t D>
struct Places {
    uint32_t key, key_scale, value, value_scale;
    __device__ __forceinline__ Places(uint32_t page_size) {
        const uint32_t m = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
        key = m * (D / 2) + g * (D / 8);
        key_scale = page_size * D + m * (D / 32) + (D == 64 ? g / 2 : g * (D / 128));
        value = page_size * (D / 2) + g * (2 * D) + m * (D / 8);
        value_scale = page_size * D + page_size * (D / 32) + g * (D / 8) + m * D / 512 * 4;
    }
    __device__ __forceinline__ void load(Keys<D> &k, gbytes head, uint32_t slot) const {
        load_words<D>(k.w, head + slot * (D / 2), key);
        const gbytes s = head + slot * (D / 32);
        k.scale = D == 256 ? *(const GLOBAL uint16_t *)(s + key_scale) : s[key_scale];
    }
    __device__ __forceinline__ void load(Values<D> &v, gbytes head, uint32_t slot) const {
        load_words<D>(v.w, head + slot * (D / 2), value);
        v.scale = *(const GLOBAL uint32_t *)(head + slot * (D / 32) + value_scale);
    }
};

// The halves of a wavefront's steps, their pages and their places in them: a
// lane per half, read once for 32 steps, so that a step's loads do not wait
// for the table.
struct Halves {
    uint32_t page, slot;
};
__device__ __forceinline__ Halves load_halves(const uint32_t *table, uint32_t t0, uint32_t stride, uint32_t end, uint32_t page_size) {
    const uint32_t lane = threadIdx.x & 63, t = t0 + lane / 2 * stride + lane % 2 * 16;
    Halves h;
    h.page = t < end ? table[t / page_size] : 0;
    h.slot = t % page_size;
    return h;
}

// FIT: chunks by the lengths (attention_part).
template <uint32_t D, bool BF, int R, bool FIT>
__global__ __launch_bounds__(256, D * R == 64 ? 4 : D * R == 128 ? 3 : 2) void attention_kernel(AttentionArgs a, uint32_t tiles) {
    constexpr int KW = D / 32, NT = D / 16;  // key words per lane and token; tiles of 16 columns
    using H = Half<BF>;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    // Workgroups of a head in a row of 8 kv_heads apart share an XCD's L2 (heads come first); the tiles with most to do start first.
    uint32_t id = blockIdx.x;
    const uint32_t h = id % a.b.kv_heads;
    id /= a.b.kv_heads;
    uint32_t s, tile, chunk, size = a.chunk;
    CacheSpan span;
    if constexpr (FIT) {
        const AttentionPart part = a.b.sequences <= 64 ? attention_part<16 * R, 1>(a, id) : attention_part<16 * R, 4>(a, id);
        s = part.sequence;
        chunk = part.chunk;
        size = part.size;
        span = part.span;
        tile = part.tile;
        if (blockIdx.x == 0 && threadIdx.x == 0) *gp((uint32_t *)(a.parts + (uint64_t)a.b.rows * a.heads * a.chunks * (D + 2))) = size;
        if (s >= a.b.sequences) return;
    } else {
        chunk = id % a.chunks;
        id /= a.chunks;
        if constexpr (R == 2) {
            const AttentionPlace place = attention_place<16 * R>(a, id, tiles);
            s = place.sequence;
            tile = place.tile;
            span = place.span;
            if (s >= a.b.sequences) return;
        } else {  // three tiles at most, by the rule
            s = id % a.b.sequences;
            tile = tiles - 1 - id / a.b.sequences;
            span = cache_span(a.b, s);
        }
    }
    const AttentionTile range = attention_tile(span, tile, 16 * R, a.group, a.window);
    const uint32_t row0 = range.first_row, rows = range.rows;
    if (row0 >= rows) return;
    const int32_t least = range.least, most = range.most;
    const uint32_t first = range.first + chunk * size, end = min(first + size, range.end);  // this chunk's tokens
    if (chunk && first >= range.end) return;  // the tile has fewer chunks
    const uint32_t head_bytes = cache_head_bytes(a.b.page_size, D);
    const uint32_t *const table = a.b.table + (uint64_t)s * a.b.table_stride;
    uint32_t t0 = first + 32 * wave, step = 0;
    Halves halves = load_halves(table, t0, 128, end, a.b.page_size);
    // the rows' positions (-1: no token). A lane without a row is the last row once more, and is not written: such lanes take
    // part in the votes on the maxima, and a row of another tile may already be the result where that takes the queries' place.
    int32_t at[R];
    constexpr bool SHARED = R > 1;  // the queries in LDS, by fragment
    constexpr int QF = SHARED ? R * KW * 64 : 1, OF = 4 * NT * 64;
    __shared__ __attribute__((aligned(16))) u32x4 lds[QF > OF ? QF : OF];
    u32x4 q[R][SHARED ? 1 : KW];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const uint32_t i = min(row0 + 16 * r + n, rows - 1), token = i / a.group, head = h * a.group + i % a.group;
        at[r] = (int32_t)(span.length + token) - (int32_t)span.rows;
        const uint16_t *const row = (const uint16_t *)a.q + (uint64_t)(span.first + token) * a.q_stride + (uint64_t)head * D + g * (D / 4);
        if constexpr (SHARED) {
            if (r == (int)wave)
#pragma unroll
                for (int w = 0; w < KW; w++) lds[(r * KW + w) * 64 + lane] = *(const GLOBAL u32x4_u *)gp(row + 8 * w);
        } else {
#pragma unroll
            for (int w = 0; w < KW; w++) q[r][w] = *(const GLOBAL u32x4_u *)gp(row + 8 * w);
        }
    }
    if constexpr (SHARED) __syncthreads();
    float m[R], l[R];
    f32x4 o[R][NT];
#pragma unroll
    for (int r = 0; r < R; r++) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int j = 0; j < NT; j++) o[r][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // A step's tokens are requested before the step before it is computed; where that does not leave the
    // registers for it (STAGED), the keys once that step's are used up, and its values likewise.
    constexpr bool STAGED = D * R >= 384;  // 256 wide, 32 rows
    struct Step {
        Keys<D> k[2];
        Values<D> v[2];
        gbytes head[2];
        uint32_t slot[2];
        bool lost[2];  // not in the pool
    };
    const Places<D> places(a.b.page_size);
    auto request_keys = [&](Step &x) {  // of step `step`
        if (step && step % 32 == 0) halves = load_halves(table, t0, 128, end, a.b.page_size);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)halves.page, 2 * (step % 32) + e);
            x.slot[e] = (uint32_t)__builtin_amdgcn_readlane((int)halves.slot, 2 * (step % 32) + e);
            x.lost[e] = page >= a.b.pages;
            page = x.lost[e] ? 0 : page;
            x.head[e] = (gbytes)gp(a.cache) + ((uint64_t)page * a.b.kv_heads + h) * head_bytes;
            places.load(x.k[e], x.head[e], x.slot[e]);
        }
        step++;
        t0 += 128;
    };
    auto request_values = [&](Step &x) {
#pragma unroll
        for (int e = 0; e < 2; e++) places.load(x.v[e], x.head[e], x.slot[e]);
    };
    auto request = [&](Step &x) {
        request_keys(x);
        request_values(x);
    };
    auto compute = [&](Step &x, const uint32_t now) {
        Keys<D>(&k)[2] = x.k;
        Values<D>(&v)[2] = x.v;
        const bool lost[2] = {x.lost[0], x.lost[1]}, more = now + 128 < end;
        // scores: lane (n, g) has row n's tokens 16 e + 4 g + i
        f32x4 sc[R][2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (lost[e]) k[e].scale = 0xffff;
#pragma unroll
            for (int r = 0; r < R; r++) sc[r][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int w = 0; w < KW; w++) {
            u32x4 x[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float scale = block_scale<H::LIMIT>(D == 256 ? (w < 4 ? k[e].scale & 0xff : k[e].scale >> 8) : k[e].scale & 0xff);
                x[e] = u32x4{H::template pair<0>(k[e].w[w], scale), H::template pair<1>(k[e].w[w], scale),
                             H::template pair<2>(k[e].w[w], scale), H::template pair<3>(k[e].w[w], scale)};
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                const u32x4 f = SHARED ? lds[(r * KW + w) * 64 + lane] : q[r][SHARED ? 0 : w];
#pragma unroll
                for (int e = 0; e < 2; e++) sc[r][e] = H::product(x[e], f, sc[r][e]);
            }
            if constexpr (STAGED)
                if (w % 2) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (STAGED)
            if (more) request_keys(x);
        const bool edge = (int32_t)now + 31 > least || (a.window && (int32_t)now + (int32_t)a.window <= most);
        u32x4 p[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (edge) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int32_t t = (int32_t)now + 16 * (i / 4) + 4 * (int32_t)g + i % 4;
                    if (!(t <= at[r] && (!a.window || t + (int32_t)a.window > at[r]))) sc[r][i / 4][i % 4] = -INFINITY;
                }
            }
            const f32x4 x = sc[r][0], y = sc[r][1];
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
            top = row_max(top) * a.c;
            // A maximum may lag by 8 (probabilities up to 256) before the sums are rescaled
            if (__any(top > m[r] + 8.f)) {
                top = fmaxf(top, m[r]);
                const float f = carry(m[r], top);
                m[r] = top;
                l[r] *= f;
#pragma unroll
                for (int j = 0; j < NT; j++) o[r][j] *= f;
            }
            const float ref = m[r] > -INFINITY ? m[r] : 0.f;
            float u[8];
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = __builtin_amdgcn_exp2f(fmaf(sc[r][i / 4][i % 4], a.c, -ref));
            p[r] = u32x4{H::pack(u[0], u[1]), H::pack(u[2], u[3]), H::pack(u[4], u[5]), H::pack(u[6], u[7])};
            // of the rounded probabilities: their roundings cancel where few tokens have all the weight
            l[r] += H::add(p[r].y, H::add(p[r].x, 0.f)) + H::add(p[r].w, H::add(p[r].z, 0.f));
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (lost[e]) v[e].scale = 0xffffffffu;
        if (__any((bytes_past<H::LIMIT>(v[0].scale) | bytes_past<H::LIMIT>(v[1].scale)) != 0)) {
            // 0 * NaN is NaN: a NaN block enters the product as numbers, and the rows that see
            // it (counted by a product of their own) become NaN in its columns
            u32x4 lost_at;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t lo = byte_of(v[i / 2].scale, 2 * i % 4) > H::LIMIT, hi = byte_of(v[i / 2].scale, 2 * i % 4 + 1) > H::LIMIT;
                lost_at[i] = lo * H::ONE | hi * (H::ONE << 16);
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                u32x4 sees;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int32_t t = (int32_t)now + 16 * (i / 4) + 4 * (int32_t)g + i % 4;
                    const uint32_t one = t <= at[r] && (!a.window || t + (int32_t)a.window > at[r]) ? H::ONE : 0;
                    sees[i / 2] = i % 2 ? sees[i / 2] | one << 16 : one;
                }
                const f32x4 count = H::product(lost_at, sees, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < NT; j++) o[r][j][i] = count[i] > 0.f ? __uint_as_float(0x7fc00000u) : o[r][j][i];
            }
#pragma unroll
            for (int e = 0; e < 2; e++) v[e].scale ^= bytes_past<H::LIMIT>(v[e].scale);
        }
        float scale[8];  // of the tokens' column block
#pragma unroll
        for (int i = 0; i < 8; i++) scale[i] = __uint_as_float(byte_of(v[i / 4].scale, i % 4) << 23);
        // byte b of a token's piece: columns 2b and 2b + 1 of the piece
#pragma unroll
        for (int b = 0; b < NT / 2; b++) {
            uint32_t c[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                constexpr int W = D / 128;  // words per token, 0: two tokens share one
                const int byte = D == 64 ? 2 * (i % 2) + b : b % 4;
                const uint32_t w = D == 64 ? v[i / 4].w[i % 4 / 2] : v[i / 4].w[i % 4 * W + b / 4];
                c[i] = byte == 0 ? H::template pair<0>(w, scale[i]) : byte == 1 ? H::template pair<1>(w, scale[i])
                     : byte == 2 ? H::template pair<2>(w, scale[i]) : H::template pair<3>(w, scale[i]);
            }
            const u32x2 l0 = low_halves(c), l1 = low_halves(c + 4), h0 = high_halves(c), h1 = high_halves(c + 4);
            const u32x4 lo = {l0.x, l0.y, l1.x, l1.y}, hi = {h0.x, h0.y, h1.x, h1.y};
#pragma unroll
            for (int r = 0; r < R; r++) {
                o[r][2 * b] = H::product(lo, p[r], o[r][2 * b]);
                o[r][2 * b + 1] = H::product(hi, p[r], o[r][2 * b + 1]);
            }
            if constexpr (STAGED) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (STAGED)
            if (more) request_values(x);
    };
    Step x, y;
    if (t0 < end) request(x);
    for (uint32_t now = first + 32 * wave; now < end; now += 256) {
        if constexpr (!STAGED)
            if (t0 < end) request(y);
        compute(x, now);
        if (now + 128 >= end) break;
        if constexpr (!STAGED) {
            if (t0 < end) request(x);
            compute(y, now + 128);
        } else {
            compute(x, now + 128);
        }
    }
    // The four wavefronts' parts: each writes all of its own and joins a quarter, NT consecutive
    // columns of every lane's row.
    f32x4(*const so)[4][NT / 4][64] = (f32x4(*)[4][NT / 4][64])lds;
    __shared__ float sm[4][64], sl[4][64];
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (r || SHARED) __syncthreads();
        sm[wave][lane] = m[r];
        sl[wave][lane] = row_sum(l[r]);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < NT / 4; j++) so[wave][i][j][lane] = f32x4{o[r][4 * j][i], o[r][4 * j + 1][i], o[r][4 * j + 2][i], o[r][4 * j + 3][i]};
        __syncthreads();
        const uint32_t i = row0 + 16 * r + n;
        if (i >= rows) continue;
        const float top = fmaxf(fmaxf(sm[0][lane], sm[1][lane]), fmaxf(sm[2][lane], sm[3][lane]));
        float total = 0.f, f[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = carry(sm[w][lane], top);
            total += sl[w][lane] * f[w];
        }
        f32x4 sum[NT / 4];
#pragma unroll
        for (int j = 0; j < NT / 4; j++) {
            sum[j] = so[0][wave][j][lane] * f[0];
#pragma unroll
            for (int w = 1; w < 4; w++) sum[j] += so[w][wave][j][lane] * f[w];
        }
        const uint32_t row = span.first + i / a.group, head = h * a.group + i % a.group, column = (4 * g + wave) * NT;
        if (a.chunks > 1) {
            const uint64_t index = ((uint64_t)row * a.heads + head) * a.chunks + chunk;
#pragma unroll
            for (int j = 0; j < NT / 4; j++) *(GLOBAL f32x4 *)gp(a.parts + index * D + column + 4 * j) = sum[j];
            if (g == 0 && wave == 0) *(GLOBAL f32x2 *)gp(a.parts + (uint64_t)a.b.rows * a.heads * a.chunks * D + index * 2) = f32x2{top, total};
        } else {
            float end_top = top;
            if (a.sinks) {
                const float sink = a.sinks[head] * 1.44269504088896341f;
                end_top = fmaxf(top, sink);
                total = total * carry(top, end_top) + carry(sink, end_top);
            }
            const float by = part_of(carry(top, end_top), total, at[r] >= 0);
            uint16_t *const out = (uint16_t *)a.out + (uint64_t)row * a.out_stride + (uint64_t)head * D + column;
#pragma unroll
            for (int j = 0; j < NT / 4; j++)
                *(GLOBAL u32x2_u *)gp(out + 4 * j) = u32x2_u{H::pack(sum[j][0] * by, sum[j][1] * by), H::pack(sum[j][2] * by, sum[j][3] * by)};
        }
    }
}

// ---- chunks joined: a workgroup per row and head, or a wavefront -------------------------

// Groups of 32 lanes (D = 64: 16) take the chunks in turn.  W = 4: a workgroup per row and head, the least latency; W = 1:
// a wavefront, from 2048 of them on, where the lookups of a row's place bound it (160 rows of 64 heads of 64 in 6 chunks:
// 62.7 -> 53.7 us with the attention; 64 rows of 32 of 128 20.9 -> 19.5; 32 rows of 32 40.2, 40.8 so).
template <uint32_t D, bool BF, int W>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a) {
    constexpr uint32_t N = D / 64, LANES = D / (4 * (N > 1 ? N / 2 : 1)), GROUPS = 64 * W / LANES;  // 16, 32 and 32 lanes
    constexpr uint32_t V = D / LANES / 4;                                                            // of 4, 4 and 8 values
    const uint32_t item = W == 1 ? blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    const uint32_t row = item / a.heads, head = item % a.heads, group = threadIdx.x % (64 * W) / LANES, lane = threadIdx.x % LANES;
    if (W == 1 && row >= a.b.rows) return;
    const uint64_t index = (uint64_t)item * a.chunks;
    const float *const ml = a.parts + (uint64_t)a.b.rows * a.heads * a.chunks * D + index * 2;
    const f32x4 *const parts = (const f32x4 *)(a.parts + index * D) + lane * V;
    // The first chunks are requested before it is known how many the row has; a place in the workspace that was not
    // written is read and not used.
    constexpr uint32_t AHEAD = 4 / V;
    f32x4 part[AHEAD][V];
    f32x2 of[AHEAD], tops = {-INFINITY, 0.f};
    if ((threadIdx.x & 63) < a.chunks) tops = *(const GLOBAL f32x2 *)gp(ml + 2 * (threadIdx.x & 63));
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; k++) {
        const uint32_t c = group + k * GROUPS;
        if (c < a.chunks) {
            of[k] = *(const GLOBAL f32x2 *)gp(ml + 2 * c);
#pragma unroll
            for (uint32_t j = 0; j < V; j++) part[k][j] = ((const GLOBAL f32x4 *)gp(parts))[(uint64_t)c * (D / 4) + j];
        }
    }
    const uint32_t size = a.works ? *gp((const uint32_t *)(a.parts + (uint64_t)a.b.rows * a.heads * a.chunks * (D + 2))) : a.chunk;
    const CacheRow at_row = cache_row(a.b, row);
    const CacheSpan span = at_row.span;
    if (at_row.sequence >= a.b.sequences) return;
    if (row - span.first >= span.rows) return;
    const AttentionTile range = attention_tile(span, ((row - span.first) * a.group + head % a.group) / a.tile_rows, a.tile_rows, a.group, a.window);
    const uint32_t used = range.end > range.first ? (range.end - range.first + size - 1) / size : 0;
    const bool sees = span.length + (row - span.first) >= span.rows;
    const float sink = a.sinks ? a.sinks[head] * 1.44269504088896341f : -INFINITY;
    float top = sink;
    if ((threadIdx.x & 63) < used) top = fmaxf(top, tops[0]);
    for (uint32_t c = 64 + (threadIdx.x & 63); c < used; c += 64) top = fmaxf(top, ml[2 * c]);
    top = wave_max(top);
    float total = 0.f;
    f32x4 o[V];
#pragma unroll
    for (uint32_t j = 0; j < V; j++) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t k = 0; k < AHEAD; k++) {
        if (group + k * GROUPS >= used) break;
        const float f = carry(of[k][0], top);
        total += of[k][1] * f;
#pragma unroll
        for (uint32_t j = 0; j < V; j++) o[j] += part[k][j] * f;
    }
    for (uint32_t c = group + AHEAD * GROUPS; c < used; c += GROUPS) {
        const float f = carry(ml[2 * c], top);
        total += ml[2 * c + 1] * f;
#pragma unroll
        for (uint32_t j = 0; j < V; j++) o[j] += parts[(uint64_t)c * (D / 4) + j] * f;
    }
    uint16_t *const out = (uint16_t *)a.out + (uint64_t)row * a.out_stride + (uint64_t)head * D;
    if constexpr (W == 1) {
        total = (GROUPS == 4 ? row_sum(total) : half_sum(total)) + carry(sink, top);
        const float f = part_of(1.f, total, sees);
#pragma unroll
        for (uint32_t j = 0; j < V; j++) {
#pragma unroll
            for (int i = 0; i < 4; i++) o[j][i] = (GROUPS == 4 ? row_sum(o[j][i]) : half_sum(o[j][i])) * f;
            if (group == 0) *(GLOBAL u32x2_u *)gp(out + 4 * (lane * V + j)) = u32x2_u{Half<BF>::pack(o[j][0], o[j][1]), Half<BF>::pack(o[j][2], o[j][3])};
        }
    } else {
        __shared__ __attribute__((aligned(16))) f32x4 so[GROUPS][LANES * V];
        __shared__ float st[GROUPS];
#pragma unroll
        for (uint32_t j = 0; j < V; j++) so[group][lane * V + j] = o[j];
        if (lane == 0) st[group] = total;
        __syncthreads();
        if (threadIdx.x >= D / 4) return;
        f32x4 sum = so[0][threadIdx.x];
        total = carry(sink, top) + st[0];
#pragma unroll
        for (uint32_t i = 1; i < GROUPS; i++) {
            sum += so[i][threadIdx.x];
            total += st[i];
        }
        const float f = part_of(1.f, total, sees);
        *(GLOBAL u32x2_u *)gp(out + 4 * threadIdx.x) = u32x2_u{Half<BF>::pack(sum[0] * f, sum[1] * f), Half<BF>::pack(sum[2] * f, sum[3] * f)};
    }
}

// ---- choices and launches -------------------------------------------------------------------

struct AttentionPlan {
    uint32_t tile, tiles, chunks, chunk;  // tile: its rows / 16
    uint32_t seen, works, pieces[2];  // as in AttentionArgs
    uint64_t grid;                    // workgroups per head
    uint64_t bytes;
};
// The tiles' split along the tokens (split: chunks of a prompt's tiles; chunk: their tokens, if not 0).
static AttentionPlan attention_split(const oco_cache *p, uint32_t tile, uint64_t rows, uint32_t split, uint32_t chunk, bool starts) {
    AttentionPlan l;
    l.tile = tile;
    l.tiles = (uint32_t)((rows + 16 * tile - 1) / (16 * tile));
    const uint64_t tile_tokens = (16 * tile + p->heads / p->kv_heads - 1) / (p->heads / p->kv_heads);
    uint64_t seen = p->max_length;
    if (p->window && p->window + tile_tokens + 31 < seen) seen = p->window + tile_tokens + 31;
    l.seen = (uint32_t)seen;
    const uint64_t blocks = (uint64_t)p->sequences * p->kv_heads * l.tiles;
    const bool prompt = tile >= 8;
    // Chunks at most and their tokens at least: twelve workgroups of few rows per compute unit, of at least two steps per
    // wavefront (one sequence of 4101: 256 tokens 8.5 us, 384 9.1, 512 9.7).
    uint64_t chunks = split;
    if (!prompt) {
        chunks = blocks ? (12 * 256 + blocks - 1) / blocks : 1;
        uint64_t most = (seen + 255) / 256;
        // what the chunks write and the join reads, in proportion to the rows: 16 MB at most
        const uint64_t part = (uint64_t)p->rows * p->heads * (p->head_dim + 2) * 4;
        if (part && (16ull << 20) / part < most) most = (16ull << 20) / part;
        if (chunks > most) chunks = most;
    }
    // Whole where the join costs more than a split saves: up to 6 tokens for each tile of 16 rows, 12 for each larger one, whose
    // rows the join all reads, but no more than 512 tiles of 16 rows give; from 1024 tiles on, which fill the card by
    // themselves, 3 for each, up to what 4096 of them give; and 768 tokens, 512 of 256 wide heads, however few tiles there
    // are.  Fitted to these (us, split / whole, 128 wide, tokens x tiles):
    // 505 x 8 8.8 / 6.7, 755 x 8 8.5 / 8.2, 1005 x 8 8.4 / 9.6; 505 x 256 12.2 / 7.9, 1255 x 256 15.8 / 13.1, 3005 x 256 28.6 /
    // 29.8; 3005 x 512 47.8 / 41.6; up to 2005 x 256 17.2 / 18.0; 256 wide 755 x 32 10.0 / 11.1, 1255 x 128 19.4 / 16.6;
    // up to 8005 x 1024 128 / 153, up to 4005 x 2048 164 / 138; tiles of 32 rows 1304 x 104 19.7 / 16.5, 2200 x 200
    // 31.1 / 23.9, 2505 x 256 37.5 / 30.8, up to 2505 x 256 26.6 / 28.5.
    const uint64_t several = (tile == 1 ? 6 : 12) * blocks, whole = blocks < 1024 ? (several < 6 * 512 ? several : 6 * 512) : 3 * (blocks < 4096 ? blocks : 4096);
    if (!prompt && seen <= (whole > 768 ? whole : p->head_dim > 128 ? 512 : 768)) chunks = 1;
    if (chunks < 1) chunks = 1;
    l.chunk = chunk ? chunk : (uint32_t)(((seen + chunks - 1) / chunks + 127) / 128 * 128);
    if (l.chunk == 0) l.chunk = 128;
    l.chunks = (uint32_t)((seen + l.chunk - 1) / l.chunk);
    if (l.chunks < 1) l.chunks = 1;
    l.grid = (uint64_t)p->sequences * l.tiles * l.chunks;
    const uint64_t places = (uint64_t)p->rows * (p->heads / p->kv_heads) / (16 * tile) + p->sequences;
    if (tile != 1 && tile != 3 && attention_counts(p->sequences, starts, l.tiles) && places * l.chunks < l.grid) l.grid = places * l.chunks;
    l.pieces[0] = l.pieces[1] = l.works = 0;
    // With few tiles per sequence and enough to do, over 640 tokens of a head for each compute unit, the kernel sizes the
    // chunks by the lengths as they are, which may be far under max_length and far apart, and numbers those that there are one
    // after the other: workgroups that end at once leave the others unevenly spread.  As many as the card holds at once, or a
    // multiple of it, or two per compute unit where that leaves them under 700 tokens or so.  From 1024 tiles of more than 64
    // sequences on the gaps cost less than the count (96 sequences of up to 8005 126 -> 102, 128 128 -> 132).
    // us, by max_length alone -> so, 128 wide, a row of 4 heads: 8 sequences of 4101 tokens 17.1 -> 15.0, 32 of them 41.4 ->
    // 35.6, 32 of up to 4101 26.9 -> 22.9, one of 64001 31.6 -> 21.2 (3 per compute unit 23.7), 32 of up to 16384 80.1 -> 76 (2:
    // 83.6, 4: 88.5); 256 wide, 2 80.2 -> 72.4 (3: 84.4); 64 wide, 4 54.4 -> 49.8 (3: 56.4); 5 x 4 rows, 4 112.9 -> 105 (2: 121);
    // 16 x 8 rows of 8 sequences, 2 52.3 -> 45.4 (4: 52.2); 64 wide, 8 x 8 rows of 16, 3 39.0 -> 36.5 (2: 40.2, 4: 39.4), 5 x 8 rows
    // of 8 20.8 -> 20.1.
    const uint64_t all = (uint64_t)p->sequences * l.tiles * ((seen + 127) / 128);
    if (l.chunks > 1 && !chunk && !prompt && l.tiles <= 4 && (p->sequences <= 64 || (p->sequences <= 256 && blocks < 1024)) && all * p->kv_heads > 640 * 2) {
        const uint32_t held = tile == 1 ? (p->head_dim == 64 ? 4 : p->head_dim == 128 ? 3 : 2) : tile == 2 && p->head_dim == 64 ? 3 : 2;
        // half a workgroup for each sequence's last chunk has to be small beside them
        const uint64_t times = 2ull * p->sequences * p->kv_heads / (256 * held) + (tile == 2 ? 1 : 0);
        const uint32_t per[2] = {2, held * (uint32_t)(times < 1 ? 1 : times)};
        l.works = 2048 * 2 / p->kv_heads + 1;
        uint64_t grid = 0;
        for (uint32_t i = 0; i < 2; i++) {
            l.pieces[i] = 256 * per[i] / p->kv_heads;
            if (l.pieces[i] == 0) l.pieces[i] = 1;
            // sizes of at least all / pieces make pieces and one per tile at most
            const uint64_t parts = l.pieces[i] + (uint64_t)p->sequences * l.tiles + 1;
            if ((i == 0 || all >= l.works) && parts > grid) grid = parts;
        }
        if (grid < l.grid) l.grid = grid;
    }
    l.bytes = l.chunks > 1 ? (uint64_t)p->rows * p->heads * l.chunks * (p->head_dim + 2) * 4 + 16 : 0;
    return l;
}

static AttentionPlan attention_plan(const oco_cache *p, bool starts) {
    const uint64_t rows = (uint64_t)(p->max_rows < p->rows ? p->max_rows : p->rows) * (p->heads / p->kv_heads);
    // Tiles of 16 rows while that is all, of 32 beyond (of 16 where the second one would be half empty, or one of 48 with
    // over 3000 tokens of a head for each compute unit).  With narrow heads the prompts' kernel: tiles of 128 rows from 256
    // of them on, one per compute unit, and of 256 from 512 on where all are alike: 128 wide, one or two sequences, no window.
    // us, tiles of 16 / 32 / 128 / 256:
    // 32 sequences of 5 x 4 rows over 8000 tokens, 128 wide 115 / 84 / 141; 8 of 5 x 8 rows, 64 wide 20.7 / 22.1 / 33;
    // 4 of 128 x 4 rows over 2000 (128 tiles of 128) 41 / 33 / 49; 16 of 64 x 4 over 4000 (256, 128 of 256) 142 / 108 / 86 / 113;
    // 64 of 32 x 4 over 1000 (512) 92 / 75 / 49 / 80; 2048 x 4 rows from the start on (512, 256 of 256) 65 with 32 / 52 / 63;
    // 4096 x 4 rows over 8192 (512 of 256) 715 / 567 / 376 / 365, 4096 from the start on 147 / 138, 8192 505 / 507, with a window
    // of 2048 252 / 272, 64 wide 328 / 339; 4 sequences of up to 1000 x 4 rows after 3000 142 / 150, 4 of up to 4096 after 4096
    // 1020 / 1047; 256 wide (16 heads) 623 / 443.
    // Tiles of 16 / 48, 5 x 8 rows: 32 sequences of 4005 tokens, 64 wide 52.6 / 42.3, 128 wide 71 / 56, of up to 8192 64 wide 63 /
    // 59, 128 wide 89 / 76; 8 of up to 8192, 64 wide 19.9 / 21.8; two of 2005 9.6 / 11.5.  Where rows differ too, 32 sequences of
    // up to 5 over up to 8192, 64 wide 50 / 54, 128 wide 77 / 69, and tiles of 32 would take 42 and 64.
    int32_t knob[4];
    const int set = plan_override(OCO_KNOB_ATTENTION, knob);
    const bool narrow = p->head_dim <= 128;
    const uint64_t heads = (uint64_t)p->kv_heads * p->sequences;
    uint32_t tile = rows <= 16 || (rows > 32 && rows <= 48) ? 1 : 2;
    if (narrow && rows > 32 && rows <= 48 && heads * p->max_length > 3000 * 256) tile = 3;
    const uint64_t total = (uint64_t)p->rows * (p->heads / p->kv_heads);  // of all sequences
    const bool wide_tiles = p->head_dim == 128 && p->sequences <= 2 && (p->window == 0 || p->window >= p->max_length);
    if (narrow && rows >= 128 && (total / 64 + p->sequences) * p->kv_heads >= 512) tile = wide_tiles && total / 256 * p->kv_heads >= 512 ? 16 : 8;
    // Fewer tiles of 128 than compute units over a long context: chunks of them until the card's 512 places are full or
    // nearly so, of 1536 tokens at least.  us, tiles of 32 / so: 512 rows of 32 heads after 8000 tokens (4 chunks) 109 / 92, 256
    // after 16000 (8) 118 / 88, 128 after 32000 (16) 126 / 86, 700 after 16000 (5) 314 / 242, 4 of 128 after 8000 (4) 105 / 93;
    // 512 after 2000 35 / 47.
    uint32_t split = 1;
    const uint64_t alike = (rows + 127) / 128 * heads, half = (total / 64 + p->sequences) * p->kv_heads / 2, estimate = alike < half ? alike : half;
    const uint64_t reach = p->window ? (p->window < p->max_length ? p->window : p->max_length) : p->max_length;
    if (narrow && rows >= 128 && estimate < 256) {
        while (split < 64 && 20 * split * estimate < 17 * ((split * estimate + 511) / 512) * 512) split++;
        if (reach / split >= 1536)
            tile = 8;
        else
            split = 1;
    }
    if (set && (knob[0] == 1 || knob[0] == 2 || ((knob[0] == 3 || knob[0] == 8) && narrow) || (knob[0] == 16 && p->head_dim == 128))) tile = (uint32_t)knob[0];
    const uint32_t chunk = set > 1 && knob[1] > 0 && knob[1] % 128 == 0 ? (uint32_t)knob[1] : 0;
    return attention_split(p, tile, rows, split, chunk, starts);
}

template <uint32_t D, bool BF>
static int attention_launch(const AttentionArgs &a, const AttentionPlan &l, hipStream_t stream) {
    const uint64_t grid = l.grid * a.b.kv_heads;
    if (grid > 0x7fffffffull) return fail(OCO_ERR_INVALID, "oco_cache_attention: too many rows for one call");
#define GO(R, FIT) hipLaunchKernelGGL((attention_kernel<D, BF, R, FIT>), dim3((uint32_t)grid), dim3(256), 0, stream, a, l.tiles)
    if (l.tile >= 8) {
        OCO_TRY(attention_prompt_launch(a, D, BF, l.tiles, (uint32_t)grid, stream));
    } else if (l.tile == 3) {
        if constexpr (D <= 128) {
            if (l.works)
                GO(3, true);
            else
                GO(3, false);
        }
    } else if (l.tile == 2) {
        if (l.works)
            GO(2, true);
        else
            GO(2, false);
    } else {
        if (l.works)
            GO(1, true);
        else
            GO(1, false);
    }
#undef GO
    OCO_TRY(launch_check("oco_cache_attention"));
    if (l.chunks > 1) {
        if (a.b.rows * a.heads >= 2048)
            hipLaunchKernelGGL((attention_join_kernel<D, BF, 1>), dim3((a.b.rows * a.heads + 3) / 4), dim3(256), 0, stream, a);
        else
            hipLaunchKernelGGL((attention_join_kernel<D, BF, 4>), dim3(a.b.rows * a.heads), dim3(256), 0, stream, a);
        OCO_TRY(launch_check("oco_cache_attention (join)"));
    }
    return OCO_OK;
}

static const char *attention_problem(const oco_cache *p) {
    if (const char *why = cache_problem(p)) return why;
    if (p->heads == 0) return "no heads";
    if ((uint64_t)p->rows * p->heads > 0x7fffffffull || (uint64_t)p->sequences * p->kv_heads > 0x7fffffffull) return "too many rows for one call";
    return nullptr;
}

}  // namespace oco

using namespace oco;

extern "C" uint64_t oco_cache_attention_workspace(const oco_cache *p) {
    return p && !attention_problem(p) ? attention_plan(p, false).bytes : 0;
}

extern "C" int oco_cache_attention(const void *q, const void *pages, const uint32_t *table, const uint32_t *starts,
                                   const uint32_t *lengths, const float *sinks, void *out, const oco_cache *p, void *workspace,
                                   uint64_t workspace_bytes, oco_stream stream) {
    if (!p) return fail(OCO_ERR_INVALID, "oco_cache_attention: null description");
    if (const char *why = attention_problem(p)) return fail(OCO_ERR_INVALID, "oco_cache_attention: %s", why);
    if (p->dtype != OCO_DT_BF16 && p->dtype != OCO_DT_F16) return fail(OCO_ERR_UNSUPPORTED, "oco_cache_attention: type %u", p->dtype);
    if (p->rows == 0 || p->sequences == 0 || p->max_rows == 0) return OCO_OK;
    if (!q || !pages || !table || !lengths || !out) return fail(OCO_ERR_INVALID, "oco_cache_attention: null pointer");
    if ((uintptr_t)pages & 15u) return fail(OCO_ERR_INVALID, "oco_cache_attention: pages must be 16-byte aligned");
    if (!starts && p->rows % p->sequences)
        return fail(OCO_ERR_INVALID, "oco_cache_attention: %u rows of %u sequences without starts", p->rows, p->sequences);
    const AttentionPlan l = attention_plan(p, starts);
    if (l.bytes && (!workspace || ((uintptr_t)workspace & 15u) || workspace_bytes < l.bytes))
        return fail(OCO_ERR_INVALID, "oco_cache_attention: workspace of %llu bytes, need %llu, 16-byte aligned",
                    (unsigned long long)workspace_bytes, (unsigned long long)l.bytes);
    AttentionArgs a;
    a.b = cache_batch(p, table, starts, lengths);
    a.cache = (const uint8_t *)pages;
    a.q = q;
    a.out = out;
    a.sinks = sinks;
    a.parts = (float *)workspace;
    a.q_stride = p->q_stride ? p->q_stride : (uint64_t)p->heads * p->head_dim;
    a.out_stride = p->out_stride ? p->out_stride : (uint64_t)p->heads * p->head_dim;
    if (q == out && a.q_stride != a.out_stride) return fail(OCO_ERR_INVALID, "oco_cache_attention: in place with another stride");
    a.heads = p->heads;
    a.group = p->heads / p->kv_heads;
    a.window = p->window >= p->max_length ? 0 : p->window;
    a.tile_rows = 16 * l.tile;
    a.chunks = l.chunks;
    a.chunk = l.chunk;
    a.seen = l.seen;
    a.works = l.works;
    for (int i = 0; i < 2; i++) {
        a.pieces[i] = l.pieces[i];
        a.inverse[i] = 1.f / (float)l.pieces[i];
        a.relaxed[i] = l.pieces[i] > p->sequences * l.tiles / 2 + 1 ? 1.f / (float)(l.pieces[i] - p->sequences * l.tiles / 2) : 1.f;
    }
    a.c = (p->scale != 0.f ? p->scale : 1.f / sqrtf((float)p->head_dim)) * 1.44269504088896341f;
    hipStream_t st = (hipStream_t)stream;
    const bool bf = p->dtype == OCO_DT_BF16;
    switch (p->head_dim) {
    case 64: return bf ? attention_launch<64, true>(a, l, st) : attention_launch<64, false>(a, l, st);
    case 128: return bf ? attention_launch<128, true>(a, l, st) : attention_launch<128, false>(a, l, st);
    default: return bf ? attention_launch<256, true>(a, l, st) : attention_launch<256, false>(a, l, st);
    }
}
