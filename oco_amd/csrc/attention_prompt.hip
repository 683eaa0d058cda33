// Attention over the paged cache for many rows: the matrix cores' side.
//
// A workgroup's four or eight wavefronts hold 32 rows each and share steps of
// 64 tokens, whose codes are converted once for all of them into LDS: keys as
// rows, values transposed, so that both products read 16 bytes per lane.  As
// in the kernel for few rows a lane is a row throughout (here of two), and the
// products' inner indexes are in the order in which the scores leave the first
// product.  A wavefront converts 16 tokens of a buffer, which lie in one page.
//
// Bound by how well matrix cores, vector units and LDS run beside each other,
// each about half of the time busy with the two wavefronts per SIMD that the
// registers leave: a step of a wavefront is 32 products of 32 x 32 x 16 (1024
// clocks), 32 KB from LDS, 32 exponentials per lane and its share of the
// conversions (190 to 210 vector instructions).  So a step computes the next
// one's scores beside its own exponentials and converts beside the second
// product, in groups that each request the next group's fragments (4096 rows
// of 32 heads over 8192 tokens: 670 us with the steps one after the other and
// in three chunks, 476 whole, 435 with the scores of the next step, 412 in
// groups and without copies between turns, 381 with the chunk grid by tile).
// Eight wavefronts on twice the tokens halve the conversions' share: 365 us,
// 1.13 PFLOP/s (a large library product of bf16 reaches 1.2 to 1.35), 807 over
// 16000 tokens.  Measured and lost: wavefront priorities around the products
// (no change), other paddings of the rows in LDS (413 to 430 against 412).
#include "attention.h"

namespace oco {

template <uint32_t D, bool BF, int W>
__global__ __launch_bounds__(64 * W, 2) void attention_prompt_kernel(AttentionArgs a, uint32_t tiles) {
    using H = Half<BF>;
    constexpr uint32_t KT = 64, BT = 16 * W;  // tokens of a step, of a buffer: a step or two
    constexpr int SUBS = BT / KT;
    constexpr int KN = KT / 32, NS = D / 16, NO = D / 32;       // key tiles, key steps, column tiles
    constexpr uint32_t PIECE = D / 16;                          // columns of a value's piece
    // rows of 16-byte pieces, one piece of padding: eight consecutive rows fall into different banks
    constexpr uint32_t KROW = D / 8 + 1, VROW = BT / 8 + 1;
    __shared__ __attribute__((aligned(16))) u32x4 keys[2][BT * KROW], values[2][D * VROW];
    __shared__ uint32_t flags[3];  // the buffer's number, from 1, whose values hold a block of NaN; the last one is not read

    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, g = lane >> 5;
    uint32_t id = blockIdx.x;
    const uint32_t h = id % a.b.kv_heads;
    id /= a.b.kv_heads;
    const uint32_t chunk = id % a.chunks;
    id /= a.chunks;
    const AttentionPlace place = attention_place<32 * W>(a, id, tiles);
    const uint32_t s = place.sequence, tile = place.tile;
    const CacheSpan span = place.span;
    if (s >= a.b.sequences) return;
    const AttentionTile range = attention_tile(span, tile, 32 * W, a.group, a.window);
    const uint32_t rows = range.rows;
    if (range.first_row >= rows) return;
    const int32_t before = (int32_t)span.length - (int32_t)span.rows;
    const uint32_t first = range.first + chunk * a.chunk, end = min(first + a.chunk, range.end);
    if (chunk && first >= range.end) return;
    const uint32_t head_bytes = cache_head_bytes(a.b.page_size, D);
    const uint32_t *const table = a.b.table + (uint64_t)s * a.b.table_stride;

    // this lane's row, or the last one once more (as in the kernel for few rows)
    const uint32_t row0 = range.first_row + 32 * wave;
    const bool live = row0 + n < rows;
    const uint32_t i0 = live ? row0 + n : rows - 1;
    const uint32_t token = i0 / a.group, head = h * a.group + i0 % a.group;
    const int32_t at = before + (int32_t)token;
    const int32_t least = before + (int32_t)(row0 / a.group), most = before + (int32_t)((min(row0 + 32, rows) - 1) / a.group);
    u32x4 q[NS];
    {
        const uint16_t *const row = (const uint16_t *)a.q + (uint64_t)(span.first + token) * a.q_stride + (uint64_t)head * D + 8 * g;
#pragma unroll
        for (int i = 0; i < NS; i++) q[i] = *(const GLOBAL u32x4_u *)gp(row + 16 * i);
    }
    float m = -INFINITY, l = 0.f;
    f32x16 o[NO];
#pragma unroll
    for (int j = 0; j < NO; j++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[j][i] = 0.f;

    // ---- converting: a thread's share of a step
    const uint32_t half = wave;  // the 16 tokens that this wavefront converts
    constexpr uint32_t KB = D == 64 ? 8 : 16, KPIECES = D / 2 / KB;  // bytes of a key per thread, threads per key
    const uint32_t kt = threadIdx.x / KPIECES, kp = threadIdx.x % KPIECES;
    const uint32_t vg = threadIdx.x / 16, vm = threadIdx.x % 16;  // four tokens, a piece
    struct Raw {
        uint32_t w[4], scale;
        bool lost;
    };
    const uint32_t k_at = kt % 16 * (D / 2) + kp * KB, ks_at = a.b.page_size * D + kt % 16 * (D / 32) + kp * KB / 16;
    const uint32_t v_at = a.b.page_size * (D / 2) + vg % 4 * (2 * D) + vm * (D / 8);
    const uint32_t vs_at = a.b.page_size * D + a.b.page_size * (D / 32) + vg % 4 * (D / 8) + vm * D / 512 * 4;
    uint32_t page_of = 0, slot_of = 0;  // lane i: of buffer 64 c + i
    auto read_table = [&](uint32_t step) {
        const uint32_t t = first + (step + lane) * BT + 16 * half;  // step: the first of 64
        page_of = t < end ? table[t / a.b.page_size] : 0;
        slot_of = t % a.b.page_size;
    };
    // the head's bytes in a step's page, and the step's place there
    struct Place {
        gbytes head;
        uint32_t slot;
        bool lost;
    };
    auto find = [&](uint32_t step) {
        Place x;
        uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)page_of, step % 64);
        x.slot = (uint32_t)__builtin_amdgcn_readlane((int)slot_of, step % 64);
        x.lost = page >= a.b.pages;
        page = x.lost ? 0 : page;
        x.head = (gbytes)gp(a.cache) + ((uint64_t)page * a.b.kv_heads + h) * head_bytes;
        return x;
    };
    auto request_keys = [&](Raw &x, const Place &p) {
        const gbytes words = p.head + p.slot * (D / 2);
        if constexpr (D == 64) {
            const u32x2 k = *(const GLOBAL u32x2 *)(words + k_at);
            x.w[0] = k.x;
            x.w[1] = k.y;
        } else {
            const u32x4 k = *(const GLOBAL u32x4 *)(words + k_at);
#pragma unroll
            for (int i = 0; i < 4; i++) x.w[i] = k[i];
        }
        x.scale = (p.head + p.slot * (D / 32))[ks_at];
        x.lost = p.lost;
    };
    auto request_values = [&](Raw &x, const Place &p) {
        const gbytes words = p.head + p.slot * (D / 2);
        if constexpr (D == 64) {
            const u32x2 v = *(const GLOBAL u32x2 *)(words + v_at);
            x.w[0] = v.x;
            x.w[1] = v.y;
        } else {
            const u32x4 v = *(const GLOBAL u32x4 *)(words + v_at);
#pragma unroll
            for (int i = 0; i < 4; i++) x.w[i] = v[i];
        }
        x.scale = *(const GLOBAL uint32_t *)(p.head + p.slot * (D / 32) + vs_at);
        x.lost = p.lost;
    };
    auto convert_keys = [&](const Raw &x, uint32_t into) {
        const float ks = block_scale<H::LIMIT>(x.lost ? 255 : x.scale);
#pragma unroll
        for (int i = 0; i < (int)KB / 4; i++)
            keys[into][kt * KROW + kp * (KB / 4) + i] = u32x4{H::template pair<0>(x.w[i], ks), H::template pair<1>(x.w[i], ks),
                                                            H::template pair<2>(x.w[i], ks), H::template pair<3>(x.w[i], ks)};
    };
    auto convert_values = [&](const Raw &x, uint32_t into, uint32_t number) {
        uint32_t vs = x.lost ? 0xffffffffu : x.scale;
        // a NaN block enters as numbers, for 0 * NaN is NaN; without a branch, which would keep the
        // products before it from running beside
        const uint32_t bad = bytes_past<H::LIMIT>(vs);
        vs ^= bad;
        flags[__any(bad != 0) ? into : 2] = number;
        float scale[4];
#pragma unroll
        for (int i = 0; i < 4; i++) scale[i] = __uint_as_float(byte_of(vs, i) << 23);
        // column PIECE m + c is in row 16 c + m; groups of four tokens of 16 in the order 0, 2, 1, 3
        u32x2 *const out = (u32x2 *)&values[into][0] + (vg / 4 * 4 + vg % 2 * 2 + vg % 4 / 2);
#pragma unroll
        for (int b = 0; b < (D == 64 ? 2 : 4); b++) {
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int byte = D == 64 ? 2 * (i % 2) + b : b;
                const uint32_t w = D == 64 ? x.w[i / 2] : x.w[i];
                c[i] = byte == 0 ? H::template pair<0>(w, scale[i]) : byte == 1 ? H::template pair<1>(w, scale[i])
                     : byte == 2 ? H::template pair<2>(w, scale[i]) : H::template pair<3>(w, scale[i]);
            }
            out[(2 * b * 16 + vm) * (2 * VROW)] = low_halves(c);
            out[((2 * b + 1) * 16 + vm) * (2 * VROW)] = high_halves(c);
        }
    };
    auto scores = [&](f32x16 *sc) {  // of the first step
#pragma unroll
        for (int k = 0; k < KN; k++)
#pragma unroll
            for (int i = 0; i < 16; i++) sc[k][i] = 0.f;
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int k = 0; k < KN; k++) sc[k] = H::product32(keys[0][(32 * k + n) * KROW + 2 * i + g], q[i], sc[k]);
    };

    // A step computes the scores of the next one beside its own probabilities.  With a step per buffer it
    // converts the keys of the buffer after the next and the values of the next; with two, the first
    // one the next buffer's keys and the second its values.  The ones after those are on their way.
    // Past the last buffer the first page is read again.
    const uint32_t steps = end > first ? (end - first + KT - 1) / KT : 0;
    Raw rk, rv;
    Place ahead;
    f32x16 sc[KN];
    if (steps) {
        read_table(0);
        Place p = find(0);
        request_keys(rk, p);
        request_values(rv, p);
        p = find(1);
        Raw second;
        if constexpr (SUBS == 1) request_keys(second, p);
        convert_keys(rk, 0);
        if (threadIdx.x < 2) flags[threadIdx.x] = 0;
        __syncthreads();
        convert_values(rv, 0, 1);
        request_values(rv, p);
        if constexpr (SUBS == 1) {
            ahead = find(2);
            request_keys(rk, ahead);
            convert_keys(second, 1);
        } else {
            request_keys(rk, p);
        }
        __syncthreads();
        scores(sc);
        // step 0 converts the keys of step 2 over those that every wavefront has just read
        if constexpr (SUBS == 1) __syncthreads();
    }
    // step, its scores, where the next step's go, its buffer's number and place, its place in the buffer
    auto compute = [&](const uint32_t step, f32x16 *sc, f32x16 *next, const uint32_t number, const uint32_t buffer, const int sub) {
        const uint32_t t0 = first + step * KT, next_buffer = sub + 1 == SUBS ? buffer ^ 1 : buffer;
        const int next_sub = sub + 1 == SUBS ? 0 : sub + 1;
        const u32x4 *const next_keys = &keys[next_buffer][(next_sub * KT + n) * KROW + g];
        const u32x4 *const own_values = &values[buffer][n * VROW + sub * (KT / 8) + g];
        if constexpr (SUBS == 1) {
            if ((step + 3) % 64 == 0) read_table(step + 3);
        } else {
            if (sub == 0 && (number + 2) % 64 == 0) read_table(number + 2);
        }
        if ((int32_t)(t0 + KT) - 1 > least || t0 + KT > end || (a.window && (int32_t)t0 + (int32_t)a.window <= most)) {
#pragma unroll
            for (int k = 0; k < KN; k++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int32_t t = (int32_t)t0 + 32 * k + 8 * (i / 4) + 4 * (int32_t)g + i % 4;
                    if (!(t <= at && (uint32_t)t < end && (!a.window || t + (int32_t)a.window > at))) sc[k][i] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < KN; k++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, sc[k][i]);
        {
            auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])) * a.c;
        }
        if (__any(top > m + 8.f)) {
            top = fmaxf(top, m);
            const float f = carry(m, top);
            m = top;
            l *= f;
#pragma unroll
            for (int j = 0; j < NO; j++) o[j] *= f;
        }
        if (flags[buffer] == number + 1) {
            // rows that see a block of NaN: every lane looks at the step's tokens itself
            uint32_t bad = 0;
            for (uint32_t t = t0; t < min(t0 + KT, end); t++) {
                if (!((int32_t)t <= at && (!a.window || (int32_t)(t + a.window) > at))) continue;
                const uint32_t page = table[t / a.b.page_size];
                for (uint32_t b = 0; b < D / 32; b++)
                    if (page >= a.b.pages ||
                        a.cache[((uint64_t)page * a.b.kv_heads + h) * head_bytes + cache_value_scale_at(a.b.page_size, t % a.b.page_size, b, D)] > H::LIMIT)
                        bad |= 1u << b;
            }
#pragma unroll
            for (int j = 0; j < NO; j++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const uint32_t r = 32 * j + 8 * (i / 4) + 4 * g + i % 4;
                    if (bad >> ((PIECE * (r % 16) + r / 16) / 32) & 1) o[j][i] = __uint_as_float(0x7fc00000u);
                }
        }
        // Scores of the next step between the exponentials of this one, then the second product between
        // the conversions.  Each group requests the next one's fragments, and nothing moves across groups.
        const float ref = m > -INFINITY ? m : 0.f;
        u32x4 p[2 * KN], kf[2][KN], vf[2][NO];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KN; k++) {
#pragma unroll
            for (int i = 0; i < 16; i++) next[k][i] = 0.f;
            kf[0][k] = next_keys[32 * k * KROW];
        }
#pragma unroll
        for (int i = 0; i < NS; i++) {
            if (i + 1 < NS) {
#pragma unroll
                for (int k = 0; k < KN; k++) kf[(i + 1) % 2][k] = next_keys[32 * k * KROW + 2 * (i + 1)];
            } else {
#pragma unroll
                for (int j = 0; j < NO; j++) vf[0][j] = own_values[32 * j * VROW];
            }
#pragma unroll
            for (int k = 0; k < KN; k++) next[k] = H::product32(kf[i % 2][k], q[i], next[k]);
            constexpr int E = KN * 16 / NS;  // a group's exponentials
#pragma unroll
            for (int e = E * i; e < E * i + E; e++) {
                const float u = __builtin_amdgcn_exp2f(fmaf(sc[e / 16][e % 16], a.c, -ref));
                sc[e / 16][e % 16] = u;
                if (e % 2) {
                    const uint32_t pair = H::pack(sc[e / 16][e % 16 - 1], u);
                    p[e / 8][e % 8 / 2] = pair;
                    sum[e / 2 % 2] = H::add(pair, sum[e / 2 % 2]);  // the rounded probabilities, as they weigh
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum[0] + sum[1];
#pragma unroll
        for (int t = 0; t < 2 * KN; t++) {
            if (t + 1 < 2 * KN) {
#pragma unroll
                for (int j = 0; j < NO; j++) vf[(t + 1) % 2][j] = own_values[32 * j * VROW + 2 * (t + 1)];
            }
#pragma unroll
            for (int j = 0; j < NO; j++) o[j] = H::product32(vf[t % 2][j], p[t], o[j]);
            if constexpr (SUBS == 1) {
                if (t == 0) {
                    convert_keys(rk, buffer);
                } else if (t == KN) {
                    convert_values(rv, buffer ^ 1, number + 2);
                    request_values(rv, ahead);
                    ahead = find(step + 3);
                    request_keys(rk, ahead);
                }
            } else if (t == 1) {
                if (sub == 0) {
                    convert_keys(rk, buffer ^ 1);
                    ahead = find(number + 2);
                    request_keys(rk, ahead);
                } else {
                    convert_values(rv, buffer ^ 1, number + 2);
                    request_values(rv, ahead);
                }
            }
            if (t + 1 < 2 * KN && (t == 0 || t + 1 == KN)) __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
    };
    f32x16 other[KN];
    if constexpr (SUBS == 1) {
        for (uint32_t step = 0; step < steps; step += 2) {
            compute(step, sc, other, step, 0, 0);
            if (step + 1 == steps) break;
            compute(step + 1, other, sc, step + 1, 1, 0);
        }
    } else {
        for (uint32_t step = 0, number = 0; step < steps; step += 2, number++) {
            compute(step, sc, other, number, number & 1, 0);
            if (step + 1 == steps) break;
            compute(step + 1, other, sc, number, number & 1, 1);
        }
    }
    if (!live) return;
    {
        auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    }
    const uint32_t row = span.first + token;
    float by = 1.f;
    const uint64_t index = ((uint64_t)row * a.heads + head) * a.chunks + chunk;
    if (a.chunks > 1) {
        if (g == 0) *(GLOBAL f32x2 *)gp(a.parts + (uint64_t)a.b.rows * a.heads * a.chunks * D + index * 2) = f32x2{m, l};
    } else {
        float top = m, total = l;
        if (a.sinks) {
            const float sink = a.sinks[head] * 1.44269504088896341f;
            top = fmaxf(m, sink);
            total = l * carry(m, top) + carry(sink, top);
        }
        by = part_of(carry(m, top), total, at >= 0);
    }
    // accumulator row 16 c + m is column PIECE m + c: a lane has all columns of a piece
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t column = PIECE * (8 * (i / 4) + 4 * g + i % 4);
        float v[PIECE];
#pragma unroll
        for (uint32_t c = 0; c < PIECE; c++) v[c] = o[c / 2][i + 8 * (c % 2)] * by;
        if (a.chunks > 1) {
            float *const out = a.parts + index * D + column;
#pragma unroll
            for (uint32_t c = 0; c < PIECE; c += 4) *(GLOBAL f32x4 *)gp(out + c) = f32x4{v[c], v[c + 1], v[c + 2], v[c + 3]};
        } else {
            uint16_t *const out = (uint16_t *)a.out + (uint64_t)row * a.out_stride + (uint64_t)head * D + column;
#pragma unroll
            for (uint32_t c = 0; c < PIECE; c += 4) *(GLOBAL u32x2_u *)gp(out + c) = u32x2_u{H::pack(v[c], v[c + 1]), H::pack(v[c + 2], v[c + 3])};
        }
    }
}

int attention_prompt_launch(const AttentionArgs &a, uint32_t head_dim, bool bf, uint32_t tiles, uint32_t grid, hipStream_t stream) {
#define GO(D, BF, W) hipLaunchKernelGGL((attention_prompt_kernel<D, BF, W>), dim3(grid), dim3(64 * W), 0, stream, a, tiles)
    if (head_dim == 64) {
        if (bf)
            GO(64, true, 4);
        else
            GO(64, false, 4);
    } else if (a.tile_rows == 256) {
        if (bf)
            GO(128, true, 8);
        else
            GO(128, false, 8);
    } else {
        if (bf)
            GO(128, true, 4);
        else
            GO(128, false, 4);
    }
#undef GO
    return launch_check("oco_cache_attention (prompt)");
}

}  // namespace oco
