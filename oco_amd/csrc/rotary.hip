// Rotary positions, and the pages of a cache in 4 bits: appending rows with
// their rotation on the way, and reading them back.
//
// Angles are position * frequency in 64 bits, at most 2^-53 of themselves off
// (1e-10 at a million radians, where f32 would be off by 0.06), their cosines
// and sines by Taylor series on a quarter turn, and the products are 64-bit
// too.  They are rounded to f32 and from there to the type, so that a key next
// to a border between two codes falls where the exact one does unless it is
// within half a step of f32 of a middle between two numbers of the type.  One
// token's pairs are the same for all its heads, so a wavefront takes a token,
// or a part of its heads, keeps them in LDS and waits for no other.
//
// Bound by memory where there are many rows (8192 rows of 32 heads of 128 f16
// 22.6 us, 5.9 TB/s; 8192 tokens of 32 + 2 * 8 heads appended 37 us, 4.5 TB/s,
// and read back 8.5), and by the loads that wait for each other where there are
// few (a row 2.2 us, 64 tokens appended 6.0 and read back 3.1).
#include "cache.h"
#include "eight.h"

namespace oco {

// cos and sin of a: a - k pi/2 with pi/2 in two parts, then Taylor series for
// |r| <= pi/4, whose first terms left out are r^19 / 19! and r^20 / 20! (1e-19).
__device__ __forceinline__ double2 cos_sin(double a) {
    const double k = __builtin_rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-k, 1.57079632679489655800, a);
    r = __builtin_fma(-k, 6.12323399573676603587e-17, r);
    const double q = r * r;
    constexpr double S[8] = {1.0 / 355687428096000.0, -1.0 / 1307674368000.0, 1.0 / 6227020800.0, -1.0 / 39916800.0,
                             1.0 / 362880.0, -1.0 / 5040.0, 1.0 / 120.0, -1.0 / 6.0};
    constexpr double C[9] = {-1.0 / 6402373705728000.0, 1.0 / 20922789888000.0, -1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0,
                             1.0 / 40320.0, -1.0 / 720.0, 1.0 / 24.0, -0.5};
    double s = S[0], c = C[0];
#pragma unroll
    for (int i = 1; i < 9; i++) {
        // constants in scalar registers: as vector ones they cost the callers 30, and spills
        double si = S[i < 8 ? i : 7], ci = C[i];
        asm("" : "+s"(si), "+s"(ci));
        if (i < 8) s = __builtin_fma(s, q, si);
        c = __builtin_fma(c, q, ci);
    }
    s = __builtin_fma(s * q, r, r);
    c = __builtin_fma(c, q, 1.0);
    const uint32_t quarter = (uint32_t)(long long)k & 3;
    const double x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
    return make_double2(quarter == 1 || quarter == 2 ? -x : x, quarter & 2 ? -y : y);
}

struct Rotation {
    const double *frequencies;
    double magnitude;
    uint32_t dim;
};

// Between what a wavefront's lanes write to LDS and what other lanes of it read there. LDS takes a wavefront's accesses in
// order; this keeps the compiler from moving them past each other, and is no instruction.
__device__ __forceinline__ void lanes_wrote() { __builtin_amdgcn_wave_barrier(); }

// The pairs' cosines and sines of one position, by one wavefront for itself.
struct Angles {
    double first;  // a lane's first frequency, which can be read before the position is known
    __device__ __forceinline__ Angles(const Rotation &r) {
        const uint32_t lane = threadIdx.x & 63;
        first = lane < r.dim / 2 ? r.frequencies[lane] : 0.0;
    }
    __device__ __forceinline__ void table(const Rotation &r, uint32_t position, double2 *out) const {
        for (uint32_t i = threadIdx.x & 63; i < r.dim / 2; i += 64) {
            const double2 t = cos_sin((double)position * (i < 64 ? first : r.frequencies[i]));
            out[i] = make_double2(t.x * r.magnitude, t.y * r.magnitude);
        }
    }
};

// A head as units of work: eight pairs (four interleaved), then runs of eight
// values that stay.  A unit reads what it writes and nothing else, so the
// result may take the place of the row.
struct HeadUnits {
    uint32_t turns, all;
    bool whole;  // every unit has all its values
};
template <bool INTERLEAVED>
__device__ __forceinline__ HeadUnits head_units(const Rotation &r, uint32_t head_dim) {
    HeadUnits u;
    u.turns = INTERLEAVED ? (r.dim + 7) / 8 : (r.dim / 2 + 7) / 8;
    u.all = u.turns + (head_dim - r.dim + 7) / 8;
    u.whole = r.dim % (INTERLEAVED ? 8 : 16) == 0 && head_dim % 8 == 0;
    return u;
}

// A unit's values: a from column `first` on, and b (of a turning unit in halves) half further.
struct Unit {
    float a[8], b[8];
};
template <class T, bool INTERLEAVED>
struct RawUnit {  // the same as they are loaded
    Eight<T> a, b;
    __device__ __forceinline__ void values(Unit &x) const {
        a.values(x.a);
        if constexpr (!INTERLEAVED) b.values(x.b);
    }
};
struct UnitPlace {
    uint32_t first;
    bool turns, pairs;  // pairs: b is there
};
template <bool INTERLEAVED>
__device__ __forceinline__ UnitPlace unit_place(uint32_t u, const HeadUnits &n, const Rotation &r) {
    UnitPlace p;
    p.turns = u < n.turns;
    p.pairs = p.turns && !INTERLEAVED;
    p.first = p.turns ? 8 * u : r.dim + 8 * (u - n.turns);
    return p;
}
template <class T, bool INTERLEAVED>
__device__ __forceinline__ void load_unit(RawUnit<T, INTERLEAVED> &x, const T *head, const UnitPlace &p, const Rotation &r) {
    x.a.load(head + p.first);
    if constexpr (!INTERLEAVED) x.b.load(head + p.first + (p.pairs ? r.dim / 2 : 0));
}
template <class T>
__device__ __forceinline__ void load_unit_tail(Unit &x, const T *head, const UnitPlace &p, const Rotation &r, uint32_t head_dim) {
    load_run(head, p.first, p.pairs ? r.dim / 2 : p.turns ? r.dim : head_dim, x.a);
    if (p.pairs) load_run(head + r.dim / 2, p.first, r.dim / 2, x.b);
}
// To f32; the type's conversion is the second rounding, kept apart from the first by the empty statement: for a pair in eight
// of f16 the compiler made one of the two, in integer code (8192 rows of 32 x 128 f16, half turned, 24.2 us, so 22.6; about
// 1300 tokens of 64 wide heads appended and read back 13.0, 12.4).
__device__ __forceinline__ void turn_pair(float &x, float &y, const double2 &t) {
    const double v = x, w = y;
    x = (float)__builtin_fma(v, t.x, -(w * t.y));
    y = (float)__builtin_fma(w, t.x, v * t.y);
    asm("" : "+v"(x), "+v"(y));
}
template <bool INTERLEAVED, bool WHOLE>
__device__ __forceinline__ void turn_unit(Unit &x, const UnitPlace &p, const Rotation &r, const double2 *table) {
    if (!p.turns) return;
    const uint32_t first = INTERLEAVED ? p.first / 2 : p.first, last = r.dim / 2 - 1;  // pairs past it are not stored
    if constexpr (!INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < 8; j++) turn_pair(x.a[j], x.b[j], table[WHOLE ? first + j : min(first + j, last)]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) turn_pair(x.a[2 * j], x.a[2 * j + 1], table[WHOLE ? first + j : min(first + j, last)]);
    }
}
// Past the caches, where rows still to be read stay: 8192 rows of 32 x 128 f16 33.4 -> 24.1 us, 8192 tokens appended and
// read back 55 -> 47; the attention that reads the turned queries next takes as long (64 sequences of one token after
// their append 21.7 us either way, 8192 tokens 574 against 569).  Loads past them lost (24 -> 31).
template <class T>
__device__ __forceinline__ void store_unit(T *head, const Unit &x, const UnitPlace &p, const Rotation &r) {
    Eight<T> y;
    y.round(x.a);
    y.stream(head + p.first);
    if (p.pairs) {
        y.round(x.b);
        y.stream(head + p.first + r.dim / 2);
    }
}
template <class T>
__device__ __forceinline__ void store_unit_tail(T *head, const Unit &x, const UnitPlace &p, const Rotation &r, uint32_t head_dim) {
    const uint32_t n = (p.pairs ? r.dim / 2 : p.turns ? r.dim : head_dim) - p.first;
    Eight<T> y;
    y.round(x.a);
    y.store_some(head + p.first, n);
    if (p.pairs) {
        y.round(x.b);
        y.store_some(head + p.first + r.dim / 2, n);
    }
}

// A unit among those of `heads` consecutive heads, and the one `step` on.
struct Cursor {
    uint32_t head, unit;
    __device__ __forceinline__ Cursor(uint32_t i, const HeadUnits &n) : head(i / n.all), unit(i % n.all) {}
    __device__ __forceinline__ void advance(uint32_t dh, uint32_t du, const HeadUnits &n) {
        unit += du;
        const bool over = unit >= n.all;
        head += dh + over;
        unit -= over ? n.all : 0;
    }
};

// Turns the units first, first + step, ... of `heads` heads.  Whole units go N
// at a time, and the loads of the first ones are out before the table of
// angles is made (false: there is nothing to turn).
template <class T, bool INTERLEAVED, class In, class Out, class Table>
__device__ __forceinline__ bool turn_heads(uint32_t first, uint32_t step, uint32_t heads, uint32_t head_dim, const HeadUnits &n, const Rotation &r,
                                           const double2 *table, In in, Out out, Table make_table) {
    constexpr int N = sizeof(T) == 4 ? 1 : 2;
    Cursor now(first, n);
    const uint32_t dh = step / n.all, du = step % n.all;
    if (n.whole) {
        RawUnit<T, INTERLEAVED> x[N];
        bool first_time = true;
        do {
            Cursor ahead = now;
#pragma unroll
            for (int k = 0; k < N; k++) {
                const bool live = ahead.head < heads;
                if (heads) load_unit<T, INTERLEAVED>(x[k], in(live ? ahead.head : 0), unit_place<INTERLEAVED>(live ? ahead.unit : 0, n, r), r);
                ahead.advance(dh, du, n);
            }
            if (first_time && !make_table()) return false;
            first_time = false;
            lanes_wrote();  // in every turn: behind the condition, the same statement costs 22 spilled scalars and 2% of a prompt
#pragma unroll
            for (int k = 0; k < N; k++) {
                if (now.head < heads) {
                    const UnitPlace p = unit_place<INTERLEAVED>(now.unit, n, r);
                    Unit y;
                    x[k].values(y);
                    turn_unit<INTERLEAVED, true>(y, p, r, table);
                    store_unit<T>(out(now.head), y, p, r);
                }
                now.advance(dh, du, n);
                __builtin_amdgcn_sched_barrier(0);  // one unit's angles and 64-bit values at a time
            }
        } while (__any(now.head < heads));
    } else {
        if (!make_table()) return false;
        lanes_wrote();
        for (; now.head < heads; now.advance(dh, du, n)) {
            const UnitPlace p = unit_place<INTERLEAVED>(now.unit, n, r);
            Unit x;
            load_unit_tail<T>(x, in(now.head), p, r, head_dim);
            turn_unit<INTERLEAVED, false>(x, p, r, table);
            store_unit_tail<T>(out(now.head), x, p, r, head_dim);
        }
    }
    return true;
}

// ---- rotation alone ----------------------------------------------------------------

struct RotateArgs {
    const void *x;
    void *out;
    const uint32_t *positions;
    uint64_t x_stride, out_stride;
    uint32_t heads, head_dim, parts;
    Rotation r;
};

// A wavefront takes a row, or some of its units.
template <class T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a, uint32_t rows) {
    extern __shared__ double2 tables[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), id = blockIdx.x * 4 + wave;
    const uint32_t row = id / a.parts, part = id % a.parts;
    if (row >= rows) return;
    double2 *const table = tables + wave * (a.r.dim / 2);
    const Angles angles(a.r);
    const HeadUnits n = head_units<INTERLEAVED>(a.r, a.head_dim);
    const T *const x = (const T *)a.x + row * a.x_stride;
    T *const out = (T *)a.out + row * a.out_stride;
    turn_heads<T, INTERLEAVED>(part * 64 + lane, a.parts * 64, a.heads, a.head_dim, n, a.r, table, [&](uint32_t h) { return x + (uint64_t)h * a.head_dim; },
                  [&](uint32_t h) { return out + (uint64_t)h * a.head_dim; }, [&] {
                      angles.table(a.r, a.positions[row], table);
                      return true;
                  });
}

// ---- appending -----------------------------------------------------------------------

struct AppendArgs {
    CacheBatch b;
    uint8_t *cache;
    const uint32_t *positions;
    const void *q, *k, *v;
    void *q_out;
    uint64_t q_stride, k_stride, v_stride, out_stride;
    uint32_t heads, parts, part_heads;  // part_heads: of the cache
    Rotation r;
};

// Eight values of a value's or key's word, quantised into their page.
template <uint32_t D>
__device__ __forceinline__ void append_word(uint8_t *head, uint32_t page_size, uint32_t t, uint32_t w, bool value, const float *x) {
    uint32_t scale;
    const uint32_t codes = cache_quantize(x, scale);
    if (!value) {
        *(GLOBAL uint32_t *)gp(head + cache_key_at(t, w, D)) = codes;
    } else if constexpr (D == 64) {  // a word is two pieces
        *(GLOBAL uint16_t *)gp(head + cache_value_at(page_size, t, 4 * w, D)) = (uint16_t)codes;
        *(GLOBAL uint16_t *)gp(head + cache_value_at(page_size, t, 4 * w + 2, D)) = (uint16_t)(codes >> 16);
    } else {
        *(GLOBAL uint32_t *)gp(head + cache_value_at(page_size, t, 4 * w, D)) = codes;
    }
    if (w % 4 == 0) *gp(head + (value ? cache_value_scale_at(page_size, t, w / 4, D) : cache_key_scale_at(page_size, t, w / 4, D))) = (uint8_t)scale;
}

// A wavefront takes a token, or some of its heads, and waits for no other.
constexpr uint32_t APPEND_VALUES = 1024;  // of keys in LDS per wavefront, at most

template <class T, uint32_t D, bool INTERLEAVED>
__global__ __launch_bounds__(256, 4) void append_kernel(AppendArgs a) {
    __shared__ double2 tables[4][D / 2];
    __shared__ __attribute__((aligned(16))) T all_keys[4][APPEND_VALUES];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), id = blockIdx.x * 4 + wave;
    double2 *const table = tables[wave];
    T *const keys = all_keys[wave];
    const uint32_t row = id / a.parts, part = id % a.parts;
    if (row >= a.b.rows) return;
    const HeadUnits n = head_units<INTERLEAVED>(a.r, D);
    const uint32_t h0 = part * a.part_heads, heads = min(a.part_heads, a.b.kv_heads - h0), group = a.q ? a.heads / a.b.kv_heads : 0;
    const T *const k = (const T *)a.k + row * a.k_stride + h0 * D, *const v = (const T *)a.v + row * a.v_stride + h0 * D;
    const T *const q = (const T *)a.q + row * a.q_stride + (uint64_t)h0 * group * D;
    T *const q_out = (T *)a.q_out + row * a.out_stride + (uint64_t)h0 * group * D;
    // A lane's first unit of a key and first two words of values go out with its queries' units, before the
    // row's place is looked up and the angles are computed.
    constexpr uint32_t WORDS = D / 8;
    Cursor c(lane, n);
    const Angles angles(a.r);
    RawUnit<T, INTERLEAVED> first_key;
    Eight<T> first_values[2];
    if (n.whole) load_unit<T, INTERLEAVED>(first_key, k + (c.head < heads ? c.head : 0) * D, unit_place<INTERLEAVED>(c.head < heads ? c.unit : 0, n, a.r), a.r);
#pragma unroll
    for (int i = 0; i < 2; i++) first_values[i].load(v + 8 * min(lane + 64 * i, heads * WORDS - 1));
    uint32_t page = 0xffffffffu, t = 0;
    const bool mine = turn_heads<T, INTERLEAVED>(lane, 64, heads * group, D, n, a.r, table, [&](uint32_t h) { return q + h * D; }, [&](uint32_t h) { return q_out + h * D; }, [&] {
        const CacheRow at_row = cache_row(a.b, row);
        const uint32_t s = at_row.sequence;
        const CacheSpan span = at_row.span;
        if (s >= a.b.sequences) return false;
        if (row - span.first >= span.rows) return false;
        const uint32_t back = span.rows - (row - span.first);  // the row's place from the end
        const bool token = span.length >= back;
        const uint32_t at = token ? span.length - back : 0;
        if (token) page = a.b.table[(uint64_t)s * a.b.table_stride + at / a.b.page_size];
        t = at % a.b.page_size;
        angles.table(a.r, a.positions ? a.positions[row] : at, table);
        return true;
    });
    if (!mine || page >= a.b.pages) return;
    for (bool first = true; c.head < heads; c.advance(64 / n.all, 64 % n.all, n), first = false) {
        const UnitPlace p = unit_place<INTERLEAVED>(c.unit, n, a.r);
        Unit x;
        if (n.whole) {
            if (!first) load_unit<T, INTERLEAVED>(first_key, k + c.head * D, p, a.r);
            first_key.values(x);
            turn_unit<INTERLEAVED, true>(x, p, a.r, table);
            Eight<T> y;
            y.round(x.a);
            T *const out = keys + c.head * D + p.first;
            *(Eight<T> *)out = y;
            if (p.pairs) {
                y.round(x.b);
                *(Eight<T> *)(out + a.r.dim / 2) = y;
            }
        } else {
            load_unit_tail<T>(x, k + c.head * D, p, a.r, D);
            turn_unit<INTERLEAVED, false>(x, p, a.r, table);
            store_unit_tail<T>(keys + c.head * D, x, p, a.r, D);
        }
    }
    lanes_wrote();  // the turned keys
    const uint32_t head_bytes = cache_head_bytes(a.b.page_size, D);
    uint8_t *const head = a.cache + ((uint64_t)page * a.b.kv_heads + h0) * head_bytes;
    // blocks of four words stay in four adjacent lanes
    for (uint32_t j = lane, i = 0; j < heads * WORDS; j += 64, i++) {
        float x[8];
        if (i < 2)
            first_values[i].values(x);
        else
            RowIO<T>::load8(v + 8 * j, x);
        append_word<D>(head + j / WORDS * head_bytes, a.b.page_size, t, j % WORDS, true, x);
    }
    for (uint32_t j = lane; j < heads * WORDS; j += 64) {
        float x[8];
        ((const Eight<T> *)(keys + 8 * j))->values(x);
        append_word<D>(head + j / WORDS * head_bytes, a.b.page_size, t, j % WORDS, false, x);
    }
}

// ---- reading back ----------------------------------------------------------------------

struct ReadArgs {
    CacheBatch b;
    const uint8_t *cache;
    void *k, *v;
    uint64_t k_stride, v_stride;
    uint32_t parts;
};

// A wavefront takes a token, or some of its heads.
template <class T, uint32_t D>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
    const uint32_t id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = id / a.parts;
    const uint32_t lane = id % a.parts * 64 + (threadIdx.x & 63), step = 64 * a.parts;
    if (row >= a.b.rows) return;
    const CacheRow at_row = cache_row(a.b, row);
    const uint32_t s = at_row.sequence;
    const CacheSpan span = at_row.span;
    if (s >= a.b.sequences) return;
    if (row - span.first >= span.rows) return;
    const uint32_t back = span.rows - (row - span.first);
    const bool token = span.length >= back;
    const uint32_t at = token ? span.length - back : 0, t = at % a.b.page_size;
    const uint32_t page = token ? a.b.table[(uint64_t)s * a.b.table_stride + at / a.b.page_size] : 0;
    const bool known = page < a.b.pages;
    const uint32_t head_bytes = cache_head_bytes(a.b.page_size, D);
    constexpr uint32_t WORDS = D / 8;
    T *const k = (T *)a.k + row * a.k_stride, *const v = (T *)a.v + row * a.v_stride;
    if (!token || !known) {  // no token: 0
        float x[8];
#pragma unroll
        for (int c = 0; c < 8; c++) x[c] = token ? __uint_as_float(0x7fc00000u) : 0.f;
        for (uint32_t i = lane; i < a.b.kv_heads * WORDS; i += step) {
            RowIO<T>::store8(k + 8 * i, x);
            RowIO<T>::store8(v + 8 * i, x);
        }
        return;
    }
#pragma unroll 2
    for (uint32_t i = lane; i < a.b.kv_heads * WORDS; i += step) {
        const uint32_t h = i / WORDS, w = i % WORDS;
        const gbytes head = (gbytes)gp(a.cache) + ((uint64_t)page * a.b.kv_heads + h) * head_bytes;
        const uint32_t key = *(const GLOBAL uint32_t *)(head + cache_key_at(t, w, D)), key_scale = head[cache_key_scale_at(a.b.page_size, t, w / 4, D)];
        uint32_t value;
        if constexpr (D == 64) {
            value = *(const GLOBAL uint16_t *)(head + cache_value_at(a.b.page_size, t, 4 * w, D));
            value |= (uint32_t)*(const GLOBAL uint16_t *)(head + cache_value_at(a.b.page_size, t, 4 * w + 2, D)) << 16;
        } else {
            value = *(const GLOBAL uint32_t *)(head + cache_value_at(a.b.page_size, t, 4 * w, D));
        }
        const uint32_t value_scale = head[cache_value_scale_at(a.b.page_size, t, w / 4, D)];
        float x[8];
        Eight<T> y;
        cache_dequantize(key, key_scale, x);
        y.round(x);
        y.stream(k + 8 * i);
        cache_dequantize(value, value_scale, x);
        y.round(x);
        y.stream(v + 8 * i);
    }
}

// ---- checks ------------------------------------------------------------------------------

static const char *pool_problem(const oco_cache *p) {
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return "head_dim is not 64, 128 or 256";
    if (p->kv_heads == 0 || p->kv_heads > 65535) return "kv_heads is not in 1 .. 65535";
    if (p->page_size == 0 || p->page_size % 16 || p->page_size > 65536) return "page_size is not a multiple of 16 up to 65536";
    return nullptr;
}
const char *cache_problem(const oco_cache *p) {
    if (const char *why = pool_problem(p)) return why;
    if (p->heads > 65535 || p->heads % p->kv_heads) return "heads is not a multiple of kv_heads under 65536";
    if (p->pages == 0) return "no pages";
    if ((uint64_t)p->max_length > (uint64_t)p->table_stride * p->page_size || p->max_length > 0x3fffffffu) return "max_length is past the table's pages";
    if (!(p->scale >= 0.f && p->scale < INFINITY)) return "the scale is not in 0 .. Inf";
    const uint64_t q = (uint64_t)p->heads * p->head_dim, kv = (uint64_t)p->kv_heads * p->head_dim;
    if ((p->q_stride && p->q_stride < q) || (p->out_stride && p->out_stride < q) || (p->k_stride && p->k_stride < kv) || (p->v_stride && p->v_stride < kv))
        return "a row stride under the row";
    return nullptr;
}

CacheBatch cache_batch(const oco_cache *p, const uint32_t *table, const uint32_t *starts, const uint32_t *lengths) {
    return CacheBatch{table, starts, lengths, p->sequences, p->rows, p->max_rows, p->max_length, p->table_stride, p->page_size, p->pages, p->kv_heads};
}

static const char *rotation_problem(const oco_rotation *r, uint32_t head_dim) {
    if (r->dim % 2 || r->dim > head_dim || r->dim > OCO_ROTATION_DIM) return "dim is odd or past the head";
    if (r->layout > OCO_ROTATION_INTERLEAVED) return "unknown layout";
    if (r->dim && !r->frequencies) return "no frequencies";
    return nullptr;
}
static Rotation rotation_of(const oco_rotation *r) {
    return r ? Rotation{r->frequencies, r->magnitude, r->dim} : Rotation{nullptr, 1.0, 0};
}

// What append and read share: 0 rows or a refusal end the call (done).
static int cache_call(const char *name, const oco_cache *p, const void *pages, const uint32_t *table, const uint32_t *starts,
                      const uint32_t *lengths, bool rest, bool *done) {
    *done = true;
    if (!p) return fail(OCO_ERR_INVALID, "%s: null description", name);
    if (const char *why = cache_problem(p)) return fail(OCO_ERR_INVALID, "%s: %s", name, why);
    if (p->dtype > OCO_DT_F16) return fail(OCO_ERR_UNSUPPORTED, "%s: type %u", name, p->dtype);
    if (p->rows == 0 || p->sequences == 0 || p->max_rows == 0) return OCO_OK;
    if (!pages || !table || !lengths || !rest) return fail(OCO_ERR_INVALID, "%s: null pointer", name);
    if ((uintptr_t)pages & 15u) return fail(OCO_ERR_INVALID, "%s: pages must be 16-byte aligned", name);
    if (!starts && p->rows % p->sequences)
        return fail(OCO_ERR_INVALID, "%s: %u rows of %u sequences without starts", name, p->rows, p->sequences);
    *done = false;
    return OCO_OK;
}

}  // namespace oco

using namespace oco;

extern "C" int oco_rotation_frequencies(const oco_frequencies *p, double *out, double *magnitude) {
    if (!p || !out) return fail(OCO_ERR_INVALID, "oco_rotation_frequencies: null pointer");
    if (p->dim % 2 || p->dim > OCO_ROTATION_DIM) return fail(OCO_ERR_INVALID, "oco_rotation_frequencies: dim %u is odd or past %u", p->dim, OCO_ROTATION_DIM);
    if (p->scaling > OCO_SCALING_BANDS) return fail(OCO_ERR_INVALID, "oco_rotation_frequencies: scaling %u", p->scaling);
    if (!(p->base > 1.0 && p->base < INFINITY)) return fail(OCO_ERR_INVALID, "oco_rotation_frequencies: the base is not past 1");
    const bool bands = p->scaling >= OCO_SCALING_YARN;
    if (p->scaling != OCO_SCALING_NONE && !(p->factor >= 1.0 && p->factor < INFINITY))
        return fail(OCO_ERR_INVALID, "oco_rotation_frequencies: the factor is under 1");
    if (bands && !(p->original >= 1.0 && p->original < INFINITY && p->slow > 0.0 && p->fast > p->slow && p->fast < INFINITY))
        return fail(OCO_ERR_INVALID, "oco_rotation_frequencies: original, fast and slow");
    const uint32_t n = p->dim / 2;
    const double pi = 3.14159265358979323846;
    // the pair that turns `turns` times over the original context, as a real number
    auto pair_of = [&](double turns) { return p->dim * log(p->original / (turns * 2.0 * pi)) / (2.0 * log(p->base)); };
    double low = 0.0, high = 0.0;
    if (p->scaling == OCO_SCALING_YARN) {
        low = fmax(floor(pair_of(p->fast)), 0.0);
        high = fmin(ceil(pair_of(p->slow)), p->dim - 1.0);
    }
    for (uint32_t j = 0; j < n; j++) {
        double f = pow(p->base, -2.0 * j / p->dim);
        if (p->factors) {
            if (!(p->factors[j] > 0.f && p->factors[j] < INFINITY)) return fail(OCO_ERR_INVALID, "oco_rotation_frequencies: factor of pair %u", j);
            f /= (double)p->factors[j];
        }
        if (p->scaling == OCO_SCALING_LINEAR) {
            f /= p->factor;
        } else if (bands) {
            // how far the pair is from `stays` (0) to `divided` (1)
            const double ramp = p->scaling == OCO_SCALING_YARN ? (j - low) / fmax(high - low, 0.001)
                                                               : (p->fast - p->original * f / (2.0 * pi)) / (p->fast - p->slow);
            const double r = fmin(fmax(ramp, 0.0), 1.0);
            f = f / p->factor * r + f * (1.0 - r);
        }
        out[j] = f;
    }
    if (magnitude) *magnitude = p->scaling == OCO_SCALING_YARN ? 0.1 * log(p->factor) + 1.0 : 1.0;
    return OCO_OK;
}

extern "C" int oco_rotate(const void *x, oco_dtype dtype, uint32_t rows, uint32_t heads, uint32_t head_dim, uint64_t x_stride,
                          const uint32_t *positions, void *out, uint64_t out_stride, const oco_rotation *rotation, oco_stream stream) {
    if (!rotation) return fail(OCO_ERR_INVALID, "oco_rotate: null rotation");
    if (const char *why = rotation_problem(rotation, head_dim)) return fail(OCO_ERR_INVALID, "oco_rotate: %s", why);
    if ((uint32_t)dtype > OCO_DT_F16) return fail(OCO_ERR_UNSUPPORTED, "oco_rotate: type %u", (uint32_t)dtype);
    const uint64_t width = (uint64_t)heads * head_dim;
    if ((x_stride && x_stride < width) || (out_stride && out_stride < width)) return fail(OCO_ERR_INVALID, "oco_rotate: a row stride under the row");
    if (width > 0x7fffffffull) return fail(OCO_ERR_INVALID, "oco_rotate: rows of %llu values", (unsigned long long)width);
    if (rows == 0 || width == 0) return OCO_OK;
    if (!x || !out || !positions) return fail(OCO_ERR_INVALID, "oco_rotate: null pointer");
    RotateArgs a;
    a.x = x;
    a.out = out;
    a.positions = positions;
    a.x_stride = x_stride ? x_stride : width;
    a.out_stride = out_stride ? out_stride : width;
    if (x == out && a.x_stride != a.out_stride) return fail(OCO_ERR_INVALID, "oco_rotate: in place with another stride");
    a.heads = heads;
    a.head_dim = head_dim;
    a.r = rotation_of(rotation);
    // few rows: their units over 1024 wavefronts, one per SIMD (one row of 32 heads 2.2 us, 3.5 by one; 512 rows 4.9, 5.2)
    a.parts = 1;
    while ((uint64_t)a.parts * 512 < width && (uint64_t)rows * a.parts < 1024) a.parts *= 2;
    if ((uint64_t)rows * a.parts > 0x7fffffffull) return fail(OCO_ERR_INVALID, "oco_rotate: %u rows", rows);
    const dim3 grid((rows * a.parts + 3) / 4);
    const uint32_t lds = 4 * (rotation->dim / 2) * sizeof(double2);
    hipStream_t st = (hipStream_t)stream;
#define GO(T)                                                                                                   \
    if (rotation->layout == OCO_ROTATION_INTERLEAVED)                                                           \
        hipLaunchKernelGGL((rotate_kernel<T, true>), grid, dim3(256), lds, st, a, rows);                        \
    else                                                                                                        \
        hipLaunchKernelGGL((rotate_kernel<T, false>), grid, dim3(256), lds, st, a, rows);                       \
    break;
    switch (dtype) {
    case OCO_DT_F32: GO(float)
    case OCO_DT_BF16: GO(bf16_t)
    default: GO(f16_t)
    }
#undef GO
    return launch_check("oco_rotate");
}

extern "C" uint64_t oco_cache_page_bytes(const oco_cache *p) {
    return p && !pool_problem(p) ? (uint64_t)cache_head_bytes(p->page_size, p->head_dim) * p->kv_heads : 0;
}

extern "C" int oco_cache_append(void *pages, const uint32_t *table, const uint32_t *starts, const uint32_t *lengths,
                                const uint32_t *positions, const void *q, const void *k, const void *v, void *q_out,
                                const oco_rotation *rotation, const oco_cache *p, oco_stream stream) {
    bool done;
    const int rc = cache_call("oco_cache_append", p, pages, table, starts, lengths, k && v && (!q || q_out), &done);
    if (done) return rc;
    if (rotation)
        if (const char *why = rotation_problem(rotation, p->head_dim)) return fail(OCO_ERR_INVALID, "oco_cache_append: %s", why);
    AppendArgs a;
    a.b = cache_batch(p, table, starts, lengths);
    a.cache = (uint8_t *)pages;
    a.positions = positions;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.q_stride = p->q_stride ? p->q_stride : (uint64_t)p->heads * p->head_dim;
    a.out_stride = p->out_stride ? p->out_stride : (uint64_t)p->heads * p->head_dim;
    a.k_stride = p->k_stride ? p->k_stride : (uint64_t)p->kv_heads * p->head_dim;
    a.v_stride = p->v_stride ? p->v_stride : (uint64_t)p->kv_heads * p->head_dim;
    if (q && q == q_out && a.q_stride != a.out_stride) return fail(OCO_ERR_INVALID, "oco_cache_append: queries in place with another stride");
    a.heads = p->heads;
    a.r = rotation_of(rotation);
    // few tokens: their heads over 1024 wavefronts, one per SIMD, down to one each, and halved under 2048 of them.  us:
    // 64 tokens of 8 heads 6.0, by one each 7.6; 512 appended and read back 10.1, 12.1, over 2048 10.5; 1500 12.9, 14.1; about
    // 1300 of 64 wide 13.0, 13.7, over 4096 16.1
    uint32_t parts = 1;
    a.part_heads = APPEND_VALUES / p->head_dim;
    while (a.part_heads > 1 && (uint64_t)p->rows * (parts = (p->kv_heads + a.part_heads - 1) / a.part_heads) < (parts == 1 ? 2048 : 1024)) a.part_heads /= 2;
    a.parts = (p->kv_heads + a.part_heads - 1) / a.part_heads;
    if ((uint64_t)p->rows * a.parts > 0x7fffffffull) return fail(OCO_ERR_INVALID, "oco_cache_append: %u rows", p->rows);
    const dim3 grid((uint32_t)(((uint64_t)p->rows * a.parts + 3) / 4));
    hipStream_t st = (hipStream_t)stream;
    const bool interleaved = rotation && rotation->layout == OCO_ROTATION_INTERLEAVED;
#define GO2(T, D)                                                                                               \
    if (interleaved)                                                                                            \
        hipLaunchKernelGGL((append_kernel<T, D, true>), grid, dim3(256), 0, st, a);                             \
    else                                                                                                        \
        hipLaunchKernelGGL((append_kernel<T, D, false>), grid, dim3(256), 0, st, a);                            \
    break;
#define GO(T)                                                                                                   \
    switch (p->head_dim) {                                                                                      \
    case 64: GO2(T, 64)                                                                                         \
    case 128: GO2(T, 128)                                                                                       \
    default: GO2(T, 256)                                                                                        \
    }                                                                                                           \
    break;
    switch (p->dtype) {
    case OCO_DT_F32: GO(float)
    case OCO_DT_BF16: GO(bf16_t)
    default: GO(f16_t)
    }
#undef GO
#undef GO2
    return launch_check("oco_cache_append");
}

extern "C" int oco_cache_read(const void *pages, const uint32_t *table, const uint32_t *starts, const uint32_t *lengths, void *k,
                              void *v, const oco_cache *p, oco_stream stream) {
    bool done;
    const int rc = cache_call("oco_cache_read", p, pages, table, starts, lengths, k && v, &done);
    if (done) return rc;
    ReadArgs a;
    a.b = cache_batch(p, table, starts, lengths);
    a.cache = (const uint8_t *)pages;
    a.k = k;
    a.v = v;
    a.k_stride = p->k_stride ? p->k_stride : (uint64_t)p->kv_heads * p->head_dim;
    a.v_stride = p->v_stride ? p->v_stride : (uint64_t)p->kv_heads * p->head_dim;
    a.parts = 1;
    while (a.parts * 64 < p->kv_heads * (p->head_dim / 8) && (uint64_t)p->rows * a.parts < 1024) a.parts *= 2;
    const dim3 grid((uint32_t)(((uint64_t)p->rows * a.parts + 3) / 4));
    hipStream_t st = (hipStream_t)stream;
#define GO(T)                                                                                               \
    switch (p->head_dim) {                                                                                  \
    case 64: hipLaunchKernelGGL((read_kernel<T, 64>), grid, dim3(256), 0, st, a); break;                    \
    case 128: hipLaunchKernelGGL((read_kernel<T, 128>), grid, dim3(256), 0, st, a); break;                  \
    default: hipLaunchKernelGGL((read_kernel<T, 256>), grid, dim3(256), 0, st, a);                          \
    }                                                                                                       \
    break;
    switch (p->dtype) {
    case OCO_DT_F32: GO(float)
    case OCO_DT_BF16: GO(bf16_t)
    default: GO(f16_t)
    }
#undef GO
    return launch_check("oco_cache_read");
}
