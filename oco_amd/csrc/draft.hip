// Verification of drafted tokens (speculative decoding): beside the greedy
// choice of argmax_f32, the choice of a whole run of tokens.
//
// With p_i the target's distribution after i drafted tokens and q_i the one
// the i-th draft d_i was drawn from (a lookup has none: all of it on d_i),
// d_i is accepted while u_i q_i(d_i) < p_i(d_i).  The first refused draft is
// replaced by a token drawn from max(p_i - q_i, 0), and if none is refused
// one more is drawn from the last p: the first token whose running sum
// passes u times the whole sum.  The result is then distributed as tokens
// drawn from the target one at a time.  Temperature 0 is greedy: p_i is all
// on the row's largest value (lowest index), and no random number is used.
//
// A decision must follow from the inputs and not from the order of sums or
// the rounding of exp: the two rows that a token is drawn from are 64-bit
// exponentials (7e-12) and 64-bit running sums.  The rows' normalising sums
// are f32 exponentials, sixteen added in f32 and the rest in 64 bits: their
// error, 1e-8 to 1e-7, shifts a whole row alike, and so a decision only where u
// is within that of its border.
//
// Bound by reading the rows once where they are logits: each chunk of each
// row gives its maximum and its sum of exponentials; the decisions follow
// from those, and only the two rows at the first refused draft are read
// again.  Rows of probabilities are read at the drafted tokens and there alone.
// 32 sequences of 7 drafts, 151936 f32 logits on both sides: rows 47 us (291 MB,
// 6.2 TB/s), decisions 4.7, what is left 15.5 (64-bit exponentials: bound by
// issue), token 8.7.  One sequence: three launches of 3.1, 6.2 and 6.2 us, all latency.
#include "exp64.h"
#include "rows.h"

namespace oco {

constexpr uint32_t DRAFT_CHUNK = 4096, DRAFT_RUN = 16;  // values per workgroup and row; per thread
constexpr uint32_t DRAFT_STEP = 1024, DRAFT_STEPS = DRAFT_CHUNK / DRAFT_STEP;  // what is left of a row: sums of 1024 values
constexpr uint32_t DRAFT_NONE = 0xffffffffu;

// A chunk's part of a row: its maximum (and where it first is), and the sum
// of exp((v - max) / T).  NaN in `sum`: the chunk holds a NaN or +Inf.
struct DraftPart {
    float max;
    uint32_t at;
    double sum;
};
struct DraftRest {  // a step's sums of max(p - q, 0) and of p
    double rest, all;
};
struct DraftState {  // the row that a token is drawn from
    double inv_p, inv_q;
    float max_p, max_q;
    uint32_t accepted, refused;
    uint32_t id, pad;  // the refused draft
};

struct DraftArgs {
    const void *target, *draft;
    const uint32_t *ids, *lengths;
    const float *u;
    uint32_t *accepted, *tokens;
    float *probabilities;
    DraftPart *parts;  // [sequences * (drafts + 1)][chunks], then [sequences * drafts][chunks]
    DraftRest *rests;  // [sequences][chunks * DRAFT_STEPS]
    DraftState *states;
    uint64_t target_stride, draft_stride;
    uint32_t sequences, drafts, vocabulary, chunks;
    uint32_t target_logits, draft_logits;  // what the rows hold
    double c;  // log2(e) / T
};

__device__ __forceinline__ uint32_t draft_length(const DraftArgs &a, uint32_t s) {
    return a.lengths ? min(a.lengths[s], a.drafts) : a.drafts;
}

// ---- parts of the rows of logits ---------------------------------------------------

template <class T, bool GREEDY>
__device__ void draft_part(const T *row, uint32_t chunk, const DraftArgs &a, DraftPart *out) {
    __shared__ float smax[4];
    __shared__ uint32_t sat[4];
    __shared__ double ssum[4];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float v[DRAFT_RUN];
#pragma unroll
    for (int h = 0; h < 2; h++) load_run(row, chunk * DRAFT_CHUNK + 2048 * h + 8 * threadIdx.x, a.vocabulary, v + 8 * h, -INFINITY);
    float m = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < (int)DRAFT_RUN; j++) {
        bad |= !(v[j] < INFINITY);
        m = fmaxf(m, v[j]);
    }
    m = wave_max_f32(m);
    if (lane == 0) smax[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3]));
    uint32_t at = DRAFT_NONE;
    double s = 0.0;
    if constexpr (GREEDY) {
#pragma unroll
        for (int j = DRAFT_RUN - 1; j >= 0; j--)
            if (v[j] == m) at = chunk * DRAFT_CHUNK + 2048 * (j / 8) + 8 * threadIdx.x + j % 8;
        at = wave_min_u32(at);
        s = bad ? __builtin_nan("") : 0.0;
    } else {
        // c in two parts: its rounding would shift every term of a row the same way
        const float c = (float)a.c, rest = (float)(a.c - (double)c);
#pragma unroll
        for (int j = 0; j < (int)DRAFT_RUN; j++) {
            const float d = fmaxf(v[j] - m, -1e30f);  // -Inf: an exponential of 0, without -Inf * rest
            v[j] = __builtin_amdgcn_exp2f(fmaf(d, rest, d * c));
        }
#pragma unroll
        for (int w = DRAFT_RUN / 2; w; w /= 2)
#pragma unroll
            for (int j = 0; j < w; j++) v[j] += v[j + w];
        s = bad ? __builtin_nan("") : m > -INFINITY ? (double)v[0] : 0.0;  // a chunk of -Inf alone has sum 0
    }
    s = wave_sum_f64(s);
    if (lane == 0) {
        sat[wave] = at;
        ssum[wave] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        out->max = m;
        out->at = min(min(sat[0], sat[1]), min(sat[2], sat[3]));
        out->sum = ((ssum[0] + ssum[1]) + ssum[2]) + ssum[3];
    }
}

// One workgroup per (row, chunk): the target's rows, then the drafter's.
template <class TT, class TD, bool GREEDY>
__global__ __launch_bounds__(256) void draft_parts_kernel(DraftArgs a, uint32_t target_rows) {
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    if (row < target_rows) {
        const uint32_t s = row / (a.drafts + 1), i = row % (a.drafts + 1);
        if (i > draft_length(a, s)) return;
        draft_part<TT, GREEDY>((const TT *)a.target + row * a.target_stride, chunk, a, a.parts + (uint64_t)row * a.chunks + chunk);
    } else {
        const uint32_t r = row - target_rows, s = r / a.drafts, i = r % a.drafts;
        if (i >= draft_length(a, s)) return;
        DraftPart *parts = a.parts + (uint64_t)a.sequences * (a.drafts + 1) * a.chunks;
        draft_part<TD, false>((const TD *)a.draft + r * a.draft_stride, chunk, a, parts + (uint64_t)r * a.chunks + chunk);
    }
}

// ---- decisions ---------------------------------------------------------------------

struct DraftRow {
    float max;
    double inv;  // 1 / sum of exp((v - max) / T); NaN for a row without a distribution
    uint32_t at;
};
// A row from its parts, by one wavefront; `first`: the lane's part of the first 64.
__device__ __forceinline__ DraftRow draft_row(const DraftPart *parts, const DraftPart &first, const DraftArgs &a) {
    const uint32_t lane = threadIdx.x & 63;
    float m = first.max;
    for (uint32_t i = 64 + lane; i < a.chunks; i += 64) m = fmaxf(m, parts[i].max);
    m = wave_max_f32(m);
    // a NaN or +Inf in the row stays a NaN sum
    auto scaled = [&](const DraftPart &p) { return p.sum * (p.max > -INFINITY ? exp2_f64<9>(((double)p.max - (double)m) * a.c) : 1.0); };
    double s = scaled(first);
    uint32_t at = first.max == m ? first.at : DRAFT_NONE;
    for (uint32_t i = 64 + lane; i < a.chunks; i += 64) {
        const DraftPart p = parts[i];
        if (p.max == m) at = min(at, p.at);
        s += scaled(p);
    }
    s = wave_sum_f64(s);
    DraftRow r;
    r.max = m;
    r.inv = m > -INFINITY ? 1.0 / s : __builtin_nan("");
    r.at = wave_min_u32(at);
    return r;
}
__device__ __forceinline__ DraftPart draft_first(const DraftPart *parts, const DraftArgs &a) {
    const uint32_t lane = threadIdx.x & 63;
    DraftPart p = {-INFINITY, DRAFT_NONE, 0.0};
    if (lane < a.chunks) p = parts[lane];
    return p;
}

// A probability as it counts: 0 for a value under 0 (a NaN stays).
__device__ __forceinline__ double draft_probability(float v) { return v < 0.f ? 0.0 : (double)v; }
__device__ __forceinline__ double draft_value(float v, bool logits, float max, double inv, double c) {
    return logits ? exp2_f64<9>(((double)v - (double)max) * c) * inv : draft_probability(v);
}

template <class TT, class TD>
struct DraftRows {
    const DraftArgs &a;
    uint32_t s;
    __device__ const TT *target(uint32_t i) const { return (const TT *)a.target + ((uint64_t)s * (a.drafts + 1) + i) * a.target_stride; }
    __device__ const TD *draft(uint32_t i) const { return (const TD *)a.draft + ((uint64_t)s * a.drafts + i) * a.draft_stride; }
    __device__ const DraftPart *target_parts(uint32_t i) const { return a.parts + ((uint64_t)s * (a.drafts + 1) + i) * a.chunks; }
    __device__ const DraftPart *draft_parts(uint32_t i) const {
        return a.parts + ((uint64_t)a.sequences * (a.drafts + 1) + (uint64_t)s * a.drafts + i) * a.chunks;
    }
};

constexpr uint32_t DRAFT_MOST = OCO_DRAFT_MAX;

// Greedy: one workgroup per sequence, from the rows' first maxima.
__global__ __launch_bounds__(256) void draft_greedy_kernel(DraftArgs a) {
    __shared__ uint32_t best[DRAFT_MOST + 1];
    const uint32_t s = blockIdx.x, wave = threadIdx.x >> 6, length = draft_length(a, s);
    const DraftRows<float, float> rows{a, s};
    for (uint32_t i = wave; i <= length; i += 4) {
        const DraftRow r = draft_row(rows.target_parts(i), draft_first(rows.target_parts(i), a), a);
        if ((threadIdx.x & 63) == 0) best[i] = r.inv == r.inv && (a.target_logits || r.max > 0.f) ? r.at : DRAFT_NONE;
    }
    __syncthreads();
    uint32_t n = 0;  // drafts that are their row's first maximum, from the front
    while (n < length && best[n] != DRAFT_NONE && a.ids[(uint64_t)s * a.drafts + n] == best[n]) n++;
    if (threadIdx.x == 0) a.accepted[s] = n;
    for (uint32_t i = threadIdx.x; i <= a.drafts; i += 256) {
        const uint32_t token = i <= n ? best[i] : DRAFT_NONE;
        a.tokens[(uint64_t)s * (a.drafts + 1) + i] = token;
        if (a.probabilities)
            a.probabilities[(uint64_t)s * (a.drafts + 1) + i] = i > n ? 0.f : token == DRAFT_NONE ? __uint_as_float(0x7fc00000u) : 1.f;
    }
}

// What the token is drawn from at four places: x = p, and d = max(p - q, 0)
// (minus: p - q, else p).  NaN stays.
template <class TT, class TD>
__device__ __forceinline__ void draft_left(const DraftArgs &a, const DraftRows<TT, TD> &rows, const DraftState &st, bool minus, uint32_t c0,
                                           float *pv, double *x, double *d) {
    float qv[4];
    load_four(rows.target(st.accepted), c0, a.vocabulary, pv, a.target_logits ? -INFINITY : 0.f);
    if (minus && a.draft) load_four(rows.draft(st.accepted), c0, a.vocabulary, qv, a.draft_logits ? -INFINITY : 0.f);
    // both rows' exponentials side by side
    double at[8], e[8], y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        at[j] = ((double)pv[j] - (double)st.max_p) * a.c;
        at[4 + j] = minus && a.draft ? ((double)qv[j] - (double)st.max_q) * a.c : 0.0;
    }
    if (minus && a.draft)
        exp2_clamped<9, 8>(at, e);
    else
        exp2_clamped<9, 4>(at, e);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        x[j] = a.target_logits ? (at[j] < -1000.0 ? 0.0 : e[j]) * st.inv_p : draft_probability(pv[j]);
        y[j] = 0.0;
        if (minus) {
            if (a.draft)
                y[j] = a.draft_logits ? (at[4 + j] < -1000.0 ? 0.0 : e[4 + j]) * st.inv_q : draft_probability(qv[j]);
            else
                y[j] = c0 + j == st.id ? 1.0 : 0.0;
        }
        const double left = x[j] - y[j];
        d[j] = left <= 0.0 ? left * 0.0 : left;  // an infinite q: NaN
    }
}

// The decisions of a sequence, by 1024 threads: a wavefront per row, then a
// thread per draft.  `write`: this workgroup stores them.
template <class TT, class TD>
__device__ __forceinline__ DraftState draft_decide(const DraftArgs &a, uint32_t s, bool write) {
    __shared__ DraftRow row_of[2 * DRAFT_MOST + 1];  // the target's rows, then the drafter's
    __shared__ uint32_t good[DRAFT_MOST], refused_id;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, length = draft_length(a, s), i = threadIdx.x;
    const DraftRows<TT, TD> rows{a, s};
    // thread i: the drafted token i
    uint32_t id = DRAFT_NONE;
    float u = 0.f, pd = 0.f, qd = 0.f;
    if (i < length) {
        id = a.ids[(uint64_t)s * a.drafts + i];
        u = a.u[(uint64_t)s * (a.drafts + 1) + i];
        if (id < a.vocabulary) {
            pd = RowIO<TT>::one(rows.target(i) + id);
            if (a.draft) qd = RowIO<TD>::one(rows.draft(i) + id);
        }
    }
    const uint32_t first = a.target_logits ? 0 : length + 1, last = a.draft && a.draft_logits ? 2 * length + 1 : length + 1;
#pragma unroll 1
    for (uint32_t r = first + wave; r < last; r += 16) {
        const DraftPart *const parts = r <= length ? rows.target_parts(r) : rows.draft_parts(r - length - 1);
        const DraftRow row = draft_row(parts, draft_first(parts, a), a);
        if (lane == 0) row_of[r] = row;
    }
    __syncthreads();
    if (i < length) {
        const DraftRow p = row_of[i], q = row_of[length + 1 + i];
        // an id past the vocabulary has no probability; without a draft's distribution q is 1
        const double pr = id < a.vocabulary ? draft_value(pd, a.target_logits, p.max, p.inv, a.c) : 0.0;
        const double qr = id < a.vocabulary && a.draft ? draft_value(qd, a.draft_logits, q.max, q.inv, a.c) : 1.0;
        good[i] = (double)u * qr < pr && pr < __builtin_inf();
        pd = (float)pr;
    }
    __syncthreads();
    const uint64_t refusals = ~__ballot(lane < length && good[lane]);
    const uint32_t n = min(length, refusals ? (uint32_t)__builtin_ctzll(refusals) : 64u);
    if (i == n && n < length) refused_id = id;
    __syncthreads();
    const DraftRow &q = row_of[min(length + 1 + n, 2 * length)];
    DraftState st;
    st.accepted = n;
    st.refused = n < length;
    st.id = n < length ? refused_id : DRAFT_NONE;
    st.pad = 0;
    st.max_p = row_of[n].max;
    st.inv_p = row_of[n].inv;
    st.max_q = q.max;
    st.inv_q = q.inv;
    if (write) {
        if (i == 0) {
            a.states[s] = st;
            a.accepted[s] = n;
        }
        if (i <= a.drafts && i != n) {  // at n: the token that is drawn next
            const uint64_t at = (uint64_t)s * (a.drafts + 1) + i;
            a.tokens[at] = i < n ? id : DRAFT_NONE;
            if (a.probabilities) a.probabilities[at] = i < n ? pd : 0.f;
        }
    }
    return st;
}

template <class TT, class TD>
__global__ __launch_bounds__(1024) void draft_decide_kernel(DraftArgs a) {
    draft_decide<TT, TD>(a, blockIdx.x, true);
}

// What is left of the target at the first refused draft, in steps of 1024
// values: four wavefronts with four values per thread.  FUSED: one workgroup
// per (sequence, chunk of four steps), each of which makes its sequence's
// decisions itself; bound by latency, and one launch less.  Else one workgroup per
// (sequence, step), from decisions that are there.
template <class TT, class TD, bool FUSED>
__global__ __launch_bounds__(FUSED ? 1024 : 256) void draft_rest_kernel(DraftArgs a) {
    constexpr uint32_t STEPS = FUSED ? DRAFT_STEPS : 1;
    __shared__ double sums[2][4 * STEPS];
    const uint32_t per = FUSED ? a.chunks : a.chunks * DRAFT_STEPS, s = blockIdx.x / per, part = blockIdx.x % per;
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const DraftRows<TT, TD> rows{a, s};
    DraftState st;
    if constexpr (FUSED)
        st = draft_decide<TT, TD>(a, s, part == 0);
    else
        st = a.states[s];
    float pv[4];
    double x[4], d[4];
    draft_left(a, rows, st, st.refused != 0, part * STEPS * DRAFT_STEP + 4 * threadIdx.x, pv, x, d);
    const double rest = wave_sum_f64((d[0] + d[1]) + (d[2] + d[3])), all = wave_sum_f64((x[0] + x[1]) + (x[2] + x[3]));
    if (lane == 0) {
        sums[0][wave] = rest;
        sums[1][wave] = all;
    }
    __syncthreads();
    if (threadIdx.x < STEPS) {
        const double *const r = sums[0] + 4 * threadIdx.x, *const t = sums[1] + 4 * threadIdx.x;
        a.rests[((uint64_t)s * per + part) * STEPS + threadIdx.x] = DraftRest{((r[0] + r[1]) + r[2]) + r[3], ((t[0] + t[1]) + t[2]) + t[3]};
    }
}

// One workgroup per sequence: the step of 1024 values, then the token in it,
// where the running sum passes u times the whole.
template <class TT, class TD>
__global__ __launch_bounds__(256) void draft_token_kernel(DraftArgs a) {
    __shared__ double sat_before, mark_of, swave[4];
    __shared__ uint32_t sat[3], from_rest;
    const uint32_t s = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, steps = a.chunks * DRAFT_STEPS;
    const DraftRest *rests = a.rests + (uint64_t)s * steps;
    const DraftState st = a.states[s];
    const uint32_t n = st.accepted;
    const double u = (double)a.u[(uint64_t)s * (a.drafts + 1) + a.drafts];
    if (wave == 0) {
        double rest = 0.0, all = 0.0;
        constexpr int HELD = 4;  // steps per lane that are read once
        DraftRest held[HELD];
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            held[h] = DraftRest{0.0, 0.0};
            if (64 * h + lane < steps) held[h] = rests[64 * h + lane];
        }
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            rest += held[h].rest;
            all += held[h].all;
        }
        for (uint32_t i = 64 * HELD + lane; i < steps; i += 64) {
            rest += rests[i].rest;
            all += rests[i].all;
        }
        rest = wave_sum_f64(rest);
        all = wave_sum_f64(all);
        const bool left = !(rest <= 0.0);  // nothing left (p == q): draw from p
        const double whole = left ? rest : all, mark = u * whole;
        // the first step whose running sum passes the mark, or the last one that holds anything
        double before = 0.0, at_before = 0.0;
        uint32_t found = DRAFT_NONE;
        bool passed = false;
#pragma unroll 1
        for (uint32_t base = 0; base < steps && !passed; base += 64) {
            const uint32_t i = base + lane;
            DraftRest r = {0.0, 0.0};
            if (base >= 64 * HELD) {
                if (i < steps) r = rests[i];
            } else {
#pragma unroll
                for (int h = 0; h < HELD; h++)
                    if (base == 64u * h) r = held[h];
            }
            const double w = left ? r.rest : r.all;
            const double sum = before + wave_scan_f64(w);
            const uint64_t pass = __ballot(sum > mark && w > 0.0), some = __ballot(w > 0.0);
            passed = pass != 0;
            if (some) {
                const int l = passed ? __builtin_ctzll(pass) : 63 - __builtin_clzll(some);
                found = base + l;
                at_before = lane_f64(sum, l) - lane_f64(w, l);
            }
            before = lane_f64(sum, 63);
        }
        if (lane == 0) {
            sat[0] = whole > 0.0 && whole < __builtin_inf() ? found : DRAFT_NONE;
            sat[1] = DRAFT_NONE;
            sat[2] = 0;
            sat_before = at_before;
            mark_of = mark;
            from_rest = left;
        }
    }
    __syncthreads();
    const uint32_t step = sat[0];
    const uint64_t out = (uint64_t)s * (a.drafts + 1) + n;
    if (step == DRAFT_NONE) {  // no distribution: a NaN, an infinity, or nothing but zeros
        if (threadIdx.x == 0) {
            a.tokens[out] = DRAFT_NONE;
            if (a.probabilities) a.probabilities[out] = __uint_as_float(0x7fc00000u);
        }
        return;
    }
    const DraftRows<TT, TD> rows{a, s};
    const bool left = from_rest != 0;
    const uint32_t c0 = step * DRAFT_STEP + 4 * threadIdx.x;
    float pv[4];
    double x[4], d[4];
    draft_left(a, rows, st, st.refused && left, c0, pv, x, d);
    const double sum = (d[0] + d[1]) + (d[2] + d[3]), scan = wave_scan_f64(sum);
    if (lane == 63) swave[wave] = scan;
    __syncthreads();
    double before = sat_before;
#pragma unroll
    for (uint32_t w = 0; w < 3; w++) before += w < wave ? swave[w] : 0.0;
    before += scan - sum;
    uint32_t first = DRAFT_NONE, last = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        before += d[j];
        if (d[j] > 0.0) {
            if (before > mark_of && first == DRAFT_NONE) first = c0 + j;
            last = c0 + j + 1;
        }
    }
    if (first != DRAFT_NONE) atomicMin(&sat[1], first);
    if (last) atomicMax(&sat[2], last);
    __syncthreads();
    const uint32_t token = sat[1] != DRAFT_NONE ? sat[1] : sat[2] - 1;
    if (token - c0 < 4) {  // the thread that holds it
        a.tokens[out] = token;
        if (a.probabilities) {
            double p = 0.0;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (token - c0 == (uint32_t)j) p = a.target_logits ? x[j] : (double)pv[j];
            a.probabilities[out] = (float)p;
        }
    }
}

struct DraftLayout {
    uint32_t chunks;
    uint64_t parts, rests, states, bytes;
};
static DraftLayout draft_layout(const oco_draft *p) {
    DraftLayout l;
    const uint64_t s = p->sequences;
    l.chunks = (uint32_t)(((uint64_t)p->vocabulary + DRAFT_CHUNK - 1) / DRAFT_CHUNK);
    l.parts = s * (2 * (uint64_t)p->drafts + 1) * l.chunks * sizeof(DraftPart);
    l.rests = s * l.chunks * DRAFT_STEPS * sizeof(DraftRest);
    l.states = s * sizeof(DraftState);
    l.bytes = l.parts + l.rests + l.states;
    return l;
}

template <class TT, class TD>
static int draft_launch(const DraftArgs &a, bool greedy, hipStream_t stream) {
    const uint64_t target_rows = greedy || a.target_logits ? (uint64_t)a.sequences * (a.drafts + 1) : 0;
    const uint64_t draft_rows = !greedy && a.draft && a.draft_logits ? (uint64_t)a.sequences * a.drafts : 0;
    if (target_rows + draft_rows) {
        const dim3 grid((uint32_t)((target_rows + draft_rows) * a.chunks));
        if (greedy)
            hipLaunchKernelGGL((draft_parts_kernel<TT, TD, true>), grid, dim3(256), 0, stream, a, (uint32_t)target_rows);
        else
            hipLaunchKernelGGL((draft_parts_kernel<TT, TD, false>), grid, dim3(256), 0, stream, a, (uint32_t)target_rows);
        OCO_TRY(launch_check("oco_draft_verify (rows)"));
    }
    if (greedy) {
        hipLaunchKernelGGL(draft_greedy_kernel, dim3(a.sequences), dim3(256), 0, stream, a);
        return launch_check("oco_draft_verify (greedy)");
    }
    // Decisions in every workgroup while they all run at once (one of 1024 threads per compute unit: its registers
    // leave six of the eight wavefronts per SIMD that two would need), in a launch of their own beyond.  The whole
    // call, logits on both sides, 7 drafts, 151936 tokens: 6 sequences (228 workgroups) 25.6 us against 27.4, 7 (266)
    // 30.9 against 29.3, 10 (380) 35.2 against 33.5; 8 and 11 lookups of 100003 bf16 logits (200, 275) 17.6 against
    // 20.8 and 22.3 against 21.6.
    if ((uint64_t)a.sequences * a.chunks <= 256) {
        hipLaunchKernelGGL((draft_rest_kernel<TT, TD, true>), dim3(a.sequences * a.chunks), dim3(1024), 0, stream, a);
    } else {
        hipLaunchKernelGGL((draft_decide_kernel<TT, TD>), dim3(a.sequences), dim3(1024), 0, stream, a);
        OCO_TRY(launch_check("oco_draft_verify (decisions)"));
        hipLaunchKernelGGL((draft_rest_kernel<TT, TD, false>), dim3(a.sequences * a.chunks * DRAFT_STEPS), dim3(256), 0, stream, a);
    }
    OCO_TRY(launch_check("oco_draft_verify (rest)"));
    hipLaunchKernelGGL((draft_token_kernel<TT, TD>), dim3(a.sequences), dim3(256), 0, stream, a);
    return launch_check("oco_draft_verify (token)");
}

static const char *draft_problem(const oco_draft *p) {
    if (p->drafts > OCO_DRAFT_MAX) return "too many drafts per sequence";
    if (p->vocabulary == 0 || p->vocabulary >= 0x80000000u) return "the vocabulary is empty or past 2^31";
    if (p->target_values > OCO_DRAFT_PROBABILITIES || p->draft_values > OCO_DRAFT_PROBABILITIES) return "unknown kind of values";
    if (p->target_dtype > OCO_DT_F16 || p->draft_dtype > OCO_DT_F16) return "unknown type";
    // the exponents' factor log2(e) / T and its remainder are f32, and -1e30 of it is an exponential of 0
    if (p->temperature != 0.f && !(p->temperature >= 0x1p-126f && p->temperature <= 0x1p64f))
        return "the temperature is neither 0 nor in 2^-126 .. 2^64";
    if ((p->target_stride && p->target_stride < p->vocabulary) || (p->draft_stride && p->draft_stride < p->vocabulary))
        return "a row stride under the vocabulary";
    const DraftLayout l = draft_layout(p);
    if ((uint64_t)p->sequences * (2ull * p->drafts + DRAFT_STEPS) * l.chunks > 0x7fffffffull) return "too many rows for one call";
    return nullptr;
}

}  // namespace oco

using namespace oco;

extern "C" uint64_t oco_draft_verify_workspace(const oco_draft *p) {
    return p && !draft_problem(p) ? draft_layout(p).bytes : 0;
}

extern "C" int oco_draft_verify(const void *target, const void *draft, const uint32_t *draft_ids, const uint32_t *lengths,
                                const float *uniforms, uint32_t *accepted, uint32_t *tokens, float *probabilities,
                                const oco_draft *p, void *workspace, uint64_t workspace_bytes, oco_stream stream) {
    if (!p) return fail(OCO_ERR_INVALID, "oco_draft_verify: null description");
    if (const char *why = draft_problem(p)) return fail(OCO_ERR_INVALID, "oco_draft_verify: %s", why);
    if (p->sequences == 0) return OCO_OK;
    const bool greedy = p->temperature == 0.f;
    if (!target || !accepted || !tokens || (p->drafts && !draft_ids) || (!greedy && !uniforms))
        return fail(OCO_ERR_INVALID, "oco_draft_verify: null pointer");
    // the first sequences' outputs are there before the last ones' inputs are read
    const uint64_t counts = (uint64_t)p->sequences * 4, places = counts * (p->drafts + 1);
    const void *const in[3] = {draft_ids, lengths, greedy ? nullptr : uniforms}, *const out[3] = {accepted, tokens, probabilities};
    const uint64_t in_bytes[3] = {counts * p->drafts, counts, places}, out_bytes[3] = {counts, places, places};
    for (int i = 0; i < 3; i++)
        for (int o = 0; o < 3; o++)
            if (in[i] && out[o] && (uintptr_t)in[i] < (uintptr_t)out[o] + out_bytes[o] && (uintptr_t)out[o] < (uintptr_t)in[i] + in_bytes[i])
                return fail(OCO_ERR_INVALID, "oco_draft_verify: an output lies over the drafted ids, the lengths or the random numbers");
    const DraftLayout l = draft_layout(p);
    if (!workspace || ((uintptr_t)workspace & 15u) || workspace_bytes < l.bytes)
        return fail(OCO_ERR_INVALID, "oco_draft_verify: workspace of %llu bytes, need %llu, 16-byte aligned",
                    (unsigned long long)workspace_bytes, (unsigned long long)l.bytes);
    DraftArgs a;
    a.target = target;
    a.draft = greedy ? nullptr : draft;
    a.ids = draft_ids;
    a.lengths = lengths;
    a.u = uniforms;
    a.accepted = accepted;
    a.tokens = tokens;
    a.probabilities = probabilities;
    a.parts = (DraftPart *)workspace;
    a.rests = (DraftRest *)((uint8_t *)workspace + l.parts);
    a.states = (DraftState *)((uint8_t *)workspace + l.parts + l.rests);
    a.target_stride = p->target_stride ? p->target_stride : p->vocabulary;
    a.draft_stride = p->draft_stride ? p->draft_stride : p->vocabulary;
    a.sequences = p->sequences;
    a.drafts = p->drafts;
    a.vocabulary = p->vocabulary;
    a.chunks = l.chunks;
    a.target_logits = p->target_values == OCO_DRAFT_LOGITS;
    a.draft_logits = p->draft_values == OCO_DRAFT_LOGITS;
    a.c = greedy ? 1.0 : 1.4426950408889634074 / (double)p->temperature;
    hipStream_t st = (hipStream_t)stream;
    const uint32_t td = a.draft ? p->draft_dtype : p->target_dtype;
#define GO(TT)                                                       \
    switch (td) {                                                    \
    case OCO_DT_F32: return draft_launch<TT, float>(a, greedy, st);  \
    case OCO_DT_BF16: return draft_launch<TT, bf16_t>(a, greedy, st); \
    default: return draft_launch<TT, f16_t>(a, greedy, st);          \
    }
    switch (p->target_dtype) {
    case OCO_DT_F32: GO(float)
    case OCO_DT_BF16: GO(bf16_t)
    default: GO(f16_t)
    }
#undef GO
}
