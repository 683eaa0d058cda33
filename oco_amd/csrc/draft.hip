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
// are f32 exponentials added in 64 bits: their error, some 1e-8, shifts a
// whole row alike, and so a decision only where u is within that of its border.
//
// Bound by reading the rows once where they are logits: each chunk of each
// row gives its maximum and its sum of exponentials; the decisions follow
// from those, and only the two rows at the first refused draft are read
// again.  Rows of probabilities are read at the drafted tokens and there alone.
#include "exp64.h"
#include "rows.h"

namespace oco {

constexpr uint32_t DRAFT_CHUNK = 4096, DRAFT_RUN = 16;  // values per workgroup and row; per thread
constexpr uint32_t DRAFT_NONE = 0xffffffffu;

// A chunk's part of a row: its maximum (and where it first is), and the sum
// of exp((v - max) / T).  NaN in `sum`: the chunk holds a NaN or +Inf.
struct DraftPart {
    float max;
    uint32_t at;
    double sum;
};
struct DraftRest {  // a chunk's sums of max(p - q, 0) and of p
    double rest, all;
};
struct DraftState {  // the row that a token is drawn from
    double inv_p, inv_q;
    float max_p, max_q;
    uint32_t accepted, refused;
};

struct DraftArgs {
    const void *target, *draft;
    const uint32_t *ids, *lengths;
    const float *u;
    uint32_t *accepted, *tokens;
    float *probabilities;
    DraftPart *parts;  // [sequences * (drafts + 1)][chunks], then [sequences * drafts][chunks]
    DraftRest *rests;  // [sequences][chunks]
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

__device__ __forceinline__ double draft_value(float v, bool logits, float max, double inv, double c) {
    return logits ? exp2_f64<9>(((double)v - (double)max) * c) * inv : (double)v;
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
        if ((threadIdx.x & 63) == 0) best[i] = r.inv == r.inv ? r.at : DRAFT_NONE;
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

// One workgroup per (sequence, chunk): every workgroup of a sequence makes
// its decisions from the rows' parts, then sums its chunk of what is left of
// the target at the first refused draft.
template <class TT, class TD>
__global__ __launch_bounds__(256) void draft_rest_kernel(DraftArgs a) {
    __shared__ DraftRow prow[DRAFT_MOST + 1], qrow[DRAFT_MOST + 1];
    __shared__ float pid[DRAFT_MOST + 1];
    __shared__ uint32_t good[DRAFT_MOST + 1];
    __shared__ double sums[2][4];
    const uint32_t s = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t length = draft_length(a, s);
    const DraftRows<TT, TD> rows{a, s};
    const bool with_q = a.draft && a.draft_logits;
    constexpr int AT_ONCE = 2;  // positions whose loads a wavefront has in flight together
    for (uint32_t base = wave; base <= length; base += 4 * AT_ONCE) {
        DraftPart pp[AT_ONCE], qp[AT_ONCE];
        float pd[AT_ONCE], qd[AT_ONCE], u[AT_ONCE];
        bool known[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) {
            const uint32_t i = base + 4 * j;
            pp[j] = qp[j] = DraftPart{-INFINITY, DRAFT_NONE, 0.0};
            pd[j] = qd[j] = u[j] = 0.f;
            known[j] = false;
            if (i <= length && a.target_logits) pp[j] = draft_first(rows.target_parts(i), a);
            if (i < length) {
                if (with_q) qp[j] = draft_first(rows.draft_parts(i), a);
                const uint32_t id = a.ids[(uint64_t)s * a.drafts + i];
                u[j] = a.u[(uint64_t)s * (a.drafts + 1) + i];
                known[j] = id < a.vocabulary;
                if (known[j]) {
                    pd[j] = RowIO<TT>::one(rows.target(i) + id);
                    if (a.draft) qd[j] = RowIO<TD>::one(rows.draft(i) + id);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) {
            const uint32_t i = base + 4 * j;
            if (i > length) break;
            DraftRow p = {0.f, 1.0, 0}, q = {0.f, 1.0, 0};
            if (a.target_logits) p = draft_row(rows.target_parts(i), pp[j], a);
            if (i < length && with_q) q = draft_row(rows.draft_parts(i), qp[j], a);
            // an id past the vocabulary has no probability
            const double pr = known[j] ? draft_value(pd[j], a.target_logits, p.max, p.inv, a.c) : 0.0;
            const double qr = known[j] && a.draft ? draft_value(qd[j], a.draft_logits, q.max, q.inv, a.c) : 1.0;
            if (lane == 0) {
                prow[i] = p;
                qrow[i] = q;
                pid[i] = (float)pr;
                good[i] = (double)u[j] * qr < pr;
            }
        }
    }
    __syncthreads();
    uint32_t n = 0;
    while (n < length && good[n]) n++;
    const bool refused = n < length;
    const DraftRow p = prow[n], q = qrow[n];
    const uint32_t id = refused ? a.ids[(uint64_t)s * a.drafts + n] : DRAFT_NONE;

    float pv[DRAFT_RUN], qv[DRAFT_RUN];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t c0 = chunk * DRAFT_CHUNK + DRAFT_RUN * threadIdx.x + 8 * h;
        load_run(rows.target(n), c0, a.vocabulary, pv + 8 * h, a.target_logits ? -INFINITY : 0.f);
        if (refused && a.draft) load_run(rows.draft(n), c0, a.vocabulary, qv + 8 * h, a.draft_logits ? -INFINITY : 0.f);
    }
    double rest = 0.0, all = 0.0;
#pragma unroll
    for (int j = 0; j < (int)DRAFT_RUN; j++) {
        const double x = draft_value(pv[j], a.target_logits, p.max, p.inv, a.c);
        double y = 0.0;
        if (refused) {
            if (a.draft)
                y = draft_value(qv[j], a.draft_logits, q.max, q.inv, a.c);
            else
                y = chunk * DRAFT_CHUNK + DRAFT_RUN * threadIdx.x + j == id ? 1.0 : 0.0;
        }
        const double d = x - y;
        rest += d <= 0.0 ? 0.0 : d;  // NaN stays
        all += x <= 0.0 ? 0.0 : x;
    }
    rest = wave_sum_f64(rest);
    all = wave_sum_f64(all);
    if (lane == 0) {
        sums[0][wave] = rest;
        sums[1][wave] = all;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        DraftRest r;
        r.rest = ((sums[0][0] + sums[0][1]) + sums[0][2]) + sums[0][3];
        r.all = ((sums[1][0] + sums[1][1]) + sums[1][2]) + sums[1][3];
        a.rests[(uint64_t)s * a.chunks + chunk] = r;
    }
    if (chunk == 0) {
        if (threadIdx.x == 0) {
            DraftState st;
            st.inv_p = p.inv;
            st.inv_q = q.inv;
            st.max_p = p.max;
            st.max_q = q.max;
            st.accepted = n;
            st.refused = refused;
            a.states[s] = st;
            a.accepted[s] = n;
        }
        for (uint32_t i = threadIdx.x; i <= a.drafts; i += 256) {
            if (i == n) continue;  // the token that is drawn next
            const uint64_t at = (uint64_t)s * (a.drafts + 1) + i;
            a.tokens[at] = i < n ? a.ids[(uint64_t)s * a.drafts + i] : DRAFT_NONE;
            if (a.probabilities) a.probabilities[at] = i < n ? pid[i] : 0.f;
        }
    }
}

// One workgroup per sequence: the chunk, then the token in it, where the
// running sum passes u times the whole.
template <class TT, class TD>
__global__ __launch_bounds__(256) void draft_token_kernel(DraftArgs a) {
    __shared__ double schunk[3];
    __shared__ uint32_t sat[3];
    __shared__ double swave[4];
    const uint32_t s = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const DraftRest *rests = a.rests + (uint64_t)s * a.chunks;
    const DraftState st = a.states[s];
    const uint32_t n = st.accepted;
    if (wave == 0) {
        double rest = 0.0, all = 0.0;
        for (uint32_t i = lane; i < a.chunks; i += 64) {
            rest += rests[i].rest;
            all += rests[i].all;
        }
        rest = wave_sum_f64(rest);
        all = wave_sum_f64(all);
        const bool left = !(rest <= 0.0);  // nothing left (p == q): draw from p
        const double whole = left ? rest : all, mark = (double)a.u[(uint64_t)s * (a.drafts + 1) + a.drafts] * whole;
        // the first chunk whose running sum passes the mark, or the last one that holds anything
        double before = 0.0, at_before = 0.0, last_before = 0.0;
        uint32_t found = DRAFT_NONE, last = DRAFT_NONE;
        for (uint32_t base = 0; base < a.chunks && found == DRAFT_NONE; base += 64) {
            const uint32_t i = base + lane;
            const double w = i < a.chunks ? (left ? rests[i].rest : rests[i].all) : 0.0;
            const double sum = before + wave_scan_f64(w);
            const uint64_t pass = __ballot(sum > mark && w > 0.0), some = __ballot(w > 0.0);
            if (pass) {
                const int l = __builtin_ctzll(pass);
                found = base + l;
                at_before = lane_f64(sum, l) - lane_f64(w, l);
            } else if (some) {
                const int l = 63 - __builtin_clzll(some);
                last = base + l;
                last_before = lane_f64(sum, l) - lane_f64(w, l);
            }
            before = lane_f64(sum, 63);
        }
        if (lane == 0) {
            const bool fine = whole > 0.0 && whole < __builtin_inf();
            sat[0] = !fine ? DRAFT_NONE : found != DRAFT_NONE ? found : last;
            sat[1] = DRAFT_NONE;
            sat[2] = 0;
            schunk[0] = found != DRAFT_NONE ? at_before : last_before;
            schunk[1] = mark;
            schunk[2] = left ? 1.0 : 0.0;
        }
    }
    __syncthreads();
    const uint32_t chunk = sat[0];
    const uint64_t out = (uint64_t)s * (a.drafts + 1) + n;
    if (chunk == DRAFT_NONE) {  // no distribution: a NaN, an infinity, or nothing but zeros
        if (threadIdx.x == 0) {
            a.tokens[out] = DRAFT_NONE;
            if (a.probabilities) a.probabilities[out] = __uint_as_float(0x7fc00000u);
        }
        return;
    }
    const DraftRows<TT, TD> rows{a, s};
    const bool minus = st.refused && schunk[2] != 0.0;
    const uint32_t id = minus ? a.ids[(uint64_t)s * a.drafts + n] : DRAFT_NONE, c0 = chunk * DRAFT_CHUNK + DRAFT_RUN * threadIdx.x;
    float pv[DRAFT_RUN], qv[DRAFT_RUN];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        load_run(rows.target(n), c0 + 8 * h, a.vocabulary, pv + 8 * h, a.target_logits ? -INFINITY : 0.f);
        if (minus && a.draft) load_run(rows.draft(n), c0 + 8 * h, a.vocabulary, qv + 8 * h, a.draft_logits ? -INFINITY : 0.f);
    }
    double r[DRAFT_RUN], sum = 0.0;
#pragma unroll
    for (int j = 0; j < (int)DRAFT_RUN; j++) {
        const double x = draft_value(pv[j], a.target_logits, st.max_p, st.inv_p, a.c);
        double y = 0.0;
        if (minus) y = a.draft ? draft_value(qv[j], a.draft_logits, st.max_q, st.inv_q, a.c) : c0 + j == id ? 1.0 : 0.0;
        r[j] = fmax(x - y, 0.0);
        sum += r[j];
    }
    const double scan = wave_scan_f64(sum);
    if (lane == 63) swave[wave] = scan;
    __syncthreads();
    double before = schunk[0];
#pragma unroll
    for (uint32_t w = 0; w < 3; w++) before += w < wave ? swave[w] : 0.0;
    before += scan - sum;
    uint32_t first = DRAFT_NONE, last = 0;
#pragma unroll
    for (int j = 0; j < (int)DRAFT_RUN; j++) {
        before += r[j];
        if (r[j] > 0.0) {
            if (before > schunk[1] && first == DRAFT_NONE) first = c0 + j;
            last = c0 + j + 1;
        }
    }
    if (first != DRAFT_NONE) atomicMin(&sat[1], first);
    if (last) atomicMax(&sat[2], last);
    __syncthreads();
    const uint32_t token = sat[1] != DRAFT_NONE ? sat[1] : sat[2] - 1;
    if (token - c0 < DRAFT_RUN) {  // the thread that holds it
        a.tokens[out] = token;
        float value = 0.f;
#pragma unroll
        for (int j = 0; j < (int)DRAFT_RUN; j++)
            if (token - c0 == (uint32_t)j) value = pv[j];
        if (a.probabilities) a.probabilities[out] = (float)draft_value(value, a.target_logits, st.max_p, st.inv_p, a.c);
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
    l.rests = s * l.chunks * sizeof(DraftRest);
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
    hipLaunchKernelGGL((draft_rest_kernel<TT, TD>), dim3(a.sequences * a.chunks), dim3(256), 0, stream, a);
    OCO_TRY(launch_check("oco_draft_verify (rest)"));
    hipLaunchKernelGGL((draft_token_kernel<TT, TD>), dim3(a.sequences), dim3(256), 0, stream, a);
    return launch_check("oco_draft_verify (token)");
}

static const char *draft_problem(const oco_draft *p) {
    if (p->drafts > OCO_DRAFT_MAX) return "too many drafts per sequence";
    if (p->vocabulary == 0 || p->vocabulary >= 0x80000000u) return "the vocabulary is empty or past 2^31";
    if (p->target_values > OCO_DRAFT_PROBABILITIES || p->draft_values > OCO_DRAFT_PROBABILITIES) return "unknown kind of values";
    if (p->target_dtype > OCO_DT_F16 || p->draft_dtype > OCO_DT_F16) return "unknown type";
    if (!(p->temperature >= 0.f) || !(p->temperature <= 3.0e38f)) return "the temperature is negative or not finite";
    if ((p->target_stride && p->target_stride < p->vocabulary) || (p->draft_stride && p->draft_stride < p->vocabulary))
        return "a row stride under the vocabulary";
    const DraftLayout l = draft_layout(p);
    if ((uint64_t)p->sequences * (2ull * p->drafts + 1) * l.chunks > 0x7fffffffull) return "too many rows for one call";
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
