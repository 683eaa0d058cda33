// Experts chosen by scores: softmax or sigmoid of the router logits, a bias
// for balance that enters the choice but not the weights, a limit to the best
// groups of experts, top-k, renormalised weights.  Stands beside
// select_topk (route.h), the reference's selection; its Nemotron-H router
// (shaders/nemotron.metal:148-212) is the sigmoid form without groups.
//
//     s_e = softmax(z)_e or 1 / (1 + exp(-z_e)),    c_e = s_e + bias_e
//     a group's rank: its largest c_e, or the sum of its two largest
//     chosen: the k largest c_e of the kept groups, ties to the lowest index
//     weight = scale * s_e [/ sum of the chosen s]
//
// The choice is made in 64 bits: with hundreds of experts two c_e within a
// few f32 roundings of each other occur in every long prompt, and which of
// them is chosen must not depend on how exp was rounded.  Without a bias
// c_e orders as z_e does, and the logits' own bits decide.
//
// Bound by issue, one wavefront per token: 8192 tokens of 256 experts with a
// bias and groups in 12.6 us, about 780 instructions each (the 8.9 MB would
// take 1.9); one token of 128 in 2.6.  A lane holds J consecutive experts
// and sorts them once; a round takes the largest head of the 64 lanes.  With a
// bias the rounds run on 64-bit keys, else on the logits' own 32 bits; then
// scores are formed for groups ranked by sums, or of the chosen alone.
#include "exp64.h"
#include "rows.h"

#include <type_traits>

namespace oco {

struct ScoresArgs {
    const void *logits;
    const float *bias;
    uint32_t *ids;
    float *weights;
    uint32_t tokens, experts, k, groups, kept, top2, sigmoid, renormalize;
    float scale;
};

constexpr int SCORE_WAVES = 4;

// What is ranked: experts and groups by their logits; groups by scores and
// experts by their logits (scores that coincide in 64 bits, as sigmoids from
// 37 on, still have an order); both by biased scores.
enum class Ranked { LOGITS, GROUPS, BIASED };

// A key and its expert take the next one's place, in their registers; the wait
// states are those of a DPP read, which the compiler does not add behind asm.
__device__ __forceinline__ void move_up(uint32_t &key, uint32_t &at, uint32_t next, uint32_t next_at) {
    asm volatile("v_mov_b32 %0, %2\n\tv_mov_b32 %1, %3\n\ts_nop 1" : "+&v"(key), "+&v"(at) : "v"(next), "v"(next_at));
}
__device__ __forceinline__ void move_up(uint64_t &key, uint32_t &at, uint64_t next, uint32_t next_at) {
    asm volatile("v_mov_b64 %0, %2\n\tv_mov_b32 %1, %3\n\ts_nop 1" : "+&v"(key), "+&v"(at) : "v"(next), "v"(next_at));
}

// Values as integers that order alike (-0 as +0); 0 is below every number, -Inf included.
__device__ __forceinline__ uint32_t order_f32(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}

// The larger and the smaller of two lanes' pairs (first >= second of disjoint sets).
template <int CTRL>
__device__ __forceinline__ void merge_dpp(double &first, double &second) {
    auto other = [](double v) {
        const uint64_t b = (uint64_t)__double_as_longlong(v);
        return words_f64((uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false),
                         (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, false));
    };
    const double a = other(first), b = other(second);
    second = fmax(fmin(first, a), fmax(second, b));
    first = fmax(first, a);
}
__device__ __forceinline__ void merge_swap(double &first, double &second, bool wide) {
    auto pair = [&](double v, double &x, double &y) {
        const uint64_t b = (uint64_t)__double_as_longlong(v);
        const uint32_t lo = (uint32_t)b, hi = (uint32_t)(b >> 32);
        if (wide) {
            auto l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
            x = words_f64(l[0], h[0]);
            y = words_f64(l[1], h[1]);
        } else {
            auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
            x = words_f64(l[0], h[0]);
            y = words_f64(l[1], h[1]);
        }
    };
    double a, b, c, d;
    pair(first, a, b);
    pair(second, c, d);
    second = fmax(fmin(a, b), fmax(c, d));
    first = fmax(a, b);
}

template <class T, int J, Ranked BY>  // J experts per lane: J lane + j
__global__ __launch_bounds__(64 * SCORE_WAVES) void scores_kernel(ScoresArgs a) {
    constexpr bool SCORED = BY != Ranked::LOGITS, WIDE = BY == Ranked::BIASED;
    using Key = std::conditional_t<WIDE, uint64_t, uint32_t>;
    __shared__ double choice_lds[SCORE_WAVES][64 * J];  // groups that are not whole lanes
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint64_t token = (uint64_t)blockIdx.x * SCORE_WAVES + wave;
    if (token >= a.tokens) return;
    const T *z = (const T *)a.logits + token * a.experts;
    float v[J];
    bool bad = false;
    if constexpr (J % 8 == 0) {
#pragma unroll
        for (int h = 0; h < J / 8; h++) load_run(z, J * lane + 8 * h, a.experts, v + 8 * h, -INFINITY);
    } else if constexpr (J == 4) {
        load_four(z, 4 * lane, a.experts, v, -INFINITY);
    } else {
#pragma unroll
        for (int j = 0; j < J; j++) v[j] = J * lane + j < a.experts ? RowIO<T>::one(z + J * lane + j) : -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; j++) {
        if (!(v[j] < INFINITY)) {  // NaN or +Inf: the token's weights are NaN
            bad = true;
            v[j] = -INFINITY;
        }
        m = fmaxf(m, v[j]);
    }
    bad = __ballot(bad) != 0;

    // e = exp(z - max) for the softmax, exp(-z) for the sigmoid; a score of 0 for an expert that is not available
    double inv = 1.0;  // softmax: the scores' common factor, where it does not cancel
    if (!a.sigmoid) m = wave_max_f32(m);
    const double from = a.sigmoid ? 0.0 : (double)m, rate = a.sigmoid ? -LOG2E : LOG2E;
    double s[J];
    if (SCORED || !(a.sigmoid || a.renormalize)) {
        double x[J];
#pragma unroll
        for (int j = 0; j < J; j++) x[j] = ((double)v[j] - from) * rate;
        exp2_clamped<12, J>(x, s);
        if (a.sigmoid) {
#pragma unroll
            for (int j = 0; j < J; j++) s[j] = v[j] > -INFINITY ? recip_f64(1.0 + s[j]) : 0.0;
        } else {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < J; j++) {
                s[j] = v[j] > -INFINITY ? s[j] : 0.0;
                sum += s[j];
            }
            sum = wave_sum_f64(sum);
            inv = sum > 0.0 ? recip_f64(sum) : 0.0;
#pragma unroll
            for (int j = 0; j < J; j++) s[j] *= inv;
        }
    }

    float bias[J];
#pragma unroll
    for (int j = 0; j < J; j++) bias[j] = WIDE && J * lane + j < a.experts ? a.bias[J * lane + j] : 0.f;

    // what is ranked, as integers: 0 for an expert that cannot be chosen
    Key key[J];
    double first = -__builtin_inf(), second = -__builtin_inf();
    const bool ranked = a.groups > 1;
    const uint32_t size = a.experts / a.groups, span = size / J;
    const bool in_lanes = size % J == 0 && (span & (span - 1)) == 0;  // a group is 1, 2, 4 .. lanes
#pragma unroll
    for (int j = 0; j < J; j++) {
        const uint32_t e = J * lane + j;
        double c = (double)v[j];
        if constexpr (SCORED) {
            c = WIDE ? s[j] + (double)bias[j] : s[j];
            if (!(v[j] > -INFINITY) || c != c) c = -__builtin_inf();
        }
        if constexpr (WIDE)
            key[j] = e < a.experts ? order_f64(c) : 0;
        else
            key[j] = e < a.experts ? order_f32(v[j]) : 0;
        if (ranked) {
            if (in_lanes) {
                second = fmax(second, fmin(first, c));
                first = fmax(first, c);
            } else {
                choice_lds[wave][e] = c;
            }
        }
    }
    if (ranked) {
        uint32_t group = lane;
        if (in_lanes) {  // each lane its own group's two largest
            group = lane / span;
            if (span > 1) merge_dpp<0xB1>(first, second);   // lanes ^ 1
            if (span > 2) merge_dpp<0x4E>(first, second);   // ^ 2
            if (span > 4) merge_dpp<0x141>(first, second);  // the mirrored half row
            if (span > 8) merge_dpp<0x140>(first, second);  // the mirrored row
            if (span > 16) merge_swap(first, second, false);
            if (span > 32) merge_swap(first, second, true);
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (lane < a.groups)
#pragma unroll 4
                for (uint32_t i = 0; i < size; i++) {
                    const double c = choice_lds[wave][lane * size + i];
                    second = fmax(second, fmin(first, c));
                    first = fmax(first, c);
                }
        }
        if (a.top2 && second > -__builtin_inf()) first += second;
        const uint64_t rank = order_f64(first);
        uint32_t better = 0;
        for (uint32_t g = 0; g < a.groups; g++) {
            const uint32_t at = in_lanes ? g * span : g;
            const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(rank >> 32), at) << 32) |
                                   (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)rank, at);
            better += other > rank || (other == rank && g < group);
        }
        if (in_lanes) {
#pragma unroll
            for (int j = 0; j < J; j++) key[j] = better < a.kept ? key[j] : 0;
        } else {
            const uint64_t kept = __ballot(lane < a.groups && better < a.kept);
            const float per = 1.0f / (float)size;
#pragma unroll
            for (int j = 0; j < J; j++) {
                // (e + 1/2) / size is at least 1 / (2 size) from an integer
                const uint32_t g = (uint32_t)(((float)(J * lane + j) + 0.5f) * per);
                if (!((kept >> (g & 63)) & 1)) key[j] = 0;
            }
        }
    }

    // each lane's experts in order: largest first, equal ones by index (adjacent exchanges that are strict)
    uint32_t at[J];
#pragma unroll
    for (int j = 0; j < J; j++) at[j] = J * lane + j;
    if constexpr (J <= 4) {
#pragma unroll
        for (int r = 0; r < J; r++)
#pragma unroll
            for (int j = r % 2; j + 1 < J; j += 2) {
                const bool swap = key[j + 1] > key[j];
                const Key k0 = key[j];
                const uint32_t a0 = at[j];
                key[j] = swap ? key[j + 1] : k0;
                key[j + 1] = swap ? k0 : key[j + 1];
                at[j] = swap ? at[j + 1] : a0;
                at[j + 1] = swap ? a0 : at[j + 1];
            }
    }
    // k rounds: the largest head; of equal ones the lowest lane's, whose experts come first
    uint32_t chosen = 0;
    for (uint32_t r = 0; r < a.k; r++) {
        Key best = key[0];
        uint32_t e = at[0];
        if constexpr (J > 4) {
#pragma unroll
            for (int j = 1; j < J; j++) {
                const bool more = key[j] > best;
                best = more ? key[j] : best;
                e = more ? at[j] : e;
            }
        }
        uint64_t lanes;
        if constexpr (WIDE) {
            const uint32_t hi = wave_max_u32((uint32_t)(best >> 32));
            const bool top = (uint32_t)(best >> 32) == hi;
            lanes = __ballot(top);
            if (__popcll(lanes) > 1) {
                const uint32_t lo = wave_max_u32(top ? (uint32_t)best : 0);
                lanes = __ballot(top && (uint32_t)best == lo);
            }
        } else {
            const uint32_t most = wave_max_u32(best);
            lanes = __ballot(best == most);
        }
        const int head = __builtin_ctzll(lanes);
        const uint32_t winner = (uint32_t)__builtin_amdgcn_readlane((int)e, head);
        if (lane == r) chosen = winner;
        if constexpr (J > 4) {
#pragma unroll
            for (int j = 0; j < J; j++) key[j] = at[j] == winner ? 0 : key[j];
        } else {
            if (lane == (uint32_t)head) {
                // in place: left to the compiler the list goes through copies (12.9 us against 12.6 for the
                // 8192 tokens), and as selects by every lane it is four times the instructions
#pragma unroll
                for (int j = 0; j + 1 < J; j++) move_up(key[j], at[j], key[j + 1], at[j + 1]);
                key[J - 1] = 0;
            }
        }
    }

    // in 64 bits: scores that f32 cannot hold still have ratios
    double w = 0.0;
    if (lane < a.k) {
        const float logit = RowIO<T>::one(z + chosen);
        const double x = ((double)logit - from) * rate;
        double e;
        exp2_clamped<12, 1>(&x, &e);
        const bool some = logit > -INFINITY && logit < INFINITY && (a.sigmoid ? x < 1000.0 : x > -1000.0);
        w = some ? a.sigmoid ? recip_f64(1.0 + e) : e * inv : 0.0;
    }
    double factor = (double)a.scale;
    if (a.renormalize) {
        const double sum = wave_sum_f64(w);
        factor = sum > 0.0 ? factor / sum : 0.0;
    }
    if (lane < a.k) {
        a.ids[token * a.k + lane] = chosen;
        a.weights[token * a.k + lane] = bad ? __uint_as_float(0x7fc00000u) : (float)(w * factor);
    }
}

typedef void (*ScoresFn)(ScoresArgs);
template <class T, Ranked BY>
static ScoresFn scores_pick(uint32_t experts) {
    if (experts <= 64) return scores_kernel<T, 1, BY>;
    if (experts <= 128) return scores_kernel<T, 2, BY>;
    if (experts <= 256) return scores_kernel<T, 4, BY>;
    if (experts <= 512) return scores_kernel<T, 8, BY>;
    return scores_kernel<T, 16, BY>;
}
template <class T>
static ScoresFn scores_pick(const ScoresArgs &a) {
    if (a.bias) return scores_pick<T, Ranked::BIASED>(a.experts);
    if (a.groups > 1 && a.top2) return scores_pick<T, Ranked::GROUPS>(a.experts);
    return scores_pick<T, Ranked::LOGITS>(a.experts);
}

}  // namespace oco

using namespace oco;

extern "C" int oco_route_scores(const void *logits, oco_dtype dtype, const float *bias, uint32_t tokens,
                                const oco_routing *p, uint32_t *ids, float *weights, oco_stream stream) {
    if (!p) return fail(OCO_ERR_INVALID, "oco_route_scores: null description");
    const uint32_t groups = p->groups ? p->groups : 1;
    if (p->experts < 1 || p->experts > OCO_ROUTING_EXPERTS || p->k < 1 || p->k > OCO_ROUTING_K || p->k > p->experts)
        return fail(OCO_ERR_INVALID, "oco_route_scores: %u of %u experts (at most %u of %u)", p->k, p->experts, OCO_ROUTING_K,
                    OCO_ROUTING_EXPERTS);
    if (p->score > OCO_SCORE_SIGMOID || p->group_rank > OCO_GROUP_TOP2)
        return fail(OCO_ERR_INVALID, "oco_route_scores: score %u, group rank %u", p->score, p->group_rank);
    if (groups > 64 || p->experts % groups)
        return fail(OCO_ERR_INVALID, "oco_route_scores: %u experts in %u groups (whole groups, at most 64)", p->experts, groups);
    if (groups > 1 && (p->groups_kept < 1 || p->groups_kept > groups || p->k > p->groups_kept * (p->experts / groups)))
        return fail(OCO_ERR_INVALID, "oco_route_scores: %u experts chosen from %u of %u groups of %u", p->k, p->groups_kept,
                    groups, p->experts / groups);
    if (tokens == 0) return OCO_OK;
    if (!logits || !ids || !weights) return fail(OCO_ERR_INVALID, "oco_route_scores: null pointer");
    ScoresArgs a;
    a.logits = logits;
    a.bias = bias;
    a.ids = ids;
    a.weights = weights;
    a.tokens = tokens;
    a.experts = p->experts;
    a.k = p->k;
    a.groups = groups > 1 && p->groups_kept < groups ? groups : 1;
    a.kept = p->groups_kept;
    a.top2 = p->group_rank == OCO_GROUP_TOP2;
    a.sigmoid = p->score == OCO_SCORE_SIGMOID;
    a.renormalize = p->renormalize != 0;
    a.scale = p->scale;
    ScoresFn fn;
    switch (dtype) {
    case OCO_DT_F32: fn = scores_pick<float>(a); break;
    case OCO_DT_BF16: fn = scores_pick<bf16_t>(a); break;
    case OCO_DT_F16: fn = scores_pick<f16_t>(a); break;
    default: return fail(OCO_ERR_UNSUPPORTED, "oco_route_scores: logits of type %d", (int)dtype);
    }
    hipLaunchKernelGGL(fn, dim3((uint32_t)(((uint64_t)tokens + SCORE_WAVES - 1) / SCORE_WAVES)), dim3(64 * SCORE_WAVES), 0,
                       (hipStream_t)stream, a);
    return launch_check("oco_route_scores");
}
