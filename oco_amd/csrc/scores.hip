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
// Bound by issue: one wavefront per token; the k rounds (a wave-wide maximum
// each) and, with a bias or ranked groups, the 64-bit exponentials.
#include "exp64.h"
#include "rows.h"

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

// 1 / d for d >= 1: the hardware's estimate and two Newton steps.
__device__ __forceinline__ double recip_f64(double d) {
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

template <class T, int J>  // J experts per lane: lane + 64 j
__global__ __launch_bounds__(64 * SCORE_WAVES) void scores_kernel(ScoresArgs a) {
    __shared__ double choice_lds[SCORE_WAVES][64 * J];
    __shared__ float score_lds[SCORE_WAVES][64 * J];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint64_t token = (uint64_t)blockIdx.x * SCORE_WAVES + wave;
    if (token >= a.tokens) return;
    const T *z = (const T *)a.logits + token * a.experts;
    const bool ranked = a.groups > 1;
    const bool wide = a.bias || (ranked && a.top2);  // the choice needs scores, not logits
    float v[J];
    bool bad = false, open[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        const uint32_t e = lane + 64 * j;
        v[j] = e < a.experts ? RowIO<T>::one(z + e) : -INFINITY;
        if (!(v[j] < INFINITY)) {  // NaN or +Inf: the token's weights are NaN
            bad = true;
            v[j] = -INFINITY;
        }
        open[j] = v[j] > -INFINITY;  // -Inf: an expert that is not available
    }
    bad = __ballot(bad) != 0;

    // scores
    double s[J];
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < J; j++) s[j] = open[j] ? recip_f64(1.0 + exp2_f64<12>(fmin((double)v[j] * -LOG2E, 999.0))) : 0.0;
    } else {
        float m = v[0];
#pragma unroll
        for (int j = 1; j < J; j++) m = fmaxf(m, v[j]);
        m = wave_max_f32(m);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < J; j++) {
            s[j] = open[j] ? exp2_f64<12>(((double)v[j] - (double)m) * LOG2E) : 0.0;
            sum += s[j];
        }
        sum = wave_sum_f64(sum);
        const double inv = sum > 0.0 ? recip_f64(sum) : 0.0;
#pragma unroll
        for (int j = 0; j < J; j++) s[j] *= inv;
    }

    // what is ranked, as integers: 0 for an expert that cannot be chosen
    uint64_t key[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        const uint32_t e = lane + 64 * j;
        double c = (double)v[j];
        if (wide) {
            c = s[j] + (a.bias && e < a.experts ? (double)a.bias[e] : 0.0);
            if (!open[j] || c != c) c = -__builtin_inf();
        }
        key[j] = e < a.experts ? order_f64(c) : 0;
        score_lds[wave][e] = (float)s[j];
        if (ranked) choice_lds[wave][e] = c;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (ranked) {
        const uint32_t size = a.experts / a.groups;
        uint64_t rank = 0;
        if (lane < a.groups) {
            double first = -__builtin_inf(), second = -__builtin_inf();
            for (uint32_t i = 0; i < size; i++) {
                const double c = choice_lds[wave][lane * size + i];
                second = fmax(second, fmin(first, c));
                first = fmax(first, c);
            }
            if (a.top2 && second > -__builtin_inf()) first += second;
            rank = order_f64(first);
        }
        uint32_t better = 0;
        for (uint32_t g = 0; g < a.groups; g++) {
            const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(rank >> 32), g) << 32) |
                                   (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)rank, g);
            better += other > rank || (other == rank && g < lane);
        }
        const uint64_t kept = __ballot(lane < a.groups && better < a.kept);
        const float per = 1.0f / (float)size;
#pragma unroll
        for (int j = 0; j < J; j++) {
            // (e + 1/2) / size is at least 1 / (2 size) from an integer
            const uint32_t g = (uint32_t)(((float)(lane + 64 * j) + 0.5f) * per);
            if (!((kept >> (g & 63)) & 1)) key[j] = 0;
        }
    }

    // k rounds: the largest high word, then, where several lanes have it, the low words
    uint32_t chosen = 0;
    for (uint32_t r = 0; r < a.k; r++) {
        uint64_t best = key[0];
        uint32_t at = 0;
#pragma unroll
        for (int j = 1; j < J; j++)
            if (key[j] > best) {
                best = key[j];
                at = j;
            }
        const uint32_t hi = wave_max_u32((uint32_t)(best >> 32));
        const bool top = (uint32_t)(best >> 32) == hi;
        uint64_t lanes = __ballot(top);
        uint32_t e = lane + 64 * at;
        if (__popcll(lanes) > 1) {
            const uint32_t lo = wave_max_u32(top ? (uint32_t)best : 0);
            e = wave_max_u32(top && (uint32_t)best == lo ? ~e : 0);
            e = ~e;
        } else {
            e = (uint32_t)__builtin_amdgcn_readlane((int)e, __builtin_ctzll(lanes));
        }
        if (lane == r) chosen = e;
#pragma unroll
        for (int j = 0; j < J; j++)
            if (e == lane + 64 * j) key[j] = 0;
    }

    const float w = lane < a.k ? score_lds[wave][chosen] : 0.f;
    float factor = a.scale;
    if (a.renormalize) {
        const float sum = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_sum(w))));
        factor = sum > 0.f ? a.scale / sum : 0.f;
    }
    if (lane < a.k) {
        a.ids[token * a.k + lane] = chosen;
        a.weights[token * a.k + lane] = bad ? __uint_as_float(0x7fc00000u) : w * factor;
    }
}

typedef void (*ScoresFn)(ScoresArgs);
template <class T>
static ScoresFn scores_pick(uint32_t experts) {
    if (experts <= 64) return scores_kernel<T, 1>;
    if (experts <= 128) return scores_kernel<T, 2>;
    if (experts <= 256) return scores_kernel<T, 4>;
    if (experts <= 512) return scores_kernel<T, 8>;
    return scores_kernel<T, 16>;
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
    case OCO_DT_F32: fn = scores_pick<float>(p->experts); break;
    case OCO_DT_BF16: fn = scores_pick<bf16_t>(p->experts); break;
    case OCO_DT_F16: fn = scores_pick<f16_t>(p->experts); break;
    default: return fail(OCO_ERR_UNSUPPORTED, "oco_route_scores: logits of type %d", (int)dtype);
    }
    hipLaunchKernelGGL(fn, dim3((uint32_t)(((uint64_t)tokens + SCORE_WAVES - 1) / SCORE_WAVES)), dim3(64 * SCORE_WAVES), 0,
                       (hipStream_t)stream, a);
    return launch_check("oco_route_scores");
}
