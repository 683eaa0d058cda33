// Rows of logits before a token is chosen from them: penalties for repeated
// tokens, biases and masks.
//
// Bound by reading and writing the rows.  A workgroup takes a chunk of a row
// and first counts in LDS which of its words the history holds, in one word
// per vocabulary entry: the history's count in the lower 20 bits, the place of
// the last bias for it (from 1) in the upper 12.  Maxima and counts do not
// hang on the order of the atomics.  Then the chunk passes through registers
// once.
#include "eight.h"

namespace oco {

struct LogitsArgs {
    const void *logits;
    void *out;
    const uint32_t *history, *history_lengths, *bias_ids, *bias_lengths, *mask;
    const float *penalties, *biases;
    uint64_t stride, out_stride;
    uint32_t vocabulary, chunks, history_stride, bias_stride, mask_stride, group, mask_group;
};

// Words per workgroup.  Every workgroup of a row reads its whole history, which costs little: 64 rows of 151936 f32 words
// take 15.1 us with 512 ids and no mask (5.2 TB/s), 16.6 with 2048 and a mask, 19.3 with 8192 (bf16, 2048 ids: 13.9).
// 1024 threads on 16384 words: 15.8 with 512 ids, 17.6 with 8192.  Copying the chunk while the ids are read, and mending
// the marked words after it: 16.8 with 2048, 22.2 with 8192, 13.4 in bf16.
constexpr uint32_t LOGITS_CHUNK = 4096;

template <class T>
__global__ __launch_bounds__(256) void logits_kernel(LogitsArgs a) {
    constexpr uint32_t THREADS = 256, CHUNK = LOGITS_CHUNK;
    __shared__ __attribute__((aligned(16))) uint32_t marks[CHUNK];
    const uint32_t row = blockIdx.x / a.chunks, first = blockIdx.x % a.chunks * CHUNK, g = row / a.group;
    const uint32_t size = min(CHUNK, a.vocabulary - first);
    float repetition = 1.f, frequency = 0.f, presence = 0.f;
    const bool marked = a.history || a.bias_ids;
    if (marked) {
        for (uint32_t i = 4 * threadIdx.x; i < CHUNK; i += 4 * THREADS) *(u32x4 *)(marks + i) = u32x4{0, 0, 0, 0};
        __syncthreads();
        if (a.bias_ids) {
            const uint32_t n = a.bias_lengths ? min(a.bias_lengths[g], a.bias_stride) : a.bias_stride;
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const uint32_t at = a.bias_ids[(uint64_t)g * a.bias_stride + i] - first;
                if (at < size) atomicMax(&marks[at], (i + 1) << 20);
            }
            __syncthreads();
        }
        if (a.history) {
            const float *const p = a.penalties + 3 * (uint64_t)g;
            repetition = p[0];
            frequency = p[1];
            presence = p[2];
            const uint32_t n = a.history_lengths ? min(a.history_lengths[g], a.history_stride) : a.history_stride;
            const uint32_t *const ids = a.history + (uint64_t)g * a.history_stride;
            for (uint32_t i = 4 * threadIdx.x; i < n; i += 4 * THREADS) {
                u32x4 id = {first - 1, first - 1, first - 1, first - 1};
                if (i + 4 <= n) {
                    id = *(const GLOBAL u32x4_u *)gp(ids + i);
                } else {
#pragma unroll
                    for (int j = 0; j < 3; j++)
                        if (i + j < n) id[j] = ids[i + j];
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (id[j] - first < size) atomicAdd(&marks[id[j] - first], 1u);
            }
        }
        __syncthreads();
    }
    const T *const x = (const T *)a.logits + row * a.stride + first;
    T *const out = (T *)a.out + row * a.out_stride + first;
    const uint32_t *const mask = a.mask ? a.mask + (uint64_t)(row / a.mask_group) * a.mask_stride + first / 32 : nullptr;
#pragma unroll
    for (uint32_t c = 8 * threadIdx.x; c < CHUNK; c += 8 * THREADS) {
        if (c >= size) break;
        float v[8];
        load_run(x, c, size, v);
        if (marked) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t m = marks[c + j];
                if (!m) continue;
                const uint32_t n = m & 0xfffffu, b = m >> 20;
                if (n) v[j] = (v[j] > 0.f ? v[j] / repetition : v[j] * repetition) - (frequency * (float)n + presence);
                if (b) v[j] += a.biases[(uint64_t)g * a.bias_stride + b - 1];
            }
        }
        if (mask) {
            const uint32_t m = mask[c / 32] >> (c % 32);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (m >> j) & 1 ? v[j] : -INFINITY;
        }
        Eight<T> y;
        y.round(v);
        if (c + 8 <= size)
            y.store(out + c);
        else
            y.store_some(out + c, size - c);
    }
}

template <class T>
static int logits_launch(LogitsArgs a, uint32_t rows, hipStream_t stream) {
    a.chunks = (a.vocabulary + LOGITS_CHUNK - 1) / LOGITS_CHUNK;
    if ((uint64_t)rows * a.chunks > 0x7fffffffull) return fail(OCO_ERR_INVALID, "oco_logits_adjust: %u rows", rows);
    hipLaunchKernelGGL((logits_kernel<T>), dim3(rows * a.chunks), dim3(256), 0, stream, a);
    return launch_check("oco_logits_adjust");
}

static const char *logits_problem(const oco_logits *p) {
    if (p->vocabulary >= 0x80000000u) return "the vocabulary is past 2^31";
    if (p->history_stride > OCO_LOGITS_HISTORY) return "the history is too long";
    if (p->bias_stride > OCO_LOGITS_BIASES) return "too many biases";
    if (p->mask_stride && p->mask_stride < (p->vocabulary + 31) / 32) return "a mask stride under the row";
    if ((p->stride && p->stride < p->vocabulary) || (p->out_stride && p->out_stride < p->vocabulary)) return "a row stride under the vocabulary";
    return nullptr;
}

}  // namespace oco

using namespace oco;

extern "C" int oco_logits_adjust(const void *logits, void *out, const uint32_t *history, const uint32_t *history_lengths,
                                 const float *penalties, const uint32_t *bias_ids, const float *biases, const uint32_t *bias_lengths,
                                 const uint32_t *mask, const oco_logits *p, oco_stream stream) {
    if (!p) return fail(OCO_ERR_INVALID, "oco_logits_adjust: null description");
    if (const char *why = logits_problem(p)) return fail(OCO_ERR_INVALID, "oco_logits_adjust: %s", why);
    if (p->dtype > OCO_DT_F16) return fail(OCO_ERR_UNSUPPORTED, "oco_logits_adjust: type %u", p->dtype);
    if (p->rows == 0 || p->vocabulary == 0) return OCO_OK;
    if (!logits || !out || (history && !penalties) || (bias_ids && !biases)) return fail(OCO_ERR_INVALID, "oco_logits_adjust: null pointer");
    LogitsArgs a;
    a.logits = logits;
    a.out = out;
    a.history = p->history_stride ? history : nullptr;
    a.history_lengths = history_lengths;
    a.bias_ids = p->bias_stride ? bias_ids : nullptr;
    a.bias_lengths = bias_lengths;
    a.mask = mask;
    a.penalties = penalties;
    a.biases = biases;
    a.stride = p->stride ? p->stride : p->vocabulary;
    a.out_stride = p->out_stride ? p->out_stride : p->vocabulary;
    if (logits == out && a.stride != a.out_stride) return fail(OCO_ERR_INVALID, "oco_logits_adjust: in place with another stride");
    a.vocabulary = p->vocabulary;
    a.history_stride = p->history_stride;
    a.bias_stride = p->bias_stride;
    a.mask_stride = p->mask_stride ? p->mask_stride : (p->vocabulary + 31) / 32;
    a.group = p->group ? p->group : 1;
    a.mask_group = p->mask_group ? p->mask_group : 1;
    hipStream_t st = (hipStream_t)stream;
    switch (p->dtype) {
    case OCO_DT_F32: return logits_launch<float>(a, p->rows, st);
    case OCO_DT_BF16: return logits_launch<bf16_t>(a, p->rows, st);
    default: return logits_launch<f16_t>(a, p->rows, st);
    }
}
