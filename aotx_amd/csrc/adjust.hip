/* Penalties, biases and grammar masks on logits (aotx_logits_adjust), before the sampler. The penalties
 * are those of the decode tick (tick.hip); there they go into the rows in place and out again, around
 * the pick, through counts of the whole vocabulary in memory. Here a workgroup takes a slice of a
 * row's tokens and counts the list's in LDS, so that one launch does all and needs no memory of its
 * own: every slice reads the whole list (at most some tens of KB, from L2) and its logits once.
 */
#include "delta_dev.h"
#include "../../include/aotx_layer.h"

#include <math.h>

#define ADJUST_SLICE 4096u
#define ADJUST_LATE  0x80000000u     /* of a token's count: it is among the last repeat_window */

struct aotx_adjust_args {
    aotx_adjust_how how;
    const float *logits;
    float *out;
    unsigned int ld, ld_out, vocab;
    unsigned int *faults;
};

/* One token's logit, as the row's penalties, bias and mask make it. */
struct aotx_adjust_row {
    bool spaced, repeated;              /* presence or frequency, repeat */
    float presence, frequency, repeat;
    const float *bias;                  /* of the row */
};
static __device__ __forceinline__ float aotx_adjust_one(const aotx_adjust_row &w, float z, unsigned int count,
                                                        unsigned int mark)
{
    const unsigned int c = count & ~ADJUST_LATE;
    if (w.spaced && c != 0u) z -= __builtin_fmaf(w.frequency, (float)c, w.presence);
    if (w.repeated && (count & ADJUST_LATE) != 0u) z = z > 0.0f ? z / w.repeat : z * w.repeat;
    if (mark != 0u) z += w.bias[mark - 1u];
    return z;
}

/* Grid: slices x rows. LDS: a count of every token of the slice, and the place in the row's biases (+ 1)
 * of the last that names it. */
__global__ __launch_bounds__(256) void aotx_adjust_kernel(aotx_adjust_args p)
{
    __shared__ unsigned int count[ADJUST_SLICE], mark[ADJUST_SLICE];
    const unsigned int r = blockIdx.y, tid = threadIdx.x;
    const unsigned int lo = blockIdx.x * ADJUST_SLICE;
    const unsigned int size = p.vocab - lo < ADJUST_SLICE ? p.vocab - lo : ADJUST_SLICE;

    aotx_adjust_row w = {false, false, 0.0f, 0.0f, 1.0f, nullptr};
    const int *list = nullptr;
    unsigned int length = 0u, first = 0u;
    if (p.how.sample != nullptr) {
        const aotx_model_how &how = p.how.sample[r];
        const unsigned int agent = p.how.agent != nullptr ? p.how.agent[r] : r;
        w.presence = how.presence_penalty;
        w.frequency = how.frequency_penalty;
        w.repeat = how.repeat_penalty;
        w.spaced = w.presence != 0.0f || w.frequency != 0.0f;
        w.repeated = how.repeat_window != 0u && w.repeat != 1.0f;
        if (agent < p.how.lists && (w.spaced || w.repeated)) {
            list = p.how.list + (unsigned long long)agent * p.how.list_stride;
            length = p.how.length[agent] < p.how.list_stride ? p.how.length[agent] : p.how.list_stride;
            first = length > how.repeat_window ? length - how.repeat_window : 0u;
        }
    }
    unsigned int biases = 0u;
    const int *named = nullptr;
    if (p.how.bias_at != nullptr) {
        unsigned int b = p.how.bias_at[r], e = p.how.bias_at[r + 1u];
        b = b < p.how.biases ? b : p.how.biases;
        e = e < p.how.biases ? e : p.how.biases;
        biases = e > b ? e - b : 0u;
        named = p.how.bias_token + b;
        w.bias = p.how.bias + b;
    }
    const unsigned int *mask = nullptr;
    if (p.how.mask != nullptr) {
        const unsigned int of = p.how.mask_of != nullptr ? p.how.mask_of[r] : r;
        if (of < p.how.masks) mask = p.how.mask + (unsigned long long)of * p.how.mask_stride;
    }

    for (unsigned int i = tid; i < size; i += 256u) count[i] = mark[i] = 0u;
    __syncthreads();
    for (unsigned int i = tid; i < length; i += 256u) {
        const unsigned int t = (unsigned int)list[i] - lo;       /* tokens below the slice wrap past it */
        if (t >= size) continue;
        atomicAdd(&count[t], 1u);
        if (i >= first) atomicOr(&count[t], ADJUST_LATE);
    }
    for (unsigned int i = tid; i < biases; i += 256u) {
        const unsigned int t = (unsigned int)named[i] - lo;
        if (t < size) atomicMax(&mark[t], i + 1u);
    }
    __syncthreads();
    const float *row = p.logits + (unsigned long long)r * p.ld + lo;
    float *out = p.out + (unsigned long long)r * p.ld_out + lo;
    for (unsigned int i = tid; i < size; i += 256u) {
        const unsigned int t = lo + i;
        const bool allowed = mask == nullptr || (mask[t / 32u] >> (t % 32u) & 1u) != 0u;
        out[i] = allowed ? aotx_adjust_one(w, row[i], count[i], mark[i]) : -INFINITY;
    }
    /* a mask that allows nothing of the vocabulary, counted once a row */
    if (blockIdx.x == 0u && mask != nullptr) {
        bool any = false;
        for (unsigned int i = tid; i * 32u < p.vocab; i += 256u) {
            const unsigned int left = p.vocab - i * 32u;
            any = any || (mask[i] & (left < 32u ? (1u << left) - 1u : 0xFFFFFFFFu)) != 0u;
        }
        if (__syncthreads_or(any) == 0 && tid == 0u) atomicAdd(p.faults, 1u);
    }
}

extern "C" int aotx_logits_adjust(const aotx_adjust_how *how, const float *logits, unsigned int ld,
                                  unsigned int rows, unsigned int vocab, float *out, unsigned int ld_out,
                                  void *stream)
{
    if (how == nullptr || logits == nullptr || out == nullptr) return 1;
    if (vocab == 0u || vocab > (1u << 20) || rows > 4096u) return 1;
    if (ld < vocab || ld > (1u << 22) || ld_out < vocab || ld_out > (1u << 22)) return 1;
    if ((const float *)out == logits && ld != ld_out) return 1;
    if (how->sample != nullptr) {
        if (how->list == nullptr || how->length == nullptr || how->list_stride > (1u << 20)) return 1;
    }
    if (how->bias_at != nullptr && how->biases != 0u && (how->bias_token == nullptr || how->bias == nullptr)) return 1;
    if (how->mask != nullptr && how->mask_stride < (vocab + 31u) / 32u) return 1;
    const void *const four[] = {logits, out, how->agent, how->list, how->length, how->bias_at, how->bias_token, how->bias,
                                how->mask, how->mask_of};
    for (const void *q : four)
        if (((uintptr_t)q & 3u) != 0u) return 1;
    if (((uintptr_t)how->sample & 7u) != 0u) return 1;
    if (rows == 0u) return 0;
    aotx_adjust_args p = {*how, logits, out, ld, ld_out, vocab, nullptr};
    if (how->mask != nullptr) {
        p.faults = aotx_faults(stream);
        if (p.faults == nullptr) return 1;
    }
    hipLaunchKernelGGL(aotx_adjust_kernel, dim3((vocab + ADJUST_SLICE - 1u) / ADJUST_SLICE, rows), dim3(256), 0,
                       aotx_stream(stream), p);
    AOTX_LAUNCH_CHECK();
    return 0;
}
