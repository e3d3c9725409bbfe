/* Penalties, biases and grammar masks on logits (aotx_logits_adjust), before the sampler. The penalties
 * are those of the decode tick (tick.hip); there they go into the rows in place and out again, around
 * the pick, through counts of the whole vocabulary in memory. Here a workgroup takes a slice of a
 * row's tokens and counts the list's in LDS, so that one launch does all and needs no memory of its
 * own: every slice reads the whole list (at most some tens of KB, from L2) and its logits once.
 */
#include "delta_dev.h"
#include "../../include/aotx_layer.h"

#include <math.h>

/* A workgroup's 512 threads take 8192 tokens of a row, 16 each. Measured with 64 rows of 128256 logits, masks and
 * lists of 6000: 16.9 us; with 256 threads 17.7 (each slice goes through the whole list), with 1024 17.9 (barriers). */
#define ADJUST_T     512u
#define ADJUST_QUADS 4u              /* times four logits of a thread */
#define ADJUST_LATE  0x80000000u     /* of a token's count: it is among the last repeat_window */
#define ADJUST_AHEAD 4u              /* loads of four of a list's tokens that a thread has under way */

typedef unsigned int aotx_u32x4 __attribute__((ext_vector_type(4)));

struct aotx_adjust_args {
    aotx_adjust_how how;
    const float *logits;
    float *out;
    unsigned int ld, ld_out, vocab, slices;
    unsigned int *faults;
};

/* A row's penalties. */
struct aotx_adjust_row {
    bool spaced, repeated;              /* presence or frequency, repeat */
    float presence, frequency, repeat;
};
static __device__ __forceinline__ float aotx_adjust_pen(const aotx_adjust_row &w, float z, unsigned int count)
{
    const unsigned int c = count & ~ADJUST_LATE;
    if (w.spaced && c != 0u) z -= __builtin_fmaf(w.frequency, (float)c, w.presence);
    if (w.repeated && (count & ADJUST_LATE) != 0u) z = z > 0.0f ? z / w.repeat : z * w.repeat;
    return z;
}

/* A list that a workgroup goes through, four tokens a load whatever the list's alignment (its ends one by one),
 * AHEAD such loads of a thread under way. */
template <unsigned int T, unsigned int AHEAD>
struct aotx_adjust_list {
    const int *list;
    unsigned int length, head, fours;
    unsigned int end;                   /* this thread's token of the ends */
    aotx_u32x4 t[AHEAD];

    __device__ __forceinline__ void load(unsigned int first)
    {
        const aotx_u32x4 *body = (const aotx_u32x4 *)(list + head);
#pragma unroll
        for (unsigned int k = 0u; k < AHEAD; ++k) {
            const unsigned int i = first + T * k;
            if (i < fours) t[k] = body[i];
        }
    }
    /* its first loads */
    __device__ __forceinline__ void open(const int *at, unsigned int n)
    {
        list = at;
        length = n;
        head = (0u - (unsigned int)((uintptr_t)list >> 2)) & 3u;
        head = head < length ? head : length;
        fours = (length - head) / 4u;
        if (threadIdx.x < length - 4u * fours) end = (unsigned int)list[threadIdx.x < head ? threadIdx.x : 4u * fours + threadIdx.x];
        load(threadIdx.x);
    }
    /* each(slot, place) for its tokens that lie in the slice of `size` from lo (those below it wrap past it) */
    template <class F>
    __device__ __forceinline__ void go(unsigned int lo, unsigned int size, F each)
    {
        const unsigned int tid = threadIdx.x;
        if (tid < length - 4u * fours && end - lo < size) each(end - lo, tid < head ? tid : 4u * fours + tid);
        for (unsigned int first = tid; first < fours;) {
#pragma unroll
            for (unsigned int k = 0u; k < AHEAD; ++k) {
                const unsigned int i = first + T * k;
                if (i >= fours) break;
#pragma unroll
                for (unsigned int e = 0u; e < 4u; ++e)
                    if (t[k][e] - lo < size) each(t[k][e] - lo, head + 4u * i + e);
            }
            first += T * AHEAD;
            load(first);
        }
    }
};

/* Grid: slices x rows, and with a mask one more workgroup a row, which looks whether the mask allows anything.
 * A row's tokens are counted from the last 16-byte boundary at or before it, so that every load of four is
 * aligned whatever the row's length: slot i of a slice is token lo + i, and the slots whose token the row does
 * not have (below 0, which is far above in 32 bits, or past its end) are never allowed. INPLACE: out
 * is logits, and only what changes is read and written. */
template <unsigned int T, bool INPLACE>
__global__ __launch_bounds__(T, 8) void aotx_adjust_kernel(aotx_adjust_args p)
{
    constexpr unsigned int SLICE = T * 4u * ADJUST_QUADS;
    __shared__ __attribute__((aligned(16))) unsigned int table[SLICE];
    const unsigned int r = blockIdx.y, tid = threadIdx.x;
    const unsigned int *mask = nullptr;
    if (p.how.mask != nullptr) {
        const unsigned int of = p.how.mask_of != nullptr ? p.how.mask_of[r] : r;
        if (of < p.how.masks) mask = p.how.mask + (unsigned long long)of * p.how.mask_stride;
    }
    const unsigned int words = (p.vocab + 31u) / 32u;
    if (blockIdx.x == p.slices) {
        if (mask == nullptr) return;
        bool any = false;
#pragma unroll 8
        for (unsigned int i = tid; i < words; i += T) {
            const unsigned int left = p.vocab - i * 32u;
            any = any || (mask[i] & (left < 32u ? (1u << left) - 1u : 0xFFFFFFFFu)) != 0u;
        }
        if (__syncthreads_or(any) == 0 && tid == 0u) atomicAdd(p.faults, 1u);
        return;
    }
    const float *row = p.logits + (unsigned long long)r * p.ld;
    float *out = p.out + (unsigned long long)r * p.ld_out;
    const unsigned int lead = (unsigned int)((uintptr_t)row >> 2) & 3u;
    const bool out_too = ((unsigned int)((uintptr_t)out >> 2) & 3u) == lead;
    const unsigned int lo = blockIdx.x * SLICE - lead;
    row += (int)lo;
    out += (int)lo;

    /* the tokens of a thread, four neighbours of every 4 T: a bit each that the row has and the mask allows */
    unsigned int live[ADJUST_QUADS], allowed[ADJUST_QUADS];
    aotx_f4 z[ADJUST_QUADS];
#pragma unroll
    for (unsigned int q = 0u; q < ADJUST_QUADS; ++q) {
        const unsigned int t = lo + q * 4u * T + 4u * tid;
        live[q] = 0u;
#pragma unroll
        for (unsigned int e = 0u; e < 4u; ++e) live[q] |= t + e < p.vocab ? 1u << e : 0u;
        allowed[q] = live[q];
        if (mask != nullptr && live[q] != 0u) {
            const int w = (int)t >> 5;
            const unsigned int w0 = mask[w < 0 ? 0 : w];
            unsigned int w1 = w0;
            if (lead != 0u) {                    /* the four may lie in two words */
                const unsigned int next = (unsigned int)((int)(t + 3u) >> 5);
                w1 = mask[next < words ? next : words - 1u];
            }
            allowed[q] &= __builtin_amdgcn_alignbit(w1, w0, t & 31u);
        }
    }
    aotx_adjust_row w = {false, false, 0.0f, 0.0f, 1.0f};
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
    unsigned int biases = 0u, bias0 = 0u;
    if (p.how.bias_at != nullptr) {
        unsigned int b = p.how.bias_at[r], e = p.how.bias_at[r + 1u];
        b = b < p.how.biases ? b : p.how.biases;
        e = e < p.how.biases ? e : p.how.biases;
        biases = e > b ? e - b : 0u;
        bias0 = b;
    }
    /* the lists' first tokens are asked for before the logits: a wave's loads come back in order, and the
     * counts are wanted first */
    aotx_adjust_list<T, ADJUST_AHEAD> tokens;
    aotx_adjust_list<T, 1u> named;
    if (length != 0u) tokens.open(list, length);
    if (biases != 0u) named.open(p.how.bias_token + bias0, biases);

    const auto load = [&](unsigned int q) {
        const float *from = row + q * 4u * T + 4u * tid;
        if (live[q] == 15u) z[q] = *(const aotx_f4 *)from;
        else
#pragma unroll
            for (unsigned int e = 0u; e < 4u; ++e) z[q][e] = live[q] >> e & 1u ? from[e] : 0.0f;
    };
    if (!INPLACE)
#pragma unroll
        for (unsigned int q = 0u; q < ADJUST_QUADS; ++q)
            if (allowed[q] != 0u) load(q);

    /* The counts, and then the places of the biases, go through one table: with two, half as many workgroups
     * would find room on a CU. */
    const auto clear = [&]() {
#pragma unroll
        for (unsigned int q = 0u; q < ADJUST_QUADS; ++q)
            *(aotx_u32x4 *)(table + q * 4u * T + 4u * tid) = (aotx_u32x4){0u, 0u, 0u, 0u};
        __syncthreads();
    };
    unsigned int held = 0u;                      /* INPLACE: a bit for every four that this thread has in z */
    const auto apply = [&](auto each) {
        __syncthreads();
#pragma unroll
        for (unsigned int q = 0u; q < ADJUST_QUADS; ++q) {
            const aotx_u32x4 v = *(const aotx_u32x4 *)(table + q * 4u * T + 4u * tid);
            unsigned int some = 0u;
#pragma unroll
            for (unsigned int e = 0u; e < 4u; ++e) some |= v[e] != 0u ? 1u << e : 0u;
            some &= allowed[q];
            if (some == 0u) continue;
            if (INPLACE && (held >> q & 1u) == 0u) {
                load(q);
                held |= 1u << q;
            }
#pragma unroll
            for (unsigned int e = 0u; e < 4u; ++e)
                if (some >> e & 1u) z[q][e] = each(z[q][e], v[e]);
        }
    };
    if (length != 0u) {
        clear();
        tokens.go(lo, SLICE, [&](unsigned int i, unsigned int at) {
            atomicAdd(&table[i], 1u);
            if (at >= first) atomicOr(&table[i], ADJUST_LATE);
        });
        apply([&](float v, unsigned int count) { return aotx_adjust_pen(w, v, count); });
    }
    if (biases != 0u) {
        if (length != 0u) __syncthreads();       /* the counts are read */
        clear();
        named.go(lo, SLICE, [&](unsigned int i, unsigned int at) {
            atomicMax(&table[i], at + 1u);
        });
        apply([&](float v, unsigned int mark) { return v + p.how.bias[bias0 + mark - 1u]; });
    }
#pragma unroll
    for (unsigned int q = 0u; q < ADJUST_QUADS; ++q) {
#pragma unroll
        for (unsigned int e = 0u; e < 4u; ++e)
            if ((allowed[q] >> e & 1u) == 0u) z[q][e] = -INFINITY;
        float *to = out + q * 4u * T + 4u * tid;
        /* in place: all four where one was changed, else those that the mask takes out */
        const unsigned int put = INPLACE && (held >> q & 1u) == 0u ? live[q] & ~allowed[q] : live[q];
        if (put == 15u && out_too) *(aotx_f4 *)to = z[q];
        else
#pragma unroll
            for (unsigned int e = 0u; e < 4u; ++e)
                if (put >> e & 1u) to[e] = z[q][e];
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
    /* (a row's slots begin up to three before its first token) */
    const unsigned int slice = ADJUST_T * 4u * ADJUST_QUADS, slices = (vocab + 3u + slice - 1u) / slice;
    aotx_adjust_args p = {*how, logits, out, ld, ld_out, vocab, slices, nullptr};
    if (how->mask != nullptr) {
        p.faults = aotx_faults(stream);
        if (p.faults == nullptr) return 1;
    }
    const dim3 grid(slices + (how->mask != nullptr ? 1u : 0u), rows);
    hipStream_t s = aotx_stream(stream);
#define AOTX_ADJUST_GO(INPLACE) \
    hipLaunchKernelGGL((aotx_adjust_kernel<ADJUST_T, INPLACE>), grid, dim3(ADJUST_T), 0, s, p)
    if ((const float *)out == logits) AOTX_ADJUST_GO(true);
    else AOTX_ADJUST_GO(false);
#undef AOTX_ADJUST_GO
    AOTX_LAUNCH_CHECK();
    return 0;
}
