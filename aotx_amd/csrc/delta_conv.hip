/* Short causal convolution with SiLU of linear layers (aotx_delta_conv).
 *
 *   out[t][c] = silu(bias[c] + sum over j < W of w[c][j] x[t - (W - 1) + j][c])
 *
 * A thread takes four channels of a run of rows and carries the last W - 1 rows of x in
 * registers, so every row is read once (and W - 1 more a run). Bound by memory, 4 B in and 2 B
 * out a value: 8192 rows of 8192 channels, 403 MB, in 77 us, 5.2 TB/s, the rate of a large copy; a
 * row of 64 sequences 5.5 us, the latency of a launch, the sequences and then their rows.
 */
#include "delta_dev.h"
#include "../../include/aotx_hybrid.h"

struct aotx_conv_args {
    const float *x, *w, *bias;
    float *state;
    unsigned short *out;
    unsigned int stride, channels, blocks, run;
    aotx_seqs seqs;
};

/* STREAM: 1, out goes past the caches; 2, and x comes past them. */
template <int W, int STREAM>
__global__ __launch_bounds__(256) void aotx_delta_conv_kernel(aotx_conv_args p)
{
    const unsigned int lane = threadIdx.x & 63u;
    /* the workgroups of a run's rows follow one another: whole rows at a time from memory */
    const unsigned int c = (blockIdx.x % p.blocks * 256u + threadIdx.x) * 4u;
    const bool live = c < p.channels;            /* whole waves stay for the sequence reads */
    const unsigned int t0 = blockIdx.x / p.blocks * p.run;
    unsigned int stop = t0 + p.run;
    if (stop > p.seqs.tokens) stop = p.seqs.tokens;

    float w[4][W];
    aotx_f4 bias = {0, 0, 0, 0};
    if (live) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < W; ++j) w[e][j] = p.w[(unsigned long long)(c + e) * W + j];
        if (p.bias != nullptr) bias = *(const aotx_f4 *)(p.bias + c);
    }
    /* the first sequence with rows from t0 on: those that end at or before t0 come first */
    const aotx_seq_lanes seqs = aotx_seqs_read(p.seqs);
    unsigned int i = (unsigned int)__popcll(__ballot(lane < p.seqs.seqs && seqs.end <= t0));
    for (; i < p.seqs.seqs; ++i) {
        const aotx_seq_view seq = aotx_seq_of(p.seqs, i, seqs);
        if (seq.start >= stop) break;
        /* The run that holds a sequence's first row takes its first W - 1 rows, so that no
         * other run needs the slot's rows, which that run replaces. */
        unsigned int t = seq.start, end = seq.start + W - 1u;
        if (end < stop) end = stop;
        if (seq.start < t0) {
            t = seq.start + W - 1u > t0 ? seq.start + W - 1u : t0;
            end = stop;
        }
        if (end > seq.end) end = seq.end;
        if (!live || t >= end) continue;
        if (seq.refused) {
            if (t == seq.start && c == 0u) atomicAdd(p.seqs.faults, 1u);
            for (; t < end; ++t)
                *(aotx_u16x4 *)(p.out + (unsigned long long)t * p.channels + c) = aotx_u16x4{0, 0, 0, 0};
            continue;
        }
        /* past[j]: row t - (W - 1) + j, from x or, before the sequence's first row, its state */
        float *kept = p.state + (unsigned long long)seq.slot * (W - 1) * p.channels + c;
        aotx_f4 past[W - 1];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            if (t != seq.start)
                past[j] = *(const aotx_f4 *)(p.x + (unsigned long long)(t - (W - 1u - j)) * p.stride + c);
            else
                past[j] = seq.fresh ? aotx_f4{0, 0, 0, 0}
                                    : *(const aotx_f4 *)(kept + (unsigned long long)j * p.channels);
        }
        if (t == seq.start) {
            /* this thread alone reads the slot's rows, so it alone may write the new ones */
            const unsigned int len = seq.end - seq.start;
            aotx_f4 next[W - 1];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                const unsigned int back = W - 1u - j;
                if (len >= back) {
                    next[j] = *(const aotx_f4 *)(p.x + (unsigned long long)(seq.end - back) * p.stride + c);
                } else {
                    next[j] = past[0];
#pragma unroll
                    for (int m = 1; m < W - 1; ++m)
                        if (j + len == (unsigned int)m) next[j] = past[m];
                }
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
                *(aotx_f4 *)(kept + (unsigned long long)j * p.channels) = next[j];
        }
        /* four rows at a time, loaded before the first is used */
        for (; t < end; t += 4u) {
            aotx_f4 now[4];
#pragma unroll
            for (unsigned int u = 0; u < 4u; ++u) {
                const unsigned int r = t + u < end ? t + u : end - 1u;
                const aotx_f4 *from = (const aotx_f4 *)(p.x + (unsigned long long)r * p.stride + c);
                now[u] = STREAM > 1 ? __builtin_nontemporal_load(from) : *from;
            }
#pragma unroll
            for (unsigned int u = 0; u < 4u; ++u) {
                if (t + u >= end) break;
                aotx_u16x4 oh;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y = bias[e];
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) y += w[e][j] * past[j][e];
                    y += w[e][W - 1] * now[u][e];
                    oh[e] = aotx_f2h(aotx_silu(y));
                }
                aotx_u16x4 *to = (aotx_u16x4 *)(p.out + (unsigned long long)(t + u) * p.channels + c);
                if (STREAM > 0) __builtin_nontemporal_store(oh, to);
                else *to = oh;
#pragma unroll
                for (int j = 0; j < W - 2; ++j) past[j] = past[j + 1];
                past[W - 2] = now[u];
            }
        }
    }
}

extern "C" int aotx_delta_conv(const float *x, unsigned int stride, const float *w,
                               const float *bias, const unsigned int *offset,
                               const unsigned int *pos, const unsigned int *agent,
                               unsigned int seqs, unsigned int tokens, unsigned int channels,
                               unsigned int width, float *state, unsigned int slots, void *out,
                               void *stream)
{
    if (x == nullptr || w == nullptr || pos == nullptr || agent == nullptr || state == nullptr
        || out == nullptr)
        return 1;
    if (channels == 0u || channels % 4u != 0u || stride % 4u != 0u || stride < channels) return 1;
    if (width < 2u || width > 4u || channels > (1u << 20) || tokens > (1u << 20)) return 1;
    if (seqs > AOTX_SLOTS || slots == 0u || slots > AOTX_SLOTS) return 1;
    if ((unsigned long long)tokens * channels > (1ull << 37)) return 1;     /* threads of a launch: below 2^32 */
    if (offset == nullptr && seqs != tokens) return 1;
    if (!aotx_aligned16(x) || !aotx_aligned16(w) || !aotx_aligned16(bias) || !aotx_aligned16(state)
        || !aotx_aligned16(out))
        return 1;
    if (tokens == 0u || seqs == 0u) return 0;
    aotx_conv_args p;
    if ((p.seqs.faults = aotx_faults(stream)) == nullptr) return 1;
    p.x = x;
    p.w = w;
    p.bias = bias;
    p.state = state;
    p.out = (unsigned short *)out;
    p.stride = stride;
    p.channels = channels;
    p.blocks = (channels / 4u + 255u) / 256u;
    /* 4 workgroups a CU where there are rows for them, and 16 rows each from there on (8192
     * channels: 64 sequences of one row 5.5 us in runs of 1 against 27 in runs of 16; 512 rows 9.3
     * in runs of 4 and 12.8 in runs of 1; 8192 rows 87 in runs of 16, 85 of 64, 92 of 32) */
    p.run = tokens * p.blocks / 1024u;
    p.run = p.run < 1u ? 1u : p.run > 16u ? 16u : p.run;
    p.seqs.offset = offset;
    p.seqs.pos = pos;
    p.seqs.agent = agent;
    p.seqs.seqs = seqs;
    p.seqs.tokens = tokens;
    p.seqs.slots = slots;
    const dim3 grid((tokens + p.run - 1u) / p.run * p.blocks);
    hipStream_t s = aotx_stream(stream);
    /* What the caches would not hold until it is used again goes past them (8192 channels: 2048
     * rows 22.3 us with out past them, 25.7 without, 25.2 with x too; 8192 rows 86, 91 and 78). */
    const unsigned long long bytes = (unsigned long long)tokens * channels * 6u;
#define AOTX_CONV_GO(W)                                                                               \
    do {                                                                                              \
        if (bytes < (32ull << 20)) hipLaunchKernelGGL((aotx_delta_conv_kernel<W, 0>), grid, dim3(256), 0, s, p); \
        else if (bytes < (256ull << 20)) hipLaunchKernelGGL((aotx_delta_conv_kernel<W, 1>), grid, dim3(256), 0, s, p); \
        else hipLaunchKernelGGL((aotx_delta_conv_kernel<W, 2>), grid, dim3(256), 0, s, p);            \
    } while (0)
    if (width == 2u) AOTX_CONV_GO(2);
    else if (width == 3u) AOTX_CONV_GO(3);
    else AOTX_CONV_GO(4);
#undef AOTX_CONV_GO
    AOTX_LAUNCH_CHECK();
    return 0;
}
