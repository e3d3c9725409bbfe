/* The gated delta rule of linear layers: one token of each slot (aotx_delta_step) and
 * sequences of any length (aotx_delta_chunk).
 *
 * With unit rows q', k' (q' also over sqrt(d)), decay g and rate beta a head's state S
 * [d keys][d values] moves on by
 *   S <- exp(g) S;  u = beta (v - S^T k');  S <- S + k' u^T;  out = S^T q'.
 * Columns of S never meet, so a head's columns are shared out over workgroups freely.
 */
#include "delta_chunk.h"
#include "../../include/aotx_hybrid.h"

template <int D, int CS>
__global__ __launch_bounds__(256) void aotx_delta_rows_kernel(aotx_delta_args p)
{
    __shared__ aotx_delta_rows_lds<D, CS> lds;
    aotx_delta_by_rows<D, CS>(p, lds, blockIdx.x);
}

template <int D>
static void aotx_delta_rows(const aotx_delta_args &p, hipStream_t s)
{
    const unsigned int units = p.seqs.seqs * p.heads;
    /* wide slices read longer pieces of a row, narrow ones make more workgroups: a token of 64
     * slots, 32 heads of 128, 50.1 us in slices of 64 and 57.2 of 32, one of 1 slot 5.1 and 4.7 */
    if (units >= 256u)
        hipLaunchKernelGGL((aotx_delta_rows_kernel<D, 64>), dim3(units * (D / 64)), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((aotx_delta_rows_kernel<D, 32>), dim3(units * (D / 32)), dim3(256), 0, s, p);
    AOTX_LAUNCH_CHECK();
}

/* The arguments that both entry points check: 1 when refused. */
static int aotx_delta_fill(aotx_delta_args *p, const void *qkv, unsigned int stride, const float *a,
                           const float *b, unsigned int ab_stride, const float *decay,
                           const float *dt, const unsigned int *pos, const unsigned int *agent,
                           unsigned int seqs, unsigned int tokens, unsigned int key_heads,
                           unsigned int heads, unsigned int head_dim, float eps, float *state,
                           unsigned int slots, void *out)
{
    if (qkv == nullptr || a == nullptr || b == nullptr || decay == nullptr || dt == nullptr
        || pos == nullptr || agent == nullptr || state == nullptr || out == nullptr)
        return 1;
    if (head_dim != 64u && head_dim != 128u) return 1;
    if (heads == 0u || heads > 256u || key_heads == 0u || heads % key_heads != 0u) return 1;
    if (stride % 8u != 0u || stride < (2u * key_heads + heads) * head_dim || stride > (1u << 22)) return 1;
    if (ab_stride < heads || !(eps >= 1e-30f)) return 1;
    if (seqs > AOTX_SLOTS || slots == 0u || slots > AOTX_SLOTS || tokens > (1u << 20)) return 1;
    if (!aotx_aligned16(qkv) || !aotx_aligned16(state) || !aotx_aligned16(out)) return 1;
    p->qkv = (const unsigned short *)qkv;
    p->a = a;
    p->b = b;
    p->decay = decay;
    p->dt = dt;
    p->state = state;
    p->out = (unsigned short *)out;
    p->stride = stride;
    p->ab_stride = ab_stride;
    p->key_heads = key_heads;
    p->heads = heads;
    p->group = heads / key_heads;
    p->eps = eps;
    p->seqs.offset = nullptr;
    p->seqs.pos = pos;
    p->seqs.agent = agent;
    p->seqs.seqs = seqs;
    p->seqs.tokens = tokens;
    p->seqs.slots = slots;
    p->few = 0xFFFFFFFFu;
    return 0;
}

extern "C" int aotx_delta_step(const void *qkv, unsigned int stride, const float *a,
                               const float *b, unsigned int ab_stride, const float *decay,
                               const float *dt, const unsigned int *pos,
                               const unsigned int *agent, unsigned int tokens,
                               unsigned int key_heads, unsigned int heads, unsigned int head_dim,
                               float eps, float *state, unsigned int slots, void *out,
                               void *stream)
{
    aotx_delta_args p;
    if (aotx_delta_fill(&p, qkv, stride, a, b, ab_stride, decay, dt, pos, agent, tokens, tokens,
                        key_heads, heads, head_dim, eps, state, slots, out) != 0)
        return 1;
    if (tokens == 0u) return 0;
    if ((p.seqs.faults = aotx_faults(stream)) == nullptr) return 1;
    if (head_dim == 128u) aotx_delta_rows<128>(p, aotx_stream(stream));
    else aotx_delta_rows<64>(p, aotx_stream(stream));
    return 0;
}

/* Chunks of a call at most: every sequence ends with a part of one. */
static unsigned int aotx_delta_chunks_max(unsigned int tokens, unsigned int seqs)
{
    return tokens / AOTX_DELTA_CHUNK + seqs;
}

extern "C" unsigned long long aotx_delta_work(unsigned int tokens, unsigned int seqs,
                                              unsigned int heads, unsigned int head_dim)
{
    /* T, P and factors for every head, K and Q for as many key heads */
    return (unsigned long long)aotx_delta_chunks_max(tokens, seqs) * heads
        * (sizeof(aotx_delta_chunk_work) + (unsigned long long)head_dim * AOTX_DELTA_CHUNK * 4u);
}

template <int D>
static void aotx_delta_one(const aotx_delta_args &p, hipStream_t s)
{
    const unsigned int units = (p.seqs.seqs * p.heads + 7u) / 8u * 8u;
    hipLaunchKernelGGL((aotx_delta_short<D>), dim3(units * (D / 16)), dim3(320), 0, s, p);
    AOTX_LAUNCH_CHECK();
}

template <int D>
static void aotx_delta_chunked(const aotx_delta_args &p, hipStream_t s)
{
    /* The sequences of few rows, if any go row by row, are workgroups of this launch in small calls,
     * where one launch less counts, and a launch of their own where the registers that they add
     * would cost the chunks more (32 heads of 128: 2 sequences of 512 rows 34.0 us in one and 36.0
     * in two, 4 of 512 rows 65.4 and 61.6, 8 of 512 rows 117 and 113). */
    const unsigned int few = p.few != 0u ? p.seqs.seqs * p.heads * (D / 64) : 0u, blocks = p.chunks * p.heads;
    if (few != 0u && blocks <= 1536u) {
        hipLaunchKernelGGL((aotx_delta_within<D, true>), dim3(blocks + few), dim3(320), 0, s, p);
    } else {
        if (few != 0u) aotx_delta_rows<D>(p, s);
        hipLaunchKernelGGL((aotx_delta_within<D, false>), dim3(blocks), dim3(320), 0, s, p);
    }
    AOTX_LAUNCH_CHECK();
    const unsigned int units = (p.seqs.seqs * p.heads + 7u) / 8u * 8u;
    /* Two chunks' loads in flight where few workgroups share a CU or sequences are long; else one,
     * in so few registers that three workgroups do (32 heads of 128: 4 sequences of 2048 rows 214
     * us with two and 233 with one, 64 of 16 rows 244 and 185, 16 of 512 rows 235 and 232). Lines
     * are asked for early where the caches of the XCDs do not hold the workspace any more (8192
     * rows 226 us with and 231 without, 4 sequences of 2048 rows 208 and 214, 4096 rows 117 and
     * 114). */
    const dim3 grid(units * (D / 16));
    if (grid.x > 512u && p.seqs.tokens < 1024u * p.seqs.seqs)
        hipLaunchKernelGGL((aotx_delta_across<D, 1>), grid, dim3(256), 0, s, p);
    else if ((unsigned long long)p.chunks * p.heads * sizeof(aotx_delta_chunk_work) < (80ull << 20))
        hipLaunchKernelGGL((aotx_delta_across<D, 2>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((aotx_delta_across<D, 3>), grid, dim3(256), 0, s, p);
    AOTX_LAUNCH_CHECK();
}

extern "C" int aotx_delta_chunk(const void *qkv, unsigned int stride, const float *a,
                                const float *b, unsigned int ab_stride, const float *decay,
                                const float *dt, const unsigned int *offset,
                                const unsigned int *pos, const unsigned int *agent,
                                unsigned int seqs, unsigned int tokens, unsigned int key_heads,
                                unsigned int heads, unsigned int head_dim, float eps,
                                float *state, unsigned int slots, void *work,
                                unsigned long long work_bytes, void *out, void *stream)
{
    aotx_delta_args p;
    if (aotx_delta_fill(&p, qkv, stride, a, b, ab_stride, decay, dt, pos, agent, seqs, tokens,
                        key_heads, heads, head_dim, eps, state, slots, out) != 0)
        return 1;
    if (offset == nullptr || work == nullptr || ((uintptr_t)work & 255u) != 0u) return 1;
    if (work_bytes < aotx_delta_work(tokens, seqs, heads, head_dim)) return 1;
    if (tokens == 0u || seqs == 0u) return 0;
    if ((p.seqs.faults = aotx_faults(stream)) == nullptr) return 1;
    p.seqs.offset = offset;
    p.chunks = aotx_delta_chunks_max(tokens, seqs);
    p.work = (aotx_delta_chunk_work *)work;
    p.rows = (aotx_h8 *)(p.work + (unsigned long long)p.chunks * heads);
    /* Sequences of few rows go row by row: no matrices to make first, and a decode row beside a
     * prompt costs what a step does. A row takes 1.7 us, a chunk 12 if the chip is idle beside (32
     * heads of 128: 4 rows 9.9 us and 12.0, 8 rows 17.0 and 12.0); a chip full of sequences is kept
     * busy longer by chunks (64 sequences of 8 rows 136 us row by row and 189 in chunks, of 12 rows
     * 175 and 190). */
    p.few = seqs * heads >= 1024u ? 12u : 4u;
    /* Calls of up to 64 rows in all go in one launch while each workgroup of it has a CU (32 heads of
     * 128: 40 rows 8.6 us, in two launches 12.5; 2 sequences of 32 rows 15.5 and 14.4, 4 of 16 rows
     * 27.7 and 19.8), where 3 rows take no longer than row by row (8.1 us and 8.2). */
    const bool one = tokens <= AOTX_DELTA_CHUNK && seqs * heads * (head_dim / 16u) <= 256u;
    hipStream_t s = aotx_stream(stream);
    if (tokens <= (one && seqs == 1u ? 2u : p.few))
        head_dim == 128u ? aotx_delta_rows<128>(p, s) : aotx_delta_rows<64>(p, s);
    else if (one) head_dim == 128u ? aotx_delta_one<128>(p, s) : aotx_delta_one<64>(p, s);
    else {
        /* The lengths are the device's: of a call's one sequence, whatever the rows that there is room
         * for. It goes in chunks at any length, so that no workgroups wait beside for few rows. */
        if (seqs == 1u) p.few = 0u;
        head_dim == 128u ? aotx_delta_chunked<128>(p, s) : aotx_delta_chunked<64>(p, s);
    }
    return 0;
}
