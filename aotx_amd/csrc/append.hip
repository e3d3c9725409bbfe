/* The rows before and behind a full layer's first product: RMSNorm of fp32 rows (aotx_norm_rows),
 * and the head norm and turn of q, k and v rows with k and v going into the pages
 * (aotx_kv_append). Both are bound by memory: every value is read once in 16-byte loads and
 * written once.
 */
#include "rope_dev.h"
#include "../../include/aotx_layer.h"

/* ---------------------------------------------------------------------------------------
 * out = half(x / sqrt(mean(x^2) + eps) * w). A lane takes 8 values at a time and keeps them while
 * the row's sum is made.
 * ------------------------------------------------------------------------------------- */
struct aotx_norm_rows_args {
    const float *x, *w;
    unsigned short *out;
    unsigned int stride, tokens, width;
    float eps;
};

static __device__ __forceinline__ void aotx_norm_put(const aotx_norm_rows_args &p, const aotx_f4 &x0, const aotx_f4 &x1,
                                                     float scale, unsigned int t, unsigned int i)
{
    const aotx_f4 w0 = *(const aotx_f4 *)(p.w + i), w1 = *(const aotx_f4 *)(p.w + i + 4);
    aotx_u16x8 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = aotx_f2h(x0[e] * scale * w0[e]);
        y[e + 4] = aotx_f2h(x1[e] * scale * w1[e]);
    }
    *(aotx_u16x8 *)(p.out + (unsigned long long)t * p.width + i) = y;
}

/* Whether fp32 lost a row's sum of squares: past its end (or NaN), or so small that squares went under and eps does
 * not outweigh them. The row times aotx_squares_by, a power of two, and eps times that twice give the same norm
 * with squares between 2^-118 and 2^111 (a row has at most 2^15 values). */
static __device__ __forceinline__ bool aotx_squares_lost(float sum, float eps)
{
    return !(sum <= 3.4028234663852886e38f) || (sum < 0x1p-80f && eps < 0x1p-80f);
}
static __device__ __forceinline__ float aotx_squares_by(float sum) { return sum < 1.0f ? 0x1p90f : 0x1p-80f; }

/* A workgroup a row, N times 2048 values: all loads are under way before the first square, and a row is read
 * once. The memory bounds it: 8192 rows of 4096 take 37 us (201 MB at 5.4 TB/s, a part of x comes from the last
 * level's cache), 64 rows 2.6, of 16384 4.5. */
template <int N>
__global__ __launch_bounds__(256) void aotx_norm_rows_kernel(aotx_norm_rows_args p)
{
    __shared__ float share[4];
    const unsigned int t = blockIdx.x;
    const float *row = p.x + (unsigned long long)t * p.stride;
    aotx_f4 x[N][2];
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const unsigned int i = n * 2048u + threadIdx.x * 8u;
        if (i < p.width) {
            x[n][0] = *(const aotx_f4 *)(row + i);
            x[n][1] = *(const aotx_f4 *)(row + i + 4);
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (n * 2048u + threadIdx.x * 8u < p.width)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += x[n][0][e] * x[n][0][e] + x[n][1][e] * x[n][1][e];
    sum = aotx_wave_sum(sum);
    if ((threadIdx.x & 63u) == 0u) share[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = share[0] + share[1] + share[2] + share[3];
    const float scale = 1.0f / sqrtf(sum / (float)p.width + p.eps);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const unsigned int i = n * 2048u + threadIdx.x * 8u;
        if (i < p.width) aotx_norm_put(p, x[n][0], x[n][1], scale, t, i);
    }
    if ((threadIdx.x & ~63u) * 8u >= p.width || !aotx_squares_lost(sum, p.eps)) return;
    /* Every wave that has values reads the row again, for itself, and writes its values again: with the values kept for
     * this, the case looked at before the stores, or the whole workgroup in it, every row would pay (8192 of 8192 75 us
     * against 72.9, of 64 5.6 against 5.3). */
    const float by = aotx_squares_by(sum), eps = p.eps * by * by;
    sum = 0.0f;
#pragma unroll 1
    for (unsigned int i = (threadIdx.x & 63u) * 4u; i < p.width; i += 256u) {
        const aotx_f4 v = *(const aotx_f4 *)(row + i) * by;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += v[e] * v[e];
    }
    const float again = 1.0f / sqrtf(aotx_wave_sum(sum) / (float)p.width + eps);
#pragma unroll 1
    for (unsigned int i = threadIdx.x * 8u; i < p.width; i += 2048u)
        aotx_norm_put(p, *(const aotx_f4 *)(row + i) * by, *(const aotx_f4 *)(row + i + 4u) * by, again, t, i);
}

extern "C" int aotx_norm_rows(const float *x, unsigned int stride, const float *w, unsigned int tokens,
                              unsigned int width, float eps, void *out, void *stream)
{
    if (x == nullptr || w == nullptr || out == nullptr) return 1;
    if (width == 0u || width % 8u != 0u || width > 32768u || tokens > (1u << 20)) return 1;
    if (stride % 4u != 0u || stride < width || !(eps >= 0.0f)) return 1;
    if (!aotx_aligned16(x) || !aotx_aligned16(w) || !aotx_aligned16(out)) return 1;
    if (tokens == 0u) return 0;
    const aotx_norm_rows_args p = {x, w, (unsigned short *)out, stride, tokens, width, eps};
    hipStream_t s = aotx_stream(stream);
#define AOTX_ROWS_GO(N) hipLaunchKernelGGL(aotx_norm_rows_kernel<N>, dim3(tokens), dim3(256), 0, s, p)
    if (width <= 2048u) AOTX_ROWS_GO(1);
    else if (width <= 4096u) AOTX_ROWS_GO(2);
    else if (width <= 8192u) AOTX_ROWS_GO(4);
    else AOTX_ROWS_GO(16);
#undef AOTX_ROWS_GO
    AOTX_LAUNCH_CHECK();
    return 0;
}

/* ---------------------------------------------------------------------------------------
 * Rows into the pages. A workgroup takes one token: its sequence, the place of its row in the
 * pages and its pairs' sines once, then all heads, a lane 8 values of one, which are 4 whole pairs (or
 * 8 values past rope_dim); the angle as in aotx_rope_axes. Where there are fewer tokens than CUs, a token has
 * a workgroup for every 2048 of its values, which takes them in one pass and makes the sines again: 32 and 8 heads of
 * 128, 64 sequences of one row with head norms, take 3.7 us so and 5.1 by a workgroup each, one row 2.9 and 3.4. Past that
 * the memory bounds it: 512 rows 7.4 us, 8192 rows 59.4 (302 MB: 5.1 TB/s, as a copy). Loads for four
 * heads ahead take 512 rows down by 0.2 and 640 up by 0.5: left out.
 * ------------------------------------------------------------------------------------- */
struct aotx_append_args {
    const float *qkv, *q_norm, *k_norm, *factor;
    const unsigned int *place;
    const unsigned long long *page;
    unsigned short *q;
    unsigned int *row_pos, *row_agent;
    unsigned int stride, heads, kv_heads, pairs, rope_dim, axes, layer;
    float eps, gain;
    aotx_kvl_shape shape;
    aotx_seqs seqs;
    aotx_rope_turns rope;
};

/* The halves of position `pos` of K head 0, or null where the slot has no page for it. */
static __device__ __forceinline__ unsigned short *aotx_append_at(const aotx_append_args &p, unsigned int slot,
                                                                 unsigned long long pos)
{
    const unsigned long long block = pos / AOTX_KVL_BLOCK * p.shape.layers + p.layer;
    if (block >= (unsigned long long)AOTX_KV_PAGES_EACH * p.shape.blocks_page) return nullptr;
    const unsigned int b = (unsigned int)block, index = b / p.shape.blocks_page;
    const unsigned long long page = p.page[slot * AOTX_KV_PAGES_EACH + index];
    if (page == 0ull) return nullptr;
    return (unsigned short *)(page + AOTX_KVL_HEADER
                              + (unsigned long long)(b - index * p.shape.blocks_page) * p.shape.block_bytes)
         + (unsigned int)(pos % AOTX_KVL_BLOCK) * p.shape.head_dim;
}

template <int D>
__global__ __launch_bounds__(256) void aotx_append_kernel(aotx_append_args p)
{
    constexpr unsigned int L = D / 8, HEADS = 256 / L;  /* lanes a head, heads at once */
    __shared__ float cs[D / 2], sn[D / 2];
    const unsigned int t = blockIdx.x;
    const unsigned int half = p.rope_dim / 2u;
    const aotx_seq_lanes lanes = aotx_seqs_read(p.seqs);
    const unsigned long long mine = __ballot(lanes.start <= t && t < lanes.end);
    if (mine == 0ull) return;                           /* outside all sequences */
    const unsigned int i = (unsigned int)__builtin_ctzll(mine);
    const aotx_seq_view seq = aotx_seq_of(p.seqs, i, lanes);
    const unsigned long long pos = (unsigned long long)(unsigned int)__builtin_amdgcn_readlane((int)lanes.pos, (int)i)
                                 + (t - seq.start);
    const unsigned int total = p.heads + 2u * p.kv_heads;
    if (seq.refused) {
        if (threadIdx.x == 0u && blockIdx.y == 0u) {
            if (t == seq.start) atomicAdd(p.seqs.faults, 1u);
            if (p.row_pos != nullptr) {
                p.row_pos[t] = 0u;
                p.row_agent[t] = AOTX_SLOTS;
            }
        }
        for (unsigned int j = blockIdx.y * 256u + threadIdx.x; j < p.heads * L; j += gridDim.y * 256u)
            *(aotx_u16x8 *)(p.q + ((unsigned long long)t * p.heads * L + j) * 8u) = (aotx_u16x8)(0);
        return;
    }
    unsigned short *at = aotx_append_at(p, seq.slot, pos);
    if (threadIdx.x == 0u && blockIdx.y == 0u) {
        if (at == nullptr) atomicAdd(p.seqs.faults, 1u);
        if (p.row_pos != nullptr) {
            p.row_pos[t] = (unsigned int)pos;
            p.row_agent[t] = pos >> 32 == 0ull ? seq.slot : AOTX_SLOTS;   /* 32 bits hold the place, or it is none */
        }
    }
    if (threadIdx.x < half) {
        const unsigned int j = threadIdx.x;
        const double place = p.place != nullptr ? (double)p.place[(unsigned long long)t * p.axes + p.rope.axis[j]]
                                                : (double)pos;
        const float f = aotx_rope_angle(place, p.rope.turns[j], p.factor, j);
        cs[j] = p.gain * cospif(2.0f * f);
        sn[j] = p.gain * sinpif(2.0f * f);
    }
    __syncthreads();
    const unsigned int j = threadIdx.x % L;
    /* the two quads of values of this lane */
    unsigned int lo = 8u * j, hi = 8u * j + 4u;
    const bool turns = j * 8u < p.rope_dim;
    if (turns && p.pairs == AOTX_ROPE_PAIRS_SPLIT) {
        lo = 4u * j;
        hi = half + 4u * j;
    }
    float c[4], s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        c[e] = turns ? cs[4u * j + e] : 1.0f;
        s[e] = turns ? sn[4u * j + e] : 0.0f;
    }
    const float *row = p.qkv + (unsigned long long)t * p.stride;
    for (unsigned int h = blockIdx.y * HEADS + threadIdx.x / L; h < total; h += gridDim.y * HEADS) {
        const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
        if (!is_q && at == nullptr) break;
        aotx_f4 x0 = *(const aotx_f4 *)(row + h * D + lo);
        aotx_f4 x1 = *(const aotx_f4 *)(row + h * D + hi);
        const float *nw = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
        if (nw != nullptr) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += x0[e] * x0[e] + x1[e] * x1[e];
#pragma unroll
            for (int off = L / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, L);
            const float scale = 1.0f / sqrtf(sum * (1.0f / D) + p.eps);
            x0 = x0 * scale * *(const aotx_f4 *)(nw + lo);
            x1 = x1 * scale * *(const aotx_f4 *)(nw + hi);
        }
        aotx_u16x4 y0, y1;
        if (is_v || !turns) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y0[e] = aotx_f2h(x0[e]);
                y1[e] = aotx_f2h(x1[e]);
            }
        } else {
            aotx_rope_pairs(p.pairs, x0, x1, c, s, y0, y1);
        }
        /* in a block of the pages the K heads come first, then the V heads, 16 positions each */
        unsigned short *to = is_q ? p.q + ((unsigned long long)t * p.heads + h) * D
                                  : at + (unsigned long long)(h - p.heads) * (AOTX_KVL_BLOCK * D);
        *(aotx_u16x4 *)(to + lo) = y0;
        *(aotx_u16x4 *)(to + hi) = y1;
    }
}

extern "C" int aotx_kv_append(const float *qkv, unsigned int stride, const float *q_norm, const float *k_norm,
                              const aotx_rope_how *how, const float *factor, float gain,
                              const unsigned int *place, const unsigned int *offset, const unsigned int *pos,
                              const unsigned int *agent, unsigned int seqs, unsigned int tokens,
                              unsigned int heads, unsigned int kv_heads, unsigned int head_dim,
                              unsigned int layer, unsigned int layers, const unsigned long long *page, void *q,
                              unsigned int *row_pos, unsigned int *row_agent, void *stream)
{
    if (qkv == nullptr || how == nullptr || pos == nullptr || agent == nullptr || page == nullptr || q == nullptr)
        return 1;
    if ((row_pos == nullptr) != (row_agent == nullptr)) return 1;
    if (head_dim != 64u && head_dim != 128u) return 1;
    if (heads == 0u || heads > 1024u || kv_heads == 0u || kv_heads > 1024u || tokens > (1u << 20)) return 1;
    if (stride % 4u != 0u || stride < (heads + 2u * kv_heads) * head_dim) return 1;
    if (seqs > AOTX_SLOTS || (offset == nullptr && seqs != tokens)) return 1;
    if (!aotx_rope_ok(how, head_dim) || (place == nullptr && how->axes != 1u)) return 1;
    if (!(gain > 0.0f) || !isfinite(gain) || layer >= layers) return 1;
    if (!aotx_aligned16(qkv) || !aotx_aligned16(q_norm) || !aotx_aligned16(k_norm) || !aotx_aligned16(q)) return 1;
    aotx_append_args p;
    p.shape = aotx_kvl_make(layers, kv_heads, head_dim);
    if (p.shape.blocks_page == 0u) return 1;            /* a block that no page holds */
    if (tokens == 0u || seqs == 0u) return 0;
    p.seqs = {offset, pos, agent, seqs, tokens, AOTX_SLOTS, aotx_faults(stream)};
    if (p.seqs.faults == nullptr) return 1;
    p.qkv = qkv;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.factor = factor;
    p.place = place;
    p.page = page;
    p.q = (unsigned short *)q;
    p.row_pos = row_pos;
    p.row_agent = row_agent;
    p.stride = stride;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.pairs = how->pairs;
    p.rope_dim = how->rope_dim;
    p.axes = how->axes;
    p.layer = layer;
    p.eps = how->eps;
    p.gain = gain;
    aotx_rope_fill(how, &p.rope);
    hipStream_t s = aotx_stream(stream);
    const unsigned int each = ((heads + 2u * kv_heads) * head_dim + 2047u) / 2048u;
    const dim3 grid(tokens, tokens <= 256u ? each : 1u);
    if (head_dim == 128u) hipLaunchKernelGGL(aotx_append_kernel<128>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(aotx_append_kernel<64>, grid, dim3(256), 0, s, p);
    AOTX_LAUNCH_CHECK();
    return 0;
}
