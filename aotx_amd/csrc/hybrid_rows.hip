/* Row operators of hybrid models' layers: the gated head norm behind a linear layer's heads
 * (aotx_norm_gate) and the turn of q and k by several axes (aotx_rope_axes). Both are bound by
 * memory: every value is read once in 16-byte loads and written once.
 */
#include "delta_dev.h"
#include "../../include/aotx_hybrid.h"

#include <math.h>

/* ---------------------------------------------------------------------------------------
 * out = half(x * rsqrt(mean(x^2) + eps) * w * silu(z)). A lane takes 8 values of a row, whose sum
 * stays within a wave up to 512 values: no LDS and no barrier, and a row's values are read once.
 * 8192 rows of 32 heads of 128, 268 MB, in 48 us, 5.6 TB/s, the rate of a large copy; 64 rows 3.1
 * us, what a launch and one trip to memory take.
 * ------------------------------------------------------------------------------------- */
struct aotx_norm_gate_args {
    const unsigned short *x;
    const float *z, *w;
    unsigned short *out;
    unsigned int z_stride, heads, width;
    unsigned long long rows;
    float eps;
};

static __device__ __forceinline__ void aotx_gate_store(const aotx_norm_gate_args &p, const float *x,
                                                       float scale, unsigned long long row, unsigned int i)
{
    const unsigned long long t = row / p.heads, h = row % p.heads;
    const float *z = p.z + t * p.z_stride + h * p.width + i;
    const aotx_f4 z0 = *(const aotx_f4 *)z, z1 = *(const aotx_f4 *)(z + 4);
    const aotx_f4 w0 = *(const aotx_f4 *)(p.w + i), w1 = *(const aotx_f4 *)(p.w + i + 4);
    aotx_u16x8 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = aotx_f2h(x[e] * scale * w0[e] * aotx_silu(z0[e]));
        y[e + 4] = aotx_f2h(x[e + 4] * scale * w1[e] * aotx_silu(z1[e]));
    }
    *(aotx_u16x8 *)(p.out + row * p.width + i) = y;
}

/* A launch has less than 2^32 threads along x: the workgroups past AOTX_GATE_X of a row of the grid
 * are in the next. */
#define AOTX_GATE_X (1u << 20)

static __device__ __forceinline__ unsigned long long aotx_gate_block()
{
    return (unsigned long long)blockIdx.y * AOTX_GATE_X + blockIdx.x;
}

/* L lanes a row (a power of two, L * 8 >= width). */
template <int L>
__global__ __launch_bounds__(256) void aotx_norm_gate_kernel(aotx_norm_gate_args p)
{
    const unsigned long long row = aotx_gate_block() * (256u / L) + threadIdx.x / L;
    const unsigned int i = (threadIdx.x % L) * 8u;
    const bool live = row < p.rows && i < p.width;
    float x[8], sum = 0.0f;
    if (live) {
        const aotx_u16x8 v = *(const aotx_u16x8 *)(p.x + row * p.width + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = aotx_h2f(v[e]);
            sum += x[e] * x[e];
        }
    }
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (live) aotx_gate_store(p, x, 1.0f / sqrtf(sum / (float)p.width + p.eps), row, i);
}

/* A workgroup a row, for widths from 520 to 8192. */
__global__ __launch_bounds__(256) void aotx_norm_gate_wide_kernel(aotx_norm_gate_args p)
{
    __shared__ float share[4];
    const unsigned long long row = aotx_gate_block();
    if (row >= p.rows) return;
    float x[4][8], sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const unsigned int i = n * 2048u + threadIdx.x * 8u;
        if (i < p.width) {
            const aotx_u16x8 v = *(const aotx_u16x8 *)(p.x + row * p.width + i);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[n][e] = aotx_h2f(v[e]);
                sum += x[n][e] * x[n][e];
            }
        }
    }
    sum = aotx_wave_sum(sum);
    if ((threadIdx.x & 63u) == 0u) share[threadIdx.x >> 6] = sum;
    __syncthreads();                             /* every value of the row is read: out may be x */
    sum = share[0] + share[1] + share[2] + share[3];
    const float scale = 1.0f / sqrtf(sum / (float)p.width + p.eps);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const unsigned int i = n * 2048u + threadIdx.x * 8u;
        if (i < p.width) aotx_gate_store(p, x[n], scale, row, i);
    }
}

static dim3 aotx_gate_grid(unsigned long long blocks)
{
    return blocks <= AOTX_GATE_X ? dim3((unsigned int)blocks)
                                 : dim3(AOTX_GATE_X, (unsigned int)((blocks + AOTX_GATE_X - 1u) / AOTX_GATE_X));
}

extern "C" int aotx_norm_gate(const void *x, const float *z, unsigned int z_stride, const float *w,
                              unsigned int tokens, unsigned int heads, unsigned int width,
                              float eps, void *out, void *stream)
{
    if (x == nullptr || z == nullptr || w == nullptr || out == nullptr) return 1;
    if (width == 0u || width % 8u != 0u || width > 8192u || heads == 0u || heads > 65536u) return 1;
    if (z_stride % 4u != 0u || z_stride < (unsigned long long)heads * width) return 1;
    if (!(eps >= 0.0f) || tokens > (1u << 20)) return 1;
    if (!aotx_aligned16(x) || !aotx_aligned16(z) || !aotx_aligned16(w) || !aotx_aligned16(out)) return 1;
    aotx_norm_gate_args p;
    p.rows = (unsigned long long)tokens * heads;
    if (p.rows == 0ull) return 0;
    p.x = (const unsigned short *)x;
    p.z = z;
    p.w = w;
    p.out = (unsigned short *)out;
    p.z_stride = z_stride;
    p.heads = heads;
    p.width = width;
    p.eps = eps;
    hipStream_t s = aotx_stream(stream);
#define AOTX_GATE_GO(L) \
    hipLaunchKernelGGL(aotx_norm_gate_kernel<L>, aotx_gate_grid((p.rows + 256 / L - 1) / (256 / L)), dim3(256), 0, s, p)
    if (width <= 64u) AOTX_GATE_GO(8);
    else if (width <= 128u) AOTX_GATE_GO(16);
    else if (width <= 256u) AOTX_GATE_GO(32);
    else if (width <= 512u) AOTX_GATE_GO(64);
    else hipLaunchKernelGGL(aotx_norm_gate_wide_kernel, aotx_gate_grid(p.rows), dim3(256), 0, s, p);
#undef AOTX_GATE_GO
    AOTX_LAUNCH_CHECK();
    return 0;
}

/* ---------------------------------------------------------------------------------------
 * Rotary turn by several axes. Pair i of a row turns by place[axis(i)] theta^(-2i/r): in
 * turns, place * freq / (2 pi) is held in 64 bits and only its fraction goes on in 32, so an
 * angle is as exact at position 2^20 as at 1 (32 bits would leave it 0.06 off there). A
 * workgroup takes one token: its pairs' sines once, then all heads, a lane 8 values of one,
 * which are 4 whole pairs (or 8 values past rope_dim). 8192 rows of 32 + 16 heads of 128, 302 MB,
 * in 57 us, 5.3 TB/s, the rate of a large copy; 64 rows 4.9 us.
 * ------------------------------------------------------------------------------------- */
struct aotx_rope_axes_args {
    const float *qkv, *q_norm, *k_norm, *factor;
    const unsigned int *place;
    unsigned short *q, *k, *v;
    unsigned int stride, tokens, heads, kv_heads, pairs, rope_dim, axes;
    float eps;
    double turns[64];           /* of pair i at place 1: theta^(-2i/r) / (2 pi) */
    unsigned char axis[64];
};

template <int D>
__global__ __launch_bounds__(256) void aotx_rope_axes_kernel(aotx_rope_axes_args p)
{
    constexpr unsigned int L = D / 8, HEADS = 256 / L;  /* lanes a head, heads at once */
    __shared__ float cs[D / 2], sn[D / 2];
    const unsigned int t = blockIdx.x;
    const unsigned int half = p.rope_dim / 2u;
    if (threadIdx.x < half) {
        const unsigned int i = threadIdx.x;
        double a = (double)p.place[(unsigned long long)t * p.axes + p.axis[i]] * p.turns[i];
        if (p.factor != nullptr) a /= (double)p.factor[i];
        const float f = (float)(a - floor(a));          /* [0, 1] turns */
        cs[i] = cospif(2.0f * f);
        sn[i] = sinpif(2.0f * f);
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
    const unsigned int total = p.heads + 2u * p.kv_heads;
    const float *row = p.qkv + (unsigned long long)t * p.stride;
    for (unsigned int h = threadIdx.x / L; h < total; h += HEADS) {
        const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
        if (is_v && p.v == nullptr) break;
        aotx_f4 x0 = *(const aotx_f4 *)(row + (unsigned long long)h * D + lo);
        aotx_f4 x1 = *(const aotx_f4 *)(row + (unsigned long long)h * D + hi);
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
        } else if (p.pairs == AOTX_ROPE_PAIRS_SPLIT) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y0[e] = aotx_f2h(x0[e] * c[e] - x1[e] * s[e]);
                y1[e] = aotx_f2h(x0[e] * s[e] + x1[e] * c[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                y0[2 * e] = aotx_f2h(x0[2 * e] * c[e] - x0[2 * e + 1] * s[e]);
                y0[2 * e + 1] = aotx_f2h(x0[2 * e] * s[e] + x0[2 * e + 1] * c[e]);
                y1[2 * e] = aotx_f2h(x1[2 * e] * c[2 + e] - x1[2 * e + 1] * s[2 + e]);
                y1[2 * e + 1] = aotx_f2h(x1[2 * e] * s[2 + e] + x1[2 * e + 1] * c[2 + e]);
            }
        }
        unsigned short *to = is_q ? p.q + ((unsigned long long)t * p.heads + h) * D
            : is_v ? p.v + ((unsigned long long)t * p.kv_heads + (h - p.heads - p.kv_heads)) * D
                   : p.k + ((unsigned long long)t * p.kv_heads + (h - p.heads)) * D;
        *(aotx_u16x4 *)(to + lo) = y0;
        *(aotx_u16x4 *)(to + hi) = y1;
    }
}

extern "C" int aotx_rope_axes(const float *qkv, unsigned int stride, const float *q_norm,
                              const float *k_norm, const aotx_rope_how *how, const float *factor,
                              const unsigned int *place, unsigned int tokens, unsigned int heads,
                              unsigned int kv_heads, unsigned int head_dim, void *q, void *k,
                              void *v, void *stream)
{
    if (qkv == nullptr || how == nullptr || place == nullptr || q == nullptr) return 1;
    if (head_dim != 64u && head_dim != 128u) return 1;
    if (heads == 0u || heads > 1024u || kv_heads > 1024u || tokens > (1u << 20)) return 1;
    if (kv_heads == 0u ? (k != nullptr || v != nullptr) : k == nullptr) return 1;
    if (stride % 4u != 0u || stride < (heads + 2u * kv_heads) * head_dim) return 1;
    const unsigned int r = how->rope_dim;
    if (r == 0u || r % 8u != 0u || r > head_dim) return 1;
    if (how->pairs != AOTX_ROPE_PAIRS_SPLIT && how->pairs != AOTX_ROPE_PAIRS_ADJACENT) return 1;
    if (how->axes == 0u || how->axes > AOTX_ROPE_AXES_MAX) return 1;
    if (how->order != AOTX_ROPE_AXES_RUNS && how->order != AOTX_ROPE_AXES_TURN) return 1;
    if (!(how->theta > 0.0f) || !isfinite(how->theta) || !(how->eps >= 0.0f)) return 1;
    unsigned long long sum = 0u;
    for (unsigned int i = 0; i < how->axes; ++i) sum += how->span[i];
    if (sum != r / 2u) return 1;
    if (!aotx_aligned16(qkv) || !aotx_aligned16(q_norm) || !aotx_aligned16(k_norm) || !aotx_aligned16(q)
        || !aotx_aligned16(k) || !aotx_aligned16(v))
        return 1;
    if (tokens == 0u) return 0;
    aotx_rope_axes_args p;
    p.qkv = qkv;
    p.q_norm = q_norm;
    p.k_norm = k_norm;
    p.factor = factor;
    p.place = place;
    p.q = (unsigned short *)q;
    p.k = (unsigned short *)k;
    p.v = (unsigned short *)v;
    p.stride = stride;
    p.tokens = tokens;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.pairs = how->pairs;
    p.rope_dim = r;
    p.axes = how->axes;
    p.eps = how->eps;
    /* powers of one step: 64 products round by less than 2^-46 of a frequency */
    const double step = pow((double)how->theta, -2.0 / (double)r);
    double turn = 0.15915494309189533577;       /* 1 / (2 pi) */
    unsigned int axis = 0u, left = how->span[0];
    for (unsigned int i = 0; i < 64u; ++i, turn *= step) {
        p.turns[i] = turn;
        p.axis[i] = 0u;
        if (i >= r / 2u) continue;
        if (how->order == AOTX_ROPE_AXES_TURN) {
            const unsigned int a = i % how->axes;
            p.axis[i] = (unsigned char)(i < how->axes * how->span[a] ? a : 0u);
        } else {
            while (left == 0u) left = how->span[++axis];
            --left;
            p.axis[i] = (unsigned char)axis;
        }
    }
    hipStream_t s = aotx_stream(stream);
    if (head_dim == 128u) hipLaunchKernelGGL(aotx_rope_axes_kernel<128>, dim3(tokens), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(aotx_rope_axes_kernel<64>, dim3(tokens), dim3(256), 0, s, p);
    AOTX_LAUNCH_CHECK();
    return 0;
}
