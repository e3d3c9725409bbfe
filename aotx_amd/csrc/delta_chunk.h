/* The chunked form of the gated delta rule (aotx_delta_chunk): device code of its two kernels.
 *
 * Within a chunk of 64 rows of one head, with K, Q the raw rows, V the values, r_k and r_q the
 * rows' inverse lengths (r_q with 1 / sqrt(d)), G the running sum of g, the rule unrolls to
 *   M_ij = beta_i r_k,i r_k,j (K_i . K_j) exp(G_i - G_j) for i > j,   T = (1 + M)^-1 diag(beta)
 *   U = T (V - diag(exp(G) r_k) K S)
 *   out = diag(exp(G) r_q) Q S + P U,   P_ij = r_q,i r_k,j (Q_i . K_j) exp(G_i - G_j) for i >= j
 *   S <- exp(G_last) S + K^T diag(r_k exp(G_last - G)) U
 * T and P need no state: aotx_delta_within makes them for every chunk at once. What is left,
 * aotx_delta_across, walks a sequence's chunks with a slice of columns of S in registers.
 *
 * Numbers. K, Q and V are fp16 and enter the matrix cores as they are; S, U, X = V - K S, T and
 * P enter as two fp16 parts (high and rest, 22 bits), so that their products are as good as
 * fp32 ones at three times the work of plain fp16 instead of sixteen times for fp32 matrix
 * instructions. The parts have fp16's range: T and P are at most 1 (the rule only ever takes
 * away from what a unit key finds), K is scaled to a length of 1 to 2 by a power of two where
 * its scale goes into U, and S, X and U are scaled by a power of two for every column that
 * follows from the column's largest entries a chunk before: |S| grows by at most the sum of 64
 * values' lengths in a chunk, so 2^7 of headroom is enough, and 15 - 7 bits above 1 leave the rest
 * part's smallest step, 2^-24, below 2^-31 of the largest entry.
 *
 * A row whose K, a or b is no number is taken out (its K, g and beta are zeros) and remembered:
 * from that row on, out and the state are NaN; the same for one column from a bad value in V on.
 */
#ifndef AOTX_DELTA_CHUNK_H
#define AOTX_DELTA_CHUNK_H

#include "delta_dev.h"

typedef _Float16 aotx_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 aotx_h8 __attribute__((ext_vector_type(8)));

#define AOTX_DELTA_CHUNK 64u

/* What aotx_delta_within leaves of one chunk and head: matrix operands in the order that a wave
 * loads them, 16 bytes a lane. Row tile w (16 rows), step s (32 columns): lane (m, g) holds row
 * 16 w + m, columns 32 s + 16 (e / 4) + 4 g + e % 4 for e < 8, which is the order in which a
 * wave's accumulators of two row tiles make the other operand. */
struct aotx_delta_chunk_work {
    aotx_h8 p_hi[4][2][64], p_lo[4][2][64], t_hi[4][2][64], t_lo[4][2][64];
    float of_k[64];         /* exp(G) r_k */
    float of_q[64];         /* exp(G) r_q */
    float of_u[64];         /* exp(G_last - G) r_k 2^e; K^T of that row is over 2^e */
    float fade;             /* exp(G_last) */
    unsigned int bad;       /* first row that is taken out, 64 for none */
    unsigned int pad[62];
};

struct aotx_delta_args {
    const unsigned short *qkv;
    const float *a, *b, *decay, *dt;
    float *state;
    unsigned short *out;
    unsigned int stride, ab_stride;
    unsigned int key_heads, heads, group;
    float eps;
    aotx_seqs seqs;
    /* chunks */
    aotx_delta_chunk_work *work;    /* [chunks][heads] */
    aotx_h8 *kt;                    /* [chunks][key_heads][d / 16][2][64]: K^T, scaled rows */
    unsigned int chunks;            /* at most: rows / 64 + sequences */
};

static __device__ __forceinline__ aotx_h8 aotx_h8_of(aotx_u16x8 v) { return __builtin_bit_cast(aotx_h8, v); }

/* x = hi + lo to 22 bits. x has to be one rounded number: where the compiler fuses the product
 * that makes x into one of its two uses, the parts belong to different roundings. */
static __device__ __forceinline__ void aotx_split(float x, _Float16 *hi, _Float16 *lo)
{
    asm("" : "+v"(x));
    *hi = (_Float16)x;
    *lo = (_Float16)(x - (float)*hi);
}

static __device__ __forceinline__ aotx_f4 aotx_mma(aotx_h8 a, aotx_h8 b, aotx_f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

/* Chunks of sequence `lane` and of the sequences before it, from the lanes' rows. */
static __device__ __forceinline__ void aotx_delta_chunks(unsigned int b, unsigned int e, unsigned int *mine,
                                                         unsigned int *before)
{
    const unsigned int lane = threadIdx.x & 63u;
    const unsigned int n = (e - b + AOTX_DELTA_CHUNK - 1u) / AOTX_DELTA_CHUNK;
    unsigned int sum = n;
    for (unsigned int off = 1u; off < 64u; off <<= 1) {
        const unsigned int o = (unsigned int)__shfl_up((int)sum, off, 64);
        if (lane >= off) sum += o;
    }
    *mine = n;
    *before = sum - n;
}

/* Place of column j in a row of a matrix that is laid out for 16-byte operand reads. */
static __device__ __forceinline__ unsigned int aotx_delta_place(unsigned int j)
{
    return (j & ~31u) + ((j >> 2) & 3u) * 8u + ((j >> 4) & 1u) * 4u + (j & 3u);
}

/* ---------------------------------------------------------------------------------------
 * T, P, K^T and the row factors of one chunk and head; a workgroup of four waves, wave w has
 * rows 16 w .. 16 w + 15.
 * ------------------------------------------------------------------------------------- */
template <int D>
__global__ __launch_bounds__(256) void aotx_delta_within(aotx_delta_args p)
{
    constexpr int KS = D / 32;
    __shared__ aotx_h8 kfrag[4][KS][64];
    __shared__ __align__(16) float M[64][68];
    __shared__ __align__(16) float Dm[4][16][20];
    __shared__ __align__(16) unsigned short tp[2][64][72];
    __shared__ float ghi[64], glo[64], beta[64], rk[64], rq[64], ks[64];
    __shared__ unsigned int badk[4], badg;
    const unsigned int lane = threadIdx.x & 63u, w = threadIdx.x >> 6, m = lane & 15u, g = lane >> 4;
    const unsigned int c = blockIdx.x / p.heads, h = blockIdx.x % p.heads;

    unsigned int b, e, mine, before;
    aotx_seq_rows(p.seqs, &b, &e);
    aotx_delta_chunks(b, e, &mine, &before);
    const unsigned int i = (unsigned int)__popcll(__ballot(lane < p.seqs.seqs && before + mine <= c));
    if (i >= p.seqs.seqs) return;
    const aotx_seq_view seq = aotx_seq_of(p.seqs, i, b, e);
    if (seq.refused) return;
    const unsigned int r0 = seq.start + (c - (unsigned int)__builtin_amdgcn_readlane((int)before, (int)i)) * 64u;
    const unsigned int n = seq.end - r0 < 64u ? seq.end - r0 : 64u;

    /* rows of K and Q, 8 columns 32 s + 8 g .. of row 16 w + m */
    const unsigned int kh = h / p.group;
    const unsigned int row = 16u * w + m;
    aotx_h8 kf[KS], qf[KS];
    float kk = 0.0f, qq = 0.0f;
    {
        const unsigned short *q = p.qkv + (unsigned long long)(r0 + (row < n ? row : n - 1u)) * p.stride + kh * D + 8u * g;
        const unsigned short *k = q + (unsigned long long)p.key_heads * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kf[s] = aotx_h8_of(*(const aotx_u16x8 *)(k + 32 * s));
            qf[s] = aotx_h8_of(*(const aotx_u16x8 *)(q + 32 * s));
        }
    }
    /* gates, a row a lane (every wave for itself; wave 0 keeps them) */
    const unsigned int gr = r0 + (lane < n ? lane : n - 1u);
    float gate = aotx_delta_gate(p.a[(unsigned long long)gr * p.ab_stride + h], p.dt[h], p.decay[h]);
    float rate = 1.0f / (1.0f + expf(-p.b[(unsigned long long)gr * p.ab_stride + h]));
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int v = 0; v < 8; ++v) {
            kk += (float)kf[s][v] * (float)kf[s][v];
            qq += (float)qf[s][v] * (float)qf[s][v];
        }
    kk += __shfl_xor(kk, 16, 64);
    kk += __shfl_xor(kk, 32, 64);
    qq += __shfl_xor(qq, 16, 64);
    qq += __shfl_xor(qq, 32, 64);
    const bool out_of = row >= n, bad = !out_of && !(kk < __builtin_inff());
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        if (out_of || bad) kf[s] = aotx_h8{0, 0, 0, 0, 0, 0, 0, 0};
        if (out_of) qf[s] = aotx_h8{0, 0, 0, 0, 0, 0, 0, 0};
        kfrag[w][s][lane] = kf[s];
    }
    const unsigned long long badrows = __ballot(bad) & 0xFFFFull;
    if (lane == 0u) badk[w] = badrows != 0ull ? 16u * w + (unsigned int)__builtin_ctzll(badrows) : 64u;
    if (g == 0u) {
        if (out_of || bad) kk = 0.0f;
        if (out_of) qq = 0.0f;
        const float len = sqrtf(kk + p.eps);
        int ex;
        (void)frexpf(len, &ex);
        rk[row] = 1.0f / len;
        ks[row] = ldexpf(1.0f, -ex);
        rq[row] = 1.0f / sqrtf(qq + p.eps) * (D == 128 ? 0.08838834764831845f : 0.125f);
    }
    {
        const bool badgate = lane < n && (gate != gate || rate != rate);
        const unsigned long long badgates = __ballot(badgate);
        if (lane >= n || badgate) gate = rate = 0.0f;
        /* sums of g in 64 bits, kept as two floats: differences of far sums stay exact */
        double sum = (double)gate;
        for (unsigned int off = 1u; off < 64u; off <<= 1) {
            const double o = __shfl_up(sum, off, 64);
            if (lane >= off) sum += o;
        }
        if (w == 0u) {
            ghi[lane] = (float)sum;
            glo[lane] = (float)(sum - (double)(float)sum);
            beta[lane] = rate;
            if (lane == 0u) badg = badgates != 0ull ? (unsigned int)__builtin_ctzll(badgates) : 64u;
        }
    }
    __syncthreads();

    aotx_delta_chunk_work *to = p.work + (unsigned long long)c * p.heads + h;
    if (w == 0u) {
        const float last = (ghi[63] - ghi[lane]) + (glo[63] - glo[lane]), all = expf(ghi[lane]);
        to->of_k[lane] = all * rk[lane];
        to->of_q[lane] = all * rq[lane];
        to->of_u[lane] = expf(last) * rk[lane] / ks[lane];
        if (lane == 0u) {
            unsigned int first = badg;
            for (int v = 0; v < 4; ++v) first = badk[v] < first ? badk[v] : first;
            to->fade = expf(ghi[63]);
            to->bad = first;
        }
    }

    /* K K^T and Q K^T of this wave's rows, and M and P from them */
    const unsigned int i0 = 16u * w + 4u * g;
    const aotx_f4 gi = *(const aotx_f4 *)&ghi[i0], gl = *(const aotx_f4 *)&glo[i0], bi = *(const aotx_f4 *)&beta[i0],
                  rki = *(const aotx_f4 *)&rk[i0], rqi = *(const aotx_f4 *)&rq[i0];
#pragma unroll
    for (unsigned int jt = 0; jt < 4u; ++jt) {
        const unsigned int j = 16u * jt + m, at = aotx_delta_place(j);
        if (jt > w) {
            if (jt == (w | 1u))
#pragma unroll
                for (int r = 0; r < 4; ++r) tp[0][i0 + r][at] = tp[1][i0 + r][at] = 0;
            continue;
        }
        aotx_f4 kks = {0, 0, 0, 0}, qks = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const aotx_h8 kj = kfrag[jt][s][lane];
            kks = aotx_mma(kf[s], kj, kks);
            qks = aotx_mma(qf[s], kj, qks);
        }
        const float gj = ghi[j], gjl = glo[j], rkj = rk[j];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned int ii = i0 + r;
            const float fade = expf((gi[r] - gj) + (gl[r] - gjl)) * rkj;
            M[ii][j] = ii > j ? bi[r] * rki[r] * kks[r] * fade : 0.0f;
            _Float16 hi, lo;
            aotx_split(ii >= j ? rqi[r] * qks[r] * fade : 0.0f, &hi, &lo);
            tp[0][ii][at] = __builtin_bit_cast(unsigned short, hi);
            tp[1][ii][at] = __builtin_bit_cast(unsigned short, lo);
        }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (unsigned int s = 0; s < 2u; ++s) {
        if (s > w / 2u) continue;
        to->p_hi[w][s][lane] = *(const aotx_h8 *)&tp[0][row][32u * s + 8u * g];
        to->p_lo[w][s][lane] = *(const aotx_h8 *)&tp[1][row][32u * s + 8u * g];
    }

    /* inverse of the diagonal block by substitution, a column a lane */
    {
        float x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float v = m == (unsigned int)r ? 1.0f : 0.0f;
#pragma unroll
            for (int q = 0; q < r; ++q) v -= M[16u * w + r][16u * w + q] * x[q];
            x[r] = v;
        }
        if (g == 0u)
#pragma unroll
            for (int r = 0; r < 16; ++r) Dm[w][r][m] = x[r];
    }
    __syncthreads();

    /* Column w of blocks of the inverse, downwards: T_b = -D_b (sum of M_bq T_q). A block in
     * accumulator order is the right operand of the next product as it stands. */
    aotx_f4 tc[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) tc[0][r] = Dm[w][4u * g + r][m];
#pragma unroll
    for (unsigned int off = 1; off < 4u; ++off) {
        const unsigned int bt = w + off;
        if (bt > 3u) break;
        aotx_f4 acc = {0, 0, 0, 0};
#pragma unroll
        for (unsigned int q = 0; q < off; ++q) {
            const aotx_f4 a = *(const aotx_f4 *)&M[16u * bt + m][16u * (w + q) + 4u * g];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], tc[q][r], acc, 0, 0, 0);
        }
        const aotx_f4 a = *(const aotx_f4 *)&Dm[bt][m][4u * g];
        aotx_f4 t = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 4; ++r) t = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], -acc[r], t, 0, 0, 0);
        tc[off] = t;
    }
    {
        const unsigned int j = 16u * w + m, at = aotx_delta_place(j);
        const float bj = beta[j];
#pragma unroll
        for (unsigned int off = 0; off < 4u; ++off) {
            const unsigned int bt = w + off;
            if (bt > 3u) break;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                _Float16 hi, lo;
                aotx_split(tc[off][r] * bj, &hi, &lo);
                tp[0][16u * bt + 4u * g + r][at] = __builtin_bit_cast(unsigned short, hi);
                tp[1][16u * bt + 4u * g + r][at] = __builtin_bit_cast(unsigned short, lo);
            }
        }
        if (w & 1u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                tp[0][16u * (w - 1u) + 4u * g + r][at] = tp[1][16u * (w - 1u) + 4u * g + r][at] = 0;
    }
    /* K^T for the state's update: rows of the identity pick its columns, which come out with
     * the rows of K along a lane's registers, the order that operand needs */
    if (h % p.group == 0u) {
        const unsigned int s = w & 1u;
        aotx_h8 *kt = p.kt + ((unsigned long long)c * p.key_heads + kh) * (D / 16) * 2 * 64;
#pragma unroll
        for (unsigned int v = 0; v < D / 32u; ++v) {
            const unsigned int t = (w >> 1) * (D / 32u) + v, st = t >> 1;
            aotx_h8 pick;
#pragma unroll
            for (unsigned int x = 0; x < 8u; ++x)
                pick[x] = g == (m >> 2) && x == 4u * (t & 1u) + (m & 3u) ? (_Float16)1.0f : (_Float16)0.0f;
            aotx_h8 o;
#pragma unroll
            for (unsigned int half = 0; half < 2u; ++half) {
                const aotx_f4 acc = aotx_mma(kfrag[2u * s + half][st][lane], pick, aotx_f4{0, 0, 0, 0});
                const aotx_f4 sc = *(const aotx_f4 *)&ks[32u * s + 16u * half + 4u * g];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[4 * half + r] = (_Float16)(acc[r] * sc[r]);
            }
            kt[(t * 2u + s) * 64u + lane] = o;
        }
    }
    __syncthreads();
#pragma unroll
    for (unsigned int s = 0; s < 2u; ++s) {
        if (s > w / 2u) continue;
        to->t_hi[w][s][lane] = *(const aotx_h8 *)&tp[0][row][32u * s + 8u * g];
        to->t_lo[w][s][lane] = *(const aotx_h8 *)&tp[1][row][32u * s + 8u * g];
    }
}

/* ---------------------------------------------------------------------------------------
 * The walk over a sequence's chunks. A workgroup has 16 NT columns of one head's S: wave w the
 * rows of S that one step of K S takes (D / 4 of them, in accumulators), and rows 16 w ..
 * 16 w + 15 of the chunk. S, X and U pass between the waves through LDS as operands, a barrier
 * each; everything else a chunk needs is loaded into registers while the one before is worked on.
 * Row x of tile t of S is key 32 (t / 2) + 8 (x / 4) + 4 (t % 2) + x % 4, so that two tiles'
 * accumulators hold keys 8 g .. 8 g + 7 of a step, as 16 bytes of a row of K do.
 * ------------------------------------------------------------------------------------- */
template <int D, int NT>
struct aotx_delta_tile {
    static constexpr int KS = D / 32, TW = D / 64;
    aotx_h8 k[KS], q[KS], th[2], tl[2], ph[2], pl[2], kt[TW][2];
    unsigned short v[4][NT];
    aotx_f4 of_k, of_q, of_u;
    float fade;
    unsigned int bad;
};

template <int D, int NT>
static __device__ __forceinline__ void aotx_delta_load(aotx_delta_tile<D, NT> &x, const aotx_delta_args &p,
                                                       unsigned int c, unsigned int r0, unsigned int n, unsigned int h,
                                                       unsigned int col, unsigned int w, unsigned int m, unsigned int g)
{
    constexpr int KS = D / 32, TW = D / 64;
    const unsigned int lane = 16u * g + m, kh = h / p.group;
    const unsigned int row = 16u * w + m;
    const unsigned short *q = p.qkv + (unsigned long long)(r0 + (row < n ? row : n - 1u)) * p.stride + kh * D + 8u * g;
    const unsigned short *k = q + (unsigned long long)p.key_heads * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        x.k[s] = aotx_h8_of(*(const aotx_u16x8 *)(k + 32 * s));
        x.q[s] = aotx_h8_of(*(const aotx_u16x8 *)(q + 32 * s));
    }
    const aotx_delta_chunk_work *from = p.work + (unsigned long long)c * p.heads + h;
#pragma unroll
    for (unsigned int s = 0; s < 2u; ++s) {
        if (s > w / 2u) continue;
        x.th[s] = from->t_hi[w][s][lane];
        x.tl[s] = from->t_lo[w][s][lane];
        x.ph[s] = from->p_hi[w][s][lane];
        x.pl[s] = from->p_lo[w][s][lane];
    }
    const aotx_h8 *kt = p.kt + ((unsigned long long)c * p.key_heads + kh) * (D / 16) * 2 * 64;
#pragma unroll
    for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s) x.kt[t][s] = kt[((w * TW + t) * 2 + s) * 64u + lane];
    const unsigned int i0 = 16u * w + 4u * g;
    const unsigned short *v = p.qkv + 2ull * p.key_heads * D + (unsigned long long)h * D + col;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t)
            x.v[r][t] = v[(unsigned long long)(r0 + (i0 + r < n ? i0 + r : n - 1u)) * p.stride + t];
    x.of_k = *(const aotx_f4 *)&from->of_k[i0];
    x.of_q = *(const aotx_f4 *)&from->of_q[i0];
    x.of_u = *(const aotx_f4 *)&from->of_u[i0];
    x.fade = from->fade;
    x.bad = from->bad;
}

/* exponent of |x|: |x| < 2^(e + 1) */
static __device__ __forceinline__ int aotx_exponent(float x)
{
    return (int)((__float_as_uint(x) >> 23) & 0xFFu) - 127;
}

template <int D, int NT>
__global__ __launch_bounds__(256) void aotx_delta_across(aotx_delta_args p)
{
    constexpr int KS = D / 32, TW = D / 64, SLICES = D / (16 * NT);
    __shared__ aotx_h8 Sx[KS][2][NT][64];           /* step of keys, part, tile of columns */
    __shared__ aotx_h8 Xx[2][2][NT][64];            /* step of rows, part, tile of columns */
    __shared__ aotx_h8 Ux[2][2][NT][64], Vx[2][2][NT][64];
    __shared__ int post[2][4][16 * NT];             /* exponents, first bad rows; by wave */
    const unsigned int lane = threadIdx.x & 63u, w = threadIdx.x >> 6, m = lane & 15u, g = lane >> 4;
    /* the slices of a head go to one XCD (workgroup b runs on XCD b % 8), whose L2 then holds
     * what they share */
    const unsigned int units = p.seqs.seqs * p.heads;
    const unsigned int unit = blockIdx.x / (8u * SLICES) * 8u + blockIdx.x % 8u;
    const unsigned int slice = blockIdx.x / 8u % SLICES;
    if (unit >= units) return;
    const unsigned int i = unit / p.heads, h = unit % p.heads;
    unsigned int b, e, mine, before;
    aotx_seq_rows(p.seqs, &b, &e);
    aotx_delta_chunks(b, e, &mine, &before);
    const aotx_seq_view seq = aotx_seq_of(p.seqs, i, b, e);
    const unsigned int c0 = (unsigned int)__builtin_amdgcn_readlane((int)before, (int)i);
    if (seq.start >= seq.end) return;
    const unsigned int col = slice * 16u * NT + m * NT;     /* this lane's NT columns */
    const unsigned long long width = (unsigned long long)p.heads * D;
    unsigned short *out = p.out + (unsigned long long)h * D + col;
    if (seq.refused) {
        if (threadIdx.x == 0u && slice == 0u && h == 0u) atomicAdd(p.seqs.faults, 1u);
        for (unsigned int t = seq.start + threadIdx.x / 16u; t < seq.end; t += 16u)
#pragma unroll
            for (int u = 0; u < NT; ++u) out[t * width + u] = 0;
        return;
    }
    const unsigned int chunks = (seq.end - seq.start + 63u) / 64u;
    const unsigned int i0 = 16u * w + 4u * g;

    aotx_f4 S[TW][NT];
    float *sp = p.state + ((unsigned long long)seq.slot * p.heads + h) * D * D + col;
#pragma unroll
    for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned int tile = w * TW + t;
            const unsigned int key = 32u * (tile >> 1) + 8u * g + 4u * (tile & 1u) + r;
#pragma unroll
            for (int u = 0; u < NT; ++u) S[t][u][r] = seq.fresh ? 0.0f : sp[key * D + u];
        }

    aotx_delta_tile<D, NT> now, next;
    aotx_delta_load<D, NT>(now, p, c0, seq.start, seq.end - seq.start < 64u ? seq.end - seq.start : 64u, h, col, w, m, g);

    /* This wave's share of the next chunk's column scales and bad rows, into `post`. */
    auto tell = [&](const aotx_delta_tile<D, NT> &x, unsigned int n, const aotx_f4 (&s)[TW][NT], const int (&floor)[NT],
                    int (&own)[NT]) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float ms = 0.0f, mv = 0.0f;
            unsigned int first = 64u;
#pragma unroll
            for (int t = 0; t < TW; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) ms = fmaxf(ms, fabsf(s[t][u][r]));
#pragma unroll
            for (int r = 3; r >= 0; --r) {
                const float v = fabsf(aotx_h2f(x.v[r][u]));
                if (v < __builtin_inff()) mv = fmaxf(mv, v);
                else if (i0 + r < n) first = i0 + r;
            }
            ms = fmaxf(ms, __shfl_xor(ms, 16, 64));
            ms = fmaxf(ms, __shfl_xor(ms, 32, 64));
            mv = fmaxf(mv, __shfl_xor(mv, 16, 64));
            mv = fmaxf(mv, __shfl_xor(mv, 32, 64));
            unsigned int o = (unsigned int)__shfl_xor((int)first, 16, 64);
            first = o < first ? o : first;
            o = (unsigned int)__shfl_xor((int)first, 32, 64);
            first = o < first ? o : first;
            own[u] = aotx_exponent(mv) + 8;
            int ex = aotx_exponent(ms) + 5;
            ex = ex > own[u] ? ex : own[u];
            ex = ex > floor[u] ? ex : floor[u];
            if (g == 0u) {
                post[0][w][m * NT + u] = ex;
                post[1][w][m * NT + u] = (int)first;
            }
        }
    };
    float up[NT], down[NT];             /* this chunk's column scales, a power of two and its inverse */
    unsigned int badv[NT];
    auto heard = [&]() {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            int ex = post[0][0][m * NT + u];
            unsigned int first = (unsigned int)post[1][0][m * NT + u];
#pragma unroll
            for (int v = 1; v < 4; ++v) {
                const int o = post[0][v][m * NT + u];
                ex = o > ex ? o : ex;
                const unsigned int f = (unsigned int)post[1][v][m * NT + u];
                first = f < first ? f : first;
            }
            ex = 14 - ex;
            ex = ex > 100 ? 100 : ex < -100 ? -100 : ex;
            up[u] = __uint_as_float((unsigned int)(ex + 127) << 23);
            down[u] = __uint_as_float((unsigned int)(127 - ex) << 23);
            badv[u] = first;
        }
    };
    int vex[NT], none[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) none[u] = -1000;
    tell(now, seq.end - seq.start < 64u ? seq.end - seq.start : 64u, S, none, vex);
    __syncthreads();
    heard();

    for (unsigned int c = 0; c < chunks; ++c) {
        const unsigned int r0 = seq.start + c * 64u;
        const unsigned int n = seq.end - r0 < 64u ? seq.end - r0 : 64u;
        const bool more = c + 1u < chunks;
        const unsigned int n1 = !more ? 0u : seq.end - r0 - 64u < 64u ? seq.end - r0 - 64u : 64u;
        if (more) aotx_delta_load<D, NT>(next, p, c0 + c + 1u, r0 + 64u, n1, h, col, w, m, g);

        /* S as an operand */
#pragma unroll
        for (int u = 0; u < NT; ++u) {
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                aotx_h4 hi, lo;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    _Float16 a, z;
                    aotx_split(S[t][u][r] * up[u], &a, &z);
                    hi[r] = a;
                    lo[r] = z;
                }
                const unsigned int tile = w * TW + t;
                *((aotx_h4 *)&Sx[tile >> 1][0][u][lane] + (tile & 1u)) = hi;
                *((aotx_h4 *)&Sx[tile >> 1][1][u][lane] + (tile & 1u)) = lo;
            }
        }
        __syncthreads();
        aotx_f4 x[NT], o[NT];
        unsigned int lim[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            aotx_f4 ks = {0, 0, 0, 0}, kl = {0, 0, 0, 0}, qs = {0, 0, 0, 0}, ql = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const aotx_h8 hi = Sx[s][0][u][lane], lo = Sx[s][1][u][lane];
                ks = aotx_mma(now.k[s], hi, ks);
                kl = aotx_mma(now.k[s], lo, kl);
                qs = aotx_mma(now.q[s], hi, qs);
                ql = aotx_mma(now.q[s], lo, ql);
            }
            lim[u] = badv[u] < now.bad ? badv[u] : now.bad;
            const unsigned int upto = lim[u] < n ? lim[u] : n;
            aotx_h4 hi, lo;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[u][r] = i0 + r < upto ? aotx_h2f(now.v[r][u]) * up[u] - now.of_k[r] * (ks[r] + kl[r]) : 0.0f;
                o[u][r] = now.of_q[r] * (qs[r] + ql[r]);
                _Float16 a, z;
                aotx_split(x[u][r], &a, &z);
                hi[r] = a;
                lo[r] = z;
            }
            *((aotx_h4 *)&Xx[w >> 1][0][u][lane] + (w & 1u)) = hi;
            *((aotx_h4 *)&Xx[w >> 1][1][u][lane] + (w & 1u)) = lo;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            aotx_f4 t = {0, 0, 0, 0}, tl = {0, 0, 0, 0};
#pragma unroll
            for (unsigned int s = 0; s < 2u; ++s) {
                if (s > w / 2u) continue;
                const aotx_h8 hi = Xx[s][0][u][lane], lo = Xx[s][1][u][lane];
                t = aotx_mma(now.th[s], hi, t);
                tl = aotx_mma(now.th[s], lo, tl);
                tl = aotx_mma(now.tl[s], hi, tl);
            }
            aotx_h4 hi, lo, vhi, vlo;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float y = t[r] + tl[r];
                _Float16 a, z;
                aotx_split(y, &a, &z);
                hi[r] = a;
                lo[r] = z;
                aotx_split(y * now.of_u[r], &a, &z);
                vhi[r] = a;
                vlo[r] = z;
            }
            *((aotx_h4 *)&Ux[w >> 1][0][u][lane] + (w & 1u)) = hi;
            *((aotx_h4 *)&Ux[w >> 1][1][u][lane] + (w & 1u)) = lo;
            *((aotx_h4 *)&Vx[w >> 1][0][u][lane] + (w & 1u)) = vhi;
            *((aotx_h4 *)&Vx[w >> 1][1][u][lane] + (w & 1u)) = vlo;
        }
        if (more) {
            int was[NT];
#pragma unroll
            for (int u = 0; u < NT; ++u) was[u] = vex[u];
            tell(next, n1, S, was, vex);
        }
        __syncthreads();
        float down_now[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            aotx_f4 lo_part = {0, 0, 0, 0};
#pragma unroll
            for (unsigned int s = 0; s < 2u; ++s) {
                if (s > w / 2u) continue;
                const aotx_h8 hi = Ux[s][0][u][lane], lo = Ux[s][1][u][lane];
                o[u] = aotx_mma(now.ph[s], hi, o[u]);
                lo_part = aotx_mma(now.ph[s], lo, lo_part);
                lo_part = aotx_mma(now.pl[s], hi, lo_part);
            }
            down_now[u] = down[u];
            const float fade = now.fade * up[u];
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                aotx_f4 acc = S[t][u] * fade, low = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    acc = aotx_mma(now.kt[t][s], Vx[s][0][u][lane], acc);
                    low = aotx_mma(now.kt[t][s], Vx[s][1][u][lane], low);
                }
                S[t][u] = (acc + low) * down[u];
                if (lim[u] < n) S[t][u] = aotx_f4{1, 1, 1, 1} * __builtin_nanf("");
            }
            o[u] = (o[u] + lo_part) * down_now[u];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (i0 + r >= n) continue;
#pragma unroll
            for (int u = 0; u < NT; ++u)
                out[(r0 + i0 + r) * width + u] = i0 + r >= lim[u] ? 0x7E00u : aotx_f2h(o[u][r]);
        }
        if (more) {
            heard();
            now = next;
        }
    }
#pragma unroll
    for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned int tile = w * TW + t;
            const unsigned int key = 32u * (tile >> 1) + 8u * g + 4u * (tile & 1u) + r;
#pragma unroll
            for (int u = 0; u < NT; ++u) sp[key * D + u] = S[t][u][r];
        }
}

#endif
