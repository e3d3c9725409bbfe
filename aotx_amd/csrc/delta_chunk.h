/* The chunked form of the gated delta rule (aotx_delta_chunk): device code of its kernels.
 *
 * Within a chunk of 64 rows of one head, with K, Q the raw rows, V the values, r_k and r_q the
 * rows' inverse lengths (r_q with 1 / sqrt(d)), G the running sum of g, the rule unrolls to
 *   M_ij = beta_i r_k,i r_k,j (K_i . K_j) exp(G_i - G_j) for i > j,   T = (1 + M)^-1
 *   X = diag(beta) (V - diag(exp(G) r_k) K S),   U = T X
 *   out = diag(exp(G) r_q) Q S + P X,   P = N T,   N_ij = r_q,i r_k,j (Q_i . K_j) exp(G_i - G_j) for i >= j
 *   S <- exp(G_last) S + K^T diag(r_k exp(G_last - G)) U
 * T and P need no state: aotx_delta_within makes them for every chunk at once. What is left,
 * aotx_delta_across, walks a sequence's chunks with a slice of columns of S in registers.
 * aotx_delta_short does both in calls of up to 64 rows, while each of its workgroups has a CU.
 *
 * Numbers. K and Q are fp16 and enter the matrix cores as they are; S, U, X and T enter as two
 * fp16 parts (high and rest, 21 bits), so that the state's products are nearly as
 * good as fp32 ones at two or three times the work of plain fp16 instead of sixteen times for
 * fp32 matrix instructions. P, which only the output sees, is rounded to fp16 once, by 2^-11 as
 * the output itself is; it is at most 1 / sqrt(d) and goes times 2^18, so that a weight that has faded
 * to 2^-32 still has its 11 bits, and none is off by more than 2^-43. (In two parts 8192 rows took 278
 * us and not 229. P X and not N U, because where keys are alike U are differences far above their sum,
 * in parts of which the weights' rounding counts: rates near 1 and keys at 0.95 of one another gave
 * outputs off by 1.2e-3.) The parts have fp16's range, below which their step is 2^-24. M and T are at
 * most 1 (the rule only ever takes away from what a unit key finds) and go times 2^14, where the step
 * is 2^-38; beta is in X, not in T, whose entries would go with its square. Rows of K are brought to
 * lengths of 1/2 to 1 by a power of two 2^e (entries below 2^-14 lose bits, 2^-24 of the length at
 * most), whose scale goes into the factors of X and U. S, X and U carry a power of two for every
 * column, set anew every four chunks from the column's largest state entry and beta |v|: a state's
 * column grows by at most the sum of the 256 rows' in that time. So their step is 2^-33 of that entry
 * or 2^-28 of that beta |v|, whichever is larger, or 2^-21 of the number itself.
 *
 * A row whose K, a or b is no number is taken out (its K, g and beta are zeros) and remembered:
 * from that row on, out and the state are NaN; the same for one column from a bad value in V on.
 */
#ifndef AOTX_DELTA_CHUNK_H
#define AOTX_DELTA_CHUNK_H

#include "delta_dev.h"

#include <stddef.h>

typedef _Float16 aotx_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 aotx_h8 __attribute__((ext_vector_type(8)));

#define AOTX_DELTA_CHUNK 64u

/* What aotx_delta_within leaves of one chunk and head: matrix operands in the order that a wave
 * loads them, 16 bytes a lane. Row tile w (16 rows), step s (32 columns): lane (m, g) holds row
 * 16 w + m, columns 32 s + 16 (e / 4) + 4 g + e % 4 for e < 8, which is the order in which a
 * wave's accumulators of two row tiles make the other operand. */
struct aotx_delta_factors {
    float of_k[64];         /* beta exp(G) r_k 2^e; the rows of K are over 2^e */
    float of_q[64];         /* exp(G) r_q 2^AOTX_DELTA_OUT_UP */
    float of_u[64];         /* exp(G_last - G) r_k 2^e / AOTX_DELTA_UP */
    float of_b[64];         /* beta */
    unsigned char vmax[128];/* of every column: its largest beta |v| is below 2^(vmax - 126), or 0 */
    float fade;             /* exp(G_last), with the sign bit set where odd is not 64 */
    unsigned int odd;       /* first row that is taken out, 64 for none; + 256 if V has a value that is no number */
    unsigned int pad[30];
};

struct aotx_delta_chunk_work {
    aotx_h8 p[4][2][64], t_hi[4][2][64], t_lo[4][2][64];
    aotx_delta_factors of;
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
    aotx_h8 *rows;                  /* [chunks][key_heads] of K and Q (aotx_delta_rows_of) */
    unsigned int chunks;            /* at most: rows / 64 + sequences */
    unsigned int few;               /* sequences of up to this many rows go row by row */
};

/* K (rows over 2^e) and Q of a chunk and key head as operands, [4 row tiles][d / 32 steps][64]
 * each. Rows of the call's tensor lie a power of two apart as a rule, so that one head's are in
 * one channel of the L2; these are not. */
static __device__ __forceinline__ aotx_h8 *aotx_delta_rows_of(const aotx_delta_args &p, unsigned int c, unsigned int kh,
                                                              unsigned int d)
{
    return p.rows + ((unsigned long long)c * p.key_heads + kh) * (16u * d);
}

#define AOTX_DELTA_UP 16384.0f      /* of M and T as operands */
#define AOTX_DELTA_OUT_UP 18        /* P, and with it the sums of outputs, go times 2^18 */

/* x = hi + lo, four of them, rounded toward zero: the rest makes up for the high part's rounding, and
 * ends 2^-21 below x at most. */
typedef _Float16 aotx_h2 __attribute__((ext_vector_type(2)));
static __device__ __forceinline__ void aotx_split4(aotx_f4 x, aotx_h4 *hi, aotx_h4 *lo)
{
    const aotx_h2 a = __builtin_bit_cast(aotx_h2, __builtin_amdgcn_cvt_pkrtz(x[0], x[1]));
    const aotx_h2 b = __builtin_bit_cast(aotx_h2, __builtin_amdgcn_cvt_pkrtz(x[2], x[3]));
    const aotx_h2 c = __builtin_bit_cast(aotx_h2, __builtin_amdgcn_cvt_pkrtz(fmaf((float)a[0], -1.0f, x[0]), fmaf((float)a[1], -1.0f, x[1])));
    const aotx_h2 d = __builtin_bit_cast(aotx_h2, __builtin_amdgcn_cvt_pkrtz(fmaf((float)b[0], -1.0f, x[2]), fmaf((float)b[1], -1.0f, x[3])));
    *hi = aotx_h4{a[0], a[1], b[0], b[1]};
    *lo = aotx_h4{c[0], c[1], d[0], d[1]};
}

static __device__ __forceinline__ aotx_f4 aotx_mma(aotx_h8 a, aotx_h8 b, aotx_f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

/* Workgroup b runs on XCD b % 8. Heads are dealt out so that those of one key head, one after
 * another, come to the same XCD, in both kernels: its L2 then fetches the rows of K and Q once. */
static __device__ __forceinline__ unsigned int aotx_delta_head(const aotx_delta_args &p, unsigned int x)
{
    return p.heads % 8u == 0u ? x % 8u * (p.heads / 8u) + x / 8u : x;
}

/* Chunks of sequence `lane` and of the sequences before it. */
static __device__ __forceinline__ void aotx_delta_chunks(const aotx_delta_args &p, const aotx_seq_lanes &l,
                                                         unsigned int *mine, unsigned int *before)
{
    const unsigned int lane = threadIdx.x & 63u, rows = l.end - l.start;
    const unsigned int n = rows > p.few ? (rows + AOTX_DELTA_CHUNK - 1u) / AOTX_DELTA_CHUNK : 0u;
    unsigned int sum = n;
    for (unsigned int off = 1u; off < p.seqs.seqs; off <<= 1) {
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
 * Row by row. A workgroup holds CS columns of one head's S in registers, four columns and
 * every RG-th row a thread; S^T k' and S^T q' come from one walk over them, since
 *   out = exp(g) S^T q' + (k' . q') u,
 * so a token costs one reduction over the rows: lanes of a wave first, then the four waves
 * through LDS with one barrier. The next token's rows are normed by wave 0 before it, into the
 * third of three places: a slower wave may still be at the S of the token before.
 *
 * Bound by the state's bytes, read and written once whatever the number of rows: a token of 64
 * slots, 32 heads of 128, moves 270 MB in 50.4 us, 5.3 TB/s, the rate of a large copy; of 1 slot 5
 * us, what a launch and one trip to memory take. Each further row of a sequence adds 1.7 us, its
 * reduction's latency. Four columns a thread: a wave's load is whole pieces of 256 bytes.
 * ------------------------------------------------------------------------------------- */
template <int D, int CS>
struct aotx_delta_rows_lds {
    __align__(16) float kq[3][2][D];
    float gate[3][4];                            /* exp(g), beta, k' . q' */
    __align__(16) float part[2][4][2][CS];
};

template <int D, int CS>
static __device__ __forceinline__ void aotx_delta_by_rows(const aotx_delta_args &p, aotx_delta_rows_lds<D, CS> &lds,
                                                          unsigned int block)
{
    constexpr int LC = CS / 4, RG = 256 / LC, NR = D / RG;
    constexpr int SLICES = D / CS;
    const unsigned int unit = block / SLICES, slice = block % SLICES;
    const unsigned int i = unit / p.heads, h = unit % p.heads;
    const unsigned int lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const aotx_seq_view seq = aotx_seq_of(p.seqs, i, aotx_seqs_read(p.seqs));
    if (seq.start >= seq.end || seq.end - seq.start > p.few) return;
    if (threadIdx.x >= 256u) {                   /* a wave that the launch has over */
        if (!seq.refused)
            for (unsigned int t = seq.start; t <= seq.end; ++t) __syncthreads();
        return;
    }
    const unsigned int c4 = (threadIdx.x % LC) * 4u, rg = threadIdx.x / LC;
    const unsigned int col = slice * CS + c4;
    const unsigned long long width = (unsigned long long)p.heads * D;
    unsigned short *out = p.out + (unsigned long long)h * D + col;
    if (seq.refused) {
        if (threadIdx.x == 0u && slice == 0u && h == 0u) atomicAdd(p.seqs.faults, 1u);
        for (unsigned int t = seq.start + rg; t < seq.end; t += RG)
            *(aotx_u16x4 *)(out + t * width) = aotx_u16x4{0, 0, 0, 0};
        return;
    }
    float *sp = p.state + ((unsigned long long)seq.slot * p.heads + h) * D * D + col;
    aotx_f4 S[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
        S[n] = seq.fresh ? aotx_f4{0, 0, 0, 0} : __builtin_nontemporal_load((const aotx_f4 *)(sp + (n * RG + rg) * D));

    const unsigned short *q = p.qkv + (unsigned long long)(h / p.group) * D;
    const unsigned short *k = q + (unsigned long long)p.key_heads * D;
    const unsigned short *v = p.qkv + 2ull * p.key_heads * D + (unsigned long long)h * D + col;
    const float decay = p.decay[h], dt = p.dt[h];
    auto stage = [&](unsigned int t, unsigned int at) {
        if (wave != 0u) return;
        const unsigned long long row = (unsigned long long)t * p.stride;
        float kv[D / 64], qv[D / 64], kk = 0.0f, qq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 64; ++n) {
            kv[n] = aotx_h2f(k[row + n * 64 + lane]);
            qv[n] = aotx_h2f(q[row + n * 64 + lane]);
            kk += kv[n] * kv[n];
            qq += qv[n] * qv[n];
            dot += kv[n] * qv[n];
        }
        const float g = aotx_delta_gate(p.a[(unsigned long long)t * p.ab_stride + h], dt, decay);
        const float beta = 1.0f / (1.0f + expf(-p.b[(unsigned long long)t * p.ab_stride + h]));
        kk = aotx_wave_sum(kk);
        qq = aotx_wave_sum(qq);
        dot = aotx_wave_sum(dot);
        const float rk = 1.0f / sqrtf(kk + p.eps);
        const float rq = 1.0f / sqrtf(qq + p.eps) * (D == 128 ? 0.08838834764831845f : 0.125f);
#pragma unroll
        for (int n = 0; n < D / 64; ++n) {
            lds.kq[at][0][n * 64 + lane] = kv[n] * rk;
            lds.kq[at][1][n * 64 + lane] = qv[n] * rq;
        }
        if (lane == 0u) {
            lds.gate[at][0] = expf(g);
            lds.gate[at][1] = beta;
            lds.gate[at][2] = dot * rk * rq;
        }
    };
    stage(seq.start, 0u);
    __syncthreads();
    unsigned int at = 0u;
    for (unsigned int t = seq.start; t < seq.end; ++t) {
        const unsigned int side = t & 1u, next = at < 2u ? at + 1u : 0u;
        const aotx_u16x4 vh = *(const aotx_u16x4 *)(v + (unsigned long long)t * p.stride);
        aotx_f4 sk = {0, 0, 0, 0}, sq = {0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float kr = lds.kq[at][0][n * RG + rg], qr = lds.kq[at][1][n * RG + rg];
            sk += S[n] * kr;
            sq += S[n] * qr;
        }
#pragma unroll
        for (int off = 32; off >= LC; off >>= 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sk[e] += __shfl_xor(sk[e], off, 64);
                sq[e] += __shfl_xor(sq[e], off, 64);
            }
        }
        if (lane < LC) {
            *(aotx_f4 *)&lds.part[side][wave][0][c4] = sk;
            *(aotx_f4 *)&lds.part[side][wave][1][c4] = sq;
        }
        if (t + 1u < seq.end) stage(t + 1u, next);
        __syncthreads();
        sk = *(const aotx_f4 *)&lds.part[side][0][0][c4];
        sq = *(const aotx_f4 *)&lds.part[side][0][1][c4];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            sk += *(const aotx_f4 *)&lds.part[side][w][0][c4];
            sq += *(const aotx_f4 *)&lds.part[side][w][1][c4];
        }
        const float fade = lds.gate[at][0], beta = lds.gate[at][1], dot = lds.gate[at][2];
        aotx_f4 u, o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            u[e] = beta * (aotx_h2f(vh[e]) - fade * sk[e]);
            o[e] = fade * sq[e] + dot * u[e];
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) S[n] = S[n] * fade + u * lds.kq[at][0][n * RG + rg];
        if (rg == 0u) {
            aotx_u16x4 oh;
#pragma unroll
            for (int e = 0; e < 4; ++e) oh[e] = aotx_f2h(o[e]);
            *(aotx_u16x4 *)(out + t * width) = oh;
        }
        at = next;
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) __builtin_nontemporal_store(S[n], (aotx_f4 *)(sp + (n * RG + rg) * D));
}

/* Rows r0 .. r0 + n - 1 of a call's qkv: what is read past them is zeros. */
struct aotx_rows_view {
    __amdgpu_buffer_rsrc_t rs;
};
static __device__ __forceinline__ aotx_rows_view aotx_rows_of(const aotx_delta_args &p, unsigned int r0, unsigned int n)
{
    aotx_rows_view v;
    v.rs = __builtin_amdgcn_make_buffer_rsrc((void *)(p.qkv + (unsigned long long)r0 * p.stride), (short)0,
                                             (int)(n * p.stride * 2u), 0x00020000);
    return v;
}
static __device__ __forceinline__ aotx_h8 aotx_rows_16(const aotx_rows_view &v, unsigned int at)
{
    return __builtin_bit_cast(aotx_h8, __builtin_amdgcn_raw_buffer_load_b128(v.rs, (int)at, 0, 0));
}
static __device__ __forceinline__ unsigned short aotx_rows_2(const aotx_rows_view &v, unsigned int at)
{
    return __builtin_amdgcn_raw_buffer_load_b16(v.rs, (int)at, 0, 0);
}

/* ---------------------------------------------------------------------------------------
 * T, P and the row factors of one chunk and head, and K and Q as operands; a workgroup of five
 * waves, wave w < 4 has rows 16 w .. 16 w + 15, wave 4 the gates of all. The products are taken
 * transposed (K_j Q_i^T), so that a lane holds one row i and four columns j along its registers, as
 * the operands above need them. (1 + M)^-1 goes by blocks of 16: substitution in the blocks on the
 * diagonal, matrix products below them. The gates have a wave of their own because their
 * exponentials and the sum over 64 rows are as long a chain as the loads that the others wait for.
 *
 * Large calls are bound by memory, the workspace above all (20 KB a chunk and head, 32 a key head):
 * 8192 rows, 32 heads of 128, read 136 MB and write 148 in 66 us, 4.3 TB/s; 512 rows, a workgroup a
 * CU, take 8.8 us of latency.
 * ------------------------------------------------------------------------------------- */
template <int D>
struct aotx_delta_within_lds {
    union {
        aotx_h8 kfrag[4][D / 32][64];                       /* rows of K, as operands */
        __align__(16) unsigned short tp[2][64][72];         /* T, to be read by rows */
    };
    __align__(16) float diag[4][16][20];                    /* M's diagonal blocks, then their inverses */
    __align__(16) unsigned short below[2][48][56];          /* M's blocks below them, rows 16 .. 63, two parts */
    __align__(16) float ghi[64], glo[64], near_end[64], beta[64], rk[64], rq[64], ks[64];
    __align__(16) unsigned int vm[4][64];
    unsigned int badk[4], badv[4];
};

/* What a wave of one chunk has in registers: its rows of K, Q, P and T as operands and, of a chunk
 * that stays in its workgroup, four rows of one column of V. */
template <int D>
struct aotx_delta_made {
    aotx_h8 k[D / 32], q[D / 32], p[2], th[2], tl[2];
    aotx_f4 qk[4];              /* N, the wave's rows by tiles of columns */
    unsigned short v[4];
    int top;                    /* of the wave's rows of the column, as vmax */
};

/* N and M of row 16 W + m. Between blocks, exp(G_i - G_j) is the product of two factors by way of
 * the last row of j's block: both are at most 1, and one exponential a row serves four columns. */
template <int D, int W>
static __device__ __forceinline__ void aotx_delta_pairs(aotx_delta_within_lds<D> &lds, aotx_delta_made<D> &made, float inv,
                                                        float qinv)
{
    constexpr int KS = D / 32;
    const unsigned int lane = threadIdx.x & 63u, m = lane & 15u, g = lane >> 4, row = 16u * W + m;
    const float gi = lds.ghi[row], gil = lds.glo[row], bi = lds.beta[row] * inv;
    aotx_f4 block;
#pragma unroll
    for (int jt = 0; jt <= W; ++jt) {
        aotx_f4 kks = {0, 0, 0, 0}, qks = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const aotx_h8 kj = lds.kfrag[jt][s][lane];
            kks = aotx_mma(kj, made.k[s], kks);
            qks = aotx_mma(kj, made.q[s], qks);
        }
        const unsigned int j0 = 16u * jt + 4u * g;
        const aotx_f4 rkj = *(const aotx_f4 *)&lds.rk[j0];
        if (jt == W) {
            const aotx_f4 gj = *(const aotx_f4 *)&lds.ghi[j0], gjl = *(const aotx_f4 *)&lds.glo[j0];
            aotx_f4 fade;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                /* above the diagonal the exponential is of a positive number, and of no use */
                fade[r] = expf((gi - gj[r]) + (gil - gjl[r])) * rkj[r];
                fade[r] = row >= j0 + r ? fade[r] : 0.0f;
                kks[r] = row > j0 + r ? kks[r] : 0.0f;
                qks[r] = row >= j0 + r ? qks[r] : 0.0f;
            }
            block = kks * fade * bi;
            made.qk[jt] = qks * fade * qinv;
        } else {
            const float from = expf((gi - lds.ghi[16 * jt + 15]) + (gil - lds.glo[16 * jt + 15]));
            const aotx_f4 fade = *(const aotx_f4 *)&lds.near_end[j0] * rkj * from;
            aotx_h4 hi, lo;
            aotx_split4(kks * fade * (bi * AOTX_DELTA_UP), &hi, &lo);
            *(aotx_h4 *)&lds.below[0][row - 16u][j0] = hi;
            *(aotx_h4 *)&lds.below[1][row - 16u][j0] = lo;
            made.qk[jt] = qks * fade * qinv;
        }
    }
    /* inverse of 1 + the diagonal block by substitution, a column a lane; every value found is
     * taken from all rows below at once, which do not wait for one another */
    *(aotx_f4 *)&lds.diag[W][m][4u * g] = block;
    __builtin_amdgcn_wave_barrier();
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = m == (unsigned int)r ? 1.0f : 0.0f;
    aotx_f4 row4[16][4];
#pragma unroll
    for (int r = 1; r < 16; ++r)
#pragma unroll
        for (int q = 0; 4 * q < r; ++q) row4[r][q] = *(const aotx_f4 *)&lds.diag[W][r][4 * q];
#pragma unroll
    for (int q = 0; q < 15; ++q)
#pragma unroll
        for (int r = q + 1; r < 16; ++r) x[r] -= row4[r][q / 4][q % 4] * x[q];
    if (g == 0u)
#pragma unroll
        for (int r = 0; r < 16; ++r) lds.diag[W][r][m] = x[r];
}

/* a b c: both in two parts, 16 x 16 blocks; b in accumulator order */
static __device__ __forceinline__ aotx_f4 aotx_mma_parts(aotx_h4 ahi, aotx_h4 alo, aotx_h4 bhi, aotx_h4 blo, aotx_f4 c)
{
    c = __builtin_amdgcn_mfma_f32_16x16x16f16(ahi, blo, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x16f16(alo, bhi, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x16f16(ahi, bhi, c, 0, 0, 0);
}

/* Column W of blocks of T, downwards: T_b = -D_b (sum of M_bq T_q). A block in accumulator order is the
 * right operand of the next product as it stands. All operands are times AOTX_DELTA_UP, and their
 * products brought back to one of it. */
template <int D, int W>
static __device__ __forceinline__ void aotx_delta_column(aotx_delta_within_lds<D> &lds)
{
    const unsigned int lane = threadIdx.x & 63u, m = lane & 15u, g = lane >> 4;
    const unsigned int at = aotx_delta_place(16u * W + m);
    aotx_f4 tc[4];
    aotx_h4 hi[4], lo[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) tc[0][r] = lds.diag[W][4u * g + r][m] * AOTX_DELTA_UP;
    aotx_split4(tc[0], &hi[0], &lo[0]);
#pragma unroll
    for (int off = 1; off < 4 - W; ++off) {
        const int bt = W + off;
        aotx_f4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < off; ++q)
            acc = aotx_mma_parts(*(const aotx_h4 *)&lds.below[0][16 * (bt - 1) + m][16 * (W + q) + 4u * g],
                                 *(const aotx_h4 *)&lds.below[1][16 * (bt - 1) + m][16 * (W + q) + 4u * g], hi[q], lo[q], acc);
        aotx_h4 dhi, dlo, yhi, ylo;
        aotx_split4(*(const aotx_f4 *)&lds.diag[bt][m][4u * g] * AOTX_DELTA_UP, &dhi, &dlo);
        aotx_split4(acc * (-1.0f / AOTX_DELTA_UP), &yhi, &ylo);
        tc[off] = aotx_mma_parts(dhi, dlo, yhi, ylo, aotx_f4{0, 0, 0, 0}) * (1.0f / AOTX_DELTA_UP);
        aotx_split4(tc[off], &hi[off], &lo[off]);
    }
#pragma unroll
    for (int off = 0; off < 4 - W; ++off) {
        aotx_h4 th, tl;
        aotx_split4(tc[off], &th, &tl);
        const aotx_u16x4 hb = __builtin_bit_cast(aotx_u16x4, th), lb = __builtin_bit_cast(aotx_u16x4, tl);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            lds.tp[0][16u * (W + off) + 4u * g + r][at] = hb[r];
            lds.tp[1][16u * (W + off) + 4u * g + r][at] = lb[r];
        }
    }
    if (W & 1)
#pragma unroll
        for (int r = 0; r < 4; ++r) lds.tp[0][16u * (W & 2) + 4u * g + r][at] = lds.tp[1][16u * (W & 2) + 4u * g + r][at] = 0;
}

/* Rows 16 W + m of P = N T, from two parts of both: taken transposed, T's columns by transposing reads
 * (as K's in the walk), so that a row stays in its lane. */
template <int D, int W>
static __device__ __forceinline__ void aotx_delta_weights(aotx_delta_within_lds<D> &lds, aotx_delta_made<D> &made)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    const unsigned int lane = threadIdx.x & 63u, m = lane & 15u, g = lane >> 4;
    aotx_h4 hi[4], lo[4];
#pragma unroll
    for (int q = 0; q <= W; ++q) aotx_split4(made.qk[q], &hi[q], &lo[q]);
    aotx_f4 pt[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        pt[c] = aotx_f4{0, 0, 0, 0};
#pragma unroll
        for (int q = c; q <= W; ++q) {
            aotx_h4 t[2];
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                unsigned short *at = &lds.tp[part][16u * q + 4u * g + (m >> 2)][32 * (c >> 1) + 4 * (c & 1) + 8u * (m & 3u)];
                t[part] = __builtin_bit_cast(aotx_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at));
            }
            pt[c] = aotx_mma_parts(t[0], t[1], hi[q], lo[q], pt[c]);
        }
        pt[c] *= 1.0f / AOTX_DELTA_UP;
    }
#pragma unroll
    for (int s = 0; s <= W / 2; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            made.p[s][r] = (_Float16)pt[2 * s][r];
            made.p[s][4 + r] = (_Float16)pt[2 * s + 1][r];
        }
}

/* The fifth wave: gates, a row a lane, and what follows from them. Sums of g are in 64 bits,
 * kept as two floats, so that differences of far sums stay exact. */
template <int D, bool STAYS>
static __device__ __forceinline__ void aotx_delta_rates(const aotx_delta_args &p, aotx_delta_within_lds<D> &lds,
                                                        aotx_delta_factors *to, unsigned int r0, unsigned int n,
                                                        unsigned int h)
{
    const unsigned int lane = threadIdx.x & 63u;
    const unsigned long long at = (unsigned long long)(r0 + (lane < n ? lane : n - 1u)) * p.ab_stride + h;
    const float a = p.a[at], b = p.b[at];
    float gate = aotx_delta_gate(a, p.dt[h], p.decay[h]);
    float rate = 1.0f / (1.0f + expf(-b));
    const bool badgate = lane < n && (gate != gate || rate != rate);
    const unsigned long long badgates = __ballot(badgate);
    if (lane >= n || badgate) gate = rate = 0.0f;
    const double sum = aotx_wave_scan((double)gate);
    const float all = expf((float)sum), last = expf((float)(__shfl(sum, 63, 64) - sum));
    lds.ghi[lane] = (float)sum;
    lds.glo[lane] = (float)(sum - (double)(float)sum);
    lds.near_end[lane] = expf((float)(__shfl(sum, (int)(lane | 15u), 64) - sum));
    lds.beta[lane] = rate;
    __syncthreads();
    to->of_k[lane] = rate * all * lds.ks[lane];
    to->of_q[lane] = all * lds.rq[lane];
    to->of_u[lane] = last * lds.ks[lane] * (1.0f / AOTX_DELTA_UP);
    to->of_b[lane] = rate;
    if (lane == 63u) {
        unsigned int first = badgates != 0ull ? (unsigned int)__builtin_ctzll(badgates) : 64u;
        for (int v = 0; v < 4; ++v) first = lds.badk[v] < first ? lds.badk[v] : first;
        const unsigned int odd = first | (lds.badv[0] | lds.badv[1] | lds.badv[2] | lds.badv[3]) << 8;
        to->fade = odd != 64u ? -all : all;
        to->odd = odd;
    }
    __syncthreads();
    if (!STAYS && lane < D / 2) {       /* two columns a lane */
        typedef unsigned short u2 __attribute__((ext_vector_type(2)));
        u2 v = __builtin_bit_cast(u2, lds.vm[0][lane]);
#pragma unroll
        for (int x = 1; x < 4; ++x) v = __builtin_elementwise_max(v, __builtin_bit_cast(u2, lds.vm[x][lane]));
        *(unsigned short *)&to->vmax[2u * lane] = (unsigned short)(v[0] | (v[1] << 8));
    }
    __syncthreads();
}

/* A wave's part of one chunk and head, of the first four waves. STAYS: its workgroup goes on with it,
 * for the 16 columns from col; else it goes to the workspace. */
template <int D, bool STAYS>
static __device__ __forceinline__ void aotx_delta_make(const aotx_delta_args &p, aotx_delta_within_lds<D> &lds,
                                                       aotx_delta_chunk_work *to, unsigned int c, unsigned int h,
                                                       unsigned int w, unsigned int r0, unsigned int n,
                                                       unsigned int col, aotx_delta_made<D> &made)
{
    constexpr int KS = D / 32;
    /* rows of K and Q, columns 32 s + 8 g .. of row 16 w + m; rows past the chunk read as zeros */
    const unsigned int lane = threadIdx.x & 63u, m = lane & 15u, g = lane >> 4;
    const unsigned int kh = h / p.group;
    const unsigned int row = 16u * w + m;
    const aotx_rows_view rows = aotx_rows_of(p, r0, n);
    const unsigned int at_q = row * p.stride * 2u + (kh * D + 8u * g) * 2u, at_k = at_q + p.key_heads * D * 2u;
    aotx_h8 (&kf)[KS] = made.k, (&qf)[KS] = made.q;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        kf[s] = aotx_rows_16(rows, at_k + 64u * s);
        qf[s] = aotx_rows_16(rows, at_q + 64u * s);
    }
    /* V: eight columns of every 256 / (D / 8)-th row a thread, or rows 16 w + 4 g .. of one */
    constexpr unsigned int VR = 256 / (D / 8);
    aotx_u16x8 vv[64 / VR];
    const unsigned int at_v = (2u * p.key_heads * D + h * D) * 2u;
    if constexpr (STAYS) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            made.v[r] = aotx_rows_2(rows, (16u * w + 4u * g + r) * p.stride * 2u + at_v + (col + m) * 2u);
    } else {
#pragma unroll
        for (unsigned int r = 0; r < 64u / VR; ++r)
            vv[r] = __builtin_bit_cast(aotx_u16x8, aotx_rows_16(rows, (r * VR + threadIdx.x / (D / 8)) * p.stride * 2u
                                       + at_v + threadIdx.x % (D / 8) * 16u));
    }
    float kk = 0.0f, qq = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int v = 0; v < 8; v += 2) {
            const aotx_h2 k2 = {kf[s][v], kf[s][v + 1]}, q2 = {qf[s][v], qf[s][v + 1]};
            kk = __builtin_amdgcn_fdot2(k2, k2, kk, false);
            qq = __builtin_amdgcn_fdot2(q2, q2, qq, false);
        }
    kk += __shfl_xor(kk, 16, 64);
    kk += __shfl_xor(kk, 32, 64);
    qq += __shfl_xor(qq, 16, 64);
    qq += __shfl_xor(qq, 32, 64);
    const bool bad = !(kk < __builtin_inff());
    if (bad) kk = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        if (bad) kf[s] = aotx_h8{0, 0, 0, 0, 0, 0, 0, 0};
        lds.kfrag[w][s][lane] = kf[s];
    }
    const unsigned long long badrows = __ballot(bad) & 0xFFFFull;
    if (lane == 0u) lds.badk[w] = badrows != 0ull ? 16u * w + (unsigned int)__builtin_ctzll(badrows) : 64u;
    const float inv = __builtin_amdgcn_rsqf(kk + p.eps);
    const float qinv = __builtin_amdgcn_rsqf(qq + p.eps) * (D == 128 ? 0.08838834764831845f : 0.125f)
        * ldexpf(1.0f, AOTX_DELTA_OUT_UP);
    /* 2^ex: the row's length over it is 1/2 to 1 */
    const int ex = __builtin_amdgcn_frexp_expf(__builtin_amdgcn_sqrtf(kk + p.eps));
    if (g == 0u) {
        lds.rk[row] = inv;
        lds.ks[row] = ldexpf(inv, ex);
        lds.rq[row] = qinv;
    }
    /* over 2^ex in two steps, each a number of fp16; ex below -28 is of rows of zeros */
    _Float16 a, z;
    {
        const int one = ex > 14 ? 14 : ex < -14 ? -14 : ex, two = ex - one < -14 ? -14 : ex - one;
        a = (_Float16)ldexpf(1.0f, -one);
        z = (_Float16)ldexpf(1.0f, -two);
    }
    if (!STAYS && h % p.group == 0u) {
        aotx_h8 *k = aotx_delta_rows_of(p, c, kh, D) + w * KS * 64u, *q = k + 8u * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            *(aotx_h8 *)((char *)(k + s * 64) + lane * 16u) = kf[s] * a * z;
            *(aotx_h8 *)((char *)(q + s * 64) + lane * 16u) = qf[s];
        }
    }
    /* V's values that are no numbers are told of, and left out of what follows */
    bool none = false;
    if constexpr (STAYS) {
#pragma unroll
        for (int r = 0; r < 4; ++r) none |= (made.v[r] & 0x7FFFu) >= 0x7C00u;
    } else {
        aotx_u16x8 top = vv[0] & (unsigned short)0x7FFF;
#pragma unroll
        for (unsigned int r = 1; r < 64u / VR; ++r) top = __builtin_elementwise_max(top, vv[r] & (unsigned short)0x7FFF);
        none = __builtin_reduce_max(top) >= 0x7C00;
        if (none)
#pragma unroll
            for (unsigned int r = 0; r < 64u / VR; ++r)
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if ((vv[r][x] & 0x7FFF) >= 0x7C00) vv[r][x] = 0;
    }
    const unsigned long long told = __ballot(none);
    if (lane == 0u) lds.badv[w] = told != 0ull ? 1u : 0u;
    __syncthreads();
    /* the largest beta |v| of V's columns, then its exponent */
    if constexpr (STAYS) {
        float top = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if ((made.v[r] & 0x7FFFu) < 0x7C00u) top = fmaxf(top, fabsf(aotx_h2f(made.v[r])) * lds.beta[16u * w + 4u * g + r]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        made.top = (int)(__float_as_uint(top) >> 23);
    } else {
        float most[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (unsigned int r = 0; r < 64u / VR; ++r) {
            const float beta = lds.beta[r * VR + threadIdx.x / (D / 8)];
#pragma unroll
            for (int x = 0; x < 8; ++x) most[x] = fmaxf(most[x], fabsf(fmaf(aotx_h2f(vv[r][x]), beta, 0.0f)));
        }
        aotx_u16x8 top;
#pragma unroll
        for (int x = 0; x < 8; ++x) top[x] = (unsigned short)(__float_as_uint(most[x]) >> 23);
        typedef unsigned int u4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (unsigned int off = D / 8; off < 64u; off <<= 1) {
            u4 o = __builtin_bit_cast(u4, top);
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = (unsigned int)__shfl_xor((int)o[x], off, 64);
            top = __builtin_elementwise_max(top, __builtin_bit_cast(aotx_u16x8, o));
        }
        if (lane < D / 8) *(aotx_u16x8 *)((unsigned short *)lds.vm[w] + lane * 8u) = top;
    }
    if (w == 0u) aotx_delta_pairs<D, 0>(lds, made, inv, qinv);
    else if (w == 1u) aotx_delta_pairs<D, 1>(lds, made, inv, qinv);
    else if (w == 2u) aotx_delta_pairs<D, 2>(lds, made, inv, qinv);
    else aotx_delta_pairs<D, 3>(lds, made, inv, qinv);
    __syncthreads();

    if (w == 0u) aotx_delta_column<D, 0>(lds);
    else if (w == 1u) aotx_delta_column<D, 1>(lds);
    else if (w == 2u) aotx_delta_column<D, 2>(lds);
    else aotx_delta_column<D, 3>(lds);
    __syncthreads();
    if (w == 0u) aotx_delta_weights<D, 0>(lds, made);
    else if (w == 1u) aotx_delta_weights<D, 1>(lds, made);
    else if (w == 2u) aotx_delta_weights<D, 2>(lds, made);
    else aotx_delta_weights<D, 3>(lds, made);
#pragma unroll
    for (unsigned int s = 0; s < 2u; ++s) {
        if (s > w / 2u) continue;
        const aotx_h8 hi = *(const aotx_h8 *)&lds.tp[0][row][32u * s + 8u * g];
        const aotx_h8 lo = *(const aotx_h8 *)&lds.tp[1][row][32u * s + 8u * g];
        if constexpr (STAYS) {
            made.th[s] = hi;
            made.tl[s] = lo;
        } else {
            to->t_hi[w][s][lane] = hi;
            to->t_lo[w][s][lane] = lo;
            to->p[w][s][lane] = made.p[s];
        }
    }
    if constexpr (STAYS)
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[s] = kf[s] * a * z;
}

/* FEW: the workgroups past those of the chunks take the sequences of few rows. Five waves a SIMD are the
 * four workgroups that LDS has room for: with 99 registers, for four waves, 2048 rows of 32 heads of 128
 * took 66.7 us, with 96 61.1. */
template <int D, bool FEW>
__global__ __launch_bounds__(320, FEW ? 1 : 5) void aotx_delta_within(aotx_delta_args p)
{
    __shared__ union {
        aotx_delta_within_lds<D> chunk;
        aotx_delta_rows_lds<D, 64> rows;
    } share;
    aotx_delta_within_lds<D> &lds = share.chunk;
    if (FEW && blockIdx.x >= p.chunks * p.heads) {      /* a sequence of few rows, the fifth wave idle */
        aotx_delta_by_rows<D, 64>(p, share.rows, blockIdx.x - p.chunks * p.heads);
        return;
    }
    const unsigned int lane = threadIdx.x & 63u;
    const unsigned int w = (unsigned int)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const unsigned int c = blockIdx.x / p.heads, h = aotx_delta_head(p, blockIdx.x % p.heads);

    unsigned int mine, before;
    const aotx_seq_lanes seqs = aotx_seqs_read(p.seqs);
    aotx_delta_chunks(p, seqs, &mine, &before);
    const unsigned int i = (unsigned int)__popcll(__ballot(lane < p.seqs.seqs && before + mine <= c));
    if (i >= p.seqs.seqs) return;
    const aotx_seq_view seq = aotx_seq_of(p.seqs, i, seqs);
    if (seq.refused) return;
    const unsigned int r0 = seq.start + (c - (unsigned int)__builtin_amdgcn_readlane((int)before, (int)i)) * 64u;
    const unsigned int n = seq.end - r0 < 64u ? seq.end - r0 : 64u;
    aotx_delta_chunk_work *to = p.work + (unsigned long long)c * p.heads + h;

    if (w == 4u) {
        aotx_delta_rates<D, false>(p, lds, &to->of, r0, n, h);
        return;
    }
    aotx_delta_made<D> made;
    aotx_delta_make<D, false>(p, lds, to, c, h, w, r0, n, 0u, made);
}

/* ---------------------------------------------------------------------------------------
 * The walk over a sequence's chunks. Four waves have 16 columns of one head's S: wave w the rows
 * of S that one step of K S takes (D / 4 of them, in accumulators), and rows 16 w .. 16 w + 15 of
 * the chunk. S, X and U pass between the waves through LDS as operands, a
 * barrier each; everything else a chunk needs is loaded into registers a chunk or two ahead. All
 * that the state's chain does not need is where the chain waits: loads beside products that are
 * under way, K's way through LDS and Q S while S and X are on theirs, P X behind the products of U, its
 * rounding and stores while the next chunk's X is read. (At other places in the chain the same
 * loads, stores and LDS writes made 8192 rows 3 to 40 us longer.)
 * Row x of tile t of S is key 32 (t / 2) + 8 (x / 4) + 4 (t % 2) + x % 4, so that two tiles'
 * accumulators hold keys 8 g .. 8 g + 7 of a step, as 16 bytes of a row of K do.
 *
 * Bound by the chain of chunks: 32 heads of 128 are 256 workgroups, one a CU, and each waits for
 * itself; 8192 rows take 178 to 194 us in a trace, 1.4 us a chunk, the latencies of its three passes
 * through LDS and of the products between them. Of that time LDS works 27 % and the matrix cores 16 %;
 * the vector caches wait for the L2 in 40 % of theirs. Columns in slices of 16 make the workgroups
 * that fill the chip: slices of 32 halve the traffic and took 369 to 400 us; eight waves, four of
 * them for the output, took as long as four.
 * ------------------------------------------------------------------------------------- */
#define AOTX_DELTA_PERIOD 4u        /* chunks for which a column's scale holds */

template <int D>
struct aotx_delta_lds {
    aotx_h8 s[D / 32][2][64];               /* S by steps of keys, two parts */
    aotx_h8 x[2][2][64];                    /* X by steps of rows */
    aotx_h8 v[2][2][64];                    /* U with the state update's factors */
    __align__(16) unsigned short k[64][D + 8];  /* the chunk's rows of K, to be read by columns */
    int size[4][16];                        /* exponents of the state's columns, by wave */
    unsigned int bad[4][16];                /* first bad rows of V's columns, by wave */
};

struct aotx_delta_walk {
    aotx_seq_view seq;
    unsigned int c0, chunks, h, col, w, m, g, lane;
};

/* 16 bytes a lane of a part of the workspace: the part's start is the wave's, and no lane has an
 * address of its own to compute. */
static __device__ __forceinline__ __amdgpu_buffer_rsrc_t aotx_part(const char *from, unsigned int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)from, (short)0, (int)bytes, 0x00020000);
}
static __device__ __forceinline__ aotx_h8 aotx_lane_16(__amdgpu_buffer_rsrc_t from, unsigned int at, unsigned int step)
{
    return __builtin_bit_cast(aotx_h8, __builtin_amdgcn_raw_buffer_load_b128(from, (int)at, (int)step, 0));
}

static __device__ __forceinline__ unsigned int aotx_delta_left(const aotx_delta_walk &k, unsigned int c)
{
    const unsigned int n = k.seq.end - k.seq.start - c * 64u;
    return n < 64u ? n : 64u;
}

/* exponent of |x|: |x| < 2^(e + 1) */
static __device__ __forceinline__ int aotx_exponent(float x)
{
    return (int)((__float_as_uint(x) >> 23) & 0xFFu) - 127;
}

template <int D, int NS>
struct aotx_delta_tile {
    aotx_h8 k[D / 32], q[D / 32], th[NS], tl[NS], p[NS];
    unsigned short v[4];
    aotx_f4 of_k, of_u, of_q, of_b;
    float fade;
    unsigned int touched;
};

/* NS: steps of 32 columns that the wave's rows of T and P have, 1 for waves 0 and 1, else 2.
 * AHEAD: how many chunks ahead the loads run, one or two; with 3, two, and their lines are asked
 * for before; with 0, there is one chunk, and it and the state are in registers (one, the column's
 * vmax, odd, one_state). */
template <int D, int NS, int AHEAD>
static __device__ __forceinline__ void aotx_delta_follow(const aotx_delta_args &p, const aotx_delta_walk k,
                                                         aotx_delta_lds<D> &lds, const aotx_delta_tile<D, NS> *one,
                                                         int one_top, unsigned int one_odd,
                                                         const aotx_f4 (*one_state)[D / 64])
{
    constexpr int KS = D / 32, TW = D / 64;
    typedef aotx_delta_tile<D, NS> tile_t;
    const unsigned int w = k.w, g = k.g, lane = k.lane, i0 = 16u * w + 4u * g, kh = k.h / p.group, l16 = lane * 16u;
    const unsigned int width = p.heads * D * 2u;        /* bytes of a row of out */
    const unsigned int at_out = i0 * width + (k.h * D + k.col) * 2u;
    /* a wave's places within a chunk's parts, in bytes */
    typedef aotx_delta_chunk_work work_t;
    const unsigned int at_k = w * KS * 1024u + l16, at_p = w * 2048u + l16;
    const unsigned int at_of = (unsigned int)offsetof(work_t, of) + i0 * 4u;
    const unsigned int at_v = i0 * p.stride * 2u + (2u * p.key_heads * D + k.h * D + k.col) * 2u;
    /* the chunk that is loaded, and 1 while there is one: past the end the loads go through views
     * of no size, which read zeros and touch no memory, so that every pass has the same in flight */
    unsigned int ahead = 0u, there = 1u;
    const char *work = (const char *)(p.work + (unsigned long long)k.c0 * p.heads + k.h);
    const char *rows = (const char *)aotx_delta_rows_of(p, k.c0, kh, D);
    const unsigned long long work_step = sizeof(work_t) * (unsigned long long)p.heads;
    const unsigned long long rows_step = 256ull * D * p.key_heads;
    auto advance = [&]() {
        ++ahead;
        there = ahead < k.chunks ? 1u : 0u;
        work += work_step;
        rows += rows_step;
    };
    /* What a chunk needs comes from memory once for the head's slices, which share an L2, and each
     * would wait for the whole of it. So each asks for its share of the lines of a chunk some
     * passes before any is loaded: a line a lane of waves 0 (K, Q and V) and 1 (P, T, factors).
     * The last chunk, which may be a part of one, is left out. */
    const char *line = rows + (k.col >> 4) * 4096u + lane * 128u;
    unsigned long long line_step = rows_step;
    unsigned int line_c = 2u;
    if constexpr (NS == 1 && AHEAD == 3) {
        constexpr unsigned int LINES = sizeof(aotx_delta_factors) / 128u;
        constexpr unsigned int SLICES = D / 16, OF_WORK = (144u + LINES + SLICES - 1u) / SLICES;
        bool some = lane < 32u;
        if (w == 0u && lane >= 32u) {
            const unsigned int l = (k.col >> 4) * 16u + (lane & 15u);
            line = (const char *)(p.qkv + (unsigned long long)(k.seq.start + l / (D / 64)) * p.stride + 2u * p.key_heads * D
                                  + k.h * D) + l % (D / 64) * 128u;
            line_step = 128ull * p.stride;
            some = lane < 48u;
        } else if (w == 1u) {
            const unsigned int l = (k.col >> 4) * OF_WORK + lane, part = l / 48u, block = l % 48u / 8u;
            line = work + (part < 3u ? part * 8192u + (block < 2u ? 2u * block : block + 2u) * 1024u + l % 8u * 128u
                                     : (unsigned int)offsetof(work_t, of) + (l - 144u) * 128u);
            line_step = work_step;
            some = lane < OF_WORK && l < 144u + LINES;
        }
        some = some && k.chunks > 3u;
        if (!some) line_step = 0ull;            /* the lane asks for a chunk's first line again */
        if (!some) line = work;
        line += 2u * line_step;
    }
    auto touch = [&]() {
        const unsigned int v = *(const unsigned int *)line;
        if (++line_c < k.chunks - 1u) line += line_step;
        return v;
    };
    auto load_k = [&](tile_t &x) {
        const __amdgpu_buffer_rsrc_t f = aotx_part(rows, there * 256u * D);
#pragma unroll
        for (int s = 0; s < KS; ++s) x.k[s] = aotx_lane_16(f, at_k, s * 1024u);
    };
    auto load_q = [&](tile_t &x) {
        const __amdgpu_buffer_rsrc_t f = aotx_part(rows, there * 256u * D);
#pragma unroll
        for (int s = 0; s < KS; ++s) x.q[s] = aotx_lane_16(f, at_k, 128u * D + s * 1024u);
    };
    auto load_t = [&](tile_t &x) {
        const __amdgpu_buffer_rsrc_t f = aotx_part(work, there * (unsigned int)sizeof(work_t));
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            x.th[s] = aotx_lane_16(f, at_p, (unsigned int)offsetof(work_t, t_hi) + s * 1024u);
            x.tl[s] = aotx_lane_16(f, at_p, (unsigned int)offsetof(work_t, t_lo) + s * 1024u);
        }
    };
    auto load_rest = [&](tile_t &x) {
        const __amdgpu_buffer_rsrc_t f = aotx_part(work, there * (unsigned int)sizeof(work_t));
#pragma unroll
        for (int s = 0; s < NS; ++s) x.p[s] = aotx_lane_16(f, at_p, s * 1024u);
        const aotx_rows_view v = aotx_rows_of(p, k.seq.start + ahead * 64u, there * aotx_delta_left(k, ahead));
#pragma unroll
        for (int r = 0; r < 4; ++r)
            x.v[r] = aotx_rows_2(v, at_v + r * p.stride * 2u);
        x.of_k = __builtin_bit_cast(aotx_f4, aotx_lane_16(f, at_of, 0u));
        x.of_q = __builtin_bit_cast(aotx_f4, aotx_lane_16(f, at_of, 256u));
        x.of_u = __builtin_bit_cast(aotx_f4, aotx_lane_16(f, at_of, 512u));
        x.of_b = __builtin_bit_cast(aotx_f4, aotx_lane_16(f, at_of, 768u));
        x.fade = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(f, 0, (int)(offsetof(work_t, of) + offsetof(aotx_delta_factors, fade)), 0));
        if constexpr (NS == 1 && AHEAD == 3) x.touched = touch();
        advance();
    };
    /* The columns' vmax in the coming period, or, one chunk ahead, in the one that begins: there four
     * registers are worth more than the wait (64 sequences of 16 rows of 32 heads of 128 185 us, with
     * them held for a period and others spilled 195). */
    unsigned char top[AOTX_DELTA_PERIOD];
    auto load_top = [&](unsigned int c) {
#pragma unroll
        for (unsigned int q = 0; q < AOTX_DELTA_PERIOD; ++q)
                top[q] = p.work[(unsigned long long)(k.c0 + (c + q < k.chunks ? c + q : k.chunks - 1u)) * p.heads
                                   + k.h].of.vmax[k.col];
    };

    aotx_f4 S[TW];                              /* times 2^shift */
    int shift = 0;
    float *sp = p.state + ((unsigned long long)k.seq.slot * p.heads + k.h) * D * D + k.col;
    if constexpr (AHEAD > 0) {
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned int tile = w * TW + t;
                const unsigned int key = 32u * (tile >> 1) + 8u * g + 4u * (tile & 1u) + r;
                S[t][r] = k.seq.fresh ? 0.0f : sp[key * D];
            }
    } else {
#pragma unroll
        for (int t = 0; t < TW; ++t) S[t] = (*one_state)[t];
    }
    /* in the order in which the passes load, so that the waits for them count alike */
    tile_t A, B;
    if constexpr (AHEAD == 0) {
        A = *one;
    } else {
        if constexpr (AHEAD > 1) load_top(0u);
        load_k(A);
        load_q(A);
        load_t(A);
        load_rest(A);
    }
    if constexpr (AHEAD > 1) {
        load_k(B);
        load_q(B);
        load_t(B);
    }

    /* the chunk before: its output, still to be stored */
    aotx_f4 o;
    int o_shift;
    auto store = [&](unsigned int c) {
        /* rows past the chunk are past the view's end: the store drops them */
        const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(
            (char *)p.out + (unsigned long long)(k.seq.start + c * 64u) * width, (short)0,
            (int)(aotx_delta_left(k, c) * width), 0x00020000);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            __builtin_amdgcn_raw_buffer_store_b16(aotx_f2h(ldexpf(o[r], -o_shift)), to, (int)(at_out + r * width), 0, 0);
    };
    auto scale = [&](unsigned int c) {
        /* in the period |S|, |X| and |U| of a column stay below sqrt(d) max|S| + 257 max(beta |v|), which
         * the exponents plus 5 and plus 10 are bounds of. Of zeros alone in V there is none. */
        float ms = 0.0f;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) ms = fmaxf(ms, fabsf(S[t][r]));
        ms = fmaxf(ms, __shfl_xor(ms, 16, 64));
        ms = fmaxf(ms, __shfl_xor(ms, 32, 64));
        if constexpr (AHEAD == 1) load_top(c);
        int ex = aotx_exponent(ms) - shift + 5, ev = one_top;
        if constexpr (AHEAD > 0)
#pragma unroll
            for (unsigned int q = 0; q < AOTX_DELTA_PERIOD; ++q) ev = top[q] > ev ? top[q] : ev;
        ev = ev != 0 ? ev - 1 + 10 - 126 : -512;
        ex = ex > ev ? ex : ev;
        if (g == 0u) lds.size[w][k.m] = ex;
        __syncthreads();
        ex = lds.size[0][k.m];
#pragma unroll
        for (int v = 1; v < 4; ++v) ex = lds.size[v][k.m] > ex ? lds.size[v][k.m] : ex;
        ex = 14 - ex;
        ex = ex > 126 ? 126 : ex < -120 ? -120 : ex;
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] = ldexpf(S[t][r], ex - shift);
        shift = ex;
        if constexpr (AHEAD > 1) load_top(c + AOTX_DELTA_PERIOD);
    };
    auto pass = [&](tile_t &x, tile_t &other, unsigned int c) {
        /* rows that are taken out, or past the chunk, have a beta or zeros in K, Q and V of 0: their X, U
         * and T are zeros by themselves. Only a chunk with values that are no numbers asks more. */
        const int fade = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x.fade));
        if constexpr (NS == 1 && AHEAD == 3) asm volatile("" ::"v"(x.touched));
        unsigned int lim = 64u;
        if (fade < 0) {
            lim = (AHEAD > 0 ? p.work[(unsigned long long)(k.c0 + c) * p.heads + k.h].of.odd : one_odd) & 0xFFu;
            unsigned int first = 64u;
#pragma unroll
            for (int r = 3; r >= 0; --r)
                if ((x.v[r] & 0x7FFFu) >= 0x7C00u) first = i0 + r;
            unsigned int f = (unsigned int)__shfl_xor((int)first, 16, 64);
            first = f < first ? f : first;
            f = (unsigned int)__shfl_xor((int)first, 32, 64);
            first = f < first ? f : first;
            if (g == 0u) lds.bad[w][k.m] = first;
            __syncthreads();
#pragma unroll
            for (int v = 0; v < 4; ++v) lim = lds.bad[v][k.m] < lim ? lds.bad[v][k.m] : lim;
        }
        /* K's rows to LDS while the state's last products run, and back by columns while the chain waits
         * for X */
#pragma unroll
        for (int s = 0; s < KS; ++s) *(aotx_h8 *)&lds.k[16u * w + k.m][32 * s + 8u * g] = x.k[s];
        aotx_h4 hi, lo;
#pragma unroll
        for (int t = 0; t < TW; ++t) {
            aotx_split4(S[t], &hi, &lo);
            const unsigned int tile = w * TW + t;
            *((aotx_h4 *)&lds.s[tile >> 1][0][lane] + (tile & 1u)) = hi;
            *((aotx_h4 *)&lds.s[tile >> 1][1][lane] + (tile & 1u)) = lo;
        }
        __syncthreads();
        aotx_h8 sh[KS], sl[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            sh[s] = lds.s[s][0][lane];
            sl[s] = lds.s[s][1][lane];
        }
        aotx_f4 a = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            a = aotx_mma(x.k[s], sl[s], a);
            a = aotx_mma(x.k[s], sh[s], a);
        }
        if constexpr (AHEAD > 1) load_rest(other);
        aotx_f4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = fmaf(aotx_h2f(x.v[r]), ldexpf(x.of_b[r], shift), -(x.of_k[r] * a[r]));
        if (fade < 0) {
            asm volatile("");               /* a branch that is not taken, no selects */
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i0 + r >= lim) y[r] = 0.0f;
        }
        aotx_split4(y, &hi, &lo);
        *((aotx_h4 *)&lds.x[w >> 1][0][lane] + (w & 1u)) = hi;
        *((aotx_h4 *)&lds.x[w >> 1][1][lane] + (w & 1u)) = lo;
        __syncthreads();
        aotx_h8 xh[NS], xl[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            xh[s] = lds.x[s][0][lane];
            xl[s] = lds.x[s][1][lane];
        }
        if (c != 0u) store(c - 1u);
        aotx_f4 qs = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qs = aotx_mma(x.q[s], sl[s], qs);
            qs = aotx_mma(x.q[s], sh[s], qs);
        }
        /* K by columns: lane (m, g) addresses row m / 4 of four, keys 8 (m % 4) .. + 3 of the
         * tile's 16, and gets key m of it for all four rows */
        aotx_h8 kt[TW][2];
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                typedef short s4 __attribute__((ext_vector_type(4)));
                const unsigned int tile = w * TW + t;
                unsigned short *at = &lds.k[32 * s + 4u * g + (k.m >> 2)][32u * (tile >> 1) + 4u * (tile & 1u) + 8u * (k.m & 3u)];
                const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at);
                const s4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(at + 16 * (D + 8)));
                kt[t][s] = __builtin_bit_cast(aotx_h8, __builtin_shufflevector(a, z, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        if constexpr (AHEAD > 0) load_k(x);
        a = aotx_f4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            a = aotx_mma(x.th[s], xl[s], a);
            a = aotx_mma(x.tl[s], xh[s], a);
            a = aotx_mma(x.th[s], xh[s], a);
        }
        o = x.of_q * qs;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            o = aotx_mma(x.p[s], xl[s], o);
            o = aotx_mma(x.p[s], xh[s], o);
        }
        o_shift = shift + AOTX_DELTA_OUT_UP;
        aotx_split4(a * x.of_u, &hi, &lo);
        *((aotx_h4 *)&lds.v[w >> 1][0][lane] + (w & 1u)) = hi;
        *((aotx_h4 *)&lds.v[w >> 1][1][lane] + (w & 1u)) = lo;
        __syncthreads();
        aotx_h8 vh[2], vl[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            vh[s] = lds.v[s][0][lane];
            vl[s] = lds.v[s][1][lane];
        }
        if constexpr (AHEAD > 0) {
            load_q(x);
            load_t(x);
        }
#pragma unroll
        for (int t = 0; t < TW; ++t) S[t] *= fabsf(__builtin_bit_cast(float, fade));
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int t = 0; t < TW; ++t) {
                S[t] = aotx_mma(kt[t][s], vl[s], S[t]);
                S[t] = aotx_mma(kt[t][s], vh[s], S[t]);
            }
        }
        if (fade < 0) {
            asm volatile("");
            const float nan = __builtin_nanf("");
#pragma unroll
            for (int t = 0; t < TW; ++t)
                if (lim < 64u) S[t] = aotx_f4{nan, nan, nan, nan};
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i0 + r >= lim) o[r] = nan;
        }
        if constexpr (AHEAD == 1) load_rest(x);
    };
    /* a period a turn: no branch but the ways out, and the loads in flight are always the same */
    for (unsigned int c = 0;;) {
        scale(c);
        pass(A, B, c);
        if (AHEAD == 0 || ++c >= k.chunks) break;
        pass(AHEAD > 1 ? B : A, A, c);
        if (++c >= k.chunks) break;
        pass(A, B, c);
        if (++c >= k.chunks) break;
        pass(AHEAD > 1 ? B : A, A, c);
        if (++c >= k.chunks) break;
    }
    store(k.chunks - 1u);
#pragma unroll
    for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned int tile = w * TW + t;
            const unsigned int key = 32u * (tile >> 1) + 8u * g + 4u * (tile & 1u) + r;
            sp[key * D] = ldexpf(S[t][r], -shift);
        }
}

template <int D, int AHEAD>
__global__ __launch_bounds__(256, AHEAD > 1 ? 2 : 3) void aotx_delta_across(aotx_delta_args p)
{
    constexpr unsigned int SLICES = D / 16;
    __shared__ aotx_delta_lds<D> lds;
    aotx_delta_walk k;
    k.lane = threadIdx.x & 63u;
    k.m = k.lane & 15u;
    k.g = k.lane >> 4;
    k.w = (unsigned int)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    /* the slices of a head go to one XCD, too, whose L2 then holds what they share */
    const unsigned int unit = blockIdx.x / (8u * SLICES) * 8u + blockIdx.x % 8u;
    const unsigned int slice = blockIdx.x / 8u % SLICES;
    if (unit >= p.seqs.seqs * p.heads) return;
    const unsigned int i = unit / p.heads;
    k.h = aotx_delta_head(p, unit % p.heads);
    unsigned int mine, before;
    const aotx_seq_lanes seqs = aotx_seqs_read(p.seqs);
    aotx_delta_chunks(p, seqs, &mine, &before);
    k.seq = aotx_seq_of(p.seqs, i, seqs);
    k.c0 = (unsigned int)__builtin_amdgcn_readlane((int)before, (int)i);
    if (k.seq.end - k.seq.start <= p.few) return;
    k.chunks = (k.seq.end - k.seq.start + 63u) / 64u;
    k.col = slice * 16u + k.m;                          /* this lane's column */
    if (k.seq.refused) {
        if (threadIdx.x == 0u && slice == 0u && k.h == 0u) atomicAdd(p.seqs.faults, 1u);
        for (unsigned int t = k.seq.start + k.w * 4u + k.g; t < k.seq.end; t += 16u)
            p.out[((unsigned long long)t * p.heads + k.h) * D + k.col] = 0;
        return;
    }
    /* (scalar: the barriers of both ways count together) */
    if (k.w < 2u) aotx_delta_follow<D, 1, AHEAD>(p, k, lds, nullptr, 0, 0u, nullptr);
    else aotx_delta_follow<D, 2, AHEAD>(p, k, lds, nullptr, 0, 0u, nullptr);
}

/* ---------------------------------------------------------------------------------------
 * A call of up to 64 rows: no sequence has more than one chunk, and a workgroup (five waves, as
 * within) makes T and P for its 16 columns by itself. They stay in the registers of the waves that
 * take them, and a second launch and the way through memory are saved; the slices of a head make
 * the same T and P, which costs nothing while the chip has room. 40 rows of 32 heads of 128 take
 * 8.6 us, the latency of a launch, the rows and one chunk's chain; in two launches 12.5.
 * ------------------------------------------------------------------------------------- */
template <int D, int NS>
static __device__ __forceinline__ void aotx_delta_go_on(const aotx_delta_args &p, const aotx_delta_walk &k,
                                                        aotx_delta_lds<D> &lds, const aotx_delta_factors &of,
                                                        const aotx_f4 (&S)[D / 64], const aotx_delta_made<D> &made)
{
    aotx_delta_tile<D, NS> x;
    const unsigned int i0 = 16u * k.w + 4u * k.g;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        x.k[s] = made.k[s];
        x.q[s] = made.q[s];
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        x.p[s] = made.p[s];
        x.th[s] = made.th[s];
        x.tl[s] = made.tl[s];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) x.v[r] = made.v[r];
    x.of_k = *(const aotx_f4 *)&of.of_k[i0];
    x.of_q = *(const aotx_f4 *)&of.of_q[i0];
    x.of_u = *(const aotx_f4 *)&of.of_u[i0];
    x.of_b = *(const aotx_f4 *)&of.of_b[i0];
    x.fade = of.fade;
    aotx_delta_follow<D, NS, 0>(p, k, lds, &x, made.top, of.odd, &S);
}

template <int D>
__global__ __launch_bounds__(320) void aotx_delta_short(aotx_delta_args p)
{
    constexpr unsigned int SLICES = D / 16;
    __shared__ aotx_delta_within_lds<D> made_lds;
    __shared__ aotx_delta_lds<D> lds;
    __shared__ __align__(16) aotx_delta_factors of;
    aotx_delta_walk k;
    k.lane = threadIdx.x & 63u;
    k.m = k.lane & 15u;
    k.g = k.lane >> 4;
    k.w = (unsigned int)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const unsigned int unit = blockIdx.x / (8u * SLICES) * 8u + blockIdx.x % 8u;
    const unsigned int slice = blockIdx.x / 8u % SLICES;
    if (unit >= p.seqs.seqs * p.heads) return;
    k.h = aotx_delta_head(p, unit % p.heads);
    k.seq = aotx_seq_of(p.seqs, unit / p.heads, aotx_seqs_read(p.seqs));
    const unsigned int n = k.seq.end - k.seq.start;
    if (n == 0u) return;
    k.c0 = 0u;
    k.chunks = 1u;
    k.col = slice * 16u + k.m;
    if (k.seq.refused) {
        if (threadIdx.x == 0u && slice == 0u && k.h == 0u) atomicAdd(p.seqs.faults, 1u);
        if (k.w < 4u)
            for (unsigned int t = k.seq.start + k.w * 4u + k.g; t < k.seq.end; t += 16u)
                p.out[((unsigned long long)t * p.heads + k.h) * D + k.col] = 0;
        return;
    }
    if (k.w == 4u) {
        aotx_delta_rates<D, true>(p, made_lds, &of, k.seq.start, n, k.h);
        /* the barriers of the others: one in scale, three in a pass, one more of an odd chunk */
        const unsigned int more = __builtin_amdgcn_readfirstlane((int)of.odd) != 64 ? 5u : 4u;
        for (unsigned int b = 0; b < more; ++b) __syncthreads();
        return;
    }
    aotx_f4 S[D / 64];
    const float *sp = p.state + ((unsigned long long)k.seq.slot * p.heads + k.h) * D * D + k.col;
#pragma unroll
    for (int t = 0; t < D / 64; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned int tile = k.w * (D / 64) + t;
            const unsigned int key = 32u * (tile >> 1) + 8u * k.g + 4u * (tile & 1u) + r;
            S[t][r] = k.seq.fresh ? 0.0f : sp[key * D];
        }
    aotx_delta_made<D> made;
    aotx_delta_make<D, true>(p, made_lds, nullptr, 0u, k.h, k.w, k.seq.start, n, slice * 16u, made);
    if (k.w < 2u) aotx_delta_go_on<D, 1>(p, k, lds, of, S, made);
    else aotx_delta_go_on<D, 2>(p, k, lds, of, S, made);
}

#endif
