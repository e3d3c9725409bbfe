/* Q8_0 products of many rows with an epilogue (aotx_q8_linear). */
#include "rgemv_dev.h"
#include "linear.h"

typedef __attribute__((address_space(3))) void lg_lds;
typedef const __attribute__((address_space(1))) void lg_global;

#define LG_TILES 16             /* weight tiles of a workgroup */

/* This wave's loads have arrived and its LDS reads too, then the workgroup's. */
static __device__ __forceinline__ void lg_barrier()
{
    __builtin_amdgcn_s_waitcnt(0x0070);          /* vmcnt(0) lgkmcnt(0) */
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

/* Where a lane reads a 16-row tile of weights (as rg_wsrc): a uniform base and an offset of 32 bits, which
 * take a register of the lane where a pointer takes two. */
template <bool FILE>
struct lg_src {
    const unsigned char *q;             /* the tile (FILE: its first row) */
    const unsigned short *s;            /* Q8R: its scales */
    unsigned int off;                   /* FILE: of the lane's row */
};
template <bool FILE>
static __device__ __forceinline__ lg_src<FILE> lg_open(const aotx_rgemv_args &a, unsigned int group, unsigned int j, unsigned int lane)
{
    lg_src<FILE> w;
    w.off = 0u;
    if constexpr (FILE) {
        const bool gated = a.epi == AOTX_EPI_SWIGLU;
        unsigned int row = rg_vrow(a, group, j, 0u, LG_TILES);
        row = row < a.n ? row : a.n - 1u;                /* past the last row: discarded */
        const unsigned int row_bytes = a.k / 32u * 34u, left = a.n - 1u - row, r = lane & 15u;
        w.q = (const unsigned char *)rg_first((unsigned long long)(rg_seg_w(a, gated && j >= LG_TILES / 2u ? 1u : 0u)
                                                                   + (unsigned long long)row * row_bytes));
        w.s = nullptr;
        w.off = (r < left ? r : left) * row_bytes;
    } else {
        unsigned int dummy = 0u;
        w.q = (const unsigned char *)rg_first((unsigned long long)rg_tile(a, group, j, LG_TILES, 0u, dummy));
        w.s = (const unsigned short *)rg_first((unsigned long long)rg_scales(a, group, j, LG_TILES, 0u));
    }
    return w;
}
/* Quad q's words: HALF 0 the first four and the ninth (Q8R: the scale; FILE: as rg_wreg, of the row's last block past its
 * end), HALF 1 the next four. */
template <bool FILE, int HALF>
static __device__ __forceinline__ void lg_load(const aotx_rgemv_args &a, const lg_src<FILE> &w, unsigned int q, unsigned int lane,
                                               rg_u4 &words, unsigned int &ninth)
{
    if constexpr (FILE) {
        const unsigned int last = a.k / 32u - 1u, at = 4u * q + (lane >> 4);
        const unsigned int byte = w.off + (at < last ? at : last) * 34u;
        const unsigned int odd = ((unsigned int)(unsigned long long)w.q + byte) & 2u;     /* the quants are aligned */
        typedef unsigned int u4d __attribute__((ext_vector_type(4), aligned(4)));
        words = *(const u4d *)(w.q + (byte + odd + HALF * 16u));
        if (HALF == 0) ninth = *(const unsigned short *)(w.q + (byte + (odd ? 0u : 32u)));
    } else {
        words = *(const rg_u4 *)(w.q + (unsigned long long)q * 2048ull + lane * 16u + HALF * 1024u);
        if (HALF == 0) ninth = *((w.s + (unsigned long long)q * 64ull) + lane);
    }
}
/* Step s's eight values of a lane as the A operand. */
template <bool FILE>
static __device__ __forceinline__ rg_h8 lg_values(const rg_wreg &o, unsigned int shift, rg_h2 scale, int s)
{
    const auto w = [&](int j) { return j < 4 ? o.w0[j] : j < 8 ? o.w1[j - 4] : o.sc; };
    const auto word = [&](int i) { return FILE ? __builtin_amdgcn_alignbit(w(i + 1), w(i), shift) ^ 0x80808080u : w(i); };
    return rg_afrag(word(2 * s), word(2 * s + 1), scale);
}

/* y = act(x w^T + bias) [* (x up^T + up_bias)] + resid over BM batch rows and 256 weight rows (of a pair 128 of each) a
 * workgroup: 8 waves, 4 along the weight rows and 2 along the batch rows, 64 x BM / 2 sums of a wave in registers.
 * A weight value is half(quant * scale), made in registers by the two waves that multiply it, so that LDS holds x
 * alone, two quads of 128 columns of it, which the loads write without passing through registers; a quad's weights
 * are loaded one quad ahead. Every weight is read m / BM times and x n / 256 times, from L2 and the last level's cache.
 * The matrix cores bound it, and the clock that they pull down: 2048 rows of the gated 14336 x 4096 take 455 us (445 to
 * 480 by the card), 1.06 PFLOP/s, where a library's fp16 product of 8192 cubed reaches 1.14 on the same card; the same rows through x and
 * weights staged in LDS in passes of 512 take 579. Instructions of 32 x 32 x 16, weights without the second buffer, a
 * fixed order of instructions and loads of weights into L2 ahead took 487 to 526. */
template <int BM, bool FILE>
__global__ __launch_bounds__(512, 2) void aotx_linear_gemm(aotx_rgemv_args a, aotx_linear_epi e, aotx_lgemm_plan p)
{
    constexpr int CB = BM / 32;                  /* column blocks of a wave */
    constexpr int DMA = BM / 32;                 /* a wave's loads of a quad of x, 4 rows each */
    constexpr unsigned int QUAD = BM * 256u;     /* LDS bytes of a quad of x */
    __shared__ __attribute__((aligned(1024))) unsigned char x0[QUAD], x1[QUAD];
    aotx_args_touch(a);
    const unsigned int tid = threadIdx.x, lane = tid & 63u;
    const unsigned int wave = (unsigned int)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const unsigned int r = lane & 15u, g = lane >> 4;
    const unsigned int wn = wave & 3u, wm = wave >> 2;
    const bool gated = a.epi == AOTX_EPI_SWIGLU;

    const unsigned int xcd = blockIdx.x & 7u, seq = blockIdx.x >> 3;
    const bool part = seq >= p.whole;
    const unsigned int t = part ? p.whole + (seq - p.whole) / p.splits : seq;
    const unsigned int split = part ? (seq - p.whole) % p.splits : 0u;
    const unsigned int group = t / p.ny * 8u + xcd, yb = t % p.ny;
    if (group >= p.groups) return;
    const unsigned int q0 = part ? split * p.qps : 0u;
    const unsigned int q1 = part && q0 + p.qps < a.qn ? q0 + p.qps : a.qn;
    const unsigned int m0 = yb * (unsigned int)BM;
    const unsigned int mrows = a.m - m0 < (unsigned int)BM ? a.m - m0 : (unsigned int)BM;

    /* a wave's 4 tiles: of a pair two of each, so that both sums of an output are in one lane */
    unsigned int tile[4];
    lg_src<FILE> src[4];
#pragma unroll
    for (unsigned int j = 0; j < 4u; ++j) {
        tile[j] = gated ? (j >> 1) * 8u + wn * 2u + (j & 1u) : wn * 4u + j;
        src[j] = lg_open<FILE>(a, group, tile[j], lane);
    }
    const unsigned int wend = rg_wend<FILE>(a, lane);
    /* FILE: as rg_wshift. Sixteen rows are a multiple of four bytes, so that a matrix has one */
    unsigned int shift[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        shift[i] = ((unsigned int)(unsigned long long)src[2 * i].q + r * (a.k / 32u * 34u) + 2u * g) & 2u ? 0u : 16u;

    /* x rows go straight to LDS, 16 bytes a lane. Piece 4g + s (8 values) of row m, which lane (m % 16, g) wants in step s,
     * is in place (4s + g) ^ (m % 16) of the row's 256 bytes: a step's reads then meet every bank once
     * in each of the hardware's groups of lanes (0-3, 12-15, 20-27 and so on; with 4g + s in place of 4s + g it is twice).
     * A row past the last one is the last again (its columns are not written). */
    const unsigned char *xb = (const unsigned char *)(a.x + (unsigned long long)m0 * a.ldx);
    const auto piece = [&](unsigned int row) {   /* in place lane % 16 of a row */
        const unsigned int at = (lane ^ row) & 15u;
        return (at & 3u) * 4u + (at >> 2);
    };
    /* a load's place in x: rows 4 apart differ by the row's length and by the two lowest bits of the piece, which are
     * made again for each load (two registers in place of one for each) */
    const unsigned int ld2 = a.ldx * 2u, last_row = (mrows - 1u) * ld2;
    unsigned int row0 = (wave * (BM / 8u) + (lane >> 4)) * ld2;
    unsigned int piece0 = piece(wave * (BM / 8u) + (lane >> 4)) * 16u;
    const auto place = [&](int i) {
        const unsigned int row = row0 + (unsigned int)i * 4u * ld2;
        return (row < last_row ? row : last_row) + (piece0 ^ (unsigned int)(i & 3) * 16u);
    };
    const auto stage = [&](unsigned char *buf, unsigned int q) {
#pragma unroll
        for (int i = 0; i < DMA; ++i)
            __builtin_amdgcn_global_load_lds((lg_global *)(xb + q * 256u + place(i)),
                                             (lg_lds *)(buf + (wave * (BM / 8u) + (unsigned int)i * 4u) * 256u), 16, 0, 0);
    };

    rg_f4 acc[4][CB];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < CB; ++c) acc[j][c] = (rg_f4){0.0f, 0.0f, 0.0f, 0.0f};
    unsigned int at = (wm * (BM / 2u) + r) * 256u + (g ^ r) * 16u;         /* the lane's reads; step s: ^ 64 s */
    const auto columns = [&](rg_h8 *B, const unsigned char *buf, int s) {
#pragma unroll
        for (int c = 0; c < CB; ++c) B[c] = *(const rg_h8 *)(buf + (at ^ (unsigned int)s * 64u) + (unsigned int)c * 4096u);
    };
    rg_wreg w0[4], w1[4];
    rg_h2 s0[4], s1[4];
    unsigned int lane_ = lane;
    const auto weights = [&](rg_wreg *w, unsigned int q) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned int none;
            lg_load<FILE, 0>(a, src[j], q, lane_, w[j].w0, w[j].sc);
            lg_load<FILE, 1>(a, src[j], q, lane_, w[j].w1, none);
        }
    };
    const auto scales = [&](rg_h2 *to, const rg_wreg *w, unsigned int q) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned int s = FILE && shift[j >> 1] != 0u ? w[j].w0[0] & 0xffffu : w[j].sc;
            if (FILE) s = q < wend ? s & 0xffffu : 0u;
            to[j] = __builtin_bit_cast(rg_h2, s | (s << 16));
        }
    };
    /* One quad, 4 steps of 4 tiles. The next step's columns are read and the next tile's values made while the
     * matrix cores have this one's. Between the steps 2 and 3 every wave has read all that it wants of the
     * quad and its loads for the next have come: after that barrier the next one but one may be loaded over this one, and
     * step 3 reads from the next. */
    rg_h8 b0[CB], b1[CB], A;
    const auto quad = [&](unsigned char *buf, const unsigned char *next, const rg_wreg *w, const rg_h2 *sc, rg_wreg *wn_, rg_h2 *scn,
                          unsigned int q, unsigned int qlast) {
        /* what a lane's addresses are made of is taken as new in every quad: kept from one to the next, the addresses
         * would take 40 registers, and sums would go to memory */
        asm volatile("" : "+v"(row0), "+v"(piece0), "+v"(at), "+v"(lane_));
        weights(wn_, q < qlast ? q + 1u : qlast);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s == 3) {
                lg_barrier();
                stage(buf, q + 2u < qlast ? q + 2u : qlast);
                scales(scn, wn_, q + 1u);
            }
            columns(s & 1 ? b0 : b1, s == 3 ? next : buf, (s + 1) & 3);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const rg_h8 now = A;
                A = j < 3 ? lg_values<FILE>(w[j + 1], shift[(j + 1) >> 1], sc[j + 1], s)
                  : s < 3 ? lg_values<FILE>(w[0], shift[0], sc[0], s + 1) : lg_values<FILE>(wn_[0], shift[0], scn[0], 0);
#pragma unroll
                for (int c = 0; c < CB; ++c)
                    acc[j][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(now, s & 1 ? b1[c] : b0[c], acc[j][c], 0, 0, 0);
            }
        }
    };

    const unsigned int qfull = a.k / 128u, q2 = q1 < qfull ? q1 : qfull;        /* whole quads [q0, q2) */
    const unsigned int qlast = q2 - 1u;
    if (q0 < q2) {
        stage(x0, q0);
        weights(w0, q0);
        stage(x1, q0 < qlast ? q0 + 1u : qlast);
        lg_barrier();
        scales(s0, w0, q0);
        columns(b0, x0, 0);
        A = lg_values<FILE>(w0[0], shift[0], s0[0], 0);
        for (unsigned int q = q0; q < q2; q += 2u) {
            quad(x0, x1, w0, s0, w1, s1, q, qlast);
            if (q + 1u >= q2) break;
            quad(x1, x0, w1, s1, w0, s0, q + 1u, qlast);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);          /* no load into LDS is under way any more */
    if (q2 < q1) {
        /* k ends inside the last quad: zeros past it, through registers */
        __syncthreads();
        weights(w0, q2);
#pragma unroll 2
        for (int i = 0; i < DMA; ++i) {
            const unsigned int row = wave * (BM / 8u) + (unsigned int)i * 4u + (lane >> 4);
            rg_u4 v = {0u, 0u, 0u, 0u};
            if (q2 * 128u + piece(row) * 8u < a.k) v = *(const rg_u4 *)(xb + q2 * 256u + place(i));
            *(rg_u4 *)(x0 + row * 256u + (lane & 15u) * 16u) = v;
        }
        __syncthreads();
        scales(s0, w0, q2);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            columns(b0, x0, s);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const rg_h8 now = lg_values<FILE>(w0[j], shift[j >> 1], s0[j], s);
#pragma unroll
                for (int c = 0; c < CB; ++c) acc[j][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(now, b0[c], acc[j][c], 0, 0, 0);
            }
        }
    }

    if (part && p.splits > 1u) {
        /* the last split of a tile to finish adds the others' sums in split order, its own from
         * registers (as rg_split_merge, whose stores and counter these are) */
        __shared__ unsigned int last;
        constexpr unsigned int FRAGS = 4u * CB;
        const unsigned int slot = xcd * (p.tiles - p.whole) + (t - p.whole);
        float *base = a.partial + (unsigned long long)slot * p.splits * (BM * 256u);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, (int)(p.splits * BM * 1024u), 0x00020000);
        const unsigned int place0 = (wave * FRAGS * 64u + lane) * 16u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < CB; ++c)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(rg_u4, acc[j][c]), rs,
                                                       (int)(split * BM * 1024u + place0 + (unsigned int)(j * CB + c) * 1024u), 0, RG_SC1);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0u) {
            const unsigned int arrived = atomicAdd(a.count + slot, 1u);
            last = arrived == p.splits - 1u ? 1u : 0u;
            if (last != 0u) atomicExch(a.count + slot, 0u);
        }
        __syncthreads();
        if (last == 0u) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            rg_f4 sum[CB];
#pragma unroll
            for (int c = 0; c < CB; ++c) sum[c] = (rg_f4){0.0f, 0.0f, 0.0f, 0.0f};
            for (unsigned int sp = 0u; sp < p.splits; ++sp) {
                rg_f4 v[CB];
#pragma unroll
                for (int c = 0; c < CB; ++c)
                    v[c] = sp == split ? acc[j][c]
                        : __builtin_bit_cast(rg_f4, __builtin_amdgcn_raw_buffer_load_b128(
                              rs, (int)(sp * BM * 1024u + place0 + (unsigned int)(j * CB + c) * 1024u), 0, RG_SC1));
#pragma unroll
                for (int c = 0; c < CB; ++c) sum[c] += v[c];
            }
#pragma unroll
            for (int c = 0; c < CB; ++c) acc[j][c] = sum[c];
        }
    }

    /* The sums go through LDS, half of the batch rows at a time: a loop of little code then writes whole lines of y
     * (from the registers, where every sum has code of its own, the activations alone would be 20000
     * instructions). Quad u of row m is in place u ^ (m % 16) of the row's kilobyte. */
    const unsigned int shift_u = gated ? 5u : 6u, units = 1u << shift_u;        /* four outputs each */
    /* Fours of y and resid at any alignment, as the memory takes such accesses whole (the outputs one at a time take
     * 1511 rows of 14029 x 256 with a residual from 88 to 109 us, 700 of 9001 x 1024 in halves from 37 to 43). */
    typedef float quad_f __attribute__((ext_vector_type(4), aligned(4)));
    typedef unsigned short quad_h __attribute__((ext_vector_type(4), aligned(2)));
    const auto sums = [&](unsigned int row, unsigned int unit) {
        return (rg_f4 *)((row < BM / 4u ? x0 : x1) + (row % (BM / 4u)) * 1024u + ((unit ^ (row & 15u)) * 16u));
    };
#pragma unroll 1
    for (unsigned int h = 0u; h < 2u; ++h) {
        __syncthreads();
        if (wm == h) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int c = 0; c < CB; ++c) *sums(16u * (unsigned int)c + r, tile[j] * 4u + g) = acc[j][c];
        }
        __syncthreads();
        const unsigned int mb = m0 + h * (BM / 2u), nb = group * units * 4u;
        const unsigned int left = a.m > mb ? a.m - mb : 0u, mend = left < BM / 2u ? left : BM / 2u;
        constexpr unsigned int U = 4u;
#pragma unroll 1
        for (unsigned int i0 = tid; i0 < units * mend; i0 += 512u * U) {
            rg_f4 res[U];
#pragma unroll
            for (unsigned int u = 0u; u < U; ++u) {
                const unsigned int i = i0 + 512u * u, unit = i & (units - 1u), row = i >> shift_u, n0 = nb + unit * 4u;
                res[u] = (rg_f4){0.0f, 0.0f, 0.0f, 0.0f};
                if (e.resid == nullptr || row >= mend || n0 >= a.n) continue;
                const float *from = e.resid + (unsigned long long)(mb + row) * e.ldr + n0;
                if (n0 + 4u <= a.n) res[u] = *(const quad_f *)from;
                else
#pragma unroll
                    for (unsigned int k = 0u; k < 4u; ++k)
                        if (n0 + k < a.n) res[u][k] = from[k];
            }
#pragma unroll
            for (unsigned int u = 0u; u < U; ++u) {
                const unsigned int i = i0 + 512u * u, unit = i & (units - 1u), row = i >> shift_u, n0 = nb + unit * 4u;
                if (row >= mend || n0 >= a.n) continue;
                rg_f4 v = *sums(row, unit), up = gated ? *sums(row, unit + 32u) : v;
#pragma unroll
                for (unsigned int k = 0u; k < 4u; ++k) {
                    const bool in = n0 + k < a.n;
                    float one = v[k];
                    if (e.bias != nullptr && in) one += e.bias[n0 + k];
                    one = rg_act(one, e.act);
                    if (gated) one *= up[k] + (e.up_bias != nullptr && in ? e.up_bias[n0 + k] : 0.0f);
                    v[k] = one + res[u][k];
                }
                const unsigned long long to = (unsigned long long)(mb + row) * a.ldy + n0;
                quad_h half = {0, 0, 0, 0};
                if (e.half)
#pragma unroll
                    for (int k = 0; k < 4; ++k) half[k] = aotx_f2h(v[k]);
                if (n0 + 4u <= a.n) {
                    if (e.half) *(quad_h *)((unsigned short *)a.y + to) = half;
                    else *(quad_f *)((float *)a.y + to) = v;
                } else {
#pragma unroll
                    for (unsigned int k = 0u; k < 4u; ++k) {
                        if (n0 + k >= a.n) continue;
                        if (e.half) ((unsigned short *)a.y)[to + k] = half[k];
                        else ((float *)a.y)[to + k] = v[k];
                    }
                }
            }
        }
    }
}

/* The plan and its time, in ns: a round of tiles on all CUs takes so long a quad of k and so long beside them, and the
 * sums of a split tile go to memory and back at 4.5 TB/s, and to the workgroup that adds them at 0.13. Measured over
 * 1000 to 14336 weight rows, 512 to 14336 columns and 64 to 2048 batch rows; on one card 2048 rows of the gated 14336 x 4096
 * take 477 us in tiles of 256 rows, 511 of 192 and 557 of 128, of 4096 square 109, 102 and 90, 1024 of 4096 square 80, 78
 * and 63. Over the file's layout, where addresses are what a quad costs, 192 rows
 * are the most whose sums stay in registers. */
unsigned long long aotx_lgemm_choose(aotx_lgemm_plan *p, unsigned int n, unsigned int k, unsigned int m, bool gated, bool file)
{
    struct form {
        unsigned int bm, quad, tile;
    };
    static const form packed[3] = {{256u, 3300u, 10000u}, {192u, 2750u, 9000u}, {128u, 2150u, 8000u}}, rows[1] = {{192u, 3900u, 9000u}};
    const unsigned int tiles = (unsigned int)aotx_q8r_tiles(n), qn = (unsigned int)aotx_q8r_quads(k);
    const unsigned int groups = gated ? (tiles + 7u) / 8u : (tiles + 15u) / 16u;
    unsigned long long best = ~0ull;
    for (unsigned int i = 0u; i < (file ? 1u : 3u); ++i) {
        const form f = file ? rows[0] : packed[i];
        aotx_lgemm_plan q;
        q.bm = f.bm;
        q.ny = (m + q.bm - 1u) / q.bm;
        q.groups = groups;
        q.tiles = (groups + 7u) / 8u * q.ny;
        q.whole = q.tiles / 32u * 32u;
        const unsigned int rest = q.tiles - q.whole;
        const unsigned long long rounds = (unsigned long long)(q.whole / 32u) * (qn * f.quad + f.tile);
        for (unsigned int s = 1u; s == 1u || (rest * s <= 32u && qn / s >= 4u); ++s) {
            q.qps = (qn + s - 1u) / s;
            q.splits = (qn + q.qps - 1u) / q.qps;
            unsigned long long time = rounds;
            if (rest != 0u) time += q.qps * f.quad + f.tile;
            if (rest != 0u && q.splits > 1u)
                time += 3000u + (unsigned long long)rest * 8u * q.splits * q.bm * 2048u / 4500u + q.splits * q.bm * 8u;
            if (time < best) {
                best = time;
                *p = q;
            }
            if (rest == 0u) break;
        }
    }
    return best;
}

size_t aotx_lgemm_partial_bytes(const aotx_lgemm_plan &p)
{
    return p.splits <= 1u ? 0u : (size_t)(p.tiles - p.whole) * 8u * p.splits * p.bm * 1024u;
}

void aotx_lgemm_launch(const aotx_lgemm_plan &p, const aotx_rgemv_args &a, const aotx_linear_epi &e, hipStream_t s)
{
    const dim3 grid((p.whole + (p.tiles - p.whole) * p.splits) * 8u);
#define LG_GO(BM, FILE) hipLaunchKernelGGL((aotx_linear_gemm<BM, FILE>), grid, dim3(512), 0, s, a, e, p)
    if (a.file) LG_GO(192, true);
    else if (p.bm == 256u) LG_GO(256, false);
    else if (p.bm == 192u) LG_GO(192, false);
    else LG_GO(128, false);
#undef LG_GO
    AOTX_LAUNCH_CHECK();
}
