/* aotx_hybrid.h — C ABI of the operators of hybrid models' layers.
 *
 * A hybrid model has linear layers, whose heads keep a matrix instead of a cache, beside full
 * attention layers whose rows carry several positions (the delta_* fields and rope_dim of
 * aotx_model_desc, and aotx_model_input.position). These are the operators that stand
 * between such a layer's products (aotx_q8_gemv, aotx_q8r_gemv):
 *
 *   linear layer   product -> aotx_delta_conv -> aotx_delta_step or aotx_delta_chunk
 *                  -> aotx_norm_gate -> product
 *   full layer     product -> aotx_rope_axes -> aotx_kv_write -> aotx_attend_paged -> product
 *
 * All pointers are device pointers of the current HIP device unless marked host; stream is a
 * hipStream_t (null = the default stream). Every call is enqueued on its stream and returns;
 * none allocates once the library's device state exists, so all may be captured into a graph
 * after a first call or aotx_kv_open (before that, a captured call is refused). They return 0
 * when they ran and 1, with nothing enqueued, for arguments they refuse: a null pointer that
 * has to be given, a shape or an alignment that is not named below.
 *
 * Sequences. A call's rows are packed one sequence after another: sequence i has the rows
 * offset[i] .. offset[i + 1] - 1, its state is that of slot agent[i], and pos[i] is the cache
 * position of its first row. A sequence at position 0 starts from zeros, whatever its slot
 * held. A sequence without rows leaves its slot as it was. Rows before offset[0] and from
 * offset[seqs] on are neither read nor written; an offset past `tokens` is taken as `tokens`, and
 * one below an earlier one as that one. A sequence that names no slot of the caller's
 * (agent[i] >= slots), or a slot that an earlier sequence with rows names too, gets rows of zeros,
 * changes no state, and adds 1 to aotx_model_faulted(). At most AOTX_SLOTS sequences and slots.
 *
 * Two calls that use the same state, or the same workspace, have to follow one another (one
 * stream, or an event between streams). What a call writes overlaps nothing that it reads, but
 * where a description says that it may.
 */
#ifndef AOTX_HYBRID_H
#define AOTX_HYBRID_H

#include "aotx_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Short causal convolution of every channel with SiLU, the q, k and v rows of a linear layer:
 *   out[t][c] = silu(bias[c] + sum over j < width of w[c][j] x[t - (width - 1) + j][c])
 * x fp32, row t at x + t * stride (stride values, at least channels); w fp32
 * [channels][width], oldest row first; bias fp32 [channels] or null; out fp16
 * [tokens][channels]. Rows before a sequence's first are those that its slot keeps:
 * state fp32 [slots][width - 1][channels], oldest first, which the call leaves holding the
 * last width - 1 rows of x. offset null: sequence i is row i alone (seqs = tokens).
 * channels (up to 2^20) and stride multiples of 4, tokens up to 2^20 and tokens times channels to
 * 2^37, width 2 to 4, x, w and state 16-byte aligned, bias and out as well. */
int aotx_delta_conv(const float *x, unsigned int stride, const float *w, const float *bias,
                    const unsigned int *offset, const unsigned int *pos,
                    const unsigned int *agent, unsigned int seqs, unsigned int tokens,
                    unsigned int channels, unsigned int width, float *state,
                    unsigned int slots, void *out, void *stream);

/* The gated delta rule. Value head h (of `heads`) has the key head h / (heads / key_heads)
 * and a state S of head_dim key rows by head_dim value columns; with q, k and v its rows of
 * one token:
 *   q' = q / sqrt(|q|^2 + eps) / sqrt(head_dim)     k' = k / sqrt(|k|^2 + eps)
 *   g = decay[h] * softplus(a + dt[h])              beta = 1 / (1 + exp(-b))
 *   S <- exp(g) S;  u = beta (v - S^T k');  S <- S + k' u^T;  out = S^T q'
 * qkv fp16: row t at qkv + t * stride values holds q [key_heads][head_dim], k
 * [key_heads][head_dim], v [heads][head_dim], as aotx_delta_conv writes them. a, b fp32: row
 * t at a + t * ab_stride, [heads] values. decay, dt fp32 [heads]; decay at most 0 (g above 0
 * is taken as 0). state fp32 [slots][heads][head_dim][head_dim]. out fp16
 * [tokens][heads][head_dim]. head_dim 64 or 128, key_heads divides heads, at most 256 heads,
 * eps at least 1e-30; stride a multiple of 8 up to 2^22; qkv, state and out 16-byte aligned. The
 * state is fp32, and its arithmetic is that or as near: the products of aotx_delta_chunk take
 * their operands as two fp16 parts, 2^-21 each, or 2^-33 of the largest state entry and 2^-28 of the
 * largest beta |v| that their column has in 256 rows, where that is more; the weights with which an
 * output takes the rows of its own 64 are rounded once, by 2^-11 of themselves or 2^-43. (Keys are taken
 * as they are while eps is at most 1/4; above that those much shorter than sqrt(eps) lose bits.) A value
 * of Inf or NaN reaches the rows from its own on and no earlier ones.
 *
 * aotx_delta_step: one token of each of `tokens` slots (row i is sequence i). */
int aotx_delta_step(const void *qkv, unsigned int stride, const float *a, const float *b,
                    unsigned int ab_stride, const float *decay, const float *dt,
                    const unsigned int *pos, const unsigned int *agent, unsigned int tokens,
                    unsigned int key_heads, unsigned int heads, unsigned int head_dim, float eps,
                    float *state, unsigned int slots, void *out, void *stream);

/* aotx_delta_chunk: sequences of any lengths, up to 2^20 rows a call. work is a workspace of
 * work_bytes bytes, at least aotx_delta_work of the same tokens, seqs, heads and head_dim,
 * 256-byte aligned; it holds nothing between calls. Those are 58 KB for every 64 rows and head of 128
 * (42 KB of 64): a prompt may be cut into calls of some thousand rows, each of which goes on where
 * the last one left the slot. */
unsigned long long aotx_delta_work(unsigned int tokens, unsigned int seqs, unsigned int heads,
                                   unsigned int head_dim);
int aotx_delta_chunk(const void *qkv, unsigned int stride, const float *a, const float *b,
                     unsigned int ab_stride, const float *decay, const float *dt,
                     const unsigned int *offset, const unsigned int *pos,
                     const unsigned int *agent, unsigned int seqs, unsigned int tokens,
                     unsigned int key_heads, unsigned int heads, unsigned int head_dim, float eps,
                     float *state, unsigned int slots, void *work, unsigned long long work_bytes,
                     void *out, void *stream);

/* RMSNorm of every head's row times its SiLU gate, the rows that a linear layer's output
 * product takes:
 *   out[t][h][i] = x[t][h][i] / sqrt(mean over i of x^2 + eps) * w[i] * silu(z[t][h][i])
 * x fp16 [tokens][heads][width]; z fp32, row t at z + t * z_stride (heads * width values); w
 * fp32 [width]; out fp16 [tokens][heads][width], which may be x itself. width a multiple of 8
 * up to 8192, up to 2^20 tokens and 65536 heads, z_stride a multiple of 4, all four 16-byte
 * aligned, eps >= 0 (with 0 a row of zeros has no norm: NaN). */
int aotx_norm_gate(const void *x, const float *z, unsigned int z_stride, const float *w,
                   unsigned int tokens, unsigned int heads, unsigned int width, float eps,
                   void *out, void *stream);

#define AOTX_ROPE_AXES_MAX  4u
#define AOTX_ROPE_AXES_RUNS 0u   /* pairs 0 .. span[0]-1 turn by axis 0, the next span[1] by axis 1, ... */
#define AOTX_ROPE_AXES_TURN 1u   /* pair i turns by axis i % axes while i < axes * span[i % axes], else by axis 0 */

typedef struct aotx_rope_how {
    float theta;                 /* base of the frequencies, > 0 */
    float eps;                   /* of the head norms */
    unsigned int rope_dim;       /* the first rope_dim values of a head turn, the others pass */
    unsigned int pairs;          /* AOTX_ROPE_PAIRS_SPLIT or AOTX_ROPE_PAIRS_ADJACENT */
    unsigned int axes;           /* 1 to AOTX_ROPE_AXES_MAX */
    unsigned int order;          /* AOTX_ROPE_AXES_RUNS or AOTX_ROPE_AXES_TURN */
    unsigned int span[AOTX_ROPE_AXES_MAX];  /* pairs of each axis; they sum to rope_dim / 2 */
} aotx_rope_how;

/* Head norm (optional) and rotary turn of q and k rows by the positions of several axes, and
 * v beside them, from the fp32 row of a product to the fp16 rows that aotx_attend_paged and
 * aotx_kv_write take. Pair i of the rope_dim / 2 pairs of a head turns by the angle
 *   place[t][axis of i] * theta^(-2 i / rope_dim) / factor[i]
 * with the angle held in 64 bits, so that far positions keep theirs. qkv: row t at
 * qkv + t * stride values, q [heads][head_dim], k [kv_heads][head_dim], v
 * [kv_heads][head_dim]; q_norm, k_norm fp32 [head_dim], each null for no norm; how host;
 * factor fp32 [rope_dim / 2] or null; place unsigned [tokens][axes]; q, k, v fp16
 * [tokens][heads or kv_heads][head_dim] (v null: not written; k and v null with kv_heads = 0).
 * head_dim 64 or 128, up to 1024 heads and kv_heads, tokens up to 2^20; rope_dim a multiple of 8,
 * 8 to head_dim; stride a multiple of 4; qkv, the norms, q, k and v 16-byte aligned. A head's norm takes
 * its squares as fp32 has them: values are below 2^60 in size, and where eps is below 2^-100 the largest of a
 * head is above 2^-50. */
int aotx_rope_axes(const float *qkv, unsigned int stride, const float *q_norm,
                   const float *k_norm, const aotx_rope_how *how, const float *factor,
                   const unsigned int *place, unsigned int tokens, unsigned int heads,
                   unsigned int kv_heads, unsigned int head_dim, void *q, void *k, void *v,
                   void *stream);

#ifdef __cplusplus
}
#endif

#endif
