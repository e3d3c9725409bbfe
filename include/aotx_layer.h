/* aotx_layer.h — C ABI of the operators of a full attention layer and of a step's answer.
 *
 * With these, a decoder's layer and its answer are calls alone, with no pass of the caller's
 * between them:
 *
 *   layer    aotx_norm_rows -> aotx_q8_linear (q, k, v with their bias) -> aotx_kv_append
 *            -> aotx_attend_paged -> aotx_q8_linear (out, with the residual)
 *            -> aotx_norm_rows -> aotx_q8_linear (gated) -> aotx_q8_linear (down, with the residual)
 *   answer   aotx_norm_rows -> aotx_q8_linear (head) -> aotx_logits_adjust -> aotx_pick
 *
 * All pointers are device pointers of the current HIP device unless marked host; stream is a
 * hipStream_t (null = the default stream). Every call is enqueued on its stream and returns;
 * none allocates once the library's device state exists, so all may be captured into a graph
 * after a first call or aotx_kv_open (before that, a captured call that may count a fault is
 * refused). They return 0 when they ran and 1, with nothing enqueued, for arguments they
 * refuse: a null pointer that has to be given, a shape or an alignment that is not named
 * below. What a call writes overlaps nothing that it reads, but where a description says
 * that it may. Two calls that use the same workspace or write the same rows have to follow
 * one another (one stream, or an event between streams).
 */
#ifndef AOTX_LAYER_H
#define AOTX_LAYER_H

#include "aotx_hip.h"
#include "aotx_hybrid.h"

#ifdef __cplusplus
extern "C" {
#endif

#define AOTX_ACT_NONE      0u
#define AOTX_ACT_SILU      1u   /* x / (1 + exp(-x)) */
#define AOTX_ACT_GELU      2u   /* x (1 + erf(x / sqrt(2))) / 2 */
#define AOTX_ACT_GELU_TANH 3u   /* x (1 + tanh(sqrt(2 / pi) (x + 0.044715 x^3))) / 2 */
#define AOTX_ACT_RELU      4u   /* x where x > 0, else 0 */

#define AOTX_LINEAR_F32 0u
#define AOTX_LINEAR_F16 1u

#define AOTX_LINEAR_ROWS_MAX (1u << 18)

typedef struct aotx_linear_how {
    const void *w;              /* Q8_0 [n][k] */
    const void *up;             /* a second matrix of that shape, or null */
    const float *bias;          /* [n], or null */
    const float *up_bias;       /* [n], or null; only with up */
    const float *resid;         /* fp32 rows, or null */
    unsigned int n;             /* 1 to AOTX_LINEAR_ROWS_MAX */
    unsigned int k;             /* a multiple of 32, up to 2^18 */
    unsigned int ldx;           /* values from one row of x to the next: a multiple of 8, k to 2^22 */
    unsigned int ldy;           /* of y: n to 2^22 */
    unsigned int ldr;           /* of resid: n to 2^22 */
    unsigned int act;           /* AOTX_ACT_* */
    unsigned int out;           /* AOTX_LINEAR_F32 or AOTX_LINEAR_F16 */
    unsigned int packed;        /* 1: w and up are repacked (aotx_q8_repack), 0: as the file has them */
} aotx_linear_how;

/* Q8_0 product with its epilogue:
 *   y = act(x w^T + bias) + resid                       up null
 *   y = act(x w^T + bias) * (x up^T + up_bias) + resid  otherwise
 * how host; x fp16, row i at x + i * ldx, m rows (up to 2^20, 0 does nothing); y fp32 or fp16,
 * row i at y + i * ldy. The weights' values are half(quant * scale), as aotx_q8_gemv has
 * them; sums, bias, activation, gate and residual are fp32, rounded once where y is fp16. resid may
 * be y itself (fp32 out, ldr = ldy): every value is read before it is written. x, and repacked
 * matrices, are 16-byte aligned, matrices in the file's layout 2-byte, the others by their type.
 * Inf and NaN reach the values whose sum holds them and no others.
 *
 * work is a workspace of work_bytes bytes, at least aotx_q8_linear_work of the same n, k, m and
 * up (fewer rows may ask for more than many do), 256-byte aligned. The caller sets its first AOTX_LINEAR_ZERO bytes to zero once, before the first
 * call that uses it; every call leaves them zero, so that calls of any shapes may use it one
 * after another. aotx_q8_linear_work returns 0 for sizes that are refused. */
#define AOTX_LINEAR_ZERO 65536ull
unsigned long long aotx_q8_linear_work(unsigned int n, unsigned int k, unsigned int m, unsigned int gated);
int aotx_q8_linear(const aotx_linear_how *how, const void *x, unsigned int m, void *y, void *work,
                unsigned long long work_bytes, void *stream);

/* RMSNorm of rows, the rows that a product takes:
 *   out[t][i] = x[t][i] / sqrt(mean over i of x^2 + eps) * w[i]
 * x fp32, row t at x + t * stride; w fp32 [width]; out fp16 [tokens][width]. width a multiple of 8
 * up to 32768, up to 2^20 tokens, stride a multiple of 4, at least width; x, w and out 16-byte
 * aligned, eps >= 0 (with 0 a row of zeros has no norm: NaN). Rows whose squares fp32 does not hold have
 * their norm too. */
int aotx_norm_rows(const float *x, unsigned int stride, const float *w, unsigned int tokens,
                   unsigned int width, float eps, void *out, void *stream);

/* Head norm (optional) and rotary turn of a product's q, k and v rows, with k and v written into
 * the pages: aotx_rope_axes and aotx_kv_write in one pass, over sequences. qkv, stride,
 * q_norm, k_norm, how (host), factor, heads, kv_heads, head_dim and tokens are those of
 * aotx_rope_axes, kv_heads at least 1. place unsigned [tokens][axes], or null: the turn goes by the
 * row's cache position (how->axes is 1). gain > 0 multiplies the turned values of q and k (those past
 * rope_dim stay), as models whose context was extended ask for; 1 for none.
 *
 * Sequences are those of aotx_hybrid.h: sequence i has the rows offset[i] .. offset[i + 1] - 1 (offset
 * null: row i alone, seqs = tokens), which stand at the cache positions pos[i], pos[i] + 1, ... of slot
 * agent[i]; at most AOTX_SLOTS of them. Rows outside all sequences are neither read nor
 * written. A sequence that names no slot (agent[i] >= AOTX_SLOTS), or one that an earlier sequence
 * with rows names too, gets q rows of zeros, writes nothing into the pages and adds 1 to
 * aotx_model_faulted(). A row whose position has no page gets its q row and adds 1 as well.
 *
 * page is the table [AOTX_SLOTS][AOTX_KV_PAGES_EACH] of the pages' addresses (0: none), as
 * aotx_kv_table_device() gives it; layer of layers as in aotx_kv_write. q fp16
 * [tokens][heads][head_dim], 16-byte aligned. row_pos and row_agent unsigned [tokens], both given or both null:
 * every row's position and slot, as aotx_attend_paged takes them (a refused sequence's rows, and those
 * whose position 32 bits do not hold: AOTX_SLOTS as their slot, where attention gives zeros). */
int aotx_kv_append(const float *qkv, unsigned int stride, const float *q_norm, const float *k_norm,
                   const aotx_rope_how *how, const float *factor, float gain,
                   const unsigned int *place, const unsigned int *offset, const unsigned int *pos,
                   const unsigned int *agent, unsigned int seqs, unsigned int tokens,
                   unsigned int heads, unsigned int kv_heads, unsigned int head_dim,
                   unsigned int layer, unsigned int layers, const unsigned long long *page, void *q,
                   unsigned int *row_pos, unsigned int *row_agent, void *stream);

typedef struct aotx_adjust_how {
    const aotx_model_how *sample;    /* [rows]: presence, frequency and repeat penalty, repeat window; null: none */
    const unsigned int *agent;       /* [rows]: the list of each row; null: row r has list r */
    const int *list;                 /* [lists][list_stride]: tokens so far, oldest first */
    const unsigned int *length;      /* [lists]: tokens in each (above list_stride: list_stride) */
    unsigned int lists;
    unsigned int list_stride;        /* up to 2^20 */
    const unsigned int *bias_at;     /* [rows + 1]: row r has the biases bias_at[r] .. bias_at[r + 1] - 1; null: none */
    const int *bias_token;           /* [biases] */
    const float *bias;               /* [biases] */
    unsigned int biases;
    const unsigned int *mask;        /* [masks][mask_stride] words: bit t % 32 of word t / 32 allows token t; null: none */
    const unsigned int *mask_of;     /* [rows]: the mask of each row (>= masks: none); null: row r has mask r */
    unsigned int masks;
    unsigned int mask_stride;        /* at least (vocab + 31) / 32 */
} aotx_adjust_how;

/* Penalties, biases and grammar masks on logits, before aotx_pick. For token t of row r, found
 * c times in the row's list:
 *   z = logits[r][t]
 *   z = z - (presence + frequency c)              where c > 0
 *   z = z > 0 ? z / repeat : z repeat             where t is among the last repeat_window of the list
 *   z = z + bias                                  of the row's last bias that names t
 *   z = -inf                                      where the mask does not allow t
 * as the decode tick's penalties go (fp32, presence + frequency c in one rounding). how host. logits
 * fp32, row r at logits + r * ld; out fp32, row r at out + r * ld_out, which may be logits itself
 * (ld_out = ld). Tokens of lists and biases that the vocabulary does not have count
 * nowhere; a row whose agent is no list has no penalties; an offset past `biases` is taken as `biases`,
 * and a row whose end is below its begin has no biases. A row with a mask that allows none of the
 * vocabulary is -inf everywhere and adds 1 to aotx_model_faulted(); aotx_pick, which has no
 * token to give, then gives 0 at temperature 0 and -1 above. rows up to 4096, vocab up to 2^20,
 * ld and ld_out from vocab to 2^22. */
int aotx_logits_adjust(const aotx_adjust_how *how, const float *logits, unsigned int ld,
                       unsigned int rows, unsigned int vocab, float *out, unsigned int ld_out,
                       void *stream);

#ifdef __cplusplus
}
#endif

#endif
