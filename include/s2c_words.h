/*
 * s2c_words.h -- C ABI of the word operators in libs2c_hip.so: what a captioner does around its word
 * logits (scan2cap_amd/csrc/s2c_vocab.hip, s2c_embed.hip; Python: scan2cap_amd/word_ops.py).
 *
 * Conventions as in s2c_ops.h: device pointers, asynchronous on `stream` (hipStream_t as void*), 0 on
 * success, S2C_EINVAL on a bad argument, a hipError_t from a failed launch.  Nothing is allocated and
 * nothing synchronises; workspaces belong to the caller and may be reused once the stream has passed
 * the call.  Element types: */
#ifndef S2C_WORDS_H
#define S2C_WORDS_H
#ifdef __cplusplus
extern "C" {
#endif

#define S2C_F32 0
#define S2C_BF16 1
#define S2C_F16 2

#define S2C_WORDS_MAX_TOP 64     /* alternatives of s2c_token_scores */
#define S2C_WORDS_MAX_SLOTS 256  /* teacher words per row of s2c_distill */
#define S2C_WORDS_MAX_DIM (1 << 24) /* columns of an embedding table */
#define S2C_WORDS_NO_PADDING (-9223372036854775807LL - 1) /* `padding` where no token is padding */

/* Word logits: `rows` rows of V elements (unit stride inside a row) of type `dtype`; row r starts at
 *   x + (r / (n1 n2)) s0 + (r / n2 % n1) s1 + (r % n2) s2        (elements)
 * so that up to three leading axes are read in place.  z = x * inv_t is what the softmax is taken of. */
typedef struct {
  int rows, V, dtype, n1, n2;
  float inv_t;
  long long s0, s1, s2;
  const void *x;
} s2c_logits;

/* Log probabilities of given words, entropy, best alternatives.  Per row, p = softmax(z):
 *   logp    = log p[token]              (token NULL: not computed)
 *   entropy = -sum p log p
 *   top_ids / top_logp (k <= S2C_WORDS_MAX_TOP, k <= V; may be 0): the k largest logits in descending
 *             order, equal ones in ascending index order, a NaN above everything
 * A row whose token equals `ignore` (has_ignore != 0) is not read: logp = entropy = top_logp = 0,
 * top_ids = -1.  A row without a finite logit (all -inf): logp = -inf, entropy = 0.  A token outside
 * [0, V): logp = NaN.  stats (rows x 4 floats, 16-byte aligned; NULL
 * where no backward follows) is what the backward needs.
 * ws: s2c_token_scores_workspace_bytes(rows, V, dtype, k) bytes, 8-byte aligned (may be 0). */
typedef struct {
  s2c_logits lg;
  int k, has_ignore;
  long long ignore;
  const long long *token;
  float *logp, *entropy, *top_logp;
  long long *top_ids;
  float *stats;
  void *ws;
} s2c_token_scores_args;
long long s2c_token_scores_workspace_bytes(int rows, int V, int dtype, int k);
int s2c_token_scores_fwd(const s2c_token_scores_args *a, void *stream);
/* dx (rows, V) contiguous, type of x:
 *   dx_v = ((g_logp [v == token] + sum_j g_top_j [v == top_ids_j])
 *           - p_v (g_logp + sum_j g_top_j + g_entropy (log p_v + entropy))) inv_t
 * any of g_logp / g_entropy / g_top may be NULL (0).  Uses a->lg, k, ignore, token, top_ids, stats.
 * Ignored rows and rows without a finite logit get zeros, a row with a bad token NaN. */
int s2c_token_scores_bwd(const s2c_token_scores_args *a, const float *g_logp, const float *g_entropy,
                         const float *g_top, void *dx, void *stream);

/* Distillation from a teacher's top logits: per row K <= S2C_WORDS_MAX_SLOTS slots of (id, logit),
 * id < 0 or a logit of -inf = an empty slot.  q = softmax over the used slots of teacher * inv_t,
 *   loss = sum_j q_j (log q_j - log p[id_j]),   p = softmax(x * inv_t) over all V words.
 * mask (rows bytes, may be NULL): rows with 0 are not read.  Masked rows and rows without a used slot:
 * loss 0, zero gradient.  A row of only -inf logits: loss +inf, zero gradient.  A used slot whose id is >= V
 * or whose logit is NaN or +inf: loss and the whole row's gradient NaN.
 * stats (rows x 4, or NULL) as above. */
typedef struct {
  s2c_logits lg;
  int K, teacher_dtype;
  const long long *ids;
  const void *teacher;
  const unsigned char *mask;
  float *loss, *stats;
  void *ws;
} s2c_distill_args;
long long s2c_distill_workspace_bytes(int rows, int V, int dtype);
int s2c_distill_fwd(const s2c_distill_args *a, void *stream);
/* dx (rows, V) contiguous: dx_v = g (p_v sum_j q_j - sum_{j: id_j = v} q_j) inv_t */
int s2c_distill_bwd(const s2c_distill_args *a, const float *g_loss, void *dx, void *stream);

/* size of s2c_logits (0), s2c_token_scores_args (1), s2c_distill_args (2) as compiled: a caller that was built
 * apart from the library compares them with its own before its first call */
long long s2c_words_args_sizeof(int which);

/* out (N, D) contiguous = scale * table[token] (table (V, D): unit column stride, row stride `ld`
 * elements); a token equal to `padding` (unless that is S2C_WORDS_NO_PADDING) gives zeros, any other one
 * outside [0, V) a row of NaN. */
int s2c_embed_fwd(long long N, int V, int D, int dtype, long long ld, const long long *token,
                  const void *table, float scale, long long padding, void *out, void *stream);
/* d_table (V, D) contiguous, every row written: scale * sum of g (N rows, row stride ldg) over the
 * places of each word, in their order, held in 32 bits and rounded once; padding and bad tokens
 * contribute nothing.  Same inputs, same bits.
 * ws: s2c_embed_grad_workspace_bytes(N, V, D) bytes, 16-byte aligned (may be 0).  N < 2^31. */
long long s2c_embed_grad_workspace_bytes(long long N, int V, int D);
int s2c_embed_grad(long long N, int V, int D, int dtype, long long ldg, const long long *token,
                   const void *g, float scale, long long padding, void *d_table, void *ws,
                   void *stream);

#ifdef __cplusplus
}
#endif
#endif
