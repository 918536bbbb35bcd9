/*
 * galvatron_ops_hip.h -- C ABI of the operators in libgalvatron_dp_hip.so
 *
 * The parts of a model that no layer covers, and that the search engine prices for every
 * vocabulary-parallel degree (the keys of other_time_cost / other_mem_cost of a DP call): the embedding
 * lookup before the first layer, the residual join and norm behind a block, the log probabilities behind the
 * head, and their gradients.  Every operator takes a shard of the vocabulary as well as all of it.
 *
 * Unlike the entry points of galvatron_dp_hip.h these take DEVICE pointers, queue their work on the stream
 * they are given (a hipStream_t; NULL is the null stream) on the calling thread's current device, and return
 * without waiting for it.  They allocate nothing, copy nothing to the host and may be captured into a graph:
 * working memory is the caller's (gdp_*_workspace says how much; 256-byte aligned, its contents do not
 * matter before or after).  Return codes and gdp_last_error() are those of galvatron_dp_hip.h; what the host
 * can see of a call (sizes, types, pointers, strides) is checked before anything is queued.
 *
 * Results do not depend on timing: the same inputs give the same bits.  Sums and statistics are held in
 * float32; what has a smaller type is rounded once, to nearest even.  Strides are in elements, between
 * rows; the elements of a row are neighbours.  Data need only be aligned to its element; rows that all start on
 * 16 bytes are read a little faster.  Outputs overlap neither inputs nor each other, but where it is said that they may.
 */
#ifndef GALVATRON_OPS_HIP_H
#define GALVATRON_OPS_HIP_H

#include "galvatron_dp_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define GDP_F32 0
#define GDP_F16 1
#define GDP_BF16 2
/* types of token numbers */
#define GDP_I32 0
#define GDP_I64 1

#define GDP_MAX_TOP 64         /* alternatives of gdp_logprob */
#define GDP_MAX_LOGPROB_PARTS 64 /* shards that gdp_logprob_join takes */
#define GDP_MAX_NORM_DIM 16384 /* width of gdp_norm */
#define GDP_MAX_VOCAB (1 << 22) /* columns of logits in one call */

/* Rows of an embedding table:  out[n] = scale * weight[tokens[n] - first] where
 * first <= tokens[n] < first + rows, and zeros where another shard of the table holds the token (or none). */
typedef struct gdp_embed {
    int64_t n;              /* tokens                                     */
    int64_t rows, dim;      /* of the table (shard)                       */
    int64_t first;          /* the token of its row 0                     */
    const void *tokens;     /* [n]                                        */
    int32_t token_type;
    int32_t weight_type, out_type;
    float scale;
    const void *weight;     /* [rows][dim]                                */
    int64_t weight_stride;
    void *out;              /* [n][dim]                                   */
    int64_t out_stride;
} gdp_embed;
int gdp_embed_forward(const gdp_embed *e, void *stream);

/* Its gradient:  out[r] = scale * sum over the n with tokens[n] == first + r of grad[n], added up in the order of n
 * over pieces of 16 to 128 tokens, and over the pieces in their order.  Every row is written, zeros where no
 * token asks for it; with `accumulate` the sums are added to what out holds, and other rows are not touched. */
typedef struct gdp_embed_grad {
    int64_t n, rows, dim, first;
    const void *tokens;
    int32_t token_type;
    int32_t grad_type, out_type;
    int32_t accumulate;
    float scale;
    const void *grad;       /* [n][dim]; a stride of 0 is a gradient that all places share */
    int64_t grad_stride;
    void *out;              /* [rows][dim]                                */
    int64_t out_stride;
    void *workspace;
    size_t workspace_bytes;
} gdp_embed_grad;
int gdp_embed_grad_workspace(int64_t n, int64_t rows, int64_t dim, size_t *bytes);
int gdp_embed_backward(const gdp_embed_grad *e, void *stream);

/* Log probabilities.  With z = scale * logits[row] and p = softmax(z):
 *   logp    = z[token] - lse      0 where the token is outside [0, vocab) ("no token here", e.g. -100)
 *   lse     = log(sum(exp(z)))
 *   entropy = -sum(p * log(p))    p = 0 contributes 0
 *   top_*   = the `top` largest logits, largest first, equal ones by number: log probability and token.
 *             NaN counts as -inf there.
 * A logit of -inf is a token that is ruled out.  Where all are, lse and logp are -inf and the entropy is 0.  A row
 * with NaN or +inf has NaN for its lse, logp and entropy.  lse is rounded to float32: -inf or inf where it is outside
 * of its range, though logp and entropy, which the row's level has no part in, are not. */
typedef struct gdp_logprob {
    int64_t n, vocab;       /* rows, columns                              */
    const void *logits;     /* [n][vocab]                                 */
    int64_t logits_stride;
    int32_t logits_type;
    int32_t token_type;
    const void *tokens;     /* [n]                                        */
    float scale;            /* > 0: 1 / temperature                       */
    int32_t top;            /* 0 .. min(GDP_MAX_TOP, vocab)               */
    float *logp, *lse, *entropy; /* [n] each                              */
    float *top_logp;        /* [n][top]                                   */
    int64_t *top_tokens;    /* [n][top]                                   */
    void *workspace;
    size_t workspace_bytes;
} gdp_logprob;
int gdp_logprob_workspace(int64_t n, int64_t vocab, int32_t logits_type, int32_t top, size_t *bytes);
int gdp_logprob_forward(const gdp_logprob *l, void *stream);
/* ... and row_stats [n][2]: the row's largest logit m, and log(sum(exp(scale * (logits[row] - m)))).  Their sum, scale * m
 * added, is lse; apart they keep the digits that lse is rounded by, which the gradient of rows far from zero needs.
 * 8-byte aligned. */
typedef struct gdp_logprob_stats {
    gdp_logprob given;
    float *row_stats;
} gdp_logprob_stats;
int gdp_logprob_forward_stats(const gdp_logprob_stats *l, void *stream);

/* The same for a vocabulary in shards: `parts` of each shard, whose first column is token `first`, are joined
 * after the ranks have exchanged them (16 + 8 * top bytes a row instead of the row).  Of a part:
 * stats [n][4] float32 (largest logit; sum of exp2; sum of exp2 times its exponent; the token's logit or
 * -inf), top_logits [n][top] float32, largest first, and top_tokens [n][top] int32, -1 behind the last of a shard with
 * fewer than `top` columns. */
typedef struct gdp_logprob_part {
    int64_t n, vocab, first;
    const void *logits;
    int64_t logits_stride;
    int32_t logits_type;
    int32_t token_type;
    const void *tokens;
    float scale;
    int32_t top;            /* 0 .. GDP_MAX_TOP                           */
    float *stats, *top_logits;
    int32_t *top_tokens;
    void *workspace;
    size_t workspace_bytes; /* gdp_logprob_workspace of the shard's sizes */
} gdp_logprob_part;
int gdp_logprob_parts(const gdp_logprob_part *l, void *stream);

typedef struct gdp_logprob_joint {
    int64_t n, vocab;       /* of the whole vocabulary                    */
    int32_t parts;          /* 1 .. GDP_MAX_LOGPROB_PARTS, in the order of their tokens */
    int32_t top;
    float scale;
    int32_t token_type;
    const void *tokens;
    const float *stats;     /* [parts][n][4]                              */
    const float *top_logits;   /* [parts][n][top]                         */
    const int32_t *top_tokens; /* [parts][n][top]                         */
    float *logp, *lse, *entropy;
    float *top_logp;
    int64_t *out_tokens;    /* [n][top]                                   */
} gdp_logprob_joint;
int gdp_logprob_join(const gdp_logprob_joint *l, void *stream);
typedef struct gdp_logprob_joint_stats {
    gdp_logprob_joint given;
    float *row_stats;       /* as of gdp_logprob_stats, of the whole row  */
} gdp_logprob_joint_stats;
int gdp_logprob_join_stats(const gdp_logprob_joint_stats *l, void *stream);

/* Gradient with respect to the logits (of a shard whose first column is token `first`), from the gradients of
 * logp, lse, entropy and top_logp:
 *   out_j = scale * (g (1[j = token] - p_j) + l p_j - h p_j (z_j - lse + entropy) + sum_i t_i (1[j = top_tokens_i] - p_j))
 * with p_j = exp(z_j - lse), of the lse that is given.  float32 rounds lse by one part in 2^24, so p_j is off by |lse| / 2^24
 * of itself; a row whose lse is below -2^24 has zeros (all of its tokens are masked, by -inf, -1e9 or the lowest value of
 * float32 or bfloat16).  gdp_logprob_backward_stats takes row_stats instead, with which rows at any level have the gradient
 * of their logp, and only one whose logits are all -inf has zeros.  A token outside the vocabulary has no g.  out may be logits itself, and does not overlap them otherwise. */
typedef struct gdp_logprob_grad {
    int64_t n, vocab, first;
    int64_t whole_vocab;       /* tokens outside [0, whole_vocab) are none */
    const void *logits;
    int64_t logits_stride;
    int32_t logits_type;       /* also out's                              */
    int32_t token_type;
    const void *tokens;
    float scale;
    int32_t top;               /* columns of top_tokens and grad_top      */
    const float *lse;          /* [n]                                     */
    const float *grad_logp, *grad_lse; /* [n] each, or NULL               */
    const float *entropy, *grad_entropy; /* [n] each, or both NULL        */
    const int64_t *top_tokens; /* [n][top], or NULL with top 0            */
    const float *grad_top;     /* [n][top]                                */
    void *out;
    int64_t out_stride;
} gdp_logprob_grad;
int gdp_logprob_backward(const gdp_logprob_grad *l, void *stream);
typedef struct gdp_logprob_grad_stats {
    gdp_logprob_grad given;    /* its lse is not read and may be NULL     */
    const float *row_stats;    /* [n][2], of the whole row                */
} gdp_logprob_grad_stats;
int gdp_logprob_backward_stats(const gdp_logprob_grad_stats *l, void *stream);

/* A block's output joined with the residual stream, with norms on both sides of the join:
 *   b      = post-norm of block (where post is not GDP_NORM_NONE), times gate
 *   stream = residual_scale * residual + block_scale * b
 *   normed = pre-norm of stream, before it is rounded            (what the next block reads)
 * norm(x) = (x - mean) * rstd * weight + bias over the row; mean is 0 for GDP_NORM_RMS, and rstd is
 * 1 / sqrt(mean of (x - mean)^2 + eps).  Without a block stream is residual_scale * residual and need not be
 * written.  A gate serves n / gates rows in turn: one gate for all rows, one for each sequence, or one a row.
 * stats [n][4]: mean and rstd of the post-norm, mean and rstd of the pre-norm (what the gradient takes).
 * Types: `type` of block and normed, `stream_type` of residual and stream -- the same, or GDP_F32. */
#define GDP_NORM_NONE 0
#define GDP_NORM_RMS 1
#define GDP_NORM_LAYER 2
typedef struct gdp_norm_params { /* of one norm */
    int32_t form;
    int32_t type;           /* of weight and bias                         */
    float eps;
    int32_t reserved;
    const void *weight;     /* [dim] or NULL: ones                        */
    const void *bias;       /* [dim] or NULL: zeros                       */
} gdp_norm_params;
typedef struct gdp_norm {
    int64_t n, dim;
    int32_t type, stream_type;
    const void *residual;   /* [n][dim]                                   */
    int64_t residual_stride;
    const void *block;      /* [n][dim] or NULL                           */
    int64_t block_stride;
    gdp_norm_params post, pre;
    const void *gate;       /* [gates][dim] or NULL                       */
    int64_t gates;          /* divides n                                  */
    int64_t gate_stride;
    int32_t gate_type;
    float residual_scale, block_scale;
    int32_t reserved;
    void *stream;           /* [n][dim]; NULL: not written                */
    int64_t stream_stride;
    void *normed;           /* [n][dim]; NULL with pre.form GDP_NORM_NONE */
    int64_t normed_stride;
    float *stats;           /* [n][4] or NULL                             */
} gdp_norm;
int gdp_norm_forward(const gdp_norm *p, void *stream);

/* Its gradients, from stream, block and stats as the forward pass left them.  Gradients of weights, biases and
 * gate are sums over their rows, in a fixed order; any of the outputs may be NULL. */
typedef struct gdp_norm_grad {
    int64_t n, dim;
    int32_t type, stream_type;
    const void *stream;     /* [n][dim]                                   */
    int64_t stream_stride;
    const void *block;      /* [n][dim] or NULL                           */
    int64_t block_stride;
    const float *stats;     /* [n][4]                                     */
    const void *grad_normed; /* [n][dim], of `type`; NULL with pre.form GDP_NORM_NONE */
    int64_t grad_normed_stride;
    const void *grad_stream; /* [n][dim], of `stream_type`, or NULL: zeros */
    int64_t grad_stream_stride;
    gdp_norm_params post, pre;
    const void *gate;
    int64_t gates, gate_stride;
    int32_t gate_type;
    float residual_scale, block_scale;
    int32_t reserved;
    void *grad_residual;    /* [n][dim], of `stream_type`                 */
    int64_t grad_residual_stride;
    void *grad_block;       /* [n][dim], of `type`                        */
    int64_t grad_block_stride;
    void *grad_pre_weight, *grad_pre_bias;   /* [dim], of pre.type        */
    void *grad_post_weight, *grad_post_bias; /* [dim], of post.type       */
    void *grad_gate;        /* [gates][dim], of gate_type                 */
    void *workspace;
    size_t workspace_bytes;
} gdp_norm_grad;
int gdp_norm_grad_workspace(int64_t n, int64_t dim, int64_t gates, size_t *bytes);
int gdp_norm_backward(const gdp_norm_grad *p, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* GALVATRON_OPS_HIP_H */
