/*
 * quamba_amd_lm.h - C ABI of the operators that a language model puts around the mixers (same library, libquamba_amd.so):
 * the residual stream with its norms, and log probabilities of tokens, of logits or of the head's int8 product.
 *
 * The conventions are those of quamba_amd.h: device pointers, strides in elements, the HIP stream as void*, QaStatus codes; no
 * allocation, no synchronisation, no state between calls.  A call over no rows returns QA_OK without a launch, and its tensors
 * may then be null.  A launch has at most 2^32 - 1 threads: calls that would need more return QA_ERR_SHAPE (rows of one wave's width: from
 * 2^26 of them on).  The parameter blocks below have a version of their own, qa_lm_abi_version().
 */
#ifndef QUAMBA_AMD_LM_H
#define QUAMBA_AMD_LM_H

#include "quamba_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QA_LM_ABI_VERSION 1
/* QA_LM_ABI_VERSION of the library: bumped on any change of the blocks below, of what a field means or of which fields a call reads. */
int qa_lm_abi_version(void);

typedef enum QaLmType { QA_LM_I8 = 0, QA_LM_F16 = 1, QA_LM_BF16 = 2, QA_LM_F32 = 3 } QaLmType;
typedef enum QaGateAct { QA_GATE_PLAIN = 0, QA_GATE_SIGMOID = 1, QA_GATE_SILU = 2 } QaGateAct;

/*
 * The end of one block and the beginning of the next, on rows of `dim` values (8 .. 32768):
 *   u = x,                      or  x / sqrt(mean(x^2) + eps) * post_weight        where post_weight is given
 *   u = u * act(gate)                                                              where gate is given
 *   v = residual + scale * u                                                       (residual null: scale * u)
 *   y = v / sqrt(mean(v^2) + eps) * weight
 * all in fp32; v is not rounded on its way into y.  residual_out (null: not wanted) gets v; it may be `residual` itself and
 * must not overlap an input otherwise.  out gets y, or with QA_LM_I8 the saturated rint(y * (1 / s)), the reciprocal rounded to
 * fp32: s is out_scale (a normal number above 0), or with dynamic_scale max(max|y|, 1e-5) / 127 of the row, written to scales.
 * A row with a NaN or an infinity, or whose
 * squares pass fp32 (values from some 1e18 on), is NaN as a whole: its y, or its scale (codes by out_scale mean nothing then).
 */
typedef struct QaAddNormParams {
    int32_t rows, dim;
    int32_t x_type;             /* QaLmType of x and gate (not I8) */
    int32_t param_type;         /* of weight, post_weight and scale_vector: x_type or F32 */
    int32_t residual_type;      /* of residual and residual_out: x_type or F32 */
    int32_t out_type;           /* x_type or I8 */
    int32_t gate_act;           /* QaGateAct */
    int32_t dynamic_scale;
    float eps, scale, out_scale;
    int32_t reserved0;
    int64_t x_row_stride, gate_row_stride /* 0: one gate for all rows */, residual_row_stride, residual_out_row_stride, out_row_stride;
    const void* x;
    const void* weight;
    const void* post_weight;    /* or null */
    const void* gate;           /* or null */
    const void* scale_vector;   /* (dim,), in place of scale; or null */
    const void* residual;       /* or null */
    void* residual_out;         /* or null */
    void* out;
    float* scales;              /* (rows,), with dynamic_scale */
} QaAddNormParams;

int qa_add_rmsnorm(const QaAddNormParams* p, void* stream);

/*
 * Of each row of logits l (vocab of them, neighbours in memory): the log probability l[token] - log sum exp l of a given token,
 * the entropy of the distribution, and the `top` (0 .. 64, at most vocab) largest logits' log probabilities and indices, the
 * lowest index first among equal ones.
 * A negative token asks for nothing: its log probability is written as 0.  A token >= vocab gets NaN.  Logits of -inf are masked
 * out (their log probability is -inf).  A row whose logits are all -inf, or hold a NaN or +inf, has no distribution: NaN, and
 * its top_tokens are indices inside the row.
 */
typedef struct QaTokenLogprobsParams {
    int32_t rows, vocab;        /* vocab up to 2^30 */
    int32_t logits_type;        /* QaLmType, not I8 */
    int32_t token_bytes;        /* 4 or 8: tokens are int32 or int64 */
    int32_t top, reserved0;
    int64_t row_stride;
    const void* logits;
    const void* tokens;         /* (rows,) */
    float* logprobs;            /* (rows,) */
    float* entropy;             /* (rows,) */
    float* top_logprobs;        /* (rows, top) */
    int64_t* top_tokens;        /* (rows, top) */
    void* workspace;            /* qa_token_logprobs_workspace_bytes, 16-byte aligned; null where that is 0 */
    int64_t workspace_bytes;
} QaTokenLogprobsParams;

/* Bytes of workspace for these sizes (rows, vocab, logits_type and top are read) on the current device; 0: none, or sizes that
 * the call refuses. */
int64_t qa_token_logprobs_workspace_bytes(const QaTokenLogprobsParams* p);
int qa_token_logprobs(const QaTokenLogprobsParams* p, void* stream);

/*
 * The same of l[m, n] = s_a[m|0] * (s_w[n|0] * sum_k a[m, k] * w[n, k]), n < vocab, of int8 a and w (the scaled product of
 * qa_gemm_w8a8, in fp32 and never written).  top is 0 or 1.
 */
typedef struct QaMmTokenLogprobsParams {
    int32_t rows, vocab, k;     /* rows up to 2^28, vocab up to 2^30, k a multiple of 16 up to 131056 (sums in 32 bits) */
    int32_t a_scale_numel, w_scale_numel;   /* 1 or rows, 1 or at least vocab */
    int32_t token_bytes;
    int32_t top, reserved0;
    int64_t lda, ldw;           /* row pitches of a (rows, k) and w (vocab, k): multiples of 16, up to 2^22 */
    const int8_t* a;
    const int8_t* w;
    const float* a_scale;
    const float* w_scale;
    const void* tokens;
    float* logprobs;
    float* entropy;
    float* top_logprobs;        /* (rows,), with top */
    int64_t* top_tokens;        /* (rows,), with top */
    void* workspace;            /* qa_mm_token_logprobs_workspace_bytes, 16-byte aligned */
    int64_t workspace_bytes;
} QaMmTokenLogprobsParams;

/* Bytes of workspace for these sizes (rows, vocab and k are read) on the current device; 0: sizes that the call refuses, or no rows. */
int64_t qa_mm_token_logprobs_workspace_bytes(const QaMmTokenLogprobsParams* p);
int qa_mm_token_logprobs(const QaMmTokenLogprobsParams* p, void* stream);

#ifdef __cplusplus
}
#endif
#endif
