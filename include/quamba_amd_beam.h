/*
 * quamba_amd_beam.h - C ABI of beam search over recurrent models (same library, libquamba_amd.so): the best continuations over the beams
 * and the vocabulary, and the mixers' states in the beams' new order.
 *
 * The conventions are those of quamba_amd.h and quamba_amd_lm.h.  The parameter blocks below have a version of their own, qa_beam_abi_version().
 */
#ifndef QUAMBA_AMD_BEAM_H
#define QUAMBA_AMD_BEAM_H

#include "quamba_amd_lm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QA_BEAM_ABI_VERSION 1
/* QA_BEAM_ABI_VERSION of the library: bumped on any change of the blocks below, of what a field means or of which fields a call reads. */
int qa_beam_abi_version(void);

/*
 * Of each of `batch` entries the `count` best continuations of its beams.  Beam i offers every token v with the score
 *   scores[b, i] + l[b, i, v] - log sum_u exp l[b, i, u]
 * in 64 bits, rounded to fp32 as it is written; larger scores come first, of equal ones the lower beam's, then the lower token's.  The exponentials
 * are good to 1e-14 of themselves, so scores of different beams that are nearer than that may come in either order; but a token that has all of its
 * beam's weight has exactly the beam's score, tokens of equal logits share it evenly, and beams whose logits differ by one number have equal scores.
 * (Tokens of one beam whose logits differ by less than 64 bits of their scores show come in either order.)
 * A beam that is done offers itself once, with its score and the token -1, and its logits are not read.  A score of -inf is no offer: masked
 * tokens, and beams whose own score is that.  A beam offers nothing either where its logits are all -inf or hold a NaN or +inf, or where
 * its score is NaN or +inf.  Places that are left without an offer get the score -inf, the token -1 and the parent -1.
 */
typedef struct QaBeamSearchParams {
    int32_t batch, beams, vocab;    /* beams 1 .. 64, vocab up to 2^20 */
    int32_t logits_type;            /* QaLmType, not I8 */
    int32_t count;                  /* 1 .. 64, at most beams * vocab */
    int32_t reserved0;
    int64_t logits_batch_stride, logits_beam_stride;    /* elements */
    const void* logits;
    const float* scores;            /* (batch, beams) */
    const uint8_t* done;            /* (batch, beams), not 0: done; or null */
    float* out_scores;              /* (batch, count) */
    int64_t* tokens;                /* (batch, count) */
    int64_t* parents;               /* (batch, count): beams */
    void* workspace;                /* qa_beam_search_workspace_bytes, 16-byte aligned */
    int64_t workspace_bytes;
} QaBeamSearchParams;

/* Bytes of workspace for these sizes (batch, beams, vocab, logits_type and count are read) on the current device; 0: sizes that the call
 * refuses, or no entries. */
int64_t qa_beam_search_workspace_bytes(const QaBeamSearchParams* p);
int qa_beam_search_step(const QaBeamSearchParams* p, void* stream);

/*
 * Rows of states in another order, in place: of every tensor, row b * beams + i becomes what row b * beams + parents[b, i] was.  A row whose
 * parent is itself, or none of its entry's beams (-1), stays as it is and is not touched; a parent may have any number of children.
 */
typedef struct QaStateRows {
    void* data;                     /* row 0 */
    int64_t row_bytes;              /* each row one piece */
    int64_t row_stride;             /* bytes, at least row_bytes */
} QaStateRows;

typedef struct QaReorderParams {
    int32_t batch, beams;           /* beams 1 .. 64 */
    int32_t tensors;                /* any number; no two may share memory */
    int32_t index_bytes;            /* 4 or 8: parents are int32 or int64 */
    const QaStateRows* states;      /* host memory, read before the call returns */
    const void* parents;            /* (batch, beams) */
} QaReorderParams;

int qa_reorder_states(const QaReorderParams* p, void* stream);

#ifdef __cplusplus
}
#endif
#endif
