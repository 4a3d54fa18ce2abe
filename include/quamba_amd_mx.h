/*
 * quamba_amd_mx.h - C ABI of the microscaled 4-bit floating-point operators (same library, libquamba_amd.so): quantisation, the
 * values back, and the product of two such operands on the matrix cores.
 *
 * An operand is a matrix of rows of k values, k a multiple of 32 along which products sum.  Of each 32 neighbours in a row (a block)
 * every value is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times the block's scale, a power of two:
 *   codes   4 bits each: bit 3 the sign, bits 0..2 the place in that list; two to a byte, the earlier value in the low half; rows of k / 2 bytes
 *   scales  a byte each: the exponent + 127 (0 .. 254), or 255: the block is NaN.  16 blocks, 512 values, are a group; scales lie
 *           as (groups, rows, 16), groups = ceil(k / 512), and block 4 j + q of a group (j, q = 0 .. 3) has byte 4 q + j: the four
 *           bytes that a lane of the matrix instruction takes with four steps are one word.  Bytes behind k are written as 0 and not looked at.
 *
 * The conventions are those of quamba_amd.h and quamba_amd_lm.h: device pointers, the HIP stream as void*, QaStatus codes; no allocation, no
 * synchronisation, no state between calls, launches of at most 2^32 - 1 threads.  A call without rows or columns returns QA_OK without a
 * launch, and its tensors may then be null.  The parameter blocks below have a version of their own, qa_mx_abi_version().
 */
#ifndef QUAMBA_AMD_MX_H
#define QUAMBA_AMD_MX_H

#include "quamba_amd_lm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QA_MX_ABI_VERSION 1
/* QA_MX_ABI_VERSION of the library: bumped on any change of the blocks below, of what a field means or of which fields a call reads. */
int qa_mx_abi_version(void);

/*
 * Codes and scales of rows of floating-point numbers.  A block's scale is 2^e, e = floor(log2(max|x|)) - 2 and at least -127 (also for a block of
 * zeros); a value becomes the nearest multiple of the scale that there is, the even code where two are as near, and at most 6 (what lies between 6 and 8
 * scales is cut).  A block with a NaN or an infinity has the scale 255.
 */
typedef struct QaMxQuantParams {
    int32_t rows, k;
    int32_t x_type;                 /* QaLmType, not I8 */
    int32_t reserved0;
    int64_t x_row_stride;           /* elements */
    int64_t code_row_stride;        /* bytes, a multiple of 16 */
    int64_t scale_group_stride;     /* bytes, a multiple of 16, at least 16 rows */
    const void* x;
    uint8_t* codes;                 /* 16-byte aligned */
    uint8_t* scales;                /* 16-byte aligned */
} QaMxQuantParams;

int qa_mxfp4_quant(const QaMxQuantParams* p, void* stream);

/* The values of an operand, rounded to the output's type. */
typedef struct QaMxDequantParams {
    int32_t rows, k;
    int32_t out_type;               /* QaLmType, not I8 */
    int32_t reserved0;
    int64_t out_row_stride, code_row_stride, scale_group_stride;
    const uint8_t* codes;
    const uint8_t* scales;
    void* out;
} QaMxDequantParams;

int qa_mxfp4_dequant(const QaMxDequantParams* p, void* stream);

/*
 * d[m, n] = sum_k a[m, k] * w[n, k], summed in fp32 and rounded once to the output's type.  w is an operand as above, n rows of it; a is one too,
 * or with an a_type other than QA_LM_I8 rows of floating-point numbers, taken as qa_mxfp4_quant leaves them (their codes
 * are written to the workspace, or to nowhere where the rows are few).  k up to 2^23, rows of codes up to 2^22 bytes apart, m and n up to 2^31 - 256; with
 * k 0 the sums are 0, and d's rows lie next to each other.
 */
typedef struct QaMxGemmParams {
    int32_t m, n, k;
    int32_t a_type;                 /* QA_LM_I8: codes and scales; else the type of the rows */
    int32_t out_type;               /* QaLmType, not I8 */
    int32_t reserved0;
    int64_t lda;                    /* bytes, a multiple of 16, for codes; elements for numbers */
    int64_t ldw;                    /* bytes, a multiple of 16 */
    int64_t ldd;                    /* elements */
    int64_t a_scale_group_stride, w_scale_group_stride;
    const void* a;                  /* codes: 16-byte aligned */
    const uint8_t* a_scales;        /* null for numbers */
    const uint8_t* w;
    const uint8_t* w_scales;
    void* d;
    void* workspace;                /* qa_mxfp4_mm_workspace_bytes, 16-byte aligned; null where that is 0 */
    int64_t workspace_bytes;
} QaMxGemmParams;

/* Bytes of workspace for these sizes (m, n, k and a_type are read) on the current device; 0: none, or sizes that the call refuses. */
int64_t qa_mxfp4_mm_workspace_bytes(const QaMxGemmParams* p);
int qa_mxfp4_mm(const QaMxGemmParams* p, void* stream);

#ifdef __cplusplus
}
#endif
#endif
