// Products of microscaled 4-bit operands on the matrix cores (qa_mxfp4_mm): what the kernels share.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 rows of 128 values from either side.  Lane l has 32 of them, one block: of row l % 16, block l / 16 of the
// four; 16 bytes of codes, and the block's scale as one byte of a register (which of the four, the instruction says).  So a word of four scales serves
// four steps of 128 values, and a lane's blocks in the group of 16 are 4 j + l / 16, j = 0 .. 3: the layout of the scales.  The weights are the first
// operand: a lane ends up with four neighbouring columns, 4 (l / 16) + 0 .. 3, of row l % 16.
#pragma once

#include "mx_common.hpp"

namespace qa {
namespace mx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// byte STEP of the scales
template <int STEP>
__device__ __forceinline__ v4f multiply(v4i w, int w_scales, v4i a, int a_scales, v4f acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1), __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1),
                                                            acc, 4, 4, STEP, w_scales, STEP, a_scales);
}

// Four neighbouring columns of a row, from n on, rounded to the output's type; those behind the last one are left out.
__device__ __forceinline__ void store_columns(const QaMxGemmParams& p, int m, int n, v4f v, bool whole_words) {
    if (m >= p.m || n >= p.n) return;
    const int64_t at = static_cast<int64_t>(m) * p.ldd + n;
    if (p.out_type == QA_LM_F32) {
        float* const d = static_cast<float*>(p.d) + at;
        if (whole_words && n + 4 <= p.n) *reinterpret_cast<v4f*>(d) = v;
        else
            for (int i = 0; i < 4 && n + i < p.n; ++i) d[i] = v[i];
        return;
    }
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    typedef uint16_t u4 __attribute__((ext_vector_type(4)));
    const u4 bits = p.out_type == QA_LM_BF16 ? __builtin_bit_cast(u4, __builtin_convertvector(v, b4)) : __builtin_bit_cast(u4, __builtin_convertvector(v, h4));
    uint16_t* const d = static_cast<uint16_t*>(p.d) + at;
    if (whole_words && n + 4 <= p.n) *reinterpret_cast<u4*>(d) = bits;
    else
        for (int i = 0; i < 4 && n + i < p.n; ++i) d[i] = bits[i];
}
// whether four columns from a multiple of four on lie on their own size
inline bool whole_words(const QaMxGemmParams& p) {
    const int four = 4 * bytes_of(p.out_type);
    return reinterpret_cast<uintptr_t>(p.d) % four == 0 && p.ldd % 4 == 0;
}

// Straight from memory (mx_gemm_direct.hip).  a_type: codes, or numbers that are quantised on the way.
int direct_launch(const QaMxGemmParams& p, hipStream_t stream);
bool direct_takes(const QaMxGemmParams& p);             // codes
bool direct_takes_numbers(const QaMxGemmParams& p);
// Of codes, in tiles through LDS (mx_gemm_tiles.hip).
int tiles_launch(const QaMxGemmParams& p, hipStream_t stream);

}  // namespace mx
}  // namespace qa
