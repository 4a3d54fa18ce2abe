// Microscaled 4-bit floating point: the layout of an operand, and a block's scale and codes.
#pragma once

#include "../../include/quamba_amd_mx.h"
#include "lm_common.hpp"

namespace qa {
namespace mx {

using lm::Raw;
using lm::bytes_of;
using lm::is_float_type;
using lm::launchable;
using lm::v4w;

constexpr int kBlock = 32;                 // values of a scale
constexpr int kGroup = 512;                // values of 16 scales that lie together
inline int64_t groups_of(int64_t k) { return (k + kGroup - 1) / kGroup; }

// The scale byte of a block from the bits of its largest magnitude: its exponent - 2, 0 at least, 255 with a NaN or an infinity.
__device__ __forceinline__ uint32_t scale_of(uint32_t most_bits) {
    const int e = static_cast<int>(most_bits >> 23);
    return e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
}
// the largest of the four lanes of a block, in all of them
__device__ __forceinline__ uint32_t most_of_block(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xb1, 0xf, 0xf, true)));
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4e, 0xf, 0xf, true)));
}
// 2^(scale - 127); 255: NaN
__device__ __forceinline__ float power_of(uint32_t scale) {
    return __uint_as_float(scale == 0 ? 0x00400000u : scale == 255 ? 0x7fc00000u : scale << 23);
}
// the codes of eight values by a scale (to nearest, ties to the even code, at most 6: the conversion's own rule), the first in the lowest bits
template <class Get>
__device__ __forceinline__ uint32_t codes_of(uint32_t scale, Get&& get) {
    const float s = power_of(min(scale, 254u));
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, get(0), get(1), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, get(2), get(3), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, get(4), get(5), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, get(6), get(7), s, 3);
    return w;
}

}  // namespace mx
}  // namespace qa
