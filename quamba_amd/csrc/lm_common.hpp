// Shared pieces of the operators around the mixers: values of a type that is chosen at run time, eight at a time.
#pragma once

#include "../../include/quamba_amd_lm.h"
#include "qa_common.hpp"

namespace qa {
namespace lm {

typedef uint32_t v4w __attribute__((ext_vector_type(4)));
typedef v4w v4w_at4 __attribute__((aligned(4)));
typedef v4w v4w_at2 __attribute__((aligned(2)));

// Type of QaLmType T.
template <int T> struct TypeOf;
template <> struct TypeOf<QA_LM_F16> { using type = _Float16; };
template <> struct TypeOf<QA_LM_BF16> { using type = __bf16; };
template <> struct TypeOf<QA_LM_F32> { using type = float; };

inline int bytes_of(int type) { return type == QA_LM_I8 ? 1 : type == QA_LM_F32 ? 4 : 2; }
inline bool is_float_type(int type) { return type == QA_LM_F16 || type == QA_LM_BF16 || type == QA_LM_F32; }

// A launch counts its threads in 32 bits.
inline bool launchable(int64_t workgroups, int64_t threads) { return workgroups <= 0xffffffffLL / threads; }

// N values of T as they lie in memory.  WIDE: on 16 bytes; else anywhere a T may lie (the hardware takes such addresses).
template <class T, int N>
struct Raw {
    static constexpr int kWords = N * static_cast<int>(sizeof(T)) / 16;
    static_assert(kWords * 16 == N * static_cast<int>(sizeof(T)), "whole 16-byte words");
    typedef std::conditional_t<sizeof(T) == 4, v4w_at4, v4w_at2> loose;
    v4w w[kWords];

    template <bool WIDE>
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (WIDE) w[i] = reinterpret_cast<const v4w*>(p)[i];
            else w[i] = *reinterpret_cast<const loose*>(reinterpret_cast<const char*>(p) + 16 * i);
        }
    }
    template <bool WIDE>
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (WIDE) reinterpret_cast<v4w*>(p)[i] = w[i];
            else *reinterpret_cast<loose*>(reinterpret_cast<char*>(p) + 16 * i) = w[i];
        }
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j / 4][j % 4]);
        const uint32_t word = w[j / 8][j % 8 / 2];
        if constexpr (std::is_same_v<T, __bf16>) return __uint_as_float(j % 2 ? word & 0xffff0000u : word << 16);
        else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(j % 2 ? word >> 16 : word & 0xffffu)));
    }
    // values j and j + 1, j even (round to nearest even; a NaN stays one)
    __device__ __forceinline__ void set2(int j, float v0, float v1) {
        if constexpr (sizeof(T) == 4) {
            w[j / 4][j % 4] = __float_as_uint(v0);
            w[j / 4][j % 4 + 1] = __float_as_uint(v1);
        } else {
            typedef float f2 __attribute__((ext_vector_type(2)));
            typedef T t2 __attribute__((ext_vector_type(2)));
            w[j / 8][j % 8 / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{v0, v1}), t2));
        }
    }
    // one value to memory
    __device__ __forceinline__ void store_one(T* p, int j) const {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = w[j / 4][j % 4];
        else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[j / 8][j % 8 / 2] >> (j % 2 * 16));
    }
};

__device__ __forceinline__ int64_t token_of(const void* tokens, int bytes, int64_t row) {
    return bytes == 8 ? static_cast<const int64_t*>(tokens)[row] : static_cast<const int32_t*>(tokens)[row];
}

}  // namespace lm
}  // namespace qa
