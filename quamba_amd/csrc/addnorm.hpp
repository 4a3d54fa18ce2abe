// The end of one block and the beginning of the next in one pass over the rows of the residual stream:
//
//   u = x  or  x * rsqrt(mean(x^2) + eps) * post_weight,   u *= act(gate),   v = residual + scale * u,
//   y = v * rsqrt(mean(v^2) + eps) * weight,               out = y, or int8 codes of it
//
// Bound by memory (x, residual and gate once in, v and y once out), with few rows by the trip there and back.  A row stays in
// the registers of its waves from the loads to the last store: W of them share a row (chosen by the host), a lane holds PIECES
// times eight neighbouring columns, so that a load of a wave is one straight run.  The sums of squares and the maximum of a row
// meet through lane exchanges and, with several waves, through LDS, one barrier each; everything is fp32.
//
// The last columns of a row whose length is no multiple of eight are loaded with some of those in front of them (every load
// stays inside the row and none is conditional); those belong to another lane and count for nothing here.
#pragma once

#include "lm_common.hpp"
#include "normgated_core.hpp"

namespace qa {
namespace lm {

constexpr int kAddNormWaves = 16;                        // of a workgroup, at most
constexpr int kAddNormDim = kAddNormWaves * 4 * 512;     // widest row

// For z above -87 within 5 + 1.25 |z| units of 2^-24 (an exponential and a reciprocal of two each, their sum's rounding, and the exponent's); below, where 1 + e^-z has
// no normal reciprocal, 0 or within 2^-126.  16-bit rows do not see that; for fp32 ones it is the choice made, as exact divisions and expf made the
// gate the larger part of the kernel's time.
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f)); }

// Pieces of a lane, waves that share a row, rows of a workgroup.  A run is what a wave loads at once, 512 columns.
struct AddNormShape {
    int pieces, waves, rows;
};
constexpr int max_waves(int pieces) { return pieces == 3 ? 9 : kAddNormWaves; }
// Two runs a wave: with one a row's barriers gather twice the waves, with more a wave holds so much that fewer of them are there
// (everything on, us with 1, 2, 3, 4 of them a wave: 8192 x 4096 bf16 73, 64, 67, 65; 4096 x 8192 bf16 with an fp32 stream 108, 91, 102, 102;
// 64 x 2560 4.6, 4.4, 4.9, 5.7).  Three where that leaves no wave without work and two would (6131 x 4099, nine runs: 95, 71, 62, 73); four
// for rows that sixteen waves do not hold otherwise.
inline AddNormShape add_norm_shape(int dim) {
    const int runs = (dim + 511) / 512;
    const int pieces = runs == 1 ? 1 : runs > 2 * kAddNormWaves ? 4 : runs % 2 != 0 && runs % 3 == 0 ? 3 : 2;
    const int waves = (runs + pieces - 1) / pieces;
    return {pieces, waves, waves >= 4 ? 1 : 4 / waves};
}

template <class X, class R, class P, int PIECES, bool WIDE, bool BLOCK>
__global__ __launch_bounds__(64 * max_waves(PIECES)) void add_rmsnorm_kernel(QaAddNormParams p, int W) {
    __shared__ float s_part[3][kAddNormWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = wave % W, first = wave - sub;
    const int64_t wanted = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 64 / W) + wave / W;
    const bool live = wanted < p.rows;                    // (the waves of a row too many walk the last one and store nothing)
    const int64_t row = live ? wanted : p.rows - 1;
    const int N = p.dim;

    int at[PIECES], skip[PIECES];                         // this lane's columns of a piece: at .. at + 7, the first `skip` another lane's
    Raw<X, 8> rx[PIECES], rg[BLOCK ? PIECES : 1];
    Raw<R, 8> rr[PIECES];
    Raw<P, 8> rw[PIECES];
    const X* const x = static_cast<const X*>(p.x) + row * p.x_row_stride;
    const X* const g = BLOCK && p.gate ? static_cast<const X*>(p.gate) + row * p.gate_row_stride : x;
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        const int col = ((c * W + sub) * 64 + lane) * 8;
        at[c] = min(col, N - 8);
        skip[c] = col - at[c];
        rx[c].template load<WIDE>(x + at[c]);
    }
    if (p.residual) {
        const R* const r = static_cast<const R*>(p.residual) + row * p.residual_row_stride;
#pragma unroll
        for (int c = 0; c < PIECES; ++c) rr[c].template load<WIDE>(r + at[c]);
    }
    if constexpr (BLOCK) {
#pragma unroll
        for (int c = 0; c < PIECES; ++c) rg[c].template load<WIDE>(g + at[c]);
    }
#pragma unroll
    for (int c = 0; c < PIECES; ++c) rw[c].template load<WIDE>(static_cast<const P*>(p.weight) + at[c]);

    // over the row's waves
    auto across = [&](float v, int slot, auto op) {
        v = op(v, -1);
        if (W > 1) {
            if (lane == 0) s_part[slot][wave] = v;
            __syncthreads();
            v = s_part[slot][first];
            for (int i = 1; i < W; ++i) v = op(v, first + i);
        }
        return v;
    };
    // (a row with a NaN, an infinity or values whose squares pass fp32 is NaN as a whole, not zeros with a NaN among them)
    auto root = [&](float ssq) { return ssq < __builtin_inff() ? rstd_of(ssq, N, p.eps) : __builtin_nanf(""); };
    auto sum = [&](float v, int slot) { return across(v, slot, [&](float a, int i) { return i < 0 ? wave_sum(a) : a + s_part[slot][i]; }); };
    auto most = [&](float v, int slot) { return across(v, slot, [&](float a, int i) { return i < 0 ? wave_max(a) : fmaxf(a, s_part[slot][i]); }); };

    float v[PIECES][8];
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = j < skip[c] ? 0.0f : rx[c].get(j);
    if constexpr (BLOCK) {
        if (p.post_weight) {
            float ssq = 0.0f;
#pragma unroll
            for (int c = 0; c < PIECES; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) ssq = ssq_step(ssq, v[c][j]);
            const float rstd = root(sum(ssq, 0));
#pragma unroll
            for (int c = 0; c < PIECES; ++c) {
                Raw<P, 8> w;
                w.template load<WIDE>(static_cast<const P*>(p.post_weight) + at[c]);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = norm_value(v[c][j], rstd, w.get(j));
            }
        }
        if (p.gate) {
#pragma unroll
            for (int c = 0; c < PIECES; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float z = rg[c].get(j);
                    v[c][j] *= p.gate_act == QA_GATE_PLAIN ? z : (p.gate_act == QA_GATE_SILU ? z : 1.0f) * sigmoid(z);
                }
        }
        if (p.scale_vector) {
#pragma unroll
            for (int c = 0; c < PIECES; ++c) {
                Raw<P, 8> s;
                s.template load<WIDE>(static_cast<const P*>(p.scale_vector) + at[c]);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] *= s.get(j);
            }
        }
    }
    const float scale = BLOCK && p.scale_vector ? 1.0f : p.scale;
    float ssq = 0.0f;
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float r = p.residual ? rr[c].get(j) : 0.0f;
            v[c][j] = j < skip[c] ? 0.0f : __builtin_fmaf(scale, v[c][j], r);
            ssq = ssq_step(ssq, v[c][j]);
        }
    ssq = sum(ssq, 1);                                    // (behind it every wave of the row has read its residual)

    auto store = [&](auto* to, const auto& raw, int c) {
        if (skip[c] == 0) raw.template store<WIDE>(to + at[c]);
        else if (!WIDE && skip[c] < 8) {
#pragma unroll
            for (int j = 1; j < 8; ++j)
                if (j >= skip[c]) raw.store_one(to + at[c] + j, j);
        }
    };
    if (p.residual_out && live) {
        R* const to = static_cast<R*>(p.residual_out) + row * p.residual_out_row_stride;
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            Raw<R, 8> o;
#pragma unroll
            for (int j = 0; j < 8; j += 2) o.set2(j, v[c][j], v[c][j + 1]);
            store(to, o, c);
        }
    }
    const float rstd = root(ssq);
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[c][j] = norm_value(v[c][j], rstd, rw[c].get(j));
            // (a column of another lane is 0 times a weight: no more than 0, or NaN where the other lane has the same NaN)
            top = fmaxf(top, fabsf(v[c][j]));
        }
    if (p.out_type != QA_LM_I8) {
        if (!live) return;
        X* const to = static_cast<X*>(p.out) + row * p.out_row_stride;
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            Raw<X, 8> o;
#pragma unroll
            for (int j = 0; j < 8; j += 2) o.set2(j, v[c][j], v[c][j + 1]);
            store(to, o, c);
        }
        return;
    }
    float s = p.out_scale;
    if (p.dynamic_scale) {
        top = most(top, 2);
        s = rstd == rstd ? fmaxf(top, 1e-5f) / 127.0f : rstd;        // (a maximum passes over NaNs)
        if (live && lane == 0 && sub == 0) p.scales[row] = s;
    }
    if (!live) return;
    const float inv = 1.0f / s;
    int8_t* const to = static_cast<int8_t*>(p.out) + row * p.out_row_stride;
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
        int8_t q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = sat8_rne(v[c][j] * inv);
        if (skip[c] == 0) {
            __builtin_memcpy(WIDE ? __builtin_assume_aligned(to + at[c], 8) : to + at[c], q, 8);
        } else if (!WIDE && skip[c] < 8) {
#pragma unroll
            for (int j = 1; j < 8; ++j)
                if (j >= skip[c]) to[at[c] + j] = q[j];
        }
    }
}

// One set of types: X of x, gate and float output, R of the residual, P of the parameters.
template <class X, class R, class P>
int add_rmsnorm_launch(const QaAddNormParams& p, const AddNormShape& s, bool wide, hipStream_t stream) {
    const int64_t blocks = (static_cast<int64_t>(p.rows) + s.rows - 1) / s.rows;
    if (!launchable(blocks, 64 * s.waves * s.rows)) return QA_ERR_SHAPE;
    const dim3 grid(static_cast<unsigned>(blocks)), block(64 * s.waves * s.rows);
    const bool of_block = p.post_weight || p.gate || p.scale_vector;
    auto go = [&](auto pieces_c) {
        constexpr int kPieces = decltype(pieces_c)::value;
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, s.waves); };
        if (wide) of_block ? launch(add_rmsnorm_kernel<X, R, P, kPieces, true, true>) : launch(add_rmsnorm_kernel<X, R, P, kPieces, true, false>);
        else of_block ? launch(add_rmsnorm_kernel<X, R, P, kPieces, false, true>) : launch(add_rmsnorm_kernel<X, R, P, kPieces, false, false>);
        return check_launch();
    };
    switch (s.pieces) {
        case 1: return go(std::integral_constant<int, 1>{});
        case 2: return go(std::integral_constant<int, 2>{});
        case 3: return go(std::integral_constant<int, 3>{});
        default: return go(std::integral_constant<int, 4>{});
    }
}

// addnorm_f16.hip, addnorm_bf16.hip: the sets of 16-bit x
int add_rmsnorm_f16(const QaAddNormParams& p, const AddNormShape& s, bool wide, hipStream_t stream);
int add_rmsnorm_bf16(const QaAddNormParams& p, const AddNormShape& s, bool wide, hipStream_t stream);

template <class X>
int add_rmsnorm_of_type(const QaAddNormParams& p, const AddNormShape& s, bool wide, hipStream_t stream) {
    const bool r32 = p.residual_type == QA_LM_F32, p32 = p.param_type == QA_LM_F32;
    if (r32) return p32 ? add_rmsnorm_launch<X, float, float>(p, s, wide, stream) : add_rmsnorm_launch<X, float, X>(p, s, wide, stream);
    return p32 ? add_rmsnorm_launch<X, X, float>(p, s, wide, stream) : add_rmsnorm_launch<X, X, X>(p, s, wide, stream);
}

}  // namespace lm
}  // namespace qa
