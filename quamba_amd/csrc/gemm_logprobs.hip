// Log probabilities of given tokens of the head's int8 product (qa_mm_token_logprobs): the tiles of gemm_core.hpp with a softmax's
// statistics in the place of the stores.
//
//   l[m, n] = s_a[m|0] * (s_w[n|0] * float(sum_k a[m, k] w[n, k]))       (the products' sum is exact, the scales are those of qa_gemm_w8a8)
//
// rows x vocabulary logits would be the largest tensor of an evaluation by far (16384 x 50280: 1.6 GB in 16 bits, written and read again).
// Here a workgroup reduces its tile to a RowStats and a best column per row: 16 bytes for each row and tile of columns go to the
// workspace, and with them the logit of the row's given token from the one lane that holds it.  A second launch joins them.
#include "gemm_core.hpp"
#include "row_stats.hpp"

#include <algorithm>

namespace qa {
namespace lm {
namespace {

using namespace gemm;

struct TilePart {
    float m, s, t;
    int best;              // the lowest column with the value m
};

// v of the lanes that hold other columns of the same row (ROWS rows: lane l has row l % ROWS), by op, in every one of them
template <int ROWS, class Op>
__device__ __forceinline__ uint32_t over_columns(uint32_t v, Op op) {
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(halves[0], halves[1]);
    if constexpr (ROWS == 16) {
        const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(rows[0], rows[1]);
    }
    return v;
}
template <int ROWS>
__device__ __forceinline__ float most_over_columns(float v) {
    return __uint_as_float(over_columns<ROWS>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int ROWS>
__device__ __forceinline__ float sum_over_columns(float v) {
    return __uint_as_float(over_columns<ROWS>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// A wave's TM x TN blocks: the statistics of each of its rows to parts[row_at + row], the given tokens' logits to `given`.
// s_lds: column scales, row scales, and the low words of the tokens, of the workgroup's tile.
//
// All waves are in here at the same time, with nothing for the matrix cores to do: what counts is instructions a value.
// PLAIN: with z = s_col * acc and c = s_row log2(e) an exponent is one fused step, z c - r for r the rounded z_max c; the rest of that
// rounding, z_max c - r, is exact in one number per row and corrects the sums.  s and t are sums of 2^d and of d 2^d until they leave.  Ten
// instructions' time a value, four of it the exponential's (fifteen with a difference, a product, a clamp and the best column each on its
// own).  This holds for columns that are all the vocabulary's, scales of rows that are none of them negative, and logits that the scales
// keep below kFarthest (plain_scales): every d is a number then, and the rest small.
// Otherwise the logits are formed as they would be written and taken as RowStats takes them: -inf is masked out (a column behind the
// vocabulary's end is that too), a NaN or +inf leaves a NaN in s.
template <bool PLAIN, bool TOP, int TM, int TN, int BM, int BN, class V, int NI, int NJ>
__device__ __forceinline__ void tile_stats(const QaMmTokenLogprobsParams& p, V (&acc)[NI][NJ], const float* s_lds, int row_at, int col_at, int m0, int n0, int n_end, int lane,
                                           TilePart* parts, float* given) {
    using Q = QuadView<V>;
    constexpr int kQuads = TN * 32 / (256 / Q::kRows), kRowBlocks = TM * 32 / Q::kRows;
    static_assert(NI * Q::kQuadsPer == kQuads && NJ == kRowBlocks, "accumulators of another tile");
    const float none = -__builtin_inff();
    const int columns = n_end - (n0 + col_at);             // of the tile, from this wave's first one on
#pragma unroll
    for (int b = 0; b < kRowBlocks; ++b) {
        const int row = row_at + b * Q::kRows + Q::row_of(lane);
        const float s_row = s_lds[BN + row], size = PLAIN ? s_row : 1.0f;      // (z: without the row's scale, or with it)
        const int token = reinterpret_cast<const int*>(s_lds)[BN + BM + row] - (n0 + col_at);      // its column among the wave's
        float z[kQuads][4], most = PLAIN ? kLowest : none;
#pragma unroll
        for (int u = 0; u < kQuads; ++u) {
            const float4 s_quad = *reinterpret_cast<const float4*>(s_lds + col_at + Q::column_of(u, lane));
            const float s_col[4] = {s_quad.x, s_quad.y, s_quad.z, s_quad.w};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                z[u][t] = s_col[t] * Q::value(acc, u, b, t);
                if constexpr (!PLAIN) z[u][t] = Q::column_of(u, lane) + t < columns ? s_row * z[u][t] : none;
                most = fmaxf(most, z[u][t]);
            }
        }
        most = most_over_columns<Q::kRows>(most);
        float s = 0.0f, w = 0.0f, m;
        if constexpr (PLAIN) {
            const float c = size * kLog2e, r = most * c, rest = __builtin_fmaf(most, c, -r);
#pragma unroll
            for (int u = 0; u < kQuads; ++u)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float d = __builtin_fmaf(z[u][t], c, -r), e = __builtin_amdgcn_exp2f(d);
                    s += e;
                    w = __builtin_fmaf(d, e, w);
                }
            s = sum_over_columns<Q::kRows>(s);
            w = sum_over_columns<Q::kRows>(w);
            const float f = __builtin_amdgcn_exp2f(-rest);
            w = (w - rest * s) * f * kLn2;
            s *= f;
            m = fmaxf(size * most, kLowest);
        } else {
            m = fmaxf(most, kLowest);                      // (nothing but masked values, or NaNs: the differences are -inf, or NaN)
            RowStats of_row = {m, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < kQuads; ++u)
#pragma unroll
                for (int t = 0; t < 4; ++t) of_row.add(z[u][t]);
            s = sum_over_columns<Q::kRows>(of_row.s);
            w = sum_over_columns<Q::kRows>(of_row.t);
        }
        uint32_t best = 0;
        if constexpr (TOP) {
            // (of the rounded logits, as they would be written)
            best = 0xffffffffu;
#pragma unroll
            for (int u = kQuads - 1; u >= 0; --u)
#pragma unroll
                for (int t = 3; t >= 0; --t)
                    if (size * z[u][t] == m) best = Q::column_of(u, lane) + t;
            best = over_columns<Q::kRows>(best, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
            if (best == 0xffffffffu) best = 0;             // (a row of NaNs, or of masked values)
        }
        if (lane < Q::kRows) parts[row] = {m, s, w, n0 + col_at + static_cast<int>(best)};
        if (__builtin_amdgcn_ballot_w64(token >= 0 && token < TN * 32)) {
            float v = 0.0f;
#pragma unroll
            for (int u = 0; u < kQuads; ++u)
#pragma unroll
                for (int t = 0; t < 4; ++t) v = token == Q::column_of(u, lane) + t ? z[u][t] : v;
            const int by = Q::kRows == 16 ? token >> 2 & 3 : token >> 2 & 1;                       // the lanes that hold it
            if (token >= 0 && token < min(columns, TN * 32) && lane / Q::kRows == by && m0 + row < p.rows) given[m0 + row] = size * v;
        }
    }
}

// Whether of a wave's COLUMNS column scales and ROWS row scales the former are numbers, the latter not negative, and no logit of theirs passes
// kFarthest.  (A row whose scale is NaN is that as a whole either way, and the rows beside it keep their bits.)
template <int ROWS, int COLUMNS>
__device__ __forceinline__ bool plain_scales(const float* s_row, const float* s_col, int k, int lane) {
    bool fine = true;
    float most_row = 0.0f, most_col = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; i += 64) {
        const float v = s_row[ROWS % 64 == 0 ? i + lane : min(i + lane, ROWS - 1)];
        fine &= !(v < 0.0f);
        most_row = fmaxf(most_row, v);
    }
#pragma unroll
    for (int i = 0; i < COLUMNS; i += 64) {
        const float v = s_col[COLUMNS % 64 == 0 ? i + lane : min(i + lane, COLUMNS - 1)];
        fine &= v == v;
        most_col = fmaxf(most_col, fabsf(v));
    }
    // (the products of two codes are at most 2^14; an infinity times 0 is not below anything either)
    fine &= wave_max(most_row) * (wave_max(most_col) * (16384.0f * k)) < kFarthest;
    return !__builtin_amdgcn_ballot_w64(!fine);
}

// A tile takes `columns` of its BN columns.  TURN: workgroups do not all start at K's beginning (in step, all of them ask for the same 128 bytes of
// rows that lie K bytes apart, which few of the memory's channels hold: 64 x 50280 x 4096 56.7 -> 50.9 us, other K the same).
template <int TM, int TN, int WGM, int WGN, int STAGES, bool TOP, bool TURN>
__global__ __launch_bounds__(64 * WGM * WGN) void mm_token_logprobs_kernel(QaMmTokenLogprobsParams p, int columns) {
    using C = Cfg<TM, TN, WGM, WGN, STAGES>;
    constexpr int BM = C::kBM, BN = C::kBN, WAVES = C::kWaves;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    static_assert(WGN * BM * static_cast<int>(sizeof(TilePart)) <= C::kLdsBytes, "the waves' statistics take the place of the operands");
    static_assert(BM % 64 == 0 && BN % 64 == 0 && BM * kChunks % C::kThreads == 0 && BN * kChunks % C::kThreads == 0, "whole requests");

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WGM, wn = wave / WGM;
    const int tiles_m = (p.rows + BM - 1) / BM, tiles_n = (p.vocab + columns - 1) / columns;
    int tile_m, tile_n;
    tile_of_workgroup<BM, BN>(blockIdx.x, tiles_m, tiles_n, tile_m, tile_n);
    const int m0 = tile_m * BM, n0 = tile_n * columns, n_end = min(n0 + columns, p.vocab);
    // (from the tile's own first row and column on: 32-bit offsets then reach over operands of any size)
    const int rows = min(BM, p.rows - m0), width = n_end - n0;
    const v4i rsrc_a = make_rsrc(p.a + m0 * p.lda, static_cast<int>((rows - 1) * p.lda + p.k));
    const v4i rsrc_w = make_rsrc(p.w + n0 * p.ldw, static_cast<int>((width - 1) * p.ldw + p.k));
    const uint32_t lds_base = lds_offset_of(lds);

    using Scales = TileScales<BM, BN, WAVES>;
    const bool one_a = p.a_scale_numel == 1, one_w = p.w_scale_numel == 1;
    Scales::request(lds_base + C::kLdsBytes, one_a ? p.a_scale : p.a_scale + m0, one_a ? 1 : 2, rows, 0, one_w ? p.w_scale : p.w_scale + n0, one_w ? 1 : 2, width, 0, wave, lane);
    const v4i rsrc_t = make_rsrc(static_cast<const uint8_t*>(p.tokens) + static_cast<int64_t>(m0) * p.token_bytes, rows * p.token_bytes);
#pragma unroll
    for (int i = 0; i < BM / 64; ++i)
        if (i % WAVES == wave) buffer_load_lds_b32(rsrc_t, lds_base + C::kLdsBytes + Scales::kBytes + i * 256, (i * 64 + lane) * p.token_bytes);
    TileLoader<C::kAInstr> load_a;
    TileLoader<C::kWInstr> load_w;
    load_a.template init<WAVES>(0, rows, p.lda, wave, lane);
    load_w.template init<WAVES>(0, width, p.ldw, wave, lane);
    const int k_tiles = (p.k + kBK - 1) / kBK;
    const int turn = TURN ? static_cast<int>(static_cast<unsigned>(blockIdx.x * 7) % static_cast<unsigned>(k_tiles)) : 0;
    auto k_of = [&](int tile) {
        if constexpr (!TURN) return tile * kBK;
        const int t = tile + turn;
        return tile >= k_tiles ? k_tiles * kBK : (t >= k_tiles ? t - k_tiles : t) * kBK;
    };

    TilePart* const parts = reinterpret_cast<TilePart*>(lds);
    TilePart* const out = static_cast<TilePart*>(p.workspace);
    auto finish = [&](auto& acc) {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        __syncthreads();
        const float* const s_lds = reinterpret_cast<const float*>(lds + C::kLdsBytes);
        float* const given = reinterpret_cast<float*>(out + static_cast<int64_t>(p.rows) * tiles_n);
        const bool plain = n_end - (n0 + wn * TN * 32) >= TN * 32 && plain_scales<TM * 32, TN * 32>(s_lds + BN + wm * TM * 32, s_lds + wn * TN * 32, p.k, lane);
        auto stats = [&](auto plain_c) __attribute__((always_inline)) {
            tile_stats<decltype(plain_c)::value, TOP, TM, TN, BM, BN>(p, acc, s_lds, wm * TM * 32, wn * TN * 32, m0, n0, n_end, lane, parts + wn * BM, given);
        };
        if (plain) stats(std::true_type{});
        else stats(std::false_type{});
        __syncthreads();
        for (int row = tid; row < BM; row += C::kThreads) {
            if (m0 + row >= p.rows) break;
            TilePart best = parts[row];
            RowStats r = {best.m, best.s, best.t};
#pragma unroll
            for (int i = 1; i < WGN; ++i) {
                const TilePart o = parts[i * BM + row];
                if (o.m > best.m) best = o;
                r.join({o.m, o.s, o.t});
            }
            out[static_cast<int64_t>(tile_n) * p.rows + m0 + row] = {r.m, r.s, r.t, best.best};
        }
    };
    if constexpr (TM * TN > 1) {
        // (requests as in the product's own kernel: one per kPace multiplications, counted from the barrier)
        using Mma = RotatedMma<TM, TN>;
        constexpr int kReq = C::kAInstr + C::kWInstr, kPace = kReq <= Mma::kPerTile / 4 ? 4 : Mma::kPerTile / kReq;
        constexpr int kEarly = Mma::kBehindBarrier / kPace < kReq ? Mma::kBehindBarrier / kPace : kReq;
        auto request = [&](int r, int k0, uint32_t stage) {
            if (r < C::kAInstr) load_a.template issue_one<WAVES>(r, rsrc_a, k0, p.k, lds_base + stage, wave);
            else if (r < kReq) load_w.template issue_one<WAVES>(r - C::kAInstr, rsrc_w, k0, p.k, lds_base + stage + BM * kBK, wave);
        };
        auto request_whole = [&](int r, int k0, uint32_t stage) {
            if (r < C::kAInstr) load_a.template issue_whole<WAVES>(r, rsrc_a, k0, lds_base + stage, wave);
            else if (r < kReq) load_w.template issue_whole<WAVES>(r - C::kAInstr, rsrc_w, k0, lds_base + stage + BM * kBK, wave);
        };
#pragma unroll
        for (int t = 0; t < STAGES - 1; ++t)
#pragma unroll
            for (int r = 0; r < kReq; ++r) request(r, k_of(t), t * C::kStageBytes);
        int k_late = k_of(STAGES - 1);                                 // of the tile STAGES - 1 further than the one at hand
#pragma unroll
        for (int r = 0; r < kEarly; ++r) request(r, k_late, (STAGES - 1) * C::kStageBytes);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((STAGES - 2) * kReq + kEarly));
        __syncthreads();
        const uint8_t* my_a = lds + (wm * TM * 32) * kBK;
        const uint8_t* my_w = lds + BM * kBK + (wn * TN * 32) * kBK;
        Mma mma;
        mma.init(lane);
        mma.start(my_a, my_w);
        uint32_t cur = 0, late = (STAGES - 1) * C::kStageBytes;
        auto multiply = [&](int kt, auto&& req) {
            const uint32_t nxt = cur + C::kStageBytes == C::kLdsBytes ? 0 : cur + C::kStageBytes;
            const int k_early = k_of(kt + STAGES);
            mma.template tile<(STAGES - 2) * kReq>(my_a + cur, my_w + cur, my_a + nxt, my_w + nxt, [&](int idx) {
                if (idx % kPace != kPace - 1) return;
                const int r = idx / kPace;
                if (r < kEarly) req(r, k_early, cur);
                else req(r, k_late, late);
            });
            k_late = k_early;
            late = cur;
            cur = nxt;
        };
        int kt = 0;
        for (const int whole = p.k / kBK - STAGES; kt < whole; ++kt) multiply(kt, request_whole);
        for (; kt < k_tiles; ++kt) multiply(kt, request);
        finish(mma.acc);
    } else {
        const int frow = lane & 31, fhalf = lane >> 5;
        v16i acc[1][1];
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[0][0][r] = 0;
        auto issue = [&](int tile) {
            const uint32_t base = lds_base + (tile % STAGES) * C::kStageBytes;
            load_a.template issue<WAVES>(rsrc_a, k_of(tile), p.k, base, wave);
            load_w.template issue<WAVES>(rsrc_w, k_of(tile), p.k, base + BM * kBK, wave);
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) issue(s);
        for (int kt = 0; kt < k_tiles; ++kt) {
            __builtin_amdgcn_s_waitcnt(vmcnt_imm((STAGES - 2) * (C::kAInstr + C::kWInstr)));
            __syncthreads();
            const uint8_t* stage = lds + (kt % STAGES) * C::kStageBytes;
            const int nt = kt + STAGES - 1;
            const uint32_t nbase = lds_base + (nt % STAGES) * C::kStageBytes;
            const int nk = k_of(nt);
            static_assert(C::kAInstr + C::kWInstr <= 4, "a request behind each of four multiplications");
            mma_tile_paced(stage + wm * 32 * kBK, stage + BM * kBK + wn * 32 * kBK, frow, fhalf, acc[0][0], [&](int r) {
                if (r < C::kAInstr) load_a.template issue_one<WAVES>(r, rsrc_a, nk, p.k, nbase, wave);
                else if (r < C::kAInstr + C::kWInstr) load_w.template issue_one<WAVES>(r - C::kAInstr, rsrc_w, nk, p.k, nbase + BM * kBK, wave);
            });
        }
        finish(acc);
    }
}

// The parts of ROWS rows, tiles_n each, by one workgroup.  A part is 16 bytes and a row's parts lie p.rows of them apart, so the rows of a
// workgroup are what its loads have in one piece; with few rows all threads go to one.  What a thread holds of a row meets through
// lane exchanges (lane l has row l % ROWS), then over the waves.
constexpr int kJoinThreads = 256, kJoinAhead = 4;
template <int ROWS>
__global__ __launch_bounds__(kJoinThreads) void mm_token_logprobs_join_kernel(QaMmTokenLogprobsParams p, int tiles_n) {
    __shared__ TilePart s_part[kJoinThreads / 64][ROWS];
    constexpr int kStep = kJoinThreads / ROWS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = threadIdx.x % ROWS;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + r, from = min(row, static_cast<int64_t>(p.rows) - 1);
    const TilePart* const parts = static_cast<const TilePart*>(p.workspace);
    RowStats all;
    all.clear();
    float best_m = -__builtin_inff();
    int best = 0x7fffffff;
    auto take = [&](float m, float s, float t, int column) {
        if (m > best_m || (m == best_m && column < best)) {
            best_m = m;
            best = column;
        }
        all.join({m, s, t});
    };
    for (int i = threadIdx.x / ROWS; i < tiles_n; i += kJoinAhead * kStep) {
        TilePart o[kJoinAhead];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) o[j] = parts[min(i + j * kStep, tiles_n - 1) * static_cast<int64_t>(p.rows) + from];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j)
            if (i + j * kStep < tiles_n) take(o[j].m, o[j].s, o[j].t, o[j].best);
    }
    auto meet = [&](auto mask_c) {
        constexpr int MASK = decltype(mask_c)::value;
        if constexpr (MASK >= ROWS) {
            auto other = [&](float v) { return __uint_as_float(word_across<MASK>(__float_as_uint(v), lane)); };
            // (an empty side has the lowest number and no column)
            const float m = other(all.m), s = other(all.s), t = other(all.t);
            take(m, s, t, static_cast<int>(word_across<MASK>(static_cast<uint32_t>(best), lane)));
        }
    };
    meet(std::integral_constant<int, 32>{});
    meet(std::integral_constant<int, 16>{});
    meet(std::integral_constant<int, 8>{});
    meet(std::integral_constant<int, 4>{});
    meet(std::integral_constant<int, 2>{});
    meet(std::integral_constant<int, 1>{});
    if (lane < ROWS) s_part[wave][lane] = {all.m, all.s, all.t, best};
    __syncthreads();
    if (threadIdx.x >= ROWS || row >= p.rows) return;
#pragma unroll
    for (int w = 1; w < kJoinThreads / 64; ++w) take(s_part[w][r].m, s_part[w][r].s, s_part[w][r].t, s_part[w][r].best);
    const int64_t token = token_of(p.tokens, p.token_bytes, row);
    float lp = token < 0 ? 0.0f : __builtin_nanf("");
    if (token >= 0 && token < p.vocab) lp = all.logprob(reinterpret_cast<const float*>(parts + static_cast<int64_t>(p.rows) * tiles_n)[row]);
    p.logprobs[row] = lp;
    p.entropy[row] = all.s > 0.0f ? all.entropy() : __builtin_nanf("");
    if (p.top) {
        p.top_logprobs[row] = all.logprob(all.m);
        p.top_tokens[row] = best;
    }
}

// The tiles, and what a launch of them takes, in us with `units` of 128 codes of K: fixed and, for each round of one tile per CU,
// per_round + per_unit x units (the launch of the join is in it).  From 65 rows on the fastest by that is taken.  Measured over 1 .. 16384
// rows, 1000 .. 256000 columns and K from 768 to 4096 the choice is the fastest of them but for 1.5 % of the time (rows x vocabulary x K,
// us by the tiles in the order below, without the third): 1000 x 4000 x 2560 25.3, 21.3, 18.2, 24.2, 34.4, 37.4; 128 x 50280 x 2560 (from
// 128 rows on) 43.7, 36.6, 45.3, 48.4; 256 x 50280 x 2560 70.9, 57.8, 49.1, 51.0; 16000 x 16000 x 768 419, 349, 360, 281, 238, 227; 16384 x
// 50280 x 2560 (the last two) 1667, 1554.
struct Tile {
    int bm, bn;
    float fixed, per_round, per_unit;
};
constexpr Tile kTiles[] = {{64, 64, 6.0f, 0.3f, 0.2f},    {64, 128, 6.0f, 1.0f, 0.31f},   {64, 256, 0.0f, 0.0f, 0.0f},   {128, 128, 4.0f, 1.6f, 0.56f},
                           {128, 256, 4.0f, 2.6f, 0.84f}, {256, 256, 5.0f, 3.6f, 1.45f}, {256, 320, 5.0f, 4.2f, 1.75f}};
constexpr int kNarrow = 0, kMiddle = 1, kWide = 2, kWideOf128 = 4;

// The tile, and how many columns of the vocabulary one takes (the rest of its width reads nothing).
//
// One row of tiles is bound by the memory's rate, of which a CU alone takes a part: all of them have to be at it all the time, with the same
// number of columns.  Those of 16 that make whole rounds, in the narrowest tile that holds them (64 rows, us with whole tiles of 128
// and so): 50280 x 2560 37.2 -> 31.5, 50280 x 4096 51.0 -> 42.9, 40000 x 2560 33.9 -> 28.1, 98304 x 2560 58.4 -> 55.8.
struct Plan {
    int tile, columns;
};
Plan plan_of(const QaMmTokenLogprobsParams& p) {
    const int cus = compute_units(), units = (p.k + kBK - 1) / kBK;
    auto even = [&](int width) {
        const int64_t places = static_cast<int64_t>((p.vocab + static_cast<int64_t>(cus) * width - 1) / (static_cast<int64_t>(cus) * width)) * cus;
        return static_cast<int>((p.vocab + 16 * places - 1) / (16 * places) * 16);
    };
    if (p.rows <= 64) {
        const int columns = std::max(even(256), 64);
        // (a short K is over before the difference shows: 1 x 50280 x 768 13.4 by 128 columns, 13.8; 4 x 256000 x 768 47.9, 49.7)
        if (columns > 128 && units <= 8) return {kMiddle, 128};
        return {columns <= 64 ? kNarrow : columns <= 128 ? kMiddle : kWide, columns};
    }
    int best = 0;
    float best_us = 1e30f;
    for (int i = 0; i < static_cast<int>(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
        const Tile& t = kTiles[i];
        if (i == kWide) continue;
        const int64_t tiles = static_cast<int64_t>((p.rows + t.bm - 1) / t.bm) * ((p.vocab + t.bn - 1) / t.bn);
        const float us = t.fixed + static_cast<float>((tiles + cus - 1) / cus) * (t.per_round + t.per_unit * units);
        if (us < best_us) {
            best = i;
            best_us = us;
        }
    }
    return {best, best == kWideOf128 && p.rows <= 128 ? even(256) : kTiles[best].bn};
}

// a tile's operands are addressed with 32-bit byte offsets
constexpr int64_t kWidestRow = 4 << 20;
static_assert(320 * kWidestRow < 0x70000000LL, "the widest tile");
constexpr int kMostColumns = 1 << 30, kMostRows = 1 << 28;     // (sums of them and a tile's stay in 32 bits)

constexpr int kDeepest = 131056;                               // (a sum of so many products of codes, up to 2^14 each, stays in 32 bits)
static_assert((kDeepest + 16LL) << 14 == 1LL << 31, "the largest multiple of 16");

int check(const QaMmTokenLogprobsParams& p) {
    if (p.rows < 0 || p.rows > kMostRows || p.vocab < 1 || p.vocab > kMostColumns || p.k < 1 || p.k > kDeepest) return QA_ERR_SHAPE;
    if (p.token_bytes != 4 && p.token_bytes != 8) return QA_ERR_UNSUPPORTED;
    if (p.top != 0 && p.top != 1) return QA_ERR_UNSUPPORTED;
    return QA_OK;
}

int64_t workspace_bytes(const QaMmTokenLogprobsParams& p) {
    const int64_t columns = plan_of(p).columns, tiles_n = (p.vocab + columns - 1) / columns;
    return p.rows * (tiles_n * static_cast<int64_t>(sizeof(TilePart)) + static_cast<int64_t>(sizeof(float)));
}

template <int TILE, int TM, int TN, int WGM, int WGN, int STAGES, bool TURN>
int launch(const QaMmTokenLogprobsParams& p, int columns, hipStream_t stream) {
    using C = Cfg<TM, TN, WGM, WGN, STAGES>;
    static_assert(C::kBM == kTiles[TILE].bm && C::kBN == kTiles[TILE].bn, "the tile of the table");
    const int tiles_n = (p.vocab + columns - 1) / columns;
    const int64_t tiles = static_cast<int64_t>((p.rows + C::kBM - 1) / C::kBM) * tiles_n;
    const int at_once = p.rows >= 4096 ? 16 : p.rows >= 512 ? 4 : 1, joins = (p.rows + at_once - 1) / at_once;
    if (!launchable(tiles, C::kThreads) || !launchable(joins, kJoinThreads)) return QA_ERR_SHAPE;
    auto kernel = p.top ? mm_token_logprobs_kernel<TM, TN, WGM, WGN, STAGES, true, TURN> : mm_token_logprobs_kernel<TM, TN, WGM, WGN, STAGES, false, TURN>;
    constexpr int kLds = C::kLdsBytes + TileScales<C::kBM, C::kBN, C::kWaves>::kBytes + C::kBM * 4;
    static_assert(kLds <= 160 * 1024, "LDS of a CU");
    if (kLds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess) return check_launch();
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles)), dim3(C::kThreads), kLds, stream, p, columns);
    if (const int status = check_launch()) return status;
    const dim3 grid(static_cast<unsigned>(joins));
    auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kJoinThreads), 0, stream, p, tiles_n); };
    at_once == 16 ? join(mm_token_logprobs_join_kernel<16>) : at_once == 4 ? join(mm_token_logprobs_join_kernel<4>) : join(mm_token_logprobs_join_kernel<1>);
    return check_launch();
}

}  // namespace
}  // namespace lm
}  // namespace qa

extern "C" int64_t qa_mm_token_logprobs_workspace_bytes(const QaMmTokenLogprobsParams* p) {
    using namespace qa::lm;
    return p && check(*p) == QA_OK && p->rows > 0 ? workspace_bytes(*p) : 0;
}

extern "C" int qa_mm_token_logprobs(const QaMmTokenLogprobsParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::lm;
    if (!p) return QA_ERR_NULL;
    if (const int status = check(*p)) return status;
    if (p->rows == 0) return QA_OK;
    if (!p->a || !p->w || !p->a_scale || !p->w_scale || !p->tokens || !p->logprobs || !p->entropy || !p->workspace) return QA_ERR_NULL;
    if (p->top && (!p->top_logprobs || !p->top_tokens)) return QA_ERR_NULL;
    if ((p->a_scale_numel != 1 && p->a_scale_numel != p->rows) || (p->w_scale_numel != 1 && p->w_scale_numel < p->vocab)) return QA_ERR_SHAPE;
    if (p->k % 16 != 0 || p->lda % 16 != 0 || p->ldw % 16 != 0 || !aligned16(p->a) || !aligned16(p->w) || p->lda < p->k || p->ldw < p->k) return QA_ERR_STRIDE;
    if (!aligned4(p->a_scale) || !aligned4(p->w_scale) || reinterpret_cast<uintptr_t>(p->tokens) % p->token_bytes != 0) return QA_ERR_STRIDE;
    if (p->lda > kWidestRow || p->ldw > kWidestRow) return QA_ERR_SHAPE;
    if (!aligned16(p->workspace) || p->workspace_bytes < workspace_bytes(*p)) return QA_ERR_SCRATCH;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    const Plan plan = plan_of(*p);
    const bool turned = p->k % kBK == 0;
    switch (plan.tile) {
        case 0: return turned ? launch<0, 1, 1, 2, 2, 3, true>(*p, plan.columns, stream) : launch<0, 1, 1, 2, 2, 3, false>(*p, plan.columns, stream);
        case 1: return turned ? launch<1, 1, 2, 2, 2, 3, true>(*p, plan.columns, stream) : launch<1, 1, 2, 2, 2, 3, false>(*p, plan.columns, stream);
        case 2: return turned ? launch<2, 1, 2, 2, 4, 3, true>(*p, plan.columns, stream) : launch<2, 1, 2, 2, 4, 3, false>(*p, plan.columns, stream);
        case 3: return launch<3, 2, 1, 2, 4, 4, false>(*p, plan.columns, stream);
        case 4: return launch<4, 2, 2, 2, 4, 3, false>(*p, plan.columns, stream);
        case 5: return launch<5, 4, 2, 2, 4, 2, false>(*p, plan.columns, stream);
        default: return launch<6, 2, 5, 4, 2, 2, false>(*p, plan.columns, stream);
    }
}
