// Products of few rows: operands straight from memory into the matrix instruction's registers.
//
// What is wanted is the weights, read once: a wave takes RN x 16 columns by RM x 16 rows and a part of K, whole groups of 512 values, so that it asks for
// all of its rows' lines (256 bytes of codes and a word of scales for each) before it multiplies.  The waves of a workgroup share the columns and split K; their
// sums meet in LDS, in the order of the waves.  Bound by latency where the weights are few - 1 x 10240 x 2560 fp16 5.4 us, a launch and two trips to memory beside 2.6 of
// bytes - and by the weights' bytes behind that (1 x 20000 x 2560 7.0, 3.9 TB/s).
#include "gemm_core.hpp"
#include "mx_gemm.hpp"

#include <algorithm>

namespace qa {
namespace mx {
namespace {

constexpr int kMaxWaves = 8, kRows = 16, kSharedRows = 4;

// The group of a wave's rows of numbers as fragments, by all of its lanes: eight values each, one row after the other, and the codes through LDS.
constexpr int kPitch = kGroup / 2 + 16, kStage = kSharedRows * (kPitch + 16);         // bytes of a row's codes; of all rows and their scales
template <class T>
__device__ __forceinline__ void quantise_rows(const QaMxGemmParams& p, int g, uint8_t* stage, v4i (&av)[4], int& as, int lane) {
    const int rows = min(kSharedRows, p.m), at = g * kGroup + lane * 8, block = lane >> 2;
    uint8_t* const scales = stage + kSharedRows * kPitch;
    Raw<T, 8> raw[kSharedRows];
#pragma unroll
    for (int r = 0; r < kSharedRows; ++r) {
        if (r >= rows) break;
#pragma unroll
        for (int i = 0; i < Raw<T, 8>::kWords; ++i) raw[r].w[i] = v4w{0, 0, 0, 0};
        if (at < p.k) raw[r].template load<false>(static_cast<const T*>(p.a) + r * p.lda + at);
    }
#pragma unroll
    for (int r = 0; r < kSharedRows; ++r) {
        if (r >= rows) break;
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(raw[r].get(j)) & 0x7fffffffu);
        const uint32_t scale = scale_of(most_of_block(most));
        *reinterpret_cast<uint32_t*>(stage + r * kPitch + lane * 4) = codes_of(scale, [&](int j) { return raw[r].get(j); });
        if ((lane & 3) == 0) scales[r * 16 + 4 * (block & 3) + (block >> 2)] = static_cast<uint8_t>(scale);
    }
    gemm::wave_lds_sync();
    // (rows behind the last one: that one again)
    const int row = min(lane & 15, rows - 1), q = lane >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) av[j] = *reinterpret_cast<const v4i*>(stage + row * kPitch + (4 * j + q) * 16);
    as = *reinterpret_cast<const int*>(scales + row * 16 + 4 * q);
    gemm::wave_lds_sync();
}

// ROWS_T: type of the rows (int8_t: codes).  SHARED: numbers are quantised by all lanes together, not each fragment by its own.
template <int RM, int RN, class ROWS_T, bool SHARED>
__global__ __launch_bounds__(64 * kMaxWaves) void mxfp4_direct_kernel(QaMxGemmParams p, int tiles_m, bool words) {
    constexpr bool kCodes = std::is_same_v<ROWS_T, int8_t>;
    extern __shared__ __attribute__((aligned(16))) v4f sums[];             // [wave][RN * RM][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int row = lane & 15, q = lane >> 4;
    const int m0 = static_cast<int>(blockIdx.x % tiles_m) * (RM * 16), n0 = static_cast<int>(blockIdx.x / tiles_m) * (RN * 16);
    const int blocks = p.k / kBlock, groups = (blocks + 15) / 16;
    // (rows behind the last one: that one again, and what comes of it is not written)
    const uint8_t *w[RN], *w_scales[RN], *a_scales[RM];
    const ROWS_T* a[RM];
#pragma unroll
    for (int i = 0; i < RN; ++i) {
        const int64_t n = min(n0 + i * 16 + row, p.n - 1);
        w[i] = p.w + n * p.ldw;
        w_scales[i] = p.w_scales + n * 16 + 4 * q;
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int64_t m = min(m0 + i * 16 + row, p.m - 1);
        a[i] = static_cast<const ROWS_T*>(p.a) + m * p.lda;
        a_scales[i] = kCodes ? p.a_scales + m * 16 + 4 * q : nullptr;
    }
    v4f acc[RN][RM];
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RM; ++j) acc[i][j] = v4f{0, 0, 0, 0};
    for (int g = wave; g < groups; g += waves) {
        v4i wv[RN][4], av[RM][4];
        int ws[RN], as[RM];
        // (blocks behind K: the last one again, by scales of 2^-127 on both sides, and nothing is left of their products in fp32)
        const int mine = (blocks - g * 16 - q + 3) >> 2;
        const uint32_t mask = mine >= 4 ? 0xffffffffu : mine <= 0 ? 0u : (1u << (8 * mine)) - 1;
        int at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = min(g * 16 + 4 * j + q, blocks - 1);
#pragma unroll
        for (int i = 0; i < RN; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) wv[i][j] = *reinterpret_cast<const v4i*>(w[i] + at[j] * 16);
            ws[i] = *reinterpret_cast<const int*>(w_scales[i] + g * p.w_scale_group_stride) & mask;
        }
        if constexpr (kCodes) {
#pragma unroll
            for (int i = 0; i < RM; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) av[i][j] = *reinterpret_cast<const v4i*>(a[i] + at[j] * 16);
                as[i] = *reinterpret_cast<const int*>(a_scales[i] + g * p.a_scale_group_stride) & mask;
            }
        } else if constexpr (SHARED) {
            static_assert(RM == 1, "one tile of rows");
            quantise_rows<ROWS_T>(p, g, reinterpret_cast<uint8_t*>(sums + (waves > 1 ? waves * RM * RN * 64 : 0)) + wave * kStage, av[0], as[0], lane);
            as[0] &= mask;
        } else {
#pragma unroll
            for (int i = 0; i < RM; ++i) {
                uint32_t scales = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    Raw<ROWS_T, 32> raw;
                    raw.template load<false>(a[i] + at[j] * kBlock);
                    uint32_t most = 0;
#pragma unroll
                    for (int e = 0; e < 32; ++e) most = max(most, __float_as_uint(raw.get(e)) & 0x7fffffffu);
                    const uint32_t scale = scale_of(most);
#pragma unroll
                    for (int e = 0; e < 4; ++e) av[i][j][e] = codes_of(scale, [&](int x) { return raw.get(e * 8 + x); });
                    scales |= scale << (8 * j);
                }
                as[i] = scales & mask;
            }
        }
        static_for<0, 4>([&](auto j_c) {
            constexpr int j = decltype(j_c)::value;
#pragma unroll
            for (int x = 0; x < RN; ++x)
#pragma unroll
                for (int y = 0; y < RM; ++y) acc[x][y] = multiply<j>(wv[x][j], ws[x], av[y][j], as[y], acc[x][y]);
        });
    }
    if (waves > 1) {
#pragma unroll
        for (int i = 0; i < RN; ++i)
#pragma unroll
            for (int j = 0; j < RM; ++j) sums[(wave * RN * RM + i * RM + j) * 64 + lane] = acc[i][j];
        __syncthreads();
    }
    // a wave finishes every `waves`-th of the blocks of 16 x 16
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RM; ++j) {
            const int f = i * RM + j;
            if (f % waves != wave) continue;
            v4f v = acc[i][j];
            if (waves > 1) {
                v = sums[f * 64 + lane];
                for (int o = 1; o < waves; ++o) v += sums[(o * RN * RM + f) * 64 + lane];
            }
            store_columns(p, m0 + j * 16 + row, n0 + i * 16 + 4 * q, v, words);
        }
}

template <int RM, int RN>
int64_t blocks_of(const QaMxGemmParams& p) { return ((p.m + RM * 16 - 1) / (RM * 16)) * static_cast<int64_t>((p.n + RN * 16 - 1) / (RN * 16)); }

template <int RM, int RN, class ROWS_T, bool SHARED = false>
int launch(const QaMxGemmParams& p, hipStream_t stream) {
    const int64_t tiles_m = (p.m + RM * 16 - 1) / (RM * 16), blocks = blocks_of<RM, RN>(p);
    const int waves = static_cast<int>(std::min<int64_t>(kMaxWaves, std::max<int64_t>(1, groups_of(p.k))));
    if (!launchable(blocks, 64 * waves)) return QA_ERR_SHAPE;
    const size_t of_sums = waves > 1 ? waves * RM * RN * 64 * sizeof(v4f) : 0, of_codes = SHARED ? waves * kStage : 0;
    hipLaunchKernelGGL((mxfp4_direct_kernel<RM, RN, ROWS_T, SHARED>), dim3(static_cast<unsigned>(blocks)), dim3(64 * waves), of_sums + of_codes, stream, p,
                       static_cast<int>(tiles_m), whole_words(p));
    return check_launch();
}

}  // namespace

// The smallest blocks of which each CU has one at most, and up to 16 rows as long as the weights are not so many that
// tiles ask for them better.  (us by 16 x 16, 32 x 16, 32 x 32, 64 x 32 and in tiles: 64 x 768 x 2560 4.1, 4.5, 5.5, 8, 8; 128 x 768 x 2560 5.1, 4.6, 5.3, 8, 8;
// 64 x 2560 x 2560 6.7, 6.7, 5.3, 7.3, 7.8; 128 x 2560 x 2560 9.2, 8.8, 8.4, 7.4, 8.0; 16 x 10240 x 2560 6.4, 7.0, 7.0, 8.1, 7.8; 17 x 10240 x 2560 9.1, 7.1, 7.1, 8.3, 7.9;
// 1 x 50280 x 2560 13.8, 17, 15, 20, 12.5.)
static bool takes(const QaMxGemmParams& p, int64_t cus) { return blocks_of<4, 2>(p) <= cus || (p.m <= kRows && blocks_of<1, 1>(p) <= 10 * cus); }
bool direct_takes(const QaMxGemmParams& p) { return takes(p, compute_units()); }

// Numbers in one launch: each wave quantises its group of the rows again, up to four rows by all its lanes, more of them fragment by fragment, and that has to cost less
// than a launch in front (us by all lanes, by fragments, with a launch of its own: 1 x 2560 x 5120 4.8, 5.7, 6.4; 1 x 10240 x 2560 5.5, 7.2, 7.2; 1 x 50280 x 2560 17, 28,
// 18; 4 x 2560 x 5120 5.7, 6.2, 6.7; 4 x 20000 x 2560 8.4, 12, 9.8; 4 x 50280 x 2560 20, 29, 17; 8 x 768 x 1536 4.0, 3.4, 5.9; 8 x 10240 x 2560 7.9, 8.4, 7.8;
// 16 x 768 x 1536 5.4, 3.8, 5.8; 16 x 2560 x 5120 9.7, 8.5, 7.3; 16 x 50280 x 2560 35, 45, 18).  So for more than four rows each SIMD may have one group, and
// for fewer 32 rows of a group; and codes of as many rows are summed in the same order, so that both ways give the same bits.
bool direct_takes_numbers(const QaMxGemmParams& p) {
    if (p.m > kRows) return false;
    const int64_t cus = compute_units(), simds = 4 * cus, wanted = blocks_of<1, 1>(p) * groups_of(p.k);
    return takes(p, cus) && (p.m <= kSharedRows ? p.m * wanted <= 32 * simds : groups_of(p.k) <= kMaxWaves && wanted <= simds);
}

int direct_launch(const QaMxGemmParams& p, hipStream_t stream) {
    auto of_numbers = [&](auto t) {
        using T = decltype(t);
        return p.m <= kSharedRows ? launch<1, 1, T, true>(p, stream) : launch<1, 1, T>(p, stream);
    };
    if (p.a_type == QA_LM_F32) return of_numbers(float{});
    if (p.a_type == QA_LM_BF16) return of_numbers(__bf16{});
    if (p.a_type == QA_LM_F16) return of_numbers(_Float16{});
    if (p.m <= kRows) return launch<1, 1, int8_t>(p, stream);
    const int64_t cus = compute_units();
    if (blocks_of<1, 1>(p) <= cus) return launch<1, 1, int8_t>(p, stream);
    if (blocks_of<2, 1>(p) <= cus) return launch<2, 1, int8_t>(p, stream);
    if (blocks_of<2, 2>(p) <= cus) return launch<2, 2, int8_t>(p, stream);
    return launch<4, 2, int8_t>(p, stream);
}

}  // namespace mx
}  // namespace qa
