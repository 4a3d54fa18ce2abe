// Products of many rows: tiles of the output, operands through LDS.
//
// The structure is that of the int8 tiles (gemm_core.hpp): a k tile is 128 bytes of a row - here 256 values - brought by buffer loads straight into LDS, rows of eight
// 16-byte chunks swizzled by the row; a wave walks through the fragments of one operand with those of the other one held.  A fragment of the 4-bit instruction, 16
// rows by 64 bytes, is in the same places as that of v_mfma_i32_16x16x64_i8, so the same reads feed it.  What is new are the scales: 16 bytes of a row for two k
// tiles, which lie next to those of the next row.  They come by the same loads, with the requests of the first tile of the two, and each lane keeps one word of four for
// each fragment while the two tiles last.
//
// Register-only loops of this instruction reach 7.0 PFLOP/s with random operands (9.0 with zeros: the clock follows the power) and those of 32x32x64 6.5
// (9.5).  8192 x 10240 x 2560 takes 125 us, 3.4 PFLOP/s, where calls follow each other, and 97 to 102 after a pause: 205 thousand cycles (2.0 GHz at 102 us, 2.45 with zeros as
// operands, 86 us).  In the faster of the two the main loop is 1.82 us a k tile of 256 x 256 outputs against 1.15 on registers alone (LDS busy for more than half of
// it), the outputs 18 in all.  64 x 50280 x 2560 takes 13.5 us, its bytes at 5.5 TB/s.
#include "gemm_core.hpp"
#include "mx_gemm.hpp"

#include <algorithm>

namespace qa {
namespace mx {
namespace {

using namespace gemm;
using mx::v4i;

constexpr int kLarge = 256;                // rows and columns of the largest tile

// The main loop of a wave's TM x TN blocks of 32 x 32; the order of fetches and multiplications is that of RotatedMma.
template <int TM, int TN>
struct MxMma {
    static constexpr bool kWalkW = TN > TM;
    static constexpr int kHeld = 2 * (kWalkW ? TM : TN), kWalk = 2 * (kWalkW ? TN : TM), kRing = 4, kAhead = 3;
    static constexpr int kPerTile = 2 * kWalk * kHeld, kBehindBarrier = kAhead * kHeld;     // multiplications
    static_assert(2 * kWalk % kRing == 0 && kAhead < kWalk && kHeld <= kAhead * (kHeld - 1), "the order of the fetches");
    v4f acc[2 * TN][2 * TM];      // lane l: row 16 j + (l & 15), columns 16 i + 4 (l >> 4) + 0..3
    v4i held[2][kHeld], ring[kRing];
    int held_scales[kHeld], walk_scales[kWalk], next_scales[kHeld];        // of this group of two tiles; of the next one's held fragments
    int at, scales_at;            // this lane's 16 bytes of fragment 0, step 0, in a stage's rows; its word of fragment 0 in those of the scales

    __device__ __forceinline__ void init(int lane) {
        at = (lane & 15) * kBK + swz(lane & 15, lane >> 4) * 16;
        scales_at = (lane & 15) * 16 + (lane >> 4) * 4;
        clear();
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 2 * TN; ++i)
#pragma unroll
            for (int j = 0; j < 2 * TM; ++j) acc[i][j] = v4f{0, 0, 0, 0};
    }
    // step 1 is four chunks further, which the swizzle turns into an exchange of bit 6
    __device__ __forceinline__ v4i fragment(const uint8_t* rows, int step, int f) const {
        return *reinterpret_cast<const v4i*>(rows + ((at ^ (step * 64)) + f * 16 * kBK));
    }
    // Words of scales (bytes that `mask` leaves out are of blocks behind K).  Those of the next group are fetched where the registers are free: behind the barrier of a
    // group's second tile the walked fragments up to the one at hand, and the held ones into registers of their own; the last kAhead walked ones in the next tile.
    template <int FIRST, int LAST>
    __device__ __forceinline__ void fetch_walked(const uint8_t* from, uint32_t mask) {
#pragma unroll
        for (int f = FIRST; f < LAST; ++f) walk_scales[f] = *reinterpret_cast<const int*>(from + scales_at + f * 256) & mask;
    }
    __device__ __forceinline__ void fetch_held(const uint8_t* from, uint32_t mask) {
#pragma unroll
        for (int f = 0; f < kHeld; ++f) next_scales[f] = *reinterpret_cast<const int*>(from + scales_at + f * 256) & mask;
    }
    __device__ __forceinline__ void next_group() {
#pragma unroll
        for (int f = 0; f < kHeld; ++f) held_scales[f] = next_scales[f];
    }
    // sa / sw: this wave's rows of the first tile's stage
    __device__ __forceinline__ void start(const uint8_t* sa, const uint8_t* sw) {
#pragma unroll
        for (int h = 0; h < kHeld; ++h) held[0][h] = fragment(kWalkW ? sa : sw, 0, h);
#pragma unroll
        for (int g = 0; g < kAhead; ++g) ring[g] = fragment(kWalkW ? sw : sa, 0, g);
    }
    // PARITY: which tile of its group.  scales_w / scales_h: where the walked and held ones' scales of this group (PARITY 0) or of the next one lie.
    template <int PARITY, int IN_FLIGHT, class Hook>
    __device__ __forceinline__ void tile(const uint8_t* sa, const uint8_t* sw, const uint8_t* na, const uint8_t* nw, const uint8_t* scales_w, const uint8_t* scales_h, uint32_t mask, Hook&& hook) {
        if constexpr (PARITY == 0) fetch_walked<kWalk - kAhead, kWalk>(scales_w, mask);
        const uint8_t* const h0 = kWalkW ? sa : sw;
        const uint8_t* const h1 = kWalkW ? na : nw;
        const uint8_t* const w0 = kWalkW ? sw : sa;
        const uint8_t* const w1 = kWalkW ? nw : na;
        static_for<0, 2 * kWalk>([&](auto g_c) {
            constexpr int g = decltype(g_c)::value, step = g / kWalk, pos = g % kWalk, from_end = kWalk - pos;
            if constexpr (g == 2 * kWalk - kAhead) {
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(IN_FLIGHT));
                __syncthreads();
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (PARITY == 1) {
                    fetch_walked<0, kWalk - kAhead>(scales_w, mask);
                    fetch_held(scales_h, mask);
                }
            }
            static_for<0, kHeld>([&](auto h_c) {
                constexpr int h = decltype(h_c)::value, x = g % 2 ? kHeld - 1 - h : h;     // there and back: one operand stays at every turn
                v4f& c = acc[kWalkW ? pos : x][kWalkW ? x : pos];
                if constexpr (kWalkW) c = multiply<2 * PARITY + step>(ring[g % kRing], walk_scales[pos], held[step][x], held_scales[x], c);
                else c = multiply<2 * PARITY + step>(held[step][x], held_scales[x], ring[g % kRing], walk_scales[pos], c);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (h == 0) {
                    constexpr int n = g + kAhead;
                    ring[n % kRing] = n < 2 * kWalk ? fragment(w0, n / kWalk, n % kWalk) : fragment(w1, 0, n - 2 * kWalk);
                } else if constexpr (from_end <= kAhead) {
                    constexpr int f = (kAhead - from_end) * (kHeld - 1) + h - 1;
                    if constexpr (f < kHeld) held[1 - step][f] = step == 0 ? fragment(h0, 1, f) : fragment(h1, 0, f);
                }
                hook((g * kHeld + h + kBehindBarrier) % kPerTile);
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        if constexpr (PARITY == 1) next_group();
    }
};

// Four columns of a row as they are written
template <class T>
struct Four {
    typedef T v __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ v of(v4f x) { return __builtin_convertvector(x, v); }
};

// Accumulators to the output, 16 rows at a time through LDS that is the wave's own, in 16-byte pieces of rows (on any address: an odd width's rows lie so).
template <class T, int TM, int TN>
__device__ __forceinline__ void write_tile(const QaMxGemmParams& p, const v4f (&acc)[2 * TN][2 * TM], uint8_t* stage, int m0, int n0, int lane) {
    constexpr int kRow = TN * 32 * static_cast<int>(sizeof(T)), kPitch = kRow + 16, kPieces = kRow / 16, kEach = 16 / static_cast<int>(sizeof(T));
    const bool whole = n0 + TN * 32 <= p.n && m0 + TM * 32 <= p.m;
#pragma unroll
    for (int j = 0; j < 2 * TM; ++j) {
#pragma unroll
        for (int i = 0; i < 2 * TN; ++i)
            *reinterpret_cast<typename Four<T>::v*>(stage + (lane & 15) * kPitch + (i * 16 + 4 * (lane >> 4)) * sizeof(T)) = Four<T>::of(acc[i][j]);
        wave_lds_sync();
#pragma unroll
        for (int piece = lane; piece < 16 * kPieces; piece += 64) {
            const int r = piece / kPieces, c = piece % kPieces * kEach, m = m0 + j * 16 + r, n = n0 + c;
            Raw<T, kEach> v;
            v.w[0] = *reinterpret_cast<const lm::v4w*>(stage + r * kPitch + c * sizeof(T));
            T* const d = static_cast<T*>(p.d) + static_cast<int64_t>(m) * p.ldd + n;
            if (whole || (m < p.m && n + kEach <= p.n)) {
                v.template store<false>(d);
            } else if (m < p.m) {
#pragma unroll
                for (int e = 0; e < kEach; ++e)
                    if (n + e < p.n) v.store_one(d + e, e);
            }
        }
        wave_lds_sync();
    }
}

// The scales of a workgroup's rows and columns, 16 bytes each for a group of two k tiles: rows first.  Every wave makes the same number of requests (what
// there is no row for goes behind the last one).
template <int BM, int BN, int WAVES>
struct ScaleLoader {
    static constexpr int kEach = ((BM + BN) / 64 + WAVES - 1) / WAVES, kBytes = kEach * WAVES * 1024;
    static_assert(BM % 64 == 0 && BN % 64 == 0, "a request has rows of one operand");
    const uint8_t *a, *w;          // of the tile's first row, group 0
    int64_t a_stride, w_stride;
    int rows, columns;             // of the tile
    __device__ __forceinline__ void issue(int i, int group, int groups, uint32_t dst, int wave, int lane) const {
        const int part = i * WAVES + wave;
        const bool of_a = part < BM / 64;
        // (by arithmetic: a branch in the middle of the multiplications would tear their order apart)
        const int first = of_a ? part * 64 : part * 64 - BM, there = part >= (BM + BN) / 64 ? 0 : (of_a ? rows : columns) & -static_cast<int>(group < groups);
        const v4i rsrc = make_rsrc((of_a ? a : w) + min(group, groups - 1) * (of_a ? a_stride : w_stride), there * 16);
        buffer_load_lds_b128(rsrc, dst + part * 1024, (first + lane) * 16);
    }
};

template <int TM, int TN, int WGM, int WGN, int STAGES>
struct TileCfg : Cfg<TM, TN, WGM, WGN, STAGES> {
    using Base = Cfg<TM, TN, WGM, WGN, STAGES>;
    using Scales = ScaleLoader<Base::kBM, Base::kBN, Base::kWaves>;
    static constexpr int kScaleBuffers = 2;
    static constexpr int kLds = Base::kLdsBytes + kScaleBuffers * Scales::kBytes;
    static_assert(5 - STAGES > 0, "group g's scales are last read in tile 2 g, and those of group g + 2 requested into their buffer in tile 2 g + 4 - (STAGES - 1)");
};

// MASKED: the last group has blocks behind K.  first: the output's tiles of 256 x 256 from that one on, in smaller ones; or -1: all of it.
template <int TM, int TN, int WGM, int WGN, int STAGES, bool MASKED>
__global__ __launch_bounds__(64 * WGM * WGN) void mxfp4_tiles_kernel(QaMxGemmParams p, int first) {
    using C = TileCfg<TM, TN, WGM, WGN, STAGES>;
    using Scales = typename C::Scales;
    using Mma = MxMma<TM, TN>;
    constexpr int BM = C::kBM, BN = C::kBN, WAVES = C::kWaves;
    static_assert(WAVES * 16 * (TN * 32 * 4 + 16) <= C::kLdsBytes, "the outputs take the place of the operands");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WGM, wn = wave / WGM;
    int tile_m, tile_n;
    if (first < 0) {
        tile_of_workgroup<BM, BN>(blockIdx.x, (p.m + BM - 1) / BM, (p.n + BN - 1) / BN, tile_m, tile_n);
    } else {
        constexpr int kDown = kLarge / BM, kAcross = kLarge / BN, kOf = kDown * kAcross;
        tile_of_workgroup<kLarge, kLarge>(first + blockIdx.x / kOf, (p.m + kLarge - 1) / kLarge, (p.n + kLarge - 1) / kLarge, tile_m, tile_n);
        tile_m = tile_m * kDown + blockIdx.x % kOf % kDown;
        tile_n = tile_n * kAcross + blockIdx.x % kOf / kDown;
    }
    const int m0 = tile_m * BM, n0 = tile_n * BN, rows = min(BM, p.m - m0), columns = min(BN, p.n - n0);
    if (rows <= 0 || columns <= 0) return;                 // (of a large tile at the output's edge)
    const int bytes = p.k / 2, k_tiles = (bytes + kBK - 1) / kBK, blocks = p.k / kBlock, groups = (blocks + 15) / 16;
    // (from the tile's own first row and column on: 32-bit offsets reach over operands of any size)
    const v4i rsrc_a = make_rsrc(static_cast<const uint8_t*>(p.a) + m0 * p.lda, static_cast<int>((rows - 1) * p.lda + bytes));
    const v4i rsrc_w = make_rsrc(p.w + n0 * p.ldw, static_cast<int>((columns - 1) * p.ldw + bytes));
    const uint32_t lds_base = lds_offset_of(lds);
    TileLoader<C::kAInstr> load_a;
    TileLoader<C::kWInstr> load_w;
    load_a.template init<WAVES>(0, rows, p.lda, wave, lane);
    load_w.template init<WAVES>(0, columns, p.ldw, wave, lane);
    const Scales load_s = {p.a_scales + static_cast<int64_t>(m0) * 16, p.w_scales + static_cast<int64_t>(n0) * 16, p.a_scale_group_stride, p.w_scale_group_stride, rows, columns};

    // Requests of a tile: its operands', and the scales' behind them for the first tile of a group.  They go out one at a time, one per kPace multiplications counted
    // from the barrier: those that fit behind it, whose stage it has just freed, for tile t + STAGES, the rest during the next tile.  Past the end of K every
    // lane is out of range and stores zeros.
    constexpr int kData = C::kAInstr + C::kWInstr, kMost = kData + Scales::kEach;
    constexpr int kPace = kMost <= Mma::kPerTile / 4 ? 4 : Mma::kPerTile / kMost;
    constexpr int kEarly = Mma::kBehindBarrier / kPace < kData ? Mma::kBehindBarrier / kPace : kData;
    static_assert(kPace >= 1, "a place for every request");
    // (first_c: whether it is the first tile of a group)
    auto request = [&](int r, int tile, auto first_c, uint32_t stage) __attribute__((always_inline)) {
        const int k0 = tile * kBK;
        if (r < C::kAInstr) load_a.template issue_one<WAVES>(r, rsrc_a, k0, bytes, lds_base + stage, wave);
        else if (r < kData) load_w.template issue_one<WAVES>(r - C::kAInstr, rsrc_w, k0, bytes, lds_base + stage + BM * kBK, wave);
        else if (decltype(first_c)::value && r < kMost) load_s.issue(r - kData, tile / 2, groups, lds_base + C::kLdsBytes + tile / 2 % 2 * Scales::kBytes, wave, lane);
    };
    const uint8_t* const scales = lds + C::kLdsBytes;
    const uint8_t* const my_a = lds + (wm * TM * 32) * kBK;
    const uint8_t* const my_w = lds + BM * kBK + (wn * TN * 32) * kBK;
    Mma mma;
    mma.init(lane);
    auto scale_mask = [&](int group) {
        if (!MASKED) return 0xffffffffu;
        const int mine = (blocks - group * 16 - (lane >> 4) + 3) >> 2;
        return mine >= 4 ? 0xffffffffu : mine <= 0 ? 0u : (1u << (8 * mine)) - 1;
    };
    const int scales_of_a = wm * TM * 32 * 16, scales_of_w = (BM + wn * TN * 32) * 16;
    auto walked_scales = [&](int group) { return scales + group % 2 * Scales::kBytes + (Mma::kWalkW ? scales_of_w : scales_of_a); };
    auto held_scales = [&](int group) { return scales + group % 2 * Scales::kBytes + (Mma::kWalkW ? scales_of_a : scales_of_w); };
    constexpr int kOdd = kData, kEven = kMost;             // requests of a tile
    static_for<0, STAGES - 1>([&](auto t_c) {
        constexpr int t = decltype(t_c)::value;
#pragma unroll
        for (int r = 0; r < kMost; ++r) request(r, t, std::bool_constant<t % 2 == 0>{}, t * C::kStageBytes);
    });
#pragma unroll
    for (int r = 0; r < kEarly; ++r) request(r, STAGES - 1, std::bool_constant<STAGES % 2 == 1>{}, (STAGES - 1) * C::kStageBytes);
    // (tiles 1 .. STAGES - 2 and the early ones in flight)
    constexpr int kOddsBehindFirst = (STAGES - 1) / 2, kEvensBehindFirst = (STAGES - 2) / 2;
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(kOddsBehindFirst * kOdd + kEvensBehindFirst * kEven + kEarly));
    __syncthreads();
    mma.template fetch_walked<0, Mma::kWalk - Mma::kAhead>(walked_scales(0), scale_mask(0));
    mma.fetch_held(held_scales(0), scale_mask(0));
    mma.next_group();
    mma.start(my_a, my_w);
    uint32_t cur = 0, late = (STAGES - 1) * C::kStageBytes;        // stages of this tile and of the tile STAGES - 1 further
    auto one = [&](int t, auto parity_c) __attribute__((always_inline)) {
        constexpr int PARITY = decltype(parity_c)::value;
        // at the barrier of tile t, tiles t + 2 .. t + STAGES - 1 may be in flight
        constexpr int kTiles = STAGES - 2, kEvens = PARITY == 0 ? (kTiles + 1) / 2 : kTiles / 2;
        const uint32_t nxt = cur + C::kStageBytes == C::kLdsBytes ? 0 : cur + C::kStageBytes;
        mma.template tile<PARITY, kEvens * kEven + (kTiles - kEvens) * kOdd>(my_a + cur, my_w + cur, my_a + nxt, my_w + nxt, walked_scales((t + PARITY) / 2), held_scales((t + PARITY) / 2), scale_mask((t + PARITY) / 2), [&](int idx) {
            if (idx % kPace != kPace - 1) return;
            const int r = idx / kPace;
            if (r < kEarly) request(r, t + STAGES, std::bool_constant<(PARITY + STAGES) % 2 == 0>{}, cur);
            else request(r, t + STAGES - 1, std::bool_constant<(PARITY + STAGES) % 2 == 1>{}, late);
        });
        late = cur;
        cur = nxt;
    };
    int t = 0;
    for (; t + 2 <= k_tiles; t += 2) {
        one(t, std::integral_constant<int, 0>{});
        one(t + 1, std::integral_constant<int, 1>{});
    }
    if (t < k_tiles) one(t, std::integral_constant<int, 0>{});
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();
    uint8_t* const stage = lds + wave * (16 * (TN * 32 * 4 + 16));
    if (p.out_type == QA_LM_F32) write_tile<float, TM, TN>(p, mma.acc, stage, m0 + wm * TM * 32, n0 + wn * TN * 32, lane);
    else if (p.out_type == QA_LM_BF16) write_tile<__bf16, TM, TN>(p, mma.acc, stage, m0 + wm * TM * 32, n0 + wn * TN * 32, lane);
    else write_tile<_Float16, TM, TN>(p, mma.acc, stage, m0 + wm * TM * 32, n0 + wn * TN * 32, lane);
}

// Tiles of 256 x 256 one after the other, a workgroup for each CU that goes through them.
//
// With few values to sum the ends of a tile weigh: K 2560 is ten k tiles, 12 us at the rate of the matrix cores, and 128 KB of outputs, which the memory takes
// 6 us for when all CUs write.  So the k tiles of all output tiles are one stream: the first of the next output tile is requested during the last of this one, and the
// outputs go out, 16 rows at a time through 2 KB of LDS for each wave, while it is on its way and while the other wave of a SIMD multiplies.
// (K a multiple of 512: every output tile then has pairs of k tiles.)
struct StreamCfg {
    using C = TileCfg<4, 2, 2, 4, 2>;
    static constexpr int kStaging = 16 * 64 * 2;           // bytes of a wave
    static constexpr int kLds = C::kLds + C::kWaves * kStaging;
};
static_assert(StreamCfg::kLds <= 160 * 1024, "all of a CU's LDS");

// 16 rows by 64 columns of 16 bits, or by 32 of 32 bits, from column n on: pieces of 16 bytes, swizzled by the row as the operands are.
template <class T, int FIRST>
__device__ __forceinline__ void write_rows(const QaMxGemmParams& p, const v4f (&acc)[4][8], int j, uint8_t* stage, int m0, int n0, bool whole, int lane) {
    constexpr int kSize = static_cast<int>(sizeof(T)), kColumns = 128 / kSize, kEach = 16 / kSize;
    const int row = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int i = 0; i < kColumns / 16; ++i) {
        const int byte = (i * 16 + 4 * quad) * kSize;
        *reinterpret_cast<typename Four<T>::v*>(stage + row * 128 + swz(row, byte / 16) * 16 + byte % 16) = Four<T>::of(acc[FIRST + i][j]);
    }
    wave_lds_sync();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = half * 8 + (lane >> 3), c = lane & 7, m = m0 + j * 16 + r, n = n0 + FIRST * 16 + c * kEach;
        Raw<T, kEach> v;
        v.w[0] = *reinterpret_cast<const lm::v4w*>(stage + r * 128 + swz(r, c) * 16);
        T* const d = static_cast<T*>(p.d) + static_cast<int64_t>(m) * p.ldd + n;
        if (whole || (m < p.m && n + kEach <= p.n)) {
            v.template store<false>(d);
        } else if (m < p.m) {
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (n + e < p.n) v.store_one(d + e, e);
        }
    }
    wave_lds_sync();
}

__global__ __launch_bounds__(512) void mxfp4_stream_kernel(QaMxGemmParams p, int tiles_m, int tiles_n, int tiles) {
    using C = StreamCfg::C;
    using Scales = C::Scales;
    using Mma = MxMma<4, 2>;
    constexpr int BM = C::kBM, BN = C::kBN, WAVES = C::kWaves, WGM = 2;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WGM, wn = wave / WGM;
    const int bytes = p.k / 2, k_tiles = bytes / kBK, groups = k_tiles / 2;
    const uint32_t lds_base = lds_offset_of(lds);
    TileLoader<C::kAInstr> load_a;
    TileLoader<C::kWInstr> load_w;
    load_a.template init<WAVES>(0, BM, p.lda, wave, lane);
    load_w.template init<WAVES>(0, BN, p.ldw, wave, lane);

    // an output tile; none behind the last one (nothing is in range)
    struct Place {
        int m0, n0, rows, columns;
    };
    auto place_of = [&](int linear) {
        int tile_m, tile_n;
        tile_of_workgroup<BM, BN>(min(linear, tiles - 1), tiles_m, tiles_n, tile_m, tile_n);
        const int there = -static_cast<int>(linear < tiles);
        return Place{tile_m * BM, tile_n * BN, min(BM, p.m - tile_m * BM) & there, min(BN, p.n - tile_n * BN) & there};
    };
    // requests of k tile `tile` of an output tile: its operands', and with GROUP its group's scales
    constexpr int kData = C::kAInstr + C::kWInstr, kMost = kData + Scales::kEach, kPace = 2;
    struct Source {
        v4i a, w;
        Scales scales;
    };
    auto source_of = [&](const Place& at) {
        Source s;
        // (no rows: nothing is in range)
        s.a = make_rsrc(static_cast<const uint8_t*>(p.a) + at.m0 * p.lda, max(0, static_cast<int>((at.rows - 1) * p.lda + (bytes & -static_cast<int>(at.rows > 0)))));
        s.w = make_rsrc(p.w + at.n0 * p.ldw, max(0, static_cast<int>((at.columns - 1) * p.ldw + (bytes & -static_cast<int>(at.columns > 0)))));
        s.scales = {p.a_scales + static_cast<int64_t>(at.m0) * 16, p.w_scales + static_cast<int64_t>(at.n0) * 16, p.a_scale_group_stride, p.w_scale_group_stride, at.rows, at.columns};
        return s;
    };
    auto request = [&](int r, const Source& from, int tile, auto group_c, uint32_t stage, int buffer) __attribute__((always_inline)) {
        if (r < C::kAInstr) load_a.template issue_whole<WAVES>(r, from.a, tile * kBK, lds_base + stage, wave);
        else if (r < kData) load_w.template issue_whole<WAVES>(r - C::kAInstr, from.w, tile * kBK, lds_base + stage + BM * kBK, wave);
        else if (decltype(group_c)::value && r < kMost) from.scales.issue(r - kData, tile / 2, groups, lds_base + C::kLdsBytes + buffer * Scales::kBytes, wave, lane);
    };
    const uint8_t* const scales = lds + C::kLdsBytes;
    const uint8_t* const my_a = lds + (wm * 128) * kBK;
    const uint8_t* const my_w = lds + BM * kBK + (wn * 64) * kBK;
    uint8_t* const staging = lds + C::kLds + wave * StreamCfg::kStaging;
    const int walked_at = wm * 128 * 16, held_at = (BM + wn * 64) * 16;

    int linear = blockIdx.x;
    Place here = place_of(linear);
    Source source = source_of(here);
    Mma mma;
    mma.init(lane);
#pragma unroll
    for (int r = 0; r < kMost; ++r) request(r, source, 0, std::true_type{}, 0, 0);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();
    mma.template fetch_walked<0, Mma::kWalk - Mma::kAhead>(scales + walked_at, 0xffffffffu);
    mma.fetch_held(scales + held_at, 0xffffffffu);
    mma.next_group();
    mma.start(my_a, my_w);
    uint32_t cur = 0;
    int buffer = 0;                                        // of this group's scales
    while (true) {
        const Place next = place_of(linear + static_cast<int>(gridDim.x));
        // the pairs of k tiles; behind the last one comes the next output tile's first
        for (int t = 0; t < k_tiles; t += 2) {
            const uint8_t* const group_now = scales + buffer * Scales::kBytes;
            const uint8_t* const group_next = scales + (buffer ^ 1) * Scales::kBytes;
            uint32_t nxt = cur ^ C::kStageBytes;
            mma.template tile<0, 0>(my_a + cur, my_w + cur, my_a + nxt, my_w + nxt, group_now + walked_at, group_now + held_at, 0xffffffffu, [&](int idx) {
                const int at = (idx + Mma::kPerTile - Mma::kBehindBarrier) % Mma::kPerTile;        // counted from the tile's beginning
                if (at % kPace == kPace - 1 && at / kPace < kData) request(at / kPace, source, t + 1, std::false_type{}, nxt, 0);
            });
            cur = nxt;
            nxt = cur ^ C::kStageBytes;
            // (by arithmetic: a branch between multiplications would tear their order apart)
            const int over = -static_cast<int>(t + 2 == k_tiles), k_next = (t + 2) & ~over;
            source = source_of({here.m0 + ((next.m0 - here.m0) & over), here.n0 + ((next.n0 - here.n0) & over), here.rows + ((next.rows - here.rows) & over),
                                here.columns + ((next.columns - here.columns) & over)});
            mma.template tile<1, 0>(my_a + cur, my_w + cur, my_a + nxt, my_w + nxt, group_next + walked_at, group_next + held_at, 0xffffffffu, [&](int idx) {
                const int at = (idx + Mma::kPerTile - Mma::kBehindBarrier) % Mma::kPerTile;
                if (at % kPace == kPace - 1 && at / kPace < kMost) request(at / kPace, source, k_next, std::true_type{}, nxt, buffer ^ 1);
            });
            cur = nxt;
            buffer ^= 1;
        }
        const int m0 = here.m0 + wm * 128, n0 = here.n0 + wn * 64;
        const bool whole = m0 + 128 <= p.m && n0 + 64 <= p.n;
        auto write = [&](auto t) __attribute__((always_inline)) {
            using T = decltype(t);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                write_rows<T, 0>(p, mma.acc, j, staging, m0, n0, whole, lane);
                if constexpr (sizeof(T) == 4) write_rows<T, 2>(p, mma.acc, j, staging, m0, n0, whole, lane);
            }
        };
        if (p.out_type == QA_LM_F32) write(float{});
        else if (p.out_type == QA_LM_BF16) write(__bf16{});
        else write(_Float16{});
        linear += static_cast<int>(gridDim.x);
        if (linear >= tiles) break;
        here = next;
        mma.clear();
    }
    // (requests behind the last tile, of nothing, store zeros into LDS: not into another workgroup's)
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
}

// the first `tiles` of the output's
int stream_launch(const QaMxGemmParams& p, int64_t tiles, int cus, hipStream_t stream) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(mxfp4_stream_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, StreamCfg::kLds) != hipSuccess) return check_launch();
    hipLaunchKernelGGL(mxfp4_stream_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(tiles, cus))), dim3(512), StreamCfg::kLds, stream, p, (p.m + kLarge - 1) / kLarge,
                       (p.n + kLarge - 1) / kLarge, static_cast<int>(tiles));
    return check_launch();
}

// tiles: how many, from the `first`-th large one on where that is not -1
template <int TM, int TN, int WGM, int WGN, int STAGES>
int launch(const QaMxGemmParams& p, int64_t tiles, int first, hipStream_t stream) {
    using C = TileCfg<TM, TN, WGM, WGN, STAGES>;
    if (tiles > 0x7fffffffLL || !launchable(tiles, C::kThreads)) return QA_ERR_SHAPE;
    auto kernel = p.k % kGroup != 0 ? mxfp4_tiles_kernel<TM, TN, WGM, WGN, STAGES, true> : mxfp4_tiles_kernel<TM, TN, WGM, WGN, STAGES, false>;
    if (C::kLds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds) != hipSuccess) return check_launch();
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles)), dim3(C::kThreads), C::kLds, stream, p, first);
    return check_launch();
}

}  // namespace

// Tiles of a launch.  With at most one tile for each CU a launch takes a tile's own time, so the smallest tile that fits the part in one round is taken (us for K 1536, 2560,
// 5120 by 64 x 128: 6.2, 8.0, 12.2; 128 x 128 6.4, 8.1, 12.5; 128 x 256 8.5, 11.7, 19; 256 x 256 13.6, 20.9, 33).  Up to 64 rows the weights count, and 64 x 256 tiles ask for
// them better once 64 x 128 need more than a round (64 x 50280 x 2560 13.8 us, 17.3 by 64 x 128).
// More than a round: what counts is rounds times a tile's time.  Large tiles do not leave the last round to themselves: what is left of them behind the last full
// round goes to smaller ones, in a launch of its own, where those take less than another round of large ones.
int tiles_launch(const QaMxGemmParams& p, hipStream_t stream) {
    const int cus = compute_units();
    auto tiles = [&](int64_t bm, int64_t bn) { return ((p.m + bm - 1) / bm) * ((p.n + bn - 1) / bn); };
    if (tiles(64, 128) <= cus) return launch<1, 2, 2, 2, 4>(p, tiles(64, 128), -1, stream);
    if (p.m <= 64) return launch<1, 2, 2, 4, 3>(p, tiles(64, 256), -1, stream);
    if (tiles(128, 128) <= cus) return launch<2, 1, 2, 4, 4>(p, tiles(128, 128), -1, stream);
    if (tiles(128, 256) <= cus) return launch<2, 2, 2, 4, 3>(p, tiles(128, 256), -1, stream);
    const float k_tiles = static_cast<float>((p.k / 2 + kBK - 1) / kBK);
    auto rounds = [&](int64_t n) { return static_cast<float>((n + cus - 1) / cus); };
    const float of_large = 2.5f + 1.86f * k_tiles, of_half = 3.0f + 1.07f * k_tiles, of_quarter = 3.3f + 0.46f * k_tiles, another_launch = 1.5f;
    const int64_t large = tiles(kLarge, kLarge), full = large / cus * cus, rest = large - full;
    const bool streams = p.k % kGroup == 0;
    const float per_round = of_large + (streams ? 0.0f : 2.2f);
    const float rest_as_half = another_launch + rounds(2 * rest) * of_half, rest_as_quarters = another_launch + rounds(4 * rest) * of_quarter;
    const float rest_alone = std::min(rest_as_half, rest_as_quarters);
    const bool split = full > 0 && rest > 0 && rest_alone < per_round;
    const float by_large = split ? full / cus * per_round + rest_alone : rounds(large) * per_round;
    if (rounds(tiles(128, 256)) * of_half < by_large) return launch<2, 2, 2, 4, 3>(p, tiles(128, 256), -1, stream);
    if (large > 0x3fffffffLL) return QA_ERR_SHAPE;
    const int64_t by_256 = split ? full : large;
    if (const int status = streams && by_256 > cus ? stream_launch(p, by_256, cus, stream) : launch<4, 2, 2, 4, 2>(p, by_256, split ? 0 : -1, stream)) return status;
    if (!split) return QA_OK;
    return rest_as_half < rest_as_quarters ? launch<2, 2, 2, 4, 3>(p, 2 * rest, static_cast<int>(full), stream) : launch<2, 1, 2, 4, 4>(p, 4 * rest, static_cast<int>(full), stream);
}

}  // namespace mx
}  // namespace qa
