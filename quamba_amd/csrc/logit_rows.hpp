// How rows of logits are cut into waves and segments, and the best entries of what a workgroup holds in registers.
#pragma once

#include "row_stats.hpp"

#include <algorithm>

namespace qa {
namespace lm {
namespace {

constexpr int kWaves = 4, kUnroll = 4;
constexpr int kMaxTop = 64, kMaxSegments = 64;
constexpr int kCandidates = 256;

// How the rows are cut: waves of a segment, segments of a row, batches of a segment, loads of a lane in a batch.
struct Cut {
    int waves, segments, batches, loads;
};
Cut cut_of(int rows, int vocab, int type) {
    const int load = kWaves * 64 * (type == QA_LM_F32 ? 4 : 8), short_batches = (vocab + load - 1) / load, batches = (vocab + load * kUnroll - 1) / (load * kUnroll);
    // A wave for each row where there are waves enough for that, or little for each of them: what comes once a row then comes once, and nothing
    // waits at barriers (us by four waves and by one: 30000 x 1000 fp16 top 5 90, 36; 20000 x 4000 fp16 47, 34, top 5 82, 45; 4096 x 50280 fp16
    // 79, 79, top 5 98, 85; but 3200 x 50280 58, 64, 2000 x 20000 top 5 27, 32; 1024 x 4000 6.1, 5.6; 1024 x 4000 fp32, four batches of a wave,
    // top 5 9.4, 11.2).
    const int cus = compute_units();
    if (rows >= 16 * cus || (rows >= cus && vocab <= 2 * kUnroll * load / kWaves)) return {1, 1, batches * kWaves, kUnroll};
    const int wanted = static_cast<int>(std::min<int64_t>((4LL * cus + rows - 1) / rows, kMaxSegments));
    if (short_batches <= wanted) return {kWaves, short_batches, 1, 1};
    const int each = (batches + std::min(batches, wanted) - 1) / std::min(batches, wanted);
    return {kWaves, (batches + each - 1) / each, each, kUnroll};
}

struct Candidates {
    alignas(16) Entry at[kCandidates];
    uint32_t keys[kWaves][64];
    int count;
};

// The candidates that a workgroup has put together, by one wave.
__device__ __forceinline__ void take_candidates(BestEntries& best, const Candidates& c, int count, int top, int lane) {
    for (int i = 0; i < count; i += 64) best.offer(i + lane < count ? c.at[i + lane] : 0, top, lane);
}

// A bound that `top` of the workgroup's values or more reach and hardly more than that do, from what its lanes' largest values are (at least `top` of them are there,
// -inf ones among them).  Clears the count of candidates.
__device__ __forceinline__ float bound_of_lanes(float most, int top, Candidates& c, int wave, int lane) {
    if (threadIdx.x == 0) c.count = 0;
    c.keys[wave][lane] = sort_wave(key_of(most), lane);
    __syncthreads();
    uint32_t reached;
    if (top <= 16) {
        // a share of `top` in every wave, or all of them in one
        const int share = (top + kWaves - 1) / kWaves - 1;
        uint32_t every = c.keys[0][share], one = c.keys[0][top - 1];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            every = min(every, c.keys[w][share]);
            one = max(one, c.keys[w][top - 1]);
        }
        reached = max(every, one);
    } else {
        // the top-th largest of all of them: more steps, and fewer values than that bound lets through (1 x 50280 top 64 12 us, 17 as above;
        // 20000 x 1000 top 5, by four waves a row, 66, 56 as above)
        const uint32_t all = merge_waves(merge_waves(c.keys[0][lane], c.keys[1][lane], lane), merge_waves(c.keys[2][lane], c.keys[3][lane], lane), lane);
        reached = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(all), top - 1));
    }
    return value_of_key(reached);
}

// The best `top` of the workgroup's values: `visit(f)` calls f(values, the largest of them, whether they are there, index) for each load of a
// lane, `most` is the largest of all.  Those that reach the bound are put together in LDS (in any order) and one wave sorts them.  Where more come
// than there is room for - equal values, or as many alternatives as lanes - every wave keeps its own best instead and one wave merges them.  The result is wave 0's.
template <int V, class Visit>
__device__ __forceinline__ BestEntries pick(Visit&& visit, float most, int top, Candidates& c, Entry (&lists)[kWaves][64], Entry* waiting, int wave, int lane) {
    const float bound = bound_of_lanes(most, top, c, wave, lane);
    visit([&](const auto& v, float most_of, bool valid, uint32_t index) __attribute__((always_inline)) {
        if (!__builtin_amdgcn_ballot_w64(valid && most_of >= bound)) return;
        constexpr int N = sizeof(v) / sizeof(v[0]);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!valid || !(v[j] >= bound)) continue;
            const int at = atomicAdd(&c.count, 1);
            if (at < kCandidates) c.at[at] = entry_of(v[j], index + j);
        }
    });
    __syncthreads();
    const int count = c.count;
    BestEntries best;
    best.clear();
    // (a NaN reaches no bound)
    if (count <= kCandidates) {
        if (wave == 0) take_candidates(best, c, count, top, lane);
        return best;
    }
    BestOfBatches<V> run;
    run.clear(waiting);
    run.batch(most, top, lane);
    visit([&](const auto& v, float most_of, bool valid, uint32_t index) __attribute__((always_inline)) { run.take(v, most_of, valid, index, top, lane); });
    run.finish(top, lane);
    lists[wave][lane] = run.best.mine;
    __syncthreads();
    best = run.best;
    if (wave == 0)
        for (int w = 1; w < kWaves; ++w) best.mine = merge_waves(best.mine, lists[w][lane], lane);
    return best;
}

}  // namespace
}  // namespace lm
}  // namespace qa
