// Log probabilities of given tokens, entropies and the best alternatives of rows of logits (qa_token_logprobs).
//
// One pass over the logits, bound by memory while the vector units keep up: a value is converted, joins a maximum of a batch,
// and costs an exponential and four operations more (RowStats); a lane raises its maximum once a batch of loads, not
// once a value.
//
// A wave takes a row where there are many, four of them a segment of a row otherwise; the parts of a cut row go to the workspace and a
// second launch joins them.  With few rows a segment is one batch, and what costs is not the bytes but what happens one after the
// other: there the best entries are picked out of the registers by a bound (pick).  In a longer segment a wave keeps its own, and loads in
// which no value is above the last of them are passed over with one comparison per lane (BestOfBatches).
#include "row_stats.hpp"

#include <algorithm>

namespace qa {
namespace lm {
namespace {

constexpr int kWaves = 4, kUnroll = 4;
constexpr int kMaxTop = 64, kMaxSegments = 64;
constexpr int kCandidates = 256;

struct Part {
    float m, s, t, bound;      // (bound: within a workgroup)
};

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

__device__ __forceinline__ float logit_at(const QaTokenLogprobsParams& p, int64_t row, int64_t i) {
    const int64_t at = row * p.row_stride + i;
    if (p.logits_type == QA_LM_F32) return static_cast<const float*>(p.logits)[at];
    if (p.logits_type == QA_LM_BF16) return static_cast<float>(static_cast<const __bf16*>(p.logits)[at]);
    return static_cast<float>(static_cast<const _Float16*>(p.logits)[at]);
}

// one wave: what is asked of a row whose statistics and best entries it holds
__device__ __forceinline__ void answer(const QaTokenLogprobsParams& p, int64_t row, const RowStats& r, Entry best, int lane) {
    if (lane == 0) {
        const int64_t token = token_of(p.tokens, p.token_bytes, row);
        float lp = token < 0 ? 0.0f : __builtin_nanf("");
        if (token >= 0 && token < p.vocab) lp = r.logprob(logit_at(p, row, token));
        p.logprobs[row] = lp;
        p.entropy[row] = r.s > 0.0f ? r.entropy() : __builtin_nanf("");
    }
    if (lane < p.top) {
        // (a row with NaNs may have fewer entries than that)
        p.top_logprobs[row * p.top + lane] = r.logprob(value_of(best));
        p.top_tokens[row * p.top + lane] = best ? index_of(best) : 0;
    }
}

struct Candidates {
    Entry at[kCandidates];
    uint32_t keys[kWaves][64];
    int count;
};

// The candidates that a workgroup has put together, by one wave.
__device__ __forceinline__ void take_candidates(BestEntries& best, const Candidates& c, int count, int top, int lane) {
    for (int i = 0; i < count; i += 64) best.offer(i + lane < count ? c.at[i + lane] : 0, top, lane);
}

// The best `top` of the workgroup's values: `visit(f)` calls f(values, the largest of them, whether they are there, index) for each load of a
// lane, `most` is the largest of all.  What the lanes' largest values say is a bound that `top` values or more reach and hardly more than
// that do: those are put together in LDS (in any order) and one wave sorts them.  Where more come than there is room for - equal values,
// or as many alternatives as lanes - every wave keeps its own best instead and one wave merges them.  The result is wave 0's.
template <int V, class Visit>
__device__ __forceinline__ BestEntries pick(Visit&& visit, float most, int top, Candidates& c, Entry (&lists)[kWaves][64], Entry* waiting, int wave, int lane) {
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
    const float bound = value_of_key(reached);
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

// W waves take a segment; ONE: it is one batch.  With W = 1 a workgroup has kWaves whole rows.  Six waves a SIMD are asked for: fp16 values that are
// kept beside their loads take three registers more than that many waves have, and 12 bytes of scratch cost less than a wave (us with five and
// six: 500 x 256000 fp16 top 20 74, 66; 20000 x 4000 fp16 top 5 47.7, 45.4; but 2000 x 50280 top 5 49.2, 52.5).
template <class T, bool WIDE, bool TOP, int W, bool ONE, int LOADS>
__global__ __launch_bounds__(64 * kWaves, 6) void token_logprobs_kernel(QaTokenLogprobsParams p, int segments, int batches_each) {
    constexpr int V = 16 / sizeof(T);                      // values a load
    static_assert(W == kWaves || (W == 1 && !ONE), "rows of a workgroup, or workgroups of a row");
    __shared__ Part s_part[kWaves];
    __shared__ Entry s_best[TOP && W > 1 ? kWaves : 1][64];
    __shared__ std::conditional_t<TOP && (W > 1), Candidates, int> s_candidates;
    __shared__ Entry s_waiting[TOP ? kWaves : 1][BestOfBatches<V>::kWaiting];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = W > 1 ? wave : 0;
    const int64_t row = W > 1 ? blockIdx.x / segments : static_cast<int64_t>(blockIdx.x) * kWaves + wave;
    const int segment = W > 1 ? blockIdx.x % segments : 0;
    if (W == 1 && row >= p.rows) return;                   // (no wave waits for another one then)
    const T* const logits = static_cast<const T*>(p.logits) + row * p.row_stride;
    const int vectors = p.vocab / V, rest = p.vocab - vectors * V;
    const int first = segment * batches_each, end = ONE ? first + 1 : min(first + batches_each, (vectors + W * 64 * LOADS - 1) / (W * 64 * LOADS));
    const float none = -__builtin_inff();

    // fewer than V values behind the last whole load: one each in the first lanes of the last segment
    const int rest_at = vectors * V + lane;
    const bool has_rest = segment == segments - 1 && sub == 0 && lane < rest;
    float rest_v = none;
    if (has_rest) rest_v = static_cast<float>(logits[rest_at]);
    RowStats r;
    r.clear();
    BestEntries best;
    best.clear();
    BestOfBatches<V> run;
    if constexpr (TOP && !ONE) run.clear(s_waiting[wave]);
    // WHOLE: every lane has its loads
    auto batch = [&](int b, auto whole_c) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_c)::value;
        Raw<T, V> raw[LOADS];
        int at[LOADS];
        float v[LOADS][V], most_of[LOADS], most = none;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            at[u] = ((b * LOADS + u) * W + sub) * 64 + lane;
            if (!ONE || vectors > 0) raw[u].template load<WIDE>(logits + static_cast<int64_t>(WHOLE ? at[u] : min(at[u], vectors - 1)) * V);
        }
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            most_of[u] = none;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[u][j] = WHOLE || at[u] < vectors ? raw[u].get(j) : none;
                most_of[u] = fmaxf(most_of[u], v[u][j]);
            }
            most = fmaxf(most, most_of[u]);
        }
        if constexpr (ONE) most = fmaxf(most, rest_v);
        const int wanted = (vectors - (b * LOADS * W + sub) * 64 + W * 64 - 1) / (W * 64);         // loads with a lane that has one
        r.add_batch(v, WHOLE ? LOADS : __builtin_amdgcn_readfirstlane(wanted), most);
        if constexpr (TOP && ONE) {
            best = pick<V>([&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < LOADS; ++u) f(v[u], most_of[u], at[u] < vectors, static_cast<uint32_t>(at[u] * V));
                const float one[1] = {rest_v};
                f(one, rest_v, has_rest, static_cast<uint32_t>(rest_at));
            }, most, p.top, s_candidates, s_best, s_waiting[wave], wave, lane);
        } else if constexpr (TOP) {
            run.batch(most, p.top, lane);
#pragma unroll
            for (int u = 0; u < LOADS; ++u) run.take(v[u], most_of[u], WHOLE || at[u] < vectors, static_cast<uint32_t>(at[u] * V), p.top, lane);
        }
    };
    if constexpr (ONE) {
        batch(first, std::false_type{});
    } else {
        const int whole = min(end, vectors / (W * 64 * LOADS));
        int b = first;
        for (; b < whole; ++b) batch(b, std::true_type{});
        for (; b < end; ++b) batch(b, std::false_type{});
    }
    if (ONE) {
        r.add(rest_v);
    } else if (segment == segments - 1 && sub == 0 && rest) {
        r.raise(fmaxf(r.m, rest_v));
        r.add(rest_v);
        if constexpr (TOP) {
            // (they are all there is of a last segment that has no whole load)
            const float one[1] = {rest_v};
            run.next_batch(p.top);
            run.take(one, rest_v, has_rest, static_cast<uint32_t>(rest_at), p.top, lane);
        }
    }
    r = wave_stats(r);
    if constexpr (W == 1) {
        if constexpr (TOP) run.finish(p.top, lane);
        answer(p, row, r, run.best.mine, lane);
    } else {
        if (lane == 0) s_part[wave] = {r.m, r.s, r.t, value_of_key(run.bound)};
        bool sorted = false;                                   // (of the same value in all waves)
        if constexpr (TOP && !ONE) {
            // what waits reaches the bound of its wave; what counts, the largest of the waves' bounds
            if (threadIdx.x == 0) s_candidates.count = 0;
            if (lane == 0) s_candidates.keys[wave][0] = run.best.last != 0;
            __syncthreads();
            float bound = s_part[0].bound;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                bound = fmaxf(bound, s_part[w].bound);
                sorted |= s_candidates.keys[w][0] != 0;
            }
            if (!sorted) {
                static_assert(kCandidates >= 64 * kWaves, "room for all that wait");
                run.wave_order();
                const Entry e = lane < run.count ? s_waiting[wave][lane] : 0;
                if (e != 0 && value_of(e) >= bound) s_candidates.at[atomicAdd(&s_candidates.count, 1)] = e;
            } else {
                run.finish(p.top, lane);
                best = run.best;
                s_best[wave][lane] = best.mine;
            }
        }
        __syncthreads();
        if (wave != 0) return;
        if constexpr (TOP && !ONE) {
            if (!sorted) take_candidates(best, s_candidates, s_candidates.count, p.top, lane);
        }
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            r.join({s_part[w].m, s_part[w].s, s_part[w].t});
            if (TOP && !ONE && sorted) best.mine = merge_waves(best.mine, s_best[w][lane], lane);
        }
        if (segments == 1) {
            answer(p, row, r, best.mine, lane);
            return;
        }
        Part* const parts = static_cast<Part*>(p.workspace);
        if (lane == 0) parts[blockIdx.x] = {r.m, r.s, r.t, 0.0f};
        if (TOP && lane < p.top) reinterpret_cast<Entry*>(parts + static_cast<int64_t>(p.rows) * segments)[static_cast<int64_t>(blockIdx.x) * p.top + lane] = best.mine;
    }
}

// A row's segments.  Their best entries, each segment's in order, are shared out among the waves: whole lists, merged as they are, or with
// few alternatives 64 entries at a time, sorted first.
template <bool TOP>
__global__ __launch_bounds__(64 * kWaves) void token_logprobs_join_kernel(QaTokenLogprobsParams p, int segments) {
    static_assert(kMaxSegments <= 64, "a lane for each");
    __shared__ Entry s_best[TOP ? kWaves : 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const Part* const parts = static_cast<const Part*>(p.workspace) + row * segments;
    RowStats r;
    r.clear();
    if (lane < segments) r = {parts[lane].m, parts[lane].s, parts[lane].t};
    Entry best = 0;
    if constexpr (TOP) {
        const Entry* const from = reinterpret_cast<const Entry*>(static_cast<const Part*>(p.workspace) + static_cast<int64_t>(p.rows) * segments) + row * segments * p.top;
        if (p.top >= 16) {
            for (int i = wave; i < segments; i += kWaves) best = merge_waves(best, lane < p.top ? from[i * p.top + lane] : Entry(0), lane);
        } else {
            const int count = segments * p.top;
            for (int i = wave * 64; i < count; i += kWaves * 64) best = merge_waves(best, sort_wave(i + lane < count ? from[i + lane] : Entry(0), lane), lane);
        }
        s_best[wave][lane] = best;
        __syncthreads();
    }
    if (wave != 0) return;
    if constexpr (TOP) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) best = merge_waves(best, s_best[w][lane], lane);
    }
    answer(p, row, wave_stats(r), best, lane);
}

int check(const QaTokenLogprobsParams& p) {
    if (p.rows < 0 || p.vocab < 1 || p.vocab > 1 << 30) return QA_ERR_SHAPE;
    if (!is_float_type(p.logits_type) || (p.token_bytes != 4 && p.token_bytes != 8)) return QA_ERR_UNSUPPORTED;
    if (p.top < 0 || p.top > kMaxTop) return QA_ERR_UNSUPPORTED;
    if (p.top > p.vocab) return QA_ERR_SHAPE;
    return QA_OK;
}

int64_t workspace_bytes(const QaTokenLogprobsParams& p) {
    const int64_t segments = cut_of(p.rows, p.vocab, p.logits_type).segments;
    return segments == 1 ? 0 : p.rows * segments * (static_cast<int64_t>(sizeof(Part)) + p.top * static_cast<int64_t>(sizeof(Entry)));
}

template <class T>
int launch(const QaTokenLogprobsParams& p, hipStream_t stream) {
    const Cut cut = cut_of(p.rows, p.vocab, p.logits_type);
    const bool wide = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.row_stride * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    const bool by_waves = cut.waves == 1;
    const int64_t workgroups = by_waves ? (static_cast<int64_t>(p.rows) + kWaves - 1) / kWaves : static_cast<int64_t>(p.rows) * cut.segments;
    if (!launchable(workgroups, 64 * kWaves)) return QA_ERR_SHAPE;
    const dim3 grid(static_cast<unsigned>(workgroups)), block(64 * kWaves);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, cut.segments, cut.batches); };
    auto of_wide = [&](auto wide_c) {
        constexpr bool WIDE = decltype(wide_c)::value;
        if (by_waves) p.top ? go(token_logprobs_kernel<T, WIDE, true, 1, false, kUnroll>) : go(token_logprobs_kernel<T, WIDE, false, 1, false, kUnroll>);
        else if (cut.loads == 1) p.top ? go(token_logprobs_kernel<T, WIDE, true, kWaves, true, 1>) : go(token_logprobs_kernel<T, WIDE, false, kWaves, true, 1>);
        else if (cut.batches == 1) p.top ? go(token_logprobs_kernel<T, WIDE, true, kWaves, true, kUnroll>) : go(token_logprobs_kernel<T, WIDE, false, kWaves, true, kUnroll>);
        else p.top ? go(token_logprobs_kernel<T, WIDE, true, kWaves, false, kUnroll>) : go(token_logprobs_kernel<T, WIDE, false, kWaves, false, kUnroll>);
    };
    wide ? of_wide(std::true_type{}) : of_wide(std::false_type{});
    if (cut.segments > 1) {
        if (const int status = check_launch()) return status;
        auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(p.rows), block, 0, stream, p, cut.segments); };
        p.top ? join(token_logprobs_join_kernel<true>) : join(token_logprobs_join_kernel<false>);
    }
    return check_launch();
}

}  // namespace
}  // namespace lm
}  // namespace qa

extern "C" int64_t qa_token_logprobs_workspace_bytes(const QaTokenLogprobsParams* p) {
    using namespace qa::lm;
    return p && check(*p) == QA_OK && p->rows > 0 ? workspace_bytes(*p) : 0;
}

extern "C" int qa_token_logprobs(const QaTokenLogprobsParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::lm;
    if (!p) return QA_ERR_NULL;
    if (const int status = check(*p)) return status;
    if (p->rows == 0) return QA_OK;
    if (!p->logits || !p->tokens || !p->logprobs || !p->entropy || (p->top && (!p->top_logprobs || !p->top_tokens))) return QA_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(p->logits) % bytes_of(p->logits_type) != 0 || reinterpret_cast<uintptr_t>(p->tokens) % p->token_bytes != 0 ||
        (p->row_stride < p->vocab && p->rows > 1))
        return QA_ERR_STRIDE;
    const int64_t need = workspace_bytes(*p);
    if (need && !p->workspace) return QA_ERR_NULL;
    if (need && (!aligned16(p->workspace) || p->workspace_bytes < need)) return QA_ERR_SCRATCH;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (p->logits_type == QA_LM_F32) return launch<float>(*p, stream);
    if (p->logits_type == QA_LM_BF16) return launch<__bf16>(*p, stream);
    return launch<_Float16>(*p, stream);
}
