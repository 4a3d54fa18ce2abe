// The best continuations over the beams and the vocabulary (qa_beam_search_step).
//
// Two launches: every row of logits, cut into segments as token_logprobs cuts them, leaves for each segment the sum of its exponentials and its best
// `count` entries by logit; then a workgroup for each entry of the batch joins the segments of its beams, turns the entries into scores and merges the beams'.
//
// Scores of different beams are compared, and which of two comes first is an answer in whole numbers.  So the sums are held in 64 bits and their terms are good to
// some 1e-10: exp_wide takes 2^(n / 64) from a table and e^r, |r| <= ln 2 / 128, from a polynomial whose first missing term is r^4 / 24 < 4e-11 - nine operations in
// 64 bits, which run at the rate of those in 32.
#include "../../include/quamba_amd_beam.h"
#include "logit_rows.hpp"

namespace qa {
namespace lm {
namespace {

constexpr int kMaxBeams = 64;

struct BeamPart {
    float m;
    float pad;
    double s;
};

// e^d for d from -700 to 0 (a NaN stays one); powers[i] = 2^(i / 64)
__device__ __forceinline__ double exp_wide(double d, const double* powers) {
    constexpr double kPerUnit = 92.332482616893657, kStep = 0.010830424696249145, kRound = 6755399441055744.0;       // 64 log2 e, ln 2 / 64, 1.5 * 2^52
    const double shifted = __builtin_fma(d, kPerUnit, kRound);
    const int n = static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, shifted)));
    const double r = __builtin_fma(shifted - kRound, -kStep, d);
    double e = __builtin_fma(r, 1.0 / 6.0, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    const uint64_t power = __builtin_bit_cast(uint64_t, powers[n & 63]) + (static_cast<uint64_t>(static_cast<uint32_t>(n >> 6)) << 52);
    return e * __builtin_bit_cast(double, power);
}

// sum e^(l - m) of a part of a row, as RowStats but in 64 bits
struct WideStats {
    float m;
    double s;
    __device__ __forceinline__ void clear() { m = kLowest; s = 0.0; }
    __device__ __forceinline__ void raise(float most, const double* powers) {
        s *= exp_wide(fmax(static_cast<double>(m) - most, -700.0), powers);
        m = most;
    }
    // (a comparison, and not a maximum, which would drop a NaN)
    __device__ __forceinline__ void add(float value, const double* powers) {
        const double d = static_cast<double>(value) - m;
        s += exp_wide(d < -700.0 ? -700.0 : d, powers);
    }
    template <int A, int B>
    __device__ __forceinline__ void add_batch(const float (&v)[A][B], int loads, float most, const double* powers) {
        raise(fmaxf(m, most), powers);
        const bool far = __builtin_amdgcn_ballot_w64(!(fabsf(m) <= kFarthest));
        const float least = m - 700.0f;
#pragma unroll
        for (int i = 0; i < A; ++i) {
            if (i >= loads) break;
            if (far) {
#pragma unroll
                for (int j = 0; j < B; ++j) add(v[i][j], powers);
            } else {
                // (the same, compared in 32 bits)
#pragma unroll
                for (int j = 0; j < B; ++j) s += exp_wide(static_cast<double>(v[i][j] < least ? least : v[i][j]) - m, powers);
            }
        }
    }
};

__device__ __forceinline__ double lane_double(double v, int from) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(from * 4, static_cast<int>(static_cast<uint32_t>(u))));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(from * 4, static_cast<int>(u >> 32)));
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// over the wave, in every lane: the order of the sum is that of the lanes' numbers' bits, the same in all of them
__device__ __forceinline__ WideStats wave_stats(WideStats r, const double* powers, int lane) {
    r.raise(wave_max(r.m), powers);
#pragma unroll
    for (int mask = 1; mask < 64; mask *= 2) r.s += lane_double(r.s, lane ^ mask);
    return r;
}

__device__ __forceinline__ void fill_powers(double (&powers)[64]) {
    if (threadIdx.x < 64) powers[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) / 64.0);
}

template <class T, bool WIDE, bool ONE, int LOADS>
__global__ __launch_bounds__(64 * kWaves) void beam_rows_kernel(QaBeamSearchParams p, int top, int segments, int batches_each) {
    constexpr int V = 16 / sizeof(T), W = kWaves;
    __shared__ BeamPart s_part[kWaves];
    __shared__ float s_bound[kWaves];
    __shared__ Entry s_best[kWaves][64];
    __shared__ Candidates s_candidates;
    __shared__ Entry s_waiting[kWaves][BestOfBatches<V>::kWaiting];
    __shared__ double s_powers[64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x / segments, segment = blockIdx.x % segments, entry = row / p.beams, beam = row % p.beams;
    if (p.done && p.done[row]) return;                     // (its part is not looked at)
    const T* const logits = static_cast<const T*>(p.logits) + entry * p.logits_batch_stride + beam * p.logits_beam_stride;
    const int vectors = p.vocab / V, rest = p.vocab - vectors * V;
    const int first = segment * batches_each, end = ONE ? first + 1 : min(first + batches_each, (vectors + W * 64 * LOADS - 1) / (W * 64 * LOADS));
    const float none = -__builtin_inff();

    // fewer than V values behind the last whole load: one each in the first lanes of the last segment
    const int rest_at = vectors * V + lane;
    const bool has_rest = segment == segments - 1 && wave == 0 && lane < rest;
    float rest_v = none;
    if (has_rest) rest_v = static_cast<float>(logits[rest_at]);
    fill_powers(s_powers);
    __syncthreads();
    WideStats r;
    r.clear();
    BestEntries best;
    best.clear();
    BestOfBatches<V> run;
    if constexpr (!ONE) run.clear(s_waiting[wave]);
    // WHOLE: every lane has its loads
    auto batch = [&](int b, auto whole_c) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_c)::value;
        Raw<T, V> raw[LOADS];
        int at[LOADS];
        float v[LOADS][V], most_of[LOADS], most = none;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            at[u] = ((b * LOADS + u) * W + wave) * 64 + lane;
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
        const int wanted = (vectors - (b * LOADS * W + wave) * 64 + W * 64 - 1) / (W * 64);        // loads with a lane that has one
        r.add_batch(v, WHOLE ? LOADS : __builtin_amdgcn_readfirstlane(wanted), most, s_powers);
        if constexpr (ONE) {
            best = pick<V>([&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < LOADS; ++u) f(v[u], most_of[u], at[u] < vectors, static_cast<uint32_t>(at[u] * V));
                const float one[1] = {rest_v};
                f(one, rest_v, has_rest, static_cast<uint32_t>(rest_at));
            }, most, top, s_candidates, s_best, s_waiting[wave], wave, lane);
        } else {
            run.batch(most, top, lane);
#pragma unroll
            for (int u = 0; u < LOADS; ++u) run.take(v[u], most_of[u], WHOLE || at[u] < vectors, static_cast<uint32_t>(at[u] * V), top, lane);
        }
    };
    if constexpr (ONE) {
        batch(first, std::false_type{});
        r.add(rest_v, s_powers);
    } else {
        const int whole = min(end, vectors / (W * 64 * LOADS));
        int b = first;
        for (; b < whole; ++b) batch(b, std::true_type{});
        for (; b < end; ++b) batch(b, std::false_type{});
        if (segment == segments - 1 && wave == 0 && rest) {
            r.raise(fmaxf(r.m, rest_v), s_powers);
            r.add(rest_v, s_powers);
            const float one[1] = {rest_v};
            run.next_batch(top);
            run.take(one, rest_v, has_rest, static_cast<uint32_t>(rest_at), top, lane);
        }
    }
    r = wave_stats(r, s_powers, lane);
    if (lane == 0) {
        s_part[wave] = {r.m, 0.0f, r.s};
        if constexpr (!ONE) s_bound[wave] = value_of_key(run.bound);
    }
    bool sorted = false;                                   // (of the same value in all waves)
    if constexpr (!ONE) {
        // what waits reaches the bound of its wave; what counts, the largest of the waves' bounds
        if (threadIdx.x == 0) s_candidates.count = 0;
        if (lane == 0) s_candidates.keys[wave][0] = run.best.last != 0;
        __syncthreads();
        float bound = s_bound[0];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            bound = fmaxf(bound, s_bound[w]);
            sorted |= s_candidates.keys[w][0] != 0;
        }
        if (!sorted) {
            static_assert(kCandidates >= 64 * kWaves, "room for all that wait");
            run.wave_order();
            const Entry e = lane < run.count ? s_waiting[wave][lane] : 0;
            if (e != 0 && value_of(e) >= bound) s_candidates.at[atomicAdd(&s_candidates.count, 1)] = e;
        } else {
            run.finish(top, lane);
            best = run.best;
            s_best[wave][lane] = best.mine;
        }
    }
    __syncthreads();
    if (wave != 0) return;
    if constexpr (!ONE) {
        if (!sorted) take_candidates(best, s_candidates, s_candidates.count, top, lane);
    }
    float most = r.m;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        most = fmaxf(most, s_part[w].m);
        if (!ONE && sorted) best.mine = merge_waves(best.mine, s_best[w][lane], lane);
    }
    r.raise(most, s_powers);
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        WideStats o = {s_part[w].m, s_part[w].s};
        o.raise(most, s_powers);
        r.s += o.s;
    }
    BeamPart* const parts = static_cast<BeamPart*>(p.workspace);
    if (lane == 0) parts[blockIdx.x] = {r.m, 0.0f, r.s};
    if (lane < top) reinterpret_cast<Entry*>(parts + static_cast<int64_t>(p.batch) * p.beams * segments)[static_cast<int64_t>(blockIdx.x) * top + lane] = best.mine;
}

// An offer: larger scores first, of equal ones the lower beam, then the place in the beam's own order.  0: none.
struct Offer {
    uint64_t key;          // of the score in 64 bits
    uint32_t at;           // ~(beam * 64 + place)
    __device__ __forceinline__ bool operator>(const Offer& o) const { return key > o.key || (key == o.key && at > o.at); }
};
template <int MASK>
__device__ __forceinline__ Offer across(Offer o, int lane) {
    return {static_cast<uint64_t>(word_across<MASK>(static_cast<uint32_t>(o.key >> 32), lane)) << 32 | word_across<MASK>(static_cast<uint32_t>(o.key), lane),
            word_across<MASK>(o.at, lane)};
}
__device__ __forceinline__ uint64_t key_of_score(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000u);
}
__device__ __forceinline__ double score_of_key(uint64_t key) { return __builtin_bit_cast(double, key & 0x8000000000000000u ? key ^ 0x8000000000000000u : ~key); }

// An entry of the batch: its beams are shared out among the waves.
__global__ __launch_bounds__(64 * kWaves) void beam_join_kernel(QaBeamSearchParams p, int top, int segments) {
    static_assert(kMaxSegments <= 64 && kMaxTop <= 64, "a lane for each");
    __shared__ Offer s_offers[kWaves][64];
    __shared__ uint32_t s_tokens[kMaxBeams][64];
    __shared__ double s_powers[64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t entry = blockIdx.x;
    const BeamPart* const parts = static_cast<const BeamPart*>(p.workspace);
    const Entry* const entries = reinterpret_cast<const Entry*>(parts + static_cast<int64_t>(p.batch) * p.beams * segments);
    fill_powers(s_powers);
    __syncthreads();
    Offer best = {0, 0};
    for (int beam = wave; beam < p.beams; beam += kWaves) {
        const int64_t row = entry * p.beams + beam;
        const double own = p.scores[row];
        Offer mine = {0, 0};
        if (!(own > -__builtin_inf() && own < __builtin_inf())) continue;
        if (p.done && p.done[row]) {
            if (lane == 0) mine = {key_of_score(own), ~static_cast<uint32_t>(beam * 64)};
            s_tokens[beam][lane] = 0xffffffffu;
        } else {
            WideStats r;
            r.clear();
            if (lane < segments) r = {parts[row * segments + lane].m, parts[row * segments + lane].s};
            Entry list = 0;
            const Entry* const from = entries + row * segments * top;
            if (top >= 16) {
                for (int i = 0; i < segments; ++i) list = merge_waves(list, lane < top ? from[i * top + lane] : Entry(0), lane);
            } else {
                for (int i = 0; i < segments * top; i += 64) list = merge_waves(list, sort_wave(i + lane < segments * top ? from[i + lane] : Entry(0), lane), lane);
            }
            r = wave_stats(r, s_powers, lane);
            const float logit = value_of(list);
            if (r.s > 0.0 && list != 0 && logit > -__builtin_inff() && lane < top)
                mine = {key_of_score(own + (static_cast<double>(logit) - r.m - log(r.s))), ~static_cast<uint32_t>(beam * 64 + lane)};
            s_tokens[beam][lane] = index_of(list);
        }
        best = merge_waves(best, mine, lane);
    }
    s_offers[wave][lane] = best;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) best = merge_waves(best, s_offers[w][lane], lane);
    if (lane >= p.count) return;
    const int64_t out = entry * p.count + lane;
    const uint32_t at = ~best.at, beam = at / 64;
    const bool there = best.key != 0;
    p.out_scores[out] = there ? static_cast<float>(score_of_key(best.key)) : -__builtin_inff();
    p.tokens[out] = there ? static_cast<int64_t>(static_cast<int32_t>(s_tokens[beam][at % 64])) : -1;
    p.parents[out] = there ? static_cast<int64_t>(beam) : -1;
}

int check(const QaBeamSearchParams& p) {
    if (p.batch < 0 || p.beams < 1 || p.vocab < 1 || p.vocab > 1 << 30) return QA_ERR_SHAPE;
    if (!is_float_type(p.logits_type) || p.beams > kMaxBeams || p.count < 1 || p.count > kMaxTop) return QA_ERR_UNSUPPORTED;
    if (p.count > static_cast<int64_t>(p.beams) * p.vocab || static_cast<int64_t>(p.batch) * p.beams > 0x7fffffffLL) return QA_ERR_SHAPE;
    return QA_OK;
}
int top_of(const QaBeamSearchParams& p) { return std::min(p.count, p.vocab); }
// four waves a segment, however many rows there are
Cut beams_cut(const QaBeamSearchParams& p) {
    Cut cut = cut_of(p.batch * p.beams, p.vocab, p.logits_type);
    if (cut.waves == 1) {
        const int load = kWaves * 64 * (p.logits_type == QA_LM_F32 ? 4 : 8) * kUnroll;
        cut = {kWaves, 1, (p.vocab + load - 1) / load, kUnroll};
    }
    return cut;
}
int64_t workspace_bytes(const QaBeamSearchParams& p) {
    return static_cast<int64_t>(p.batch) * p.beams * beams_cut(p).segments * (static_cast<int64_t>(sizeof(BeamPart)) + top_of(p) * static_cast<int64_t>(sizeof(Entry)));
}

template <class T>
int launch(const QaBeamSearchParams& p, hipStream_t stream) {
    const Cut cut = beams_cut(p);
    const int top = top_of(p);
    auto whole = [&](int64_t stride, int n) { return n == 1 || stride * static_cast<int64_t>(sizeof(T)) % 16 == 0; };
    const bool wide = aligned16(p.logits) && whole(p.logits_batch_stride, p.batch) && whole(p.logits_beam_stride, p.beams);
    const int64_t workgroups = static_cast<int64_t>(p.batch) * p.beams * cut.segments;
    if (!launchable(workgroups, 64 * kWaves)) return QA_ERR_SHAPE;
    const dim3 grid(static_cast<unsigned>(workgroups)), block(64 * kWaves);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, top, cut.segments, cut.batches); };
    auto of_wide = [&](auto wide_c) {
        constexpr bool WIDE = decltype(wide_c)::value;
        if (cut.loads == 1) go(beam_rows_kernel<T, WIDE, true, 1>);
        else if (cut.batches == 1) go(beam_rows_kernel<T, WIDE, true, kUnroll>);
        else go(beam_rows_kernel<T, WIDE, false, kUnroll>);
    };
    wide ? of_wide(std::true_type{}) : of_wide(std::false_type{});
    if (const int status = check_launch()) return status;
    hipLaunchKernelGGL(beam_join_kernel, dim3(p.batch), block, 0, stream, p, top, cut.segments);
    return check_launch();
}

}  // namespace
}  // namespace lm
}  // namespace qa

extern "C" int qa_beam_abi_version(void) { return QA_BEAM_ABI_VERSION; }

extern "C" int64_t qa_beam_search_workspace_bytes(const QaBeamSearchParams* p) {
    using namespace qa::lm;
    return p && check(*p) == QA_OK && p->batch > 0 ? workspace_bytes(*p) : 0;
}

extern "C" int qa_beam_search_step(const QaBeamSearchParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::lm;
    if (!p) return QA_ERR_NULL;
    if (const int status = check(*p)) return status;
    if (p->batch == 0) return QA_OK;
    if (!p->logits || !p->scores || !p->out_scores || !p->tokens || !p->parents) return QA_ERR_NULL;
    const int64_t beams_span = (p->beams - 1) * p->logits_beam_stride + p->vocab;
    if (reinterpret_cast<uintptr_t>(p->logits) % bytes_of(p->logits_type) != 0 || reinterpret_cast<uintptr_t>(p->scores) % 4 != 0 ||
        (p->beams > 1 && p->logits_beam_stride < 0) || (p->batch > 1 && p->logits_batch_stride < 0) || beams_span <= 0)
        return QA_ERR_STRIDE;
    if (!p->workspace) return QA_ERR_NULL;
    if (!aligned16(p->workspace) || p->workspace_bytes < workspace_bytes(*p)) return QA_ERR_SCRATCH;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (p->logits_type == QA_LM_F32) return launch<float>(*p, stream);
    if (p->logits_type == QA_LM_BF16) return launch<__bf16>(*p, stream);
    return launch<_Float16>(*p, stream);
}
