// The best continuations over the beams and the vocabulary (qa_beam_search_step).
//
// Two launches: every row of logits, cut into segments, leaves for each segment the sum of its exponentials and its best `count` entries by logit; then a
// workgroup for each entry of the batch joins the sums of its beams, turns the entries into scores and ranks those that reach a bound.
//
// Scores of different beams are compared, and which of two comes first is an answer in whole numbers.  So the sums are held in 64 bits and their terms are good to
// 1e-14: e^d is 2^(n / 512) from a table by e^r, |r| <= ln 2 / 1024, from a polynomial whose first missing term is r^4 / 24 < 9e-15.
// With the difference from the largest logit that makes thirteen instructions a value, nine of them in 64 bits (5.4 cycles of a wave each, those in 32 some 4 to 5): what a launch
// on many rows takes its time for.
#include "../../include/quamba_amd_beam.h"
#include "logit_rows.hpp"

namespace qa {
namespace lm {
namespace {

constexpr int kMaxBeams = 64, kMaxVocab = 1 << 20;
constexpr int kMaxLoads = 16;              // chunks of a segment

// A sum of exponentials is s e^m, m the largest logit of what it covers: s is 1 at least, and 1 exactly where one logit has all of the weight.  Of nothing m is -inf and s 0, or
// NaN where there was one.
struct BeamPart {
    float m;
    double s;
};

// The sum of a part of a row, by one wave (all but s are the same in its lanes).  64 bits hold e^600 as well as e^-600, so the first values' largest, m, is near enough until one is
// more than kReach above it.  Terms are taken of the differences from it, exact in 64 bits (but for logits 2^29 times smaller than m): rows that differ by a number have the same terms.
constexpr float kReach = 600.0f;
constexpr int kSteps = 512;
__device__ __forceinline__ float uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
struct WideSum {
    double s;
    float m;                   // -inf: no value was seen yet
    float limit, least;        // values above the one are seen from another place, those below the other count as it
    __device__ __forceinline__ void clear() {
        s = 0.0;
        m = limit = -__builtin_inff();
        least = 0.0f;
    }
    // seen from where values up to `most` are
    __device__ __forceinline__ void place(float most) {
        if (m > -__builtin_inff()) s *= exp(fmax(static_cast<double>(m) - most, -700.0));
        m = uniform(most);
        limit = uniform(most + kReach);
        least = uniform(most - 700.0f);
    }
    // e^d, d from -700 to kReach + some (a NaN stays one), added for B values to `to`; powers those of kPowers.  In steps, so that the reads of the table are on
    // their way together: one after the other they took 130 cycles a value, most of it waiting.
    template <int B>
    static __device__ __forceinline__ double exponentials(double to, const double (&d)[B], const double* powers) {
        // 512 log2 e, ln 2 / 512; the rounded multiple of a step is in the low word of 1.5 * 2^52 and it
        constexpr double kPerUnit = 738.65986093514926, kStep = 0.0013538030870311431, kRound = 6755399441055744.0;
        int n[B];
        double value[B], power[B];
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const double shifted = __builtin_fma(d[j], kPerUnit, kRound);
            n[j] = static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, shifted)));
            const double r = __builtin_fma(shifted - kRound, -kStep, d[j]);
            value[j] = __builtin_fma(__builtin_fma(__builtin_fma(r, 1.0 / 6.0, 0.5), r, 1.0), r, 1.0);
        }
#pragma unroll
        for (int j = 0; j < B; ++j) power[j] = powers[n[j] & (kSteps - 1)];
#pragma unroll
        for (int j = 0; j < B; ++j) {
            // (into the exponent, which stays a normal one; what the compiler makes of it are five instructions)
            v2u bits = __builtin_bit_cast(v2u, power[j]);
            uint32_t high;
            asm("v_lshl_add_u32 %0, %1, 11, %2" : "=v"(high) : "v"(n[j]), "v"(bits[1]));
            bits[1] = high;
            to = __builtin_fma(value[j], __builtin_bit_cast(double, bits), to);
        }
        return to;
    }
    static_assert(kSteps == 1 << 9, "the shift into the exponent: 20 - 9");
    // values of which `most` is the largest of this lane's
    template <int B>
    __device__ __forceinline__ void add(const float (&v)[B], float most, const double* powers) {
        if (__builtin_amdgcn_ballot_w64(most > limit)) place(wave_max(most));
        if (!(m > -__builtin_inff())) {
            // (masked values alone, or NaNs)
#pragma unroll
            for (int j = 0; j < B; ++j) s = v[j] == v[j] ? s : __builtin_nan("");
            return;
        }
        double d[B];
        if (fabsf(m) <= kFarthest) {
#pragma unroll
            for (int j = 0; j < B; ++j) {
                float one;                                 // (the larger, a NaN if there is one)
                asm("v_maximum3_f32 %0, %1, %2, %2" : "=v"(one) : "v"(v[j]), "v"(least));
                d[j] = static_cast<double>(one) - m;
            }
        } else {
            // (m - 700 is no number of 32 bits here)
#pragma unroll
            for (int j = 0; j < B; ++j) {
                d[j] = static_cast<double>(v[j]) - m;
                d[j] = d[j] < -700.0 ? -700.0 : d[j];
            }
        }
        s = exponentials(s, d, powers);
    }
    // the wave's: `most` its largest value.  Divided by what its own term is, so that this one counts as 1 whatever the approximation is off by.
    __device__ __forceinline__ BeamPart part(float most, const double* powers) const {
        if (!(m > -__builtin_inff())) return {m, s};
        const double d[1] = {static_cast<double>(most) - m};
        return {most, s / exponentials(0.0, d, powers)};
    }
};

template <int MASK>
__device__ __forceinline__ double across(double v, int lane) { return __builtin_bit_cast(double, lm::across<MASK>(__builtin_bit_cast(uint64_t, v), lane)); }
// f(1), f(2), f(4) .. below `end`, each a constant of its own
template <int MASK = 1, class F>
__device__ __forceinline__ void each_mask(int end, F&& f) {
    if constexpr (MASK < 64) {
        if (MASK >= end) return;
        f(std::integral_constant<int, MASK>{});
        each_mask<2 * MASK>(end, f);
    }
}
// over the wave, in every lane: the order of the sum is that of the lanes' numbers' bits, the same in all of them
__device__ __forceinline__ double wave_sum(double s, int lane) {
    each_mask(64, [&](auto mask) { s += across<decltype(mask)::value>(s, lane); });
    return s;
}

// Both sums as one.
__device__ __forceinline__ BeamPart joined(BeamPart a, BeamPart b) {
    const BeamPart high = b.m > a.m ? b : a, low = b.m > a.m ? a : b;
    return {high.m, low.s == 0.0 ? high.s : high.s + low.s * exp(static_cast<double>(low.m) - high.m)};
}
// The sums of `lanes` neighbouring lanes as one, in all of them: the largest first, then one exponential each, and their sum.
__device__ __forceinline__ BeamPart joined_over(BeamPart r, int lanes, int lane) {
    float m = r.m;
    each_mask(lanes, [&](auto mask) { m = fmaxf(m, __uint_as_float(word_across<decltype(mask)::value>(__float_as_uint(m), lane))); });
    r.s = r.s == 0.0 ? 0.0 : r.s * exp(static_cast<double>(r.m) - m);
    each_mask(lanes, [&](auto mask) { r.s += across<decltype(mask)::value>(r.s, lane); });
    r.m = m;
    return r;
}

// powers[i] = 2^(i / kSteps), less i steps in the exponent's place: n steps added there, whatever n, make 2^(n / kSteps) of powers[n mod kSteps].  (Worked out by each
// workgroup they were half of the instructions of a row of 1000 values.)
struct Powers {
    uint64_t bits[kSteps];
};
constexpr Powers make_powers() {
    // 2^(1/2), 2^(1/4) .. 2^(1/512): products of nine of them are off by 1e-15
    constexpr double roots[9] = {1.4142135623730951, 1.189207115002721, 1.0905077326652577, 1.0442737824274138, 1.0218971486541166, 1.0108892860517005, 1.0054299011128027, 1.0027112750502025, 1.0013547198921082};
    Powers p = {};
    for (int i = 0; i < kSteps; ++i) {
        double v = 1.0;
        for (int b = 0; b < 9; ++b)
            if (i >> (8 - b) & 1) v *= roots[b];
        p.bits[i] = __builtin_bit_cast(uint64_t, v) - (static_cast<uint64_t>(i) << (52 - 9));
    }
    return p;
}
__device__ constexpr Powers kPowers = make_powers();

typedef uint64_t v2k __attribute__((ext_vector_type(2)));
// How many of the first `n` keys are larger than one, and as large; up to seven behind them are 0 (which no key that is looked at is).  first, step: some of the
// eights they are in.
struct Above {
    int larger, equal;
};
__device__ __forceinline__ Above above(const uint64_t* keys, int n, uint64_t own, int first = 0, int step = 8) {
    Above a = {0, 0};
    for (int o = first; o < n; o += step) {
        v2k k[4];                                          // (on their way together)
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const v2k*>(keys + o + 2 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a.larger += (k[i][0] > own) + (k[i][1] > own);
            a.equal += (k[i][0] == own) + (k[i][1] == own);
        }
    }
    return a;
}

// f(i, sub, lanes) for each of `count` things by four lanes, two or one, as many as there are; sums over them
template <class F>
__device__ __forceinline__ void by_lanes(int count, int threads, F&& f) {
    const int lanes = 4 * count <= threads ? 4 : 2 * count <= threads ? 2 : 1, i = threadIdx.x / lanes;
    if (threadIdx.x / 64 * 64 / lanes < static_cast<unsigned>(count)) f(i, static_cast<int>(threadIdx.x % lanes), lanes);
}
__device__ __forceinline__ int over_lanes(int v, int lanes, int lane) {
    if (lanes >= 2) v += static_cast<int>(lm::across<1>(static_cast<uint32_t>(v), lane));
    if (lanes >= 4) v += static_cast<int>(lm::across<2>(static_cast<uint32_t>(v), lane));
    return v;
}

// A workgroup has a segment of up to kMaxLoads chunks, one load a lane each; kAhead of them are under way while one is summed.  What each load's largest value is goes to LDS, and
// when all were seen a bound says which loads have one of the best entries: their values are read once more, a lane each, and what reaches the bound is ranked (each
// counts the others that are larger).  64 x 8 rows of 50280 bf16, count 16, take 21.4 us (2.4 TB/s): the loop, bound by the vector units with 20 instructions a value in all (the
// loads alone 10), and some 4 for the selection of the last of a CU's four workgroups, which the others' hide behind their loops.  (By terms of two instructions less, that do not
// keep equal scores equal, 20; by those: registers handed on from load to load, for which the compiler waits each time, 26; entries kept on the way, as token_logprobs has
// them, 35; three to five loads ahead the same; six or eight workgroups a CU 26 and 28.)
constexpr int kAhead = 2;

template <class T, bool WIDE>
__global__ __launch_bounds__(64 * kWaves, 4) void beam_rows_kernel(QaBeamSearchParams p, int top, int segments, int each) {
    constexpr int V = 16 / sizeof(T), W = kWaves, kThreads = 64 * W;
    typedef BestOfBatches<V> Run;
    __shared__ BeamPart s_part[W];
    __shared__ Candidates s_candidates;
    __shared__ union {
        float most[kMaxLoads][kThreads];
        Entry waiting[W][Run::kWaiting];
    } s;
    __shared__ uint32_t s_loads[kCandidates];              // (chunk, thread) of those that are read once more
    __shared__ double s_powers[kSteps];
    __shared__ int s_count;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x / segments, segment = blockIdx.x % segments, entry = row / p.beams, beam = row % p.beams;
    static_assert(kSteps == 2 * kThreads, "two each");
    const uint64_t powers[2] = {kPowers.bits[2 * threadIdx.x], kPowers.bits[2 * threadIdx.x + 1]};
    if (p.done && p.done[row]) return;                     // (its part is not looked at)
    const T* const logits = static_cast<const T*>(p.logits) + entry * p.logits_batch_stride + beam * p.logits_beam_stride;
    const int vectors = p.vocab / V, rest = p.vocab - vectors * V;
    const int first = segment * each, loads = min(each, (vectors + kThreads - 1) / kThreads - first);
    const float none = -__builtin_inff();

    // load u of thread `thread` (what is not there: the last one)
    auto place = [&](int u, int thread) { return (first + u) * kThreads + thread; };
    const T* const from = vectors ? logits : static_cast<const T*>(p.workspace);           // (something to load, if for nothing)
    auto load = [&](Raw<T, V>& raw, int u, int thread) __attribute__((always_inline)) {
        raw.template load<WIDE>(from + static_cast<int64_t>(max(min(place(u, thread), vectors - 1), 0)) * V);
    };
    // chunks that are there for every thread; one that is not may follow
    const int whole = max(0, min(loads, vectors / kThreads - first));
    Raw<T, V> raw[kAhead], last;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(raw[i], min(i, loads - 1), threadIdx.x);
    load(last, min(whole, loads - 1), threadIdx.x);
    // fewer than V values behind the last whole load: one each in the first lanes of the last segment
    const int rest_at = vectors * V + lane;
    const bool has_rest = segment == segments - 1 && wave == 0 && lane < rest;
    T rest_raw = static_cast<T>(0.0f);
    if (has_rest) rest_raw = logits[rest_at];
    s_powers[2 * threadIdx.x] = __builtin_bit_cast(double, powers[0]);
    s_powers[2 * threadIdx.x + 1] = __builtin_bit_cast(double, powers[1]);
    if (threadIdx.x == 0) s_count = 0;
    static_assert(kCandidates == kThreads, "one each");
    s_candidates.at[threadIdx.x] = 0;                      // (behind the last candidate none is found)
    __syncthreads();
    WideSum r;
    r.clear();
    float most = none;
    auto sum = [&](int u, const Raw<T, V>& now, auto whole_c) __attribute__((always_inline)) {
        float v[V], most_of = none;
        const bool there = decltype(whole_c)::value || place(u, threadIdx.x) < vectors;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = there ? now.get(j) : none;
#pragma unroll
        for (int j = 0; j < V; ++j) most_of = fmaxf(most_of, v[j]);
        s.most[u][threadIdx.x] = most_of;
        most = fmaxf(most, most_of);
        r.add(v, most_of, s_powers);
    };
    // (loads without a condition, behind the last one that one again: a branch around them, or registers handed on, and the compiler waits for all of them each time)
    int u = 0;
    for (; u + kAhead <= whole; u += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            sum(u + i, raw[i], std::true_type{});
            load(raw[i], min(u + i + kAhead, whole - 1), threadIdx.x);
        }
    }
#pragma unroll
    for (int i = 0; i + 1 < kAhead; ++i)
        if (u + i < whole) sum(u + i, raw[i], std::true_type{});
    if (whole < loads) sum(whole, last, std::false_type{});
    const float rest_v = has_rest ? static_cast<float>(rest_raw) : none, one[1] = {rest_v};
    most = fmaxf(most, rest_v);
    if (segment == segments - 1 && wave == 0) r.add(one, rest_v, s_powers);
    r.s = wave_sum(r.s, lane);

    const float bound = bound_of_lanes(most, top, s_candidates, wave, lane);
    const BeamPart mine = r.part(value_of_key(s_candidates.keys[wave][0]), s_powers);
    if (lane == 0) s_part[wave] = mine;
    // (of chunks that are there, in bits)
    uint32_t hits = 0, there = (1u << max(loads, 0)) - 1;
    if (whole < loads && place(whole, threadIdx.x) >= vectors) there &= ~(1u << whole);
    static_assert(kMaxLoads <= 16, "bits, and five planes of their number");
#pragma unroll
    for (int u0 = 0; u0 < kMaxLoads; u0 += 4) {
        if (u0 >= loads) break;
        float of[4];                                       // (on their way together)
#pragma unroll
        for (int i = 0; i < 4; ++i) of[i] = s.most[u0 + i][threadIdx.x];
#pragma unroll
        for (int i = 0; i < 4; ++i) hits |= of[i] >= bound ? 1u << (u0 + i) : 0u;
    }
    hits &= there;
    // (places for the wave's by one atomic; the compiler would go through the lanes one by one)
    int in_wave = 0, before = 0;
#pragma unroll
    for (int plane = 0; plane < 5; ++plane) {
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(__popc(hits) >> plane & 1);
        in_wave += __popcll(lanes) << plane;
        before += static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(lanes >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(lanes), 0))) << plane;
    }
    if (in_wave > 0) {
        int at = 0;
        if (lane == 0) at = atomicAdd(&s_count, in_wave);
        at = __builtin_amdgcn_readfirstlane(at) + before;
        for (; hits; hits &= hits - 1, ++at)
            if (at < kCandidates) s_loads[at] = static_cast<uint32_t>(__ffs(hits) - 1) << 16 | threadIdx.x;
    }
    auto candidate = [&](float value, uint32_t index) {
        if (!(value >= bound)) return;
        const int at = atomicAdd(&s_candidates.count, 1);
        if (at < kCandidates) s_candidates.at[at] = entry_of(value, index);
    };
    if (has_rest) candidate(rest_v, rest_at);
    __syncthreads();
    const int again = s_count;
    // (a lane for each value)
    if (again <= kCandidates) {
        for (int i = threadIdx.x; i < again * V; i += kThreads) {
            const int at = place(static_cast<int>(s_loads[i / V] >> 16), static_cast<int>(s_loads[i / V] & 0xffff)) * V + i % V;
            candidate(static_cast<float>(logits[at]), static_cast<uint32_t>(at));
        }
    }
    __syncthreads();
    BeamPart* const parts = static_cast<BeamPart*>(p.workspace);
    Entry* const out = reinterpret_cast<Entry*>(parts + static_cast<int64_t>(p.batch) * p.beams * segments) + static_cast<int64_t>(blockIdx.x) * top;
    // (by the last wave, which has the fewest candidates to rank)
    if (wave == W - 1) {
        const BeamPart all = joined_over(s_part[lane % W], W, lane);
        if (lane == 0) parts[blockIdx.x] = all;
    }
    const int count = s_candidates.count;
    if (again <= kCandidates && count <= kCandidates - 8) {
        by_lanes(count, kThreads, [&](int i, int sub, int lanes) {
            const Entry mine = s_candidates.at[i];
            const int before = over_lanes(above(s_candidates.at, count, mine, sub * 8, lanes * 8).larger, lanes, lane);
            if (mine != 0 && sub == 0 && before < top) out[before] = mine;
        });
        if (static_cast<int>(threadIdx.x) >= count && static_cast<int>(threadIdx.x) < top) out[threadIdx.x] = 0;
        return;
    }
    // more reach the bound than there is room for - equal values, or as many as lanes are asked for: every wave keeps its own best as it goes through its loads again
    Run run;
    run.clear(s.waiting[wave]);
    for (int u = 0; u < loads; ++u) {
        Raw<T, V> once_more;
        load(once_more, u, threadIdx.x);
        const bool there = place(u, threadIdx.x) < vectors;
        float v[V], most_of = none;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[j] = there ? once_more.get(j) : none;
            most_of = fmaxf(most_of, v[j]);
        }
        run.batch(most_of, top, lane);
        run.take(v, most_of, there, static_cast<uint32_t>(place(u, threadIdx.x) * V), top, lane);
    }
    run.next_batch(top);
    run.take(one, rest_v, has_rest, static_cast<uint32_t>(rest_at), top, lane);
    run.finish(top, lane);
    __syncthreads();
    s.waiting[wave][lane] = run.best.mine;
    __syncthreads();
    if (wave != 0) return;
    Entry best = run.best.mine;
    for (int w = 1; w < W; ++w) best = merge_waves(best, s.waiting[w][lane], lane);
    if (lane < top) out[lane] = best;
}

// An offer: larger scores first, of equal ones the lower beam, then the place in the beam's own order.  0: none.
struct Offer {
    uint64_t key;          // of the score in 64 bits
    uint32_t at;           // ~ of its place among the entries of the beams, a beam's behind those of the one before
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

// A bound that `count` of the workgroup's keys or more reach, one a lane (0: none): the count-th largest of their upper halves, by sorts of words.  0 where
// fewer lanes have a key.
template <int WAVES>
__device__ __forceinline__ uint64_t bound_of_keys(uint64_t mine, int count, uint32_t (&keys)[WAVES][64], int wave, int lane) {
    static_assert(WAVES == 4, "two pairs");
    keys[wave][lane] = sort_wave(static_cast<uint32_t>(mine >> 32), lane);
    __syncthreads();
    const uint32_t all = merge_waves(merge_waves(keys[0][lane], keys[1][lane], lane), merge_waves(keys[2][lane], keys[3][lane], lane), lane);
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(all), count - 1))) << 32;
}

// An entry of the batch.  The lanes are shared out among the beams and join their segments' sums; meanwhile the lists are on their way.  Up to kKept entries, four a lane,
// get their scores' keys at once: a bound, the `count`-th largest of what the lanes have best, leaves about as many offers, and those are ranked, each counting the
// others that are larger.  Of more than that the first entry of each list alone says whether any of it counts: a bound that `count` firsts reach leaves
// about as many lists, and a second one over their entries, a wave four lists at a time, about as many offers.  (us of this launch: 4 beams of 25 segments, count 8, 5.4,
// lists first 7.6; 5 of 63, count 10, 7.9, all entries first, 13 a lane, 10.5; 30 of 28, count 60, 18.7, the lists' entries one after the other 27; all entries sorted, 64 at a
// time, 8 and 26 for the first two; a wave eight or sixteen lists at a time 9 and 10.5 for the second.)  What is left are some ten waits, for memory and for LDS, one after the other.  Where more reach the bounds than there is room
// for - equal scores, or as many places as lanes - each wave sorts what its lanes have.
constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / 64, kOffers = 256, kFew = 48, kEach = 4, kKept = kEach * kJoinThreads;
constexpr int kSlots = kMaxBeams * kMaxSegments + 1024;
constexpr int join_lds(int entries) { return entries <= kKept ? kKept * 12 : kSlots * 8 + kMaxBeams * kMaxSegments * 2; }
__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(QaBeamSearchParams p, int top, int segments) {
    static_assert(kMaxSegments <= 64 && kMaxTop <= 64, "a lane for each");
    __shared__ double s_rest[kMaxBeams], s_base[kMaxBeams];        // of a beam: own score - ln s, -inf: it offers nothing; m
    __shared__ uint8_t s_done[kMaxBeams], s_beam[kOffers];
    __shared__ __attribute__((aligned(16))) uint64_t s_keys[kOffers + 8];
    __shared__ uint32_t s_at[kOffers], s_token[kOffers];
    // keys of this lane's entries and their tokens; or keys of the first ones of lists, then of all entries of lists, and the lists
    extern __shared__ uint64_t s_slot_keys[];
    uint32_t* const s_slot_tokens = reinterpret_cast<uint32_t*>(s_slot_keys + kKept);
    uint16_t* const s_lists = reinterpret_cast<uint16_t*>(s_slot_keys + kSlots);
    __shared__ Offer s_sorted[kJoinWaves][64];
    __shared__ uint32_t s_bounds[kJoinWaves][64];
    __shared__ int s_count, s_further;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t entry = blockIdx.x;
    const BeamPart* const parts = static_cast<const BeamPart*>(p.workspace) + entry * p.beams * segments;
    const Entry* const entries = reinterpret_cast<const Entry*>(static_cast<const BeamPart*>(p.workspace) + static_cast<int64_t>(p.batch) * p.beams * segments) +
                                 entry * p.beams * segments * top;
    const int lists = p.beams * segments;
    const int all = lists * top;
    const bool kept = all <= kKept;                        // (join_lds)
    const int slots = kept ? all : lists;
    // the entry of this lane's slot j
    auto entry_at = [&](int j) { return static_cast<int>(j * kJoinThreads + threadIdx.x) * (kept ? 1 : top); };
    Entry mine[kEach];                                     // (on their way meanwhile)
    auto fetch = [&](int first) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine[i] = entries[min(entry_at(first + i), all - 1)];
    };
    fetch(0);
    if (threadIdx.x == 0) s_count = s_further = 0;
    static_assert(kOffers == kJoinThreads, "one each");
    s_keys[threadIdx.x] = 0;                               // (behind the last offer none is found)
    if (threadIdx.x < 8) s_keys[kOffers + threadIdx.x] = 0;
    {
        // a power of two of lanes for each beam
        const int share = kJoinThreads >> (32 - __builtin_clz(max(p.beams, 4) - 1)), beam = threadIdx.x / share, part = threadIdx.x % share;
        // (all of it on its way at the same time, also what a beam that is done does not need)
        const bool there = beam < p.beams;
        const int64_t row = entry * p.beams + (there ? beam : 0);
        const double own = p.scores[row];
        const uint8_t end_reached = p.done ? p.done[row] : 0;
        BeamPart r = {-__builtin_inff(), 0.0}, second = r;
        if (there && part < segments) r = parts[beam * segments + part];
        if (there && part + share < segments) second = parts[beam * segments + part + share];
        const bool done = end_reached != 0;
        if (share < segments) r = joined(r, second);
        for (int i = part + 2 * share; there && i < segments; i += share) r = joined(r, parts[beam * segments + i]);
        r = joined_over(r, share, lane);
        if (there && part == 0) {
            const bool offers = own > -__builtin_inf() && own < __builtin_inf() && (done || r.s > 0.0);
            s_rest[beam] = !offers ? -__builtin_inf() : done ? own : own - log(r.s);
            s_base[beam] = done ? 0.0 : r.m;
            s_done[beam] = done;
        }
    }
    __syncthreads();
    const int of_beam = segments * top;
    const float per = 1.0f / static_cast<float>(of_beam);
    // (half an entry from a whole number of beams at least, 1 / 8192 of one: the product's error is far below that)
    auto beam_of = [&](int at) { return static_cast<int>((static_cast<float>(at) + 0.5f) * per); };
    // the key of an entry's score; 0: no offer
    auto key_of = [&](int at, Entry e, bool there) __attribute__((always_inline)) -> uint64_t {
        const int beam = beam_of(min(at, all - 1));
        const double rest = s_rest[beam], base = s_base[beam];
        const bool done = s_done[beam];
        const float logit = value_of(e);
        const bool offers = there & (rest > -__builtin_inf()) & (done ? at == beam * of_beam : (e != 0) & (logit > -__builtin_inff()));
        // (the difference first: next to a mask of -3e38 nothing else is left of the sum)
        const double score = rest + (done ? 0.0 : static_cast<double>(logit) - base);
        return offers ? key_of_score(score) : 0;
    };
    auto offer = [&](int at, uint64_t key, uint32_t token) {
        const int place = atomicAdd(&s_count, 1);
        if (place >= kOffers) return;
        s_keys[place] = key;
        s_at[place] = ~static_cast<uint32_t>(at);
        s_beam[place] = static_cast<uint8_t>(beam_of(at));
        s_token[place] = token;
    };
    uint64_t best_key = 0, bound = 0;
    int further = lists;                                   // lists that are looked at
    for (int first = 0; first * kJoinThreads < slots; first += kEach) {
        if (first > 0) fetch(first);
        uint64_t key[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) key[i] = key_of(entry_at(first + i), mine[i], entry_at(first + i) < all);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            s_slot_keys[(first + i) * kJoinThreads + threadIdx.x] = key[i];
            best_key = key[i] > best_key ? key[i] : best_key;
            if (kept) s_slot_tokens[(first + i) * kJoinThreads + threadIdx.x] = index_of(mine[i]);
        }
    }
    if (slots > kFew) bound = bound_of_keys(best_key, p.count, s_bounds, wave, lane);
    auto each_slot = [&](auto&& f) __attribute__((always_inline)) {
        for (int j = 0; j * kJoinThreads < slots; ++j) {
            const uint64_t key = s_slot_keys[j * kJoinThreads + threadIdx.x];
            if (key != 0 && key >= bound) f(j, key);
        }
    };
    if (kept) {
        each_slot([&](int j, uint64_t key) { offer(entry_at(j), key, s_slot_tokens[j * kJoinThreads + threadIdx.x]); });
    } else {
        each_slot([&](int j, uint64_t) { s_lists[atomicAdd(&s_further, 1)] = static_cast<uint16_t>(j * kJoinThreads + threadIdx.x); });
        __syncthreads();
        further = s_further;
        // a wave has four lists at a time, their entries from another lane on in each: what they begin with is no lane's alone
        auto each_entry = [&](auto&& f) __attribute__((always_inline)) {
            for (int first = wave * kEach; first < further; first += kJoinWaves * kEach) {
                Entry e[kEach];
                int at[kEach], slot[kEach];
                bool there[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int l = min(first + i, further - 1), place = (lane + 17 * l) & 63;
                    there[i] = (first + i < further) & (place < top);
                    slot[i] = l * top + min(place, top - 1);
                    at[i] = s_lists[l] * top + min(place, top - 1);
                    e[i] = entries[at[i]];
                }
                uint64_t key[kEach];                       // (all of them, then what comes of them: their reads are on their way together)
#pragma unroll
                for (int i = 0; i < kEach; ++i) key[i] = key_of(at[i], e[i], there[i]);
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (there[i]) f(slot[i], at[i], key[i], e[i]);
            }
        };
        // their keys take the place of the lists', if there is room for all
        const int items = further * top;
        const bool room = items <= kSlots;
        best_key = 0;
        each_entry([&](int slot, int, uint64_t key, Entry) {
            best_key = key > best_key ? key : best_key;
            if (room) s_slot_keys[slot] = key;
        });
        const uint64_t closer = bound_of_keys(best_key, p.count, s_bounds, wave, lane);
        bound = closer > bound ? closer : bound;
        if (room) {
            for (int i = threadIdx.x; i < items; i += kJoinThreads) {
                const uint64_t key = s_slot_keys[i];
                if (key == 0 || key < bound) continue;
                const int at = s_lists[i / top] * top + i % top;
                offer(at, key, index_of(entries[at]));
            }
        } else {
            each_entry([&](int, int at, uint64_t key, Entry e) {
                if (key != 0 && key >= bound) offer(at, key, index_of(e));
            });
        }
    }
    __syncthreads();
    const int offers = s_count;
    const int64_t out = entry * p.count;
    auto write = [&](int place, uint64_t key, int beam, uint32_t token) {
        p.out_scores[out + place] = static_cast<float>(score_of_key(key));
        p.tokens[out + place] = s_done[beam] ? -1 : static_cast<int64_t>(token);
        p.parents[out + place] = beam;
    };
    auto leave = [&](int place) {
        p.out_scores[out + place] = -__builtin_inff();
        p.tokens[out + place] = -1;
        p.parents[out + place] = -1;
    };
    if (offers <= kOffers) {
        by_lanes(offers, kJoinThreads, [&](int i, int sub, int lanes) {
            const uint64_t key = s_keys[i];
            const Above a = above(s_keys, offers, key, sub * 8, lanes * 8);
            int place = over_lanes(a.larger, lanes, lane);
            if (over_lanes(a.equal, lanes, lane) > 1 && i < offers) {
                const uint32_t at = s_at[i];
                int first = 0;
                for (int n = sub; n < offers; n += lanes) first += s_keys[n] == key && s_at[n] > at;
                place += over_lanes(first, lanes, lane);
            }
            if (i < offers && sub == 0 && place < p.count) write(place, key, s_beam[i], s_token[i]);
        });
        if (static_cast<int>(threadIdx.x) >= offers && static_cast<int>(threadIdx.x) < p.count) leave(threadIdx.x);
        return;
    }
    Offer best = {0, 0};
    for (int i = wave * 64; i < further * top; i += kJoinThreads) {
        Offer o = {0, 0};
        if (i + lane < further * top) {
            const int list = kept ? (i + lane) / top : s_lists[(i + lane) / top], place = (i + lane) % top;
            const uint64_t key = key_of(list * top + place, entries[list * top + place], true);
            if (key != 0) o = {key, ~static_cast<uint32_t>(list * top + place)};
        }
        if (__builtin_amdgcn_ballot_w64(o.key != 0 && o.key >= bound)) best = merge_waves(best, sort_wave(o, lane), lane);
    }
    s_sorted[wave][lane] = best;
    __syncthreads();
    if (wave != 0) return;
    for (int w = 1; w < kJoinWaves; ++w) best = merge_waves(best, s_sorted[w][lane], lane);
    if (lane < p.count) best.key != 0 ? write(lane, best.key, static_cast<int>(~best.at) / top / segments, index_of(entries[~best.at])) : leave(lane);
}

int check(const QaBeamSearchParams& p) {
    if (p.batch < 0 || p.beams < 1 || p.vocab < 1 || p.vocab > kMaxVocab) return QA_ERR_SHAPE;
    if (!is_float_type(p.logits_type) || p.beams > kMaxBeams || p.count < 1 || p.count > kMaxTop) return QA_ERR_UNSUPPORTED;
    if (p.count > static_cast<int64_t>(p.beams) * p.vocab || static_cast<int64_t>(p.batch) * p.beams > 0x7fffffffLL) return QA_ERR_SHAPE;
    return QA_OK;
}
int top_of(const QaBeamSearchParams& p) { return std::min(p.count, p.vocab); }
// How a row is cut: segments, chunks of a segment.  Four workgroups for each CU where the rows are few.
struct BeamsCut {
    int segments, each;
};
BeamsCut beams_cut(const QaBeamSearchParams& p) {
    const int chunk = kWaves * 64 * (p.logits_type == QA_LM_F32 ? 4 : 8), chunks = (p.vocab + chunk - 1) / chunk;
    static_assert(kMaxVocab / (kWaves * 64 * 4) <= kMaxSegments * kMaxLoads, "a place for every chunk");
    const int64_t rows = static_cast<int64_t>(p.batch) * p.beams;
    const int wanted = static_cast<int>(std::min<int64_t>((4LL * compute_units() + rows - 1) / rows, kMaxSegments));
    const int each = std::min(kMaxLoads, (chunks + std::min(chunks, wanted) - 1) / std::min(chunks, wanted));
    return {(chunks + each - 1) / each, each};
}
int64_t workspace_bytes(const QaBeamSearchParams& p) {
    return static_cast<int64_t>(p.batch) * p.beams * beams_cut(p).segments * (static_cast<int64_t>(sizeof(BeamPart)) + top_of(p) * static_cast<int64_t>(sizeof(Entry)));
}

template <class T>
int launch(const QaBeamSearchParams& p, hipStream_t stream) {
    const BeamsCut cut = beams_cut(p);
    const int top = top_of(p);
    auto whole = [&](int64_t stride, int n) { return n == 1 || stride * static_cast<int64_t>(sizeof(T)) % 16 == 0; };
    const bool wide = aligned16(p.logits) && whole(p.logits_batch_stride, p.batch) && whole(p.logits_beam_stride, p.beams);
    const int64_t workgroups = static_cast<int64_t>(p.batch) * p.beams * cut.segments;
    if (!launchable(workgroups, 64 * kWaves)) return QA_ERR_SHAPE;
    const dim3 grid(static_cast<unsigned>(workgroups)), block(64 * kWaves);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, top, cut.segments, cut.each); };
    wide ? go(beam_rows_kernel<T, true>) : go(beam_rows_kernel<T, false>);
    if (const int status = check_launch()) return status;
    hipLaunchKernelGGL(beam_join_kernel, dim3(p.batch), dim3(kJoinThreads), join_lds(p.beams * cut.segments * top), stream, p, top, cut.segments);
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
