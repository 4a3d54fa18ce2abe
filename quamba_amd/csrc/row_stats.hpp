// Running statistics of a softmax over a part of a row, the best entries of a row in order, and how both are joined.
//
// Stats: the largest value m, s = sum e^(l - m) and t = sum (l - m) e^(l - m), in fp32.  Two parts join at the larger m:
//   s = sum s_i f_i,   t = sum (t_i + (m_i - m) s_i) f_i,   f_i = e^(m_i - m)
// and at the end  log sum exp = m + ln s,  entropy = ln s - t / s.  Masked values (-inf) add nothing; m starts at the lowest
// finite number, so a part without a value has s = 0.  A NaN or +inf leaves a NaN in s, which joins keep.
#pragma once

#include "lm_common.hpp"
#include "normgated_core.hpp"

namespace qa {
namespace lm {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kFarthest = 1 << 20;       // (what the rounding of m log2(e) leaves out is below 2^-4 up to here)

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

struct RowStats {
    float m, s, t;
    __device__ __forceinline__ void clear() { m = kLowest; s = 0.0f; t = 0.0f; }
    // the statistics as seen from `most` >= m
    __device__ __forceinline__ void raise(float most) {
        const float d = fmaxf(m - most, -1e30f), f = exp_fast(d);          // (0 * -inf has no place here)
        t = f * __builtin_fmaf(d, s, t);
        s *= f;
        m = most;
    }
    // one value, m no smaller than it
    __device__ __forceinline__ void add(float value) {
        const float d = value - m, e = exp_fast(d);
        s += e;
        t = __builtin_fmaf(fmaxf(d, -200.0f), e, t);                       // (e is 0 from -104 on)
    }
    // a batch of values, the largest of them `most`.  With c = log2(e) and r the rounded m c an exponent is one fused step, v c - r; what the
    // rounding left out, m c - r, is exact in one number and corrects the sums.  (It is up to 2^-24 of m c: some 1e9 from 0 the sums and the
    // correction would be 0 and inf, so from kFarthest on the differences are taken as they are - for values that are masked with a large finite
    // number, and in lanes that have seen none yet.  A product of 0 and -inf has no place here, and e is 0 long before the exponent is -200.)
    // `loads` of the A groups are there (the same number in all lanes).
    template <int A, int B>
    __device__ __forceinline__ void add_batch(const float (&v)[A][B], int loads, float most) {
        raise(fmaxf(m, most));
        if (__builtin_amdgcn_ballot_w64(!(fabsf(m) <= kFarthest))) {
#pragma unroll
            for (int i = 0; i < A; ++i) {
                if (i >= loads) break;
#pragma unroll
                for (int j = 0; j < B; ++j) add(v[i][j]);
            }
            return;
        }
        const float r = m * kLog2e, rest = __builtin_fmaf(m, kLog2e, -r);
        float sum = 0.0f, weighted = 0.0f;
#pragma unroll
        for (int i = 0; i < A; ++i) {
            if (i >= loads) break;
#pragma unroll
            for (int j = 0; j < B; ++j) {
                const float d = __builtin_fmaf(v[i][j], kLog2e, -r), e = __builtin_amdgcn_exp2f(d);
                sum += e;
                weighted = __builtin_fmaf(fmaxf(d, -200.0f), e, weighted);
            }
        }
        const float f = __builtin_amdgcn_exp2f(-rest);
        s = __builtin_fmaf(sum, f, s);
        t = __builtin_fmaf((weighted - rest * sum) * f, kLn2, t);
    }
    __device__ __forceinline__ void join(RowStats o) {
        const float most = fmaxf(m, o.m);
        raise(most);
        o.raise(most);
        s += o.s;
        t += o.t;
    }
    // (s of a row with all of its weight on one value is 1 to within a rounding: neither answer may pass 0 for that, as callers take
    // logarithms of 1 - p; a NaN stays one)
    __device__ __forceinline__ float entropy() const {
        const float h = logf(s) - t / s;
        return h < 0.0f ? 0.0f : h;
    }
    // log probability of a value; NaN where the row has no distribution
    __device__ __forceinline__ float logprob(float value) const {
        const float lp = s > 0.0f ? (value - m) - logf(s) : __builtin_nanf("");
        return lp > 0.0f ? 0.0f : lp;
    }
};

// over the wave, in every lane
__device__ __forceinline__ RowStats wave_stats(RowStats r) {
    r.raise(wave_max(r.m));
    r.s = wave_sum(r.s);
    r.t = wave_sum(r.t);
    return r;
}

// An entry of a row as one number: larger values first, of equal ones (-0 and 0 are equal) the lower index.  0: no entry.  A NaN ranks with -inf.
typedef uint64_t Entry;
__device__ __forceinline__ uint32_t key_of(float value) {
    const float v = value == value ? value + 0.0f : -__builtin_inff();
    const uint32_t u = __float_as_uint(v);
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of_key(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
__device__ __forceinline__ Entry entry_of(float value, uint32_t index) { return static_cast<uint64_t>(key_of(value)) << 32 | ~index; }
__device__ __forceinline__ float value_of(Entry e) { return value_of_key(static_cast<uint32_t>(e >> 32)); }
__device__ __forceinline__ uint32_t index_of(Entry e) { return ~static_cast<uint32_t>(e); }

__device__ __forceinline__ Entry entry_of_lane(Entry e, int lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(e >> 32), lane))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(e)), lane));
}

// the entry of lane ^ MASK, MASK + 1 a power of two (a mirror) or MASK a power of two
template <int MASK>
__device__ __forceinline__ uint32_t word_across(uint32_t v, int lane) {
    auto dpp = [](uint32_t a, auto ctrl) { return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(a), decltype(ctrl)::value, 0xf, 0xf, true)); };
    if constexpr (MASK == 1) return dpp(v, std::integral_constant<int, 0xb1>{});
    else if constexpr (MASK == 2) return dpp(v, std::integral_constant<int, 0x4e>{});
    else if constexpr (MASK == 3) return dpp(v, std::integral_constant<int, 0x1b>{});
    else if constexpr (MASK == 7) return dpp(v, std::integral_constant<int, 0x141>{});
    else if constexpr (MASK == 15) return dpp(v, std::integral_constant<int, 0x140>{});
    else if constexpr (MASK == 4) return word_across<3>(word_across<7>(v, lane), lane);
    else if constexpr (MASK == 8) return dpp(v, std::integral_constant<int, 0x128>{});
    else if constexpr (MASK == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return lane & 16 ? r[0] : r[1];
    } else if constexpr (MASK == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return lane & 32 ? r[0] : r[1];
    } else if constexpr (MASK == 31) return word_across<16>(word_across<15>(v, lane), lane);
    else return word_across<32>(word_across<31>(v, lane), lane);
}
template <int MASK>
__device__ __forceinline__ uint32_t across(uint32_t v, int lane) { return word_across<MASK>(v, lane); }
template <int MASK>
__device__ __forceinline__ Entry across(Entry e, int lane) {
    return static_cast<uint64_t>(word_across<MASK>(static_cast<uint32_t>(e >> 32), lane)) << 32 | word_across<MASK>(static_cast<uint32_t>(e), lane);
}
// lane l and lane l ^ MASK in descending order: the lower lane of the two gets the larger of them (entries, or keys alone)
template <int MASK, class E>
__device__ __forceinline__ E order(E e, int lane) {
    constexpr int kTop = (MASK + 1) & MASK ? MASK : (MASK + 1) / 2;        // the highest bit of MASK
    const E o = across<MASK>(e, lane);
    return ((e > o) == !(lane & kTop)) ? e : o;
}
template <int HALF, class E>
__device__ __forceinline__ E order_from(E e, int lane) {                   // a sequence that rises and falls, in blocks of 2 HALF
    if constexpr (HALF == 0) return e;
    else return order_from<HALF / 2>(order<HALF>(e, lane), lane);
}
// the wave's in descending order: sorted runs of 2, 4 .. 64, each of two halves met as mirror images
template <class E>
__device__ __forceinline__ E sort_wave(E e, int lane) {
    e = order<1>(e, lane);
    e = order_from<1>(order<3>(e, lane), lane);
    e = order_from<2>(order<7>(e, lane), lane);
    e = order_from<4>(order<15>(e, lane), lane);
    e = order_from<8>(order<31>(e, lane), lane);
    return order_from<16>(order<63>(e, lane), lane);
}
// the best 64 of two descending sequences, descending
template <class E>
__device__ __forceinline__ E merge_waves(E a, E b, int lane) {
    const E o = across<63>(b, lane);
    return order_from<32>(a > o ? a : o, lane);
}

// The best entries of what a wave has seen, lane i the i-th best.
struct BestEntries {
    Entry mine;
    Entry last;            // the top-th best (the same in every lane): what comes in has to be larger
    __device__ __forceinline__ void clear() { mine = last = 0; }
    // one candidate per lane (0: none)
    __device__ __forceinline__ void take(Entry e, int top, int lane) {
        const Entry sorted = sort_wave(e, lane);
        mine = __builtin_amdgcn_ballot_w64(mine != 0) ? merge_waves(mine, sorted, lane) : sorted;
        last = entry_of_lane(mine, top - 1);
    }
    // the same, skipped where none comes in
    __device__ __forceinline__ void offer(Entry e, int top, int lane) {
        if (__builtin_amdgcn_ballot_w64(e > last)) take(e > last ? e : 0, top, lane);
    }
};

// The best entries of a long run of values, a batch of loads at a time: what may come in is put down in LDS, and once more than 64 are
// together they are sorted and merged.  `bound` stands for the top-th best: that many values reach it.  Until entries were merged it is the top-th
// largest of the lanes' largest values so far, looked at again in batches 1, 2, 4, 8 ..: by that of the first batch alone some `top` values of
// every later one come in (1000 x 128000 bf16 top 5 68 us, 63 so; from more than half as many alternatives as lanes the bound is too weak to pay).
// (The sorting stands behind a load of V values, not behind each of them: in 32 places its code does not stay in the instruction cache.)
template <int V>
struct BestOfBatches {
    static constexpr int kWaiting = 64 + 64 * V;
    BestEntries best;
    uint32_t bound, reach; // keys, scalars of the wave: what comes in is no smaller than `reach`
    float lane_most;       // this lane's largest value
    int batches;           // so far
    int seen;              // values so far
    int count;             // entries waiting, at most 64 between loads
    Entry* waiting;        // kWaiting of them, of this wave alone
    __device__ __forceinline__ void clear(Entry* place) {
        best.clear();
        lane_most = -__builtin_inff();
        bound = reach = key_of(lane_most);
        batches = seen = count = 0;
        waiting = place;
    }
    // what a wave has seen has lower indices than what comes: an equal value does not come in any more (once there were `top` values)
    __device__ __forceinline__ void next_batch(int top) { reach = seen >= top ? bound + 1 : bound; }
    // in front of the loads of a batch; most: the largest of the lane's in it
    __device__ __forceinline__ void batch(float most, int top, int lane) {
        next_batch(top);
        lane_most = fmaxf(lane_most, most);
        if (batches == 0 || (top <= 32 && (batches & (batches + 1)) == 0)) {
            const uint32_t b = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(sort_wave(key_of(lane_most), lane)), top - 1));
            if (b > bound) bound = reach = b;              // (reached by values of this batch too: equal ones come in)
        }
        ++batches;
    }
    // N values of each lane that says so, index and following
    template <int N>
    __device__ __forceinline__ void take(const float (&v)[N], float most, bool valid, uint32_t index, int top, int lane) {
        seen += N * __popcll(__builtin_amdgcn_ballot_w64(valid));
        const float least = value_of_key(reach);           // (behind +inf: a NaN, which nothing reaches)
        if (!__builtin_amdgcn_ballot_w64(valid && most >= least)) return;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const bool wanted = valid && v[j] >= least;
            const uint64_t which = __builtin_amdgcn_ballot_w64(wanted);
            if (which == 0) continue;
            const int before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(which >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(which), 0));
            if (wanted) waiting[count + before] = entry_of(v[j], index + j);
            count += __popcll(which);
        }
        while (count > 64) {
            count -= 64;
            wave_order();
            best.take(waiting[count + lane], top, lane);
            bound = max(bound, static_cast<uint32_t>(best.last >> 32));
            reach = max(reach, bound);
        }
    }
    __device__ __forceinline__ void finish(int top, int lane) {
        wave_order();
        best.offer(lane < count ? waiting[lane] : 0, top, lane);
    }
    // the wave's own LDS accesses in the order of the program
    static __device__ __forceinline__ void wave_order() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
};

}  // namespace lm
}  // namespace qa
