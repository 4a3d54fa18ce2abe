// Rows of states in another order, in place (qa_reorder_states).
//
// A thread has two units of 16 bytes, on any address, of all the rows of an entry, or one of the bytes behind a row's last unit: it reads what its rows are to become and
// then writes them, so that no row is read after it was written and no copy is needed.  Rows that stay are neither read nor written, and a parent of several
// rows comes from memory once and from the caches again.  One launch has up to kTensors tensors, with their addresses in its arguments.
//
// Bound by memory: 4 x 4 rows of 64 layers of 5120 x 16 fp32 states and their int8 conv states, two launches that read and write 462 MB, take 99 us, 4.7 TB/s, where other states
// were moved before, and 75 us again and again.  (2 x 16 rows of 32 layers of 4096, 434 MB: 87 and 73; one unit a thread 97 and 76, and 89 and 76.)  States that the last-level
// cache does not hold are written past it (102 and 85 us otherwise, and 98 and 66); those that it holds are read again soon (2 x 16 rows of 32 layers of 2048, 143 MB, again and
// again 32 us, 42 past it; after others 53 and 43).  Rows of 2331 bytes, 256 of them in 64 tensors, take 15.6 us and of 2352 12.2 (a byte a lane 37).
#include "../../include/quamba_amd_beam.h"
#include "lm_common.hpp"

#include <algorithm>

namespace qa {
namespace lm {
namespace {

constexpr int kTensors = 96, kThreads = 256, kMaxBeams = 64;

struct Tensors {
    uint8_t* data[kTensors];
    int64_t row_stride[kTensors];
    int32_t units[kTensors];           // of a row
    uint8_t rest[kTensors];            // bytes behind them
    int32_t first[kTensors + 1];       // workgroup of the first unit; behind the last one, all of them
    int32_t count;
};
static_assert(sizeof(Tensors) <= 4000, "arguments of a launch: 4 KB");

// units of a thread, as far as the registers go; their bytes (of more than 32 beams 16 each are more than the registers of two waves)
template <int BEAMS>
constexpr int kUnits = BEAMS <= 16 ? 2 : 1;
template <int BEAMS>
constexpr int kUnit = BEAMS <= 32 ? 16 : 4;
typedef uint32_t v4any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t any32 __attribute__((aligned(1)));

// N units, kThreads apart, of every row; left: how many there are from the first of them on
template <int N, int BEAMS, bool PAST, class U>
__device__ __forceinline__ void move_units(uint8_t* base, int64_t row_stride, const int (&from)[BEAMS], int beams, int left) {
    std::remove_cv_t<U> v[BEAMS][N];
#pragma unroll
    for (int i = 0; i < BEAMS; ++i)
        if (i < beams && from[i] != i)
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (k * kThreads < left) v[i][k] = reinterpret_cast<const U*>(base + from[i] * row_stride)[k * kThreads];
#pragma unroll
    for (int i = 0; i < BEAMS; ++i)
        if (i < beams && from[i] != i)
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (k * kThreads < left) {
                    U* const to = reinterpret_cast<U*>(base + i * row_stride) + k * kThreads;
                    if constexpr (PAST) __builtin_nontemporal_store(v[i][k], to);
                    else *to = v[i][k];
                }
}

// BEAMS: at least as many as there are; PAST: written past the last-level cache
template <int BEAMS, bool PAST>
__global__ __launch_bounds__(kThreads) void reorder_kernel(Tensors t, const void* parents, int index_bytes, int beams) {
    const int64_t entry = blockIdx.y;
    int from[BEAMS], moved = 0;
#pragma unroll
    for (int i = 0; i < BEAMS; ++i) {
        from[i] = i;
        if (i >= beams) continue;
        const int64_t parent = token_of(parents, index_bytes, entry * beams + i);
        if (parent >= 0 && parent < beams) from[i] = static_cast<int>(parent);
        moved |= from[i] ^ i;
    }
    if (!moved) return;
    int low = 0, high = t.count - 1;                       // the tensor of this workgroup
    while (low < high) {
        const int middle = (low + high + 1) / 2;
        if (t.first[middle] <= static_cast<int>(blockIdx.x)) low = middle;
        else high = middle - 1;
    }
    constexpr int N = kUnits<BEAMS>, UNIT = kUnit<BEAMS>;
    static_assert(UNIT <= kThreads, "a thread has one of the bytes at most");
    const int unit = (static_cast<int>(blockIdx.x) - t.first[low]) * (kThreads * N) + threadIdx.x, units = t.units[low];
    uint8_t* const rows = t.data[low] + entry * beams * t.row_stride[low];
    using U = std::conditional_t<UNIT == 16, v4any, any32>;
    if (unit < units) move_units<N, BEAMS, PAST, U>(rows + static_cast<int64_t>(unit) * UNIT, t.row_stride[low], from, beams, units - unit);
    const int byte = (unit >= units ? unit : unit + (N - 1) * kThreads) - units;
    if (byte >= 0 && byte < t.rest[low]) move_units<1, BEAMS, PAST, uint8_t>(rows + static_cast<int64_t>(units) * UNIT + byte, t.row_stride[low], from, beams, 1);
}

template <int BEAMS>
int launch(const QaReorderParams& p, const Tensors& t, bool past, hipStream_t stream) {
    const dim3 grid(t.first[t.count], p.batch);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, t, p.parents, p.index_bytes, p.beams); };
    past ? go(reorder_kernel<BEAMS, true>) : go(reorder_kernel<BEAMS, false>);
    return check_launch();
}

}  // namespace
}  // namespace lm
}  // namespace qa

extern "C" int qa_reorder_states(const QaReorderParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::lm;
    if (!p) return QA_ERR_NULL;
    if (p->batch < 0 || p->beams < 1 || p->tensors < 0) return QA_ERR_SHAPE;
    if (p->beams > kMaxBeams || (p->index_bytes != 4 && p->index_bytes != 8)) return QA_ERR_UNSUPPORTED;
    if (p->batch == 0 || p->tensors == 0) return QA_OK;
    if (!p->states || !p->parents) return QA_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(p->parents) % p->index_bytes != 0) return QA_ERR_STRIDE;
    if (p->batch > 65535) return QA_ERR_SHAPE;
    for (int i = 0; i < p->tensors; ++i) {
        const QaStateRows& s = p->states[i];
        if (s.row_bytes < 0) return QA_ERR_SHAPE;
        if (s.row_bytes == 0) continue;
        if (!s.data) return QA_ERR_NULL;
        if (s.row_stride < s.row_bytes && static_cast<int64_t>(p->batch) * p->beams > 1) return QA_ERR_STRIDE;
        const int64_t units = (p->beams <= 32 ? s.row_bytes / 16 : s.row_bytes / 4) + 15;              // (with the bytes behind them)
        if (units > 0x7fffffffLL || !launchable((units + kThreads - 1) / kThreads * p->batch, kThreads)) return QA_ERR_SHAPE;
    }
    if (p->beams == 1) return QA_OK;
    constexpr int64_t kCached = 224LL << 20;
    int64_t bytes = 0;
    for (int i = 0; i < p->tensors; ++i) bytes += p->states[i].row_bytes * p->batch * p->beams;
    const bool past = bytes >= kCached;
    auto of_beams = [&](auto beams_c) {
        constexpr int BEAMS = decltype(beams_c)::value, UNIT = kUnit<BEAMS>, kEach = kThreads * kUnits<BEAMS>;
        Tensors t = {};
        auto flush = [&] {
            const int status = t.count ? launch<BEAMS>(*p, t, past, static_cast<hipStream_t>(stream_)) : QA_OK;
            t.count = 0;
            return status;
        };
        for (int i = 0; i < p->tensors; ++i) {
            const QaStateRows& s = p->states[i];
            if (s.row_bytes == 0) continue;
            const int64_t units = s.row_bytes / UNIT, rest = s.row_bytes % UNIT, workgroups = (units + rest + kEach - 1) / kEach;
            if (t.count == kTensors || !launchable((t.first[t.count] + workgroups) * p->batch, kThreads))
                if (const int status = flush()) return status;
            t.data[t.count] = static_cast<uint8_t*>(s.data);
            t.row_stride[t.count] = s.row_stride;
            t.units[t.count] = static_cast<int32_t>(units);
            t.rest[t.count] = static_cast<uint8_t>(rest);
            t.first[t.count + 1] = t.first[t.count] + static_cast<int32_t>(workgroups);
            ++t.count;
        }
        return flush();
    };
    if (p->beams <= 4) return of_beams(std::integral_constant<int, 4>{});
    if (p->beams <= 8) return of_beams(std::integral_constant<int, 8>{});
    if (p->beams <= 16) return of_beams(std::integral_constant<int, 16>{});
    if (p->beams <= 32) return of_beams(std::integral_constant<int, 32>{});
    return of_beams(std::integral_constant<int, 64>{});
}
