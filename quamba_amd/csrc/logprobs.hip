// Log probabilities of given tokens, entropies and the best alternatives of rows of logits (qa_token_logprobs).
//
// One pass over the logits, bound by memory while the vector units keep up: a value is converted, joins a maximum of a batch,
// and costs an exponential and five operations more (RowStats); a lane raises its maximum once a batch of kUnroll loads, not
// once a value.  The best entries stay sorted over the lanes of a wave, and a batch in which no value is above the last of them is
// passed over with one comparison per lane.
//
// A workgroup of four waves takes a segment of a row, whole rows when there are many; the parts of a cut row go to the workspace
// and a second launch joins them.
#include "row_stats.hpp"

#include <algorithm>

namespace qa {
namespace lm {
namespace {

constexpr int kWaves = 4, kUnroll = 4;
constexpr int kMaxTop = 64, kMaxSegments = 64;

struct Part {
    float m, s, t, reserved;
};

// values of a workgroup's batch
int batch_values(int type) { return kWaves * 64 * kUnroll * (type == QA_LM_F32 ? 4 : 8); }

// segments a row is cut into
int segments_of(int rows, int vocab, int type) {
    const int batches = (vocab + batch_values(type) - 1) / batch_values(type);
    const int wanted = static_cast<int>((4LL * compute_units() + rows - 1) / rows);
    const int segments = std::min(std::min(batches, wanted), kMaxSegments);
    const int each = (batches + segments - 1) / segments;
    return (batches + each - 1) / each;
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
        p.top_logprobs[row * p.top + lane] = r.logprob(value_of(best));
        p.top_tokens[row * p.top + lane] = index_of(best);
    }
}

template <class T, bool WIDE, bool TOP>
__global__ __launch_bounds__(64 * kWaves) void token_logprobs_kernel(QaTokenLogprobsParams p, int segments, int batches_each) {
    constexpr int V = 16 / sizeof(T);                      // values a load
    __shared__ Part s_part[kWaves];
    __shared__ Entry s_best[TOP ? kWaves : 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x / segments;
    const int segment = blockIdx.x % segments;
    const T* const logits = static_cast<const T*>(p.logits) + row * p.row_stride;
    const int vectors = p.vocab / V, rest = p.vocab - vectors * V;
    const int first = segment * batches_each, end = min(first + batches_each, (vectors + kWaves * 64 * kUnroll - 1) / (kWaves * 64 * kUnroll));
    const float none = -__builtin_inff();

    RowStats r;
    r.clear();
    BestEntries best;
    best.clear();
    for (int b = first; b < end; ++b) {
        Raw<T, V> raw[kUnroll];
        int at[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            at[u] = ((b * kUnroll + u) * kWaves + wave) * 64 + lane;
            raw[u].template load<WIDE>(logits + static_cast<int64_t>(min(at[u], vectors - 1)) * V);
        }
        float v[kUnroll][V], most = none;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[u][j] = at[u] < vectors ? raw[u].get(j) : none;
                most = fmaxf(most, v[u][j]);
            }
        r.raise(fmaxf(r.m, most));
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) r.add(v[u][j]);
        if constexpr (TOP) {
            // (what a wave has seen has lower indices than what comes: an equal value does not come in)
            if (best.last == 0 || __builtin_amdgcn_ballot_w64(most > value_of(best.last))) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                    for (int j = 0; j < V; ++j) best.offer(at[u] < vectors ? entry_of(v[u][j], at[u] * V + j) : 0, p.top, lane);
            }
        }
    }
    if (segment == segments - 1 && wave == 0 && rest) {    // fewer than V values behind the last whole load
        const int i = vectors * V + lane;
        const float v = lane < rest ? static_cast<float>(logits[i]) : none;
        r.raise(fmaxf(r.m, v));
        r.add(v);
        if constexpr (TOP) best.offer(lane < rest ? entry_of(v, i) : 0, p.top, lane);
    }
    r = wave_stats(r);
    if (lane == 0) s_part[wave] = {r.m, r.s, r.t, 0.0f};
    if constexpr (TOP) s_best[wave][lane] = best.mine;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        r.join({s_part[w].m, s_part[w].s, s_part[w].t});
        if constexpr (TOP) best.mine = merge_waves(best.mine, s_best[w][lane], lane);
    }
    if (segments == 1) {
        answer(p, row, r, best.mine, lane);
        return;
    }
    Part* const parts = static_cast<Part*>(p.workspace);
    if (lane == 0) parts[blockIdx.x] = {r.m, r.s, r.t, 0.0f};
    if (TOP && lane < p.top) reinterpret_cast<Entry*>(parts + static_cast<int64_t>(p.rows) * segments)[static_cast<int64_t>(blockIdx.x) * p.top + lane] = best.mine;
}

// a row's segments, by one wave
__global__ __launch_bounds__(64) void token_logprobs_join_kernel(QaTokenLogprobsParams p, int segments) {
    static_assert(kMaxSegments <= 64, "a lane for each");
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const Part* const parts = static_cast<const Part*>(p.workspace);
    RowStats r;
    r.clear();
    if (lane < segments) {
        const Part part = parts[row * segments + lane];
        r = {part.m, part.s, part.t};
    }
    r = wave_stats(r);
    BestEntries best;
    best.clear();
    if (p.top) {
        const Entry* const from = reinterpret_cast<const Entry*>(parts + static_cast<int64_t>(p.rows) * segments) + row * segments * p.top;
        for (int i = 0; i < segments * p.top; i += 64) best.offer(i + lane < segments * p.top ? from[i + lane] : 0, p.top, lane);
    }
    answer(p, row, r, best.mine, lane);
}

int check(const QaTokenLogprobsParams& p) {
    if (p.rows < 0 || p.vocab < 1) return QA_ERR_SHAPE;
    if (!is_float_type(p.logits_type) || (p.token_bytes != 4 && p.token_bytes != 8)) return QA_ERR_UNSUPPORTED;
    if (p.top < 0 || p.top > kMaxTop) return QA_ERR_UNSUPPORTED;
    if (p.top > p.vocab) return QA_ERR_SHAPE;
    return QA_OK;
}

int64_t workspace_bytes(const QaTokenLogprobsParams& p) {
    const int segments = segments_of(p.rows, p.vocab, p.logits_type);
    return segments == 1 ? 0 : static_cast<int64_t>(p.rows) * segments * (static_cast<int64_t>(sizeof(Part)) + p.top * static_cast<int64_t>(sizeof(Entry)));
}

template <class T>
int launch(const QaTokenLogprobsParams& p, hipStream_t stream) {
    const int segments = segments_of(p.rows, p.vocab, p.logits_type);
    const int batches = (p.vocab + batch_values(p.logits_type) - 1) / batch_values(p.logits_type);
    const bool wide = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.row_stride * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p.rows) * segments)), block(64 * kWaves);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, segments, (batches + segments - 1) / segments); };
    if (wide) p.top ? go(token_logprobs_kernel<T, true, true>) : go(token_logprobs_kernel<T, true, false>);
    else p.top ? go(token_logprobs_kernel<T, false, true>) : go(token_logprobs_kernel<T, false, false>);
    if (segments > 1) {
        if (const int status = check_launch()) return status;
        hipLaunchKernelGGL(token_logprobs_join_kernel, dim3(p.rows), dim3(64), 0, stream, p, segments);
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
