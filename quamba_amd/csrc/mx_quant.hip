// Rows in microscaled 4-bit floating point (qa_mxfp4_quant), and their values back (qa_mxfp4_dequant).
//
// Bound by memory: 16384 x 2560 bf16 are quantised in 20 us (5.3 TB/s) and given back in 24 (4.4, most of it written; 18 where the last-level cache holds it), 1021 x 10240
// fp32 in 8.6 and 11.  Four lanes have a block, eight values
// each: 16 bytes of 16-bit numbers a load.  A wave has a group of 512 values of a row, whose codes are 256 bytes and whose scales 16 in one piece; a workgroup has the same
// group of eight rows, whose scales are a line (by one row after the other 16384 x 2560 bf16 took 22.8 us).  A block's largest magnitude is taken on the bits of the
// absolute values, which rank as the numbers do, NaN above all.
#include "mx_common.hpp"

namespace qa {
namespace mx {
namespace {

constexpr int kThreads = 256, kRows = 2, kTogether = kThreads / 64 * kRows;

// Row and values of a lane's load r: a workgroup has a group of kTogether rows, whose scales lie next to each other, a wave kRows of them at the same time.
struct Place {
    int64_t row;
    int at;
    bool there;
};
__device__ __forceinline__ Place place_of(int r, int group, int64_t row0, int rows, int k, int lane) {
    const int64_t row = row0 + (threadIdx.x >> 6) * kRows + r;
    const int at = group * kGroup + lane * 8;
    return {row, at, row < rows && at < k};
}

template <class T, bool WIDE>
__global__ __launch_bounds__(kThreads) void mxfp4_quant_kernel(QaMxQuantParams p, int groups) {
    const int lane = threadIdx.x & 63, group = static_cast<int>(blockIdx.x % groups);
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / groups) * kTogether;
    Raw<T, 8> raw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const Place q = place_of(r, group, row0, p.rows, p.k, lane);
#pragma unroll
        for (int i = 0; i < Raw<T, 8>::kWords; ++i) raw[r].w[i] = v4w{0, 0, 0, 0};
        if (q.there) raw[r].template load<WIDE>(static_cast<const T*>(p.x) + q.row * p.x_row_stride + q.at);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const Place q = place_of(r, group, row0, p.rows, p.k, lane);
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(raw[r].get(j)) & 0x7fffffffu);
        const uint32_t scale = scale_of(most_of_block(most));
        const uint32_t codes = codes_of(scale, [&](int j) { return raw[r].get(j); });
        if (q.there) *reinterpret_cast<uint32_t*>(p.codes + q.row * p.code_row_stride + q.at / 2) = codes;
        // block 4 j + q of the group is byte 4 q + j
        const int block = lane >> 2;
        if ((lane & 3) == 0 && q.row < p.rows) p.scales[group * p.scale_group_stride + q.row * 16 + 4 * (block & 3) + (block >> 2)] = static_cast<uint8_t>(q.there ? scale : 0);
    }
}

// (A workgroup has four groups next to each other here.)
template <class T, bool WIDE>
__global__ __launch_bounds__(kThreads) void mxfp4_dequant_kernel(QaMxDequantParams p, uint32_t groups, uint32_t pieces) {
    const int lane = threadIdx.x & 63, block = lane >> 2;
    const uint32_t piece = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (piece >= pieces) return;
    const int64_t row = piece / groups;
    const int group = static_cast<int>(piece % groups), at = group * kGroup + lane * 8;
    if (at >= p.k) return;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(p.codes + row * p.code_row_stride + at / 2);
    const float s = power_of(p.scales[group * p.scale_group_stride + row * 16 + 4 * (block & 3) + (block >> 2)]);
    Raw<T, 8> raw;
    auto two = [&](int j, auto v) { raw.set2(j, v[0] * s, v[1] * s); };
    two(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0));
    two(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1));
    two(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2));
    two(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3));
    raw.template store<WIDE>(static_cast<T*>(p.out) + row * p.out_row_stride + at);
}

int64_t workgroups_of(int64_t rows, int64_t k) { return (rows + kTogether - 1) / kTogether * groups_of(k); }

// what both check of their rows: `numbers` of `type`, and an operand
int check_rows(int rows, int k, int type, const void* numbers, int64_t row_stride, const void* codes, const void* scales, int64_t code_stride, int64_t group_stride) {
    if (rows < 0 || k < 0) return QA_ERR_SHAPE;
    if (!is_float_type(type)) return QA_ERR_UNSUPPORTED;
    if (k % kBlock != 0) return QA_ERR_SHAPE;
    if (rows == 0 || k == 0) return QA_OK;
    if (!numbers || !codes || !scales) return QA_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(numbers) % bytes_of(type) != 0 || (rows > 1 && row_stride < k)) return QA_ERR_STRIDE;
    if (!aligned16(codes) || !aligned16(scales) || code_stride % 16 != 0 || group_stride % 16 != 0) return QA_ERR_STRIDE;
    if ((rows > 1 && code_stride < k / 2) || (k > kGroup && group_stride < 16LL * rows)) return QA_ERR_STRIDE;
    return launchable((rows * groups_of(k) + kThreads / 64 - 1) / (kThreads / 64), kThreads) ? QA_OK : QA_ERR_SHAPE;
}

// kernel of T and of rows that lie on 16 bytes or anywhere
template <class P, class Launch>
int by_type(const P& p, int type, const void* numbers, int64_t row_stride, Launch&& launch) {
    const bool wide = aligned16(numbers) && (p.rows == 1 || row_stride * bytes_of(type) % 16 == 0);
    auto of_type = [&](auto t) { wide ? launch(t, std::true_type{}) : launch(t, std::false_type{}); };
    if (type == QA_LM_F32) of_type(float{});
    else if (type == QA_LM_BF16) of_type(__bf16{});
    else of_type(_Float16{});
    return check_launch();
}

}  // namespace
}  // namespace mx
}  // namespace qa

extern "C" int qa_mx_abi_version(void) { return QA_MX_ABI_VERSION; }

extern "C" int qa_mxfp4_quant(const QaMxQuantParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::mx;
    if (!p) return QA_ERR_NULL;
    if (const int status = check_rows(p->rows, p->k, p->x_type, p->x, p->x_row_stride, p->codes, p->scales, p->code_row_stride, p->scale_group_stride)) return status;
    if (p->rows == 0 || p->k == 0) return QA_OK;
    const int groups = static_cast<int>(groups_of(p->k));
    const dim3 grid(static_cast<unsigned>(workgroups_of(p->rows, p->k)));
    return by_type(*p, p->x_type, p->x, p->x_row_stride, [&](auto t, auto wide) {
        hipLaunchKernelGGL((mxfp4_quant_kernel<decltype(t), decltype(wide)::value>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream_), *p, groups);
    });
}

extern "C" int qa_mxfp4_dequant(const QaMxDequantParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::mx;
    if (!p) return QA_ERR_NULL;
    if (const int status = check_rows(p->rows, p->k, p->out_type, p->out, p->out_row_stride, p->codes, p->scales, p->code_row_stride, p->scale_group_stride)) return status;
    if (p->rows == 0 || p->k == 0) return QA_OK;
    const uint32_t groups = static_cast<uint32_t>(groups_of(p->k)), pieces = p->rows * groups;         // (as many as check_rows lets through fit)
    const dim3 grid((pieces + kThreads / 64 - 1) / (kThreads / 64));
    return by_type(*p, p->out_type, p->out, p->out_row_stride, [&](auto t, auto wide) {
        hipLaunchKernelGGL((mxfp4_dequant_kernel<decltype(t), decltype(wide)::value>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream_), *p, groups, pieces);
    });
}
