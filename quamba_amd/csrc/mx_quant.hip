// Rows in microscaled 4-bit floating point (qa_mxfp4_quant), and their values back (qa_mxfp4_dequant).
//
// Bound by memory.  Four lanes have a block, eight values each: 16 bytes of 16-bit numbers a load.  A wave has a group of 512 values of a row, whose codes are
// 256 bytes and whose scales 16 in one piece.  A block's largest magnitude is taken on the bits of the absolute values, which rank as the numbers
// do, NaN above all.
#include "mx_common.hpp"

namespace qa {
namespace mx {
namespace {

constexpr int kThreads = 256;

// the largest of the four lanes of a block, in all of them
__device__ __forceinline__ uint32_t most_of_block(uint32_t v) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xb1, 0xf, 0xf, true)));
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4e, 0xf, 0xf, true)));
}

template <class T, bool WIDE>
__global__ __launch_bounds__(kThreads) void mxfp4_quant_kernel(QaMxQuantParams p, int groups, int64_t pieces) {
    const int lane = threadIdx.x & 63;
    const int64_t piece = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    if (piece >= pieces) return;
    const int64_t row = piece / groups;
    const int group = static_cast<int>(piece - row * groups), at = group * kGroup + lane * 8;
    const bool there = at < p.k;
    Raw<T, 8> raw;
#pragma unroll
    for (int i = 0; i < Raw<T, 8>::kWords; ++i) raw.w[i] = v4w{0, 0, 0, 0};
    if (there) raw.template load<WIDE>(static_cast<const T*>(p.x) + row * p.x_row_stride + at);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(raw.get(j)) & 0x7fffffffu);
    const uint32_t scale = scale_of(most_of_block(most));
    const uint32_t codes = codes_of(scale, [&](int j) { return raw.get(j); });
    if (there) *reinterpret_cast<uint32_t*>(p.codes + row * p.code_row_stride + at / 2) = codes;
    // block 4 j + q of the group is byte 4 q + j
    const int block = lane >> 2;
    if ((lane & 3) == 0) p.scales[group * p.scale_group_stride + row * 16 + 4 * (block & 3) + (block >> 2)] = static_cast<uint8_t>(there ? scale : 0);
}

template <class T, bool WIDE>
__global__ __launch_bounds__(kThreads) void mxfp4_dequant_kernel(QaMxDequantParams p, int groups, int64_t pieces) {
    const int lane = threadIdx.x & 63;
    const int64_t piece = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    if (piece >= pieces) return;
    const int64_t row = piece / groups;
    const int group = static_cast<int>(piece - row * groups), at = group * kGroup + lane * 8, block = lane >> 2;
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
    const int64_t pieces = static_cast<int64_t>(p->rows) * groups;
    const dim3 grid(static_cast<unsigned>((pieces + kThreads / 64 - 1) / (kThreads / 64)));
    return by_type(*p, p->x_type, p->x, p->x_row_stride, [&](auto t, auto wide) {
        hipLaunchKernelGGL((mxfp4_quant_kernel<decltype(t), decltype(wide)::value>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream_), *p, groups, pieces);
    });
}

extern "C" int qa_mxfp4_dequant(const QaMxDequantParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::mx;
    if (!p) return QA_ERR_NULL;
    if (const int status = check_rows(p->rows, p->k, p->out_type, p->out, p->out_row_stride, p->codes, p->scales, p->code_row_stride, p->scale_group_stride)) return status;
    if (p->rows == 0 || p->k == 0) return QA_OK;
    const int groups = static_cast<int>(groups_of(p->k));
    const int64_t pieces = static_cast<int64_t>(p->rows) * groups;
    const dim3 grid(static_cast<unsigned>((pieces + kThreads / 64 - 1) / (kThreads / 64)));
    return by_type(*p, p->out_type, p->out, p->out_row_stride, [&](auto t, auto wide) {
        hipLaunchKernelGGL((mxfp4_dequant_kernel<decltype(t), decltype(wide)::value>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream_), *p, groups, pieces);
    });
}
