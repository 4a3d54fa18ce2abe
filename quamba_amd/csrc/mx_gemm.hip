// Product of two microscaled 4-bit operands (qa_mxfp4_mm): what it refuses, and which kernel takes it.
#include "mx_gemm.hpp"

namespace qa {
namespace mx {
namespace {

constexpr int64_t kMaxPitch = 1 << 22;     // bytes of an operand's row: those of a tile in 32 bits
constexpr int kMaxRows = 0x7fffffff - 255; // rows and columns: whole tiles of them in 32 bits

// (the workspace does not go by the output's type)
int check_rows(const QaMxGemmParams& p) {
    if (p.m < 0 || p.n < 0 || p.k < 0) return QA_ERR_SHAPE;
    if (p.a_type != QA_LM_I8 && !is_float_type(p.a_type)) return QA_ERR_UNSUPPORTED;
    if (p.k % kBlock != 0 || p.k / 2 > kMaxPitch || p.m > kMaxRows || p.n > kMaxRows) return QA_ERR_SHAPE;
    return QA_OK;
}
int check(const QaMxGemmParams& p) {
    const int status = check_rows(p);
    return status == QA_OK && !is_float_type(p.out_type) ? QA_ERR_UNSUPPORTED : status;
}
bool fused(const QaMxGemmParams& p) { return p.a_type != QA_LM_I8 && direct_takes_numbers(p); }
int64_t code_bytes(const QaMxGemmParams& p) { return static_cast<int64_t>(p.m) * ((p.k / 2 + 15) / 16 * 16); }

int64_t workspace_bytes(const QaMxGemmParams& p, bool one_launch) { return p.a_type == QA_LM_I8 || one_launch ? 0 : code_bytes(p) + groups_of(p.k) * 16 * p.m; }

}  // namespace
}  // namespace mx
}  // namespace qa

extern "C" int64_t qa_mxfp4_mm_workspace_bytes(const QaMxGemmParams* p) {
    using namespace qa::mx;
    return p && check_rows(*p) == QA_OK && p->m > 0 && p->n > 0 && p->k > 0 ? workspace_bytes(*p, fused(*p)) : 0;
}

extern "C" int qa_mxfp4_mm(const QaMxGemmParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::mx;
    if (!p) return QA_ERR_NULL;
    if (const int status = check(*p)) return status;
    if (p->m == 0 || p->n == 0) return QA_OK;
    if (!p->d) return QA_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(p->d) % bytes_of(p->out_type) != 0 || (p->m > 1 && p->ldd < p->n)) return QA_ERR_STRIDE;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (p->k == 0) {
        // (a sum over nothing)
        const int64_t row = static_cast<int64_t>(p->n) * bytes_of(p->out_type);
        if (p->m > 1 && p->ldd != p->n) return QA_ERR_STRIDE;
        return fill_zero(p->d, row * p->m, stream);
    }
    if (!p->a || !p->w || !p->w_scales || (p->a_type == QA_LM_I8 && !p->a_scales)) return QA_ERR_NULL;
    const int64_t codes = p->k / 2;
    const bool rows_of_codes = p->a_type == QA_LM_I8;
    if (p->ldw % 16 != 0 || (p->n > 1 && p->ldw < codes) || !aligned16(p->w) || !aligned16(p->w_scales) || p->w_scale_group_stride % 16 != 0) return QA_ERR_STRIDE;
    if (p->k > kGroup && p->w_scale_group_stride < 16LL * p->n) return QA_ERR_STRIDE;
    if (rows_of_codes) {
        if (p->lda % 16 != 0 || (p->m > 1 && p->lda < codes) || !aligned16(p->a) || !aligned16(p->a_scales) || p->a_scale_group_stride % 16 != 0) return QA_ERR_STRIDE;
        if (p->k > kGroup && p->a_scale_group_stride < 16LL * p->m) return QA_ERR_STRIDE;
        if (p->m > 1 && p->lda > kMaxPitch) return QA_ERR_SHAPE;
    } else if (reinterpret_cast<uintptr_t>(p->a) % bytes_of(p->a_type) != 0 || (p->m > 1 && p->lda < p->k)) {
        return QA_ERR_STRIDE;
    }
    if (p->n > 1 && p->ldw > kMaxPitch) return QA_ERR_SHAPE;
    const bool one_launch = fused(*p);
    const int64_t need = workspace_bytes(*p, one_launch);
    if (need && !p->workspace) return QA_ERR_NULL;
    if (need && (!aligned16(p->workspace) || p->workspace_bytes < need)) return QA_ERR_SCRATCH;
    auto of_codes = [&](const QaMxGemmParams& q) { return direct_takes(q) ? direct_launch(q, stream) : tiles_launch(q, stream); };
    if (one_launch) return direct_launch(*p, stream);
    if (rows_of_codes) return of_codes(*p);
    // many rows of numbers: quantised once, for all columns
    QaMxQuantParams rows = {};
    rows.rows = p->m; rows.k = p->k; rows.x_type = p->a_type;
    rows.x_row_stride = p->lda; rows.code_row_stride = (codes + 15) / 16 * 16; rows.scale_group_stride = 16LL * p->m;
    rows.x = p->a;
    rows.codes = static_cast<uint8_t*>(p->workspace);
    rows.scales = rows.codes + code_bytes(*p);
    if (const int status = qa_mxfp4_quant(&rows, stream_)) return status;
    QaMxGemmParams product = *p;
    product.a_type = QA_LM_I8;
    product.a = rows.codes; product.lda = rows.code_row_stride;
    product.a_scales = rows.scales; product.a_scale_group_stride = rows.scale_group_stride;
    return of_codes(product);
}
