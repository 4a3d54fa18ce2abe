// The residual sum with its norms: checks of the call, the shape of the launch, and fp32 rows (addnorm.hpp).
#include "addnorm.hpp"

namespace qa {
namespace lm {
namespace {

// rows, when there are any, of `type` on 16 bytes (8 for codes)
bool on_words(const void* base, int64_t row_stride, int type) {
    const int64_t bytes = bytes_of(type), unit = type == QA_LM_I8 ? 8 : 16;
    return !base || (reinterpret_cast<uintptr_t>(base) % unit == 0 && row_stride * bytes % unit == 0);
}
bool on_elements(const void* base, int type) { return reinterpret_cast<uintptr_t>(base) % bytes_of(type) == 0; }

}  // namespace
}  // namespace lm
}  // namespace qa

extern "C" int qa_lm_abi_version(void) { return QA_LM_ABI_VERSION; }

extern "C" int qa_add_rmsnorm(const QaAddNormParams* p, void* stream_) {
    using namespace qa;
    using namespace qa::lm;
    if (!p) return QA_ERR_NULL;
    if (p->rows < 0 || p->dim < 1) return QA_ERR_SHAPE;
    if (p->dim < 8 || p->dim > kAddNormDim) return QA_ERR_UNSUPPORTED;
    if (!is_float_type(p->x_type)) return QA_ERR_UNSUPPORTED;
    if ((p->param_type != p->x_type && p->param_type != QA_LM_F32) || (p->residual_type != p->x_type && p->residual_type != QA_LM_F32)) return QA_ERR_UNSUPPORTED;
    if (p->out_type != p->x_type && p->out_type != QA_LM_I8) return QA_ERR_UNSUPPORTED;
    if (p->gate_act < QA_GATE_PLAIN || p->gate_act > QA_GATE_SILU) return QA_ERR_UNSUPPORTED;
    if (p->rows == 0) return QA_OK;
    const bool dynamic = p->out_type == QA_LM_I8 && p->dynamic_scale;
    // (the reciprocal of a smaller scale is no number)
    if (p->out_type == QA_LM_I8 && !dynamic && !(p->out_scale >= 1.17549435e-38f && p->out_scale <= 3.402823466e38f)) return QA_ERR_UNSUPPORTED;
    if (!p->x || !p->weight || !p->out || (dynamic && !p->scales)) return QA_ERR_NULL;
    auto row_ok = [&](const void* base, int64_t stride, int type) { return !base || (on_elements(base, type) && (stride >= p->dim || p->rows == 1)); };
    if (!row_ok(p->x, p->x_row_stride, p->x_type) || !row_ok(p->residual, p->residual_row_stride, p->residual_type) ||
        !row_ok(p->residual_out, p->residual_out_row_stride, p->residual_type) || !row_ok(p->out, p->out_row_stride, p->out_type) ||
        (p->gate_row_stride != 0 && !row_ok(p->gate, p->gate_row_stride, p->x_type)) || !on_elements(p->gate, p->x_type) ||
        !on_elements(p->weight, p->param_type) || !on_elements(p->post_weight, p->param_type) || !on_elements(p->scale_vector, p->param_type) ||
        (dynamic && !aligned4(p->scales)))
        return QA_ERR_STRIDE;
    const bool wide = p->dim % 8 == 0 && on_words(p->x, p->x_row_stride, p->x_type) && on_words(p->gate, p->gate_row_stride, p->x_type) &&
                      on_words(p->residual, p->residual_row_stride, p->residual_type) && on_words(p->residual_out, p->residual_out_row_stride, p->residual_type) &&
                      on_words(p->out, p->out_row_stride, p->out_type) && on_words(p->weight, 0, p->param_type) &&
                      on_words(p->post_weight, 0, p->param_type) && on_words(p->scale_vector, 0, p->param_type);
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    const AddNormShape s = add_norm_shape(p->dim);
    if (p->x_type == QA_LM_F16) return add_rmsnorm_f16(*p, s, wide, stream);
    if (p->x_type == QA_LM_BF16) return add_rmsnorm_bf16(*p, s, wide, stream);
    return add_rmsnorm_launch<float, float, float>(*p, s, wide, stream);
}
