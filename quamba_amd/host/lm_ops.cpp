// The host side of the operators around the mixers: quamba_amd._lm_host.
//
// A decoding step calls them on a few rows, where the kernels take 3-5 us and the checks, allocations and parameter blocks
// 20-25 us in Python.  Each function here checks its arguments, allocates outputs and workspace, fills the block of
// include/quamba_amd_lm.h and enqueues the call on the current stream of its tensors' device.  It raises RuntimeError for arguments that
// do not fit, NotImplementedError for what the library has no kernel for.
#include "host_common.hpp"

#include "../../include/quamba_amd_lm.h"

namespace {

// What bind() was given: the library's functions.
struct Bound {
    int (*add_rmsnorm)(const QaAddNormParams*, void*) = nullptr;
    int64_t (*token_logprobs_bytes)(const QaTokenLogprobsParams*) = nullptr;
    int (*token_logprobs)(const QaTokenLogprobsParams*, void*) = nullptr;
    int64_t (*mm_token_logprobs_bytes)(const QaMmTokenLogprobsParams*) = nullptr;
    int (*mm_token_logprobs)(const QaMmTokenLogprobsParams*, void*) = nullptr;
} g;

// add_rmsnorm(x, weight, eps, residual, post_weight, gate, gate_act, residual_scale, prenorm, residual_dtype, residual_out,
// out_dtype, out_scale) -> (y, v or None, scales or None)
PyObject* add_rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 13) {
        PyErr_SetString(PyExc_TypeError, "add_rmsnorm takes 13 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "x");
        const at::Tensor& weight = tensor(a[1], "weight");
        const at::Tensor* residual = tensor_or_none(a[3], "residual");
        const at::Tensor* post = tensor_or_none(a[4], "post_weight");
        const at::Tensor* gate = tensor_or_none(a[5], "gate");
        const at::Tensor* vector = THPVariable_Check(a[7]) ? &THPVariable_Unpack(a[7]) : nullptr;
        const int prenorm = PyObject_IsTrue(a[8]);
        if (prenorm < 0) throw Raised{};
        const at::Tensor* given = tensor_or_none(a[10], "residual_out");
        require(x.dim() == 2, "x must be (rows, dim)");
        on_gpu(x, "x");
        const auto type = x.scalar_type();
        require(is_float(type), "x must be fp16, bf16 or fp32");
        in_rows(x, "x");
        const int64_t rows = x.size(0), dim = x.size(1);
        const at::Device device = x.device();
        supported(dim >= 8 && dim <= 32768, "add_rmsnorm: rows of 8 to 32768 values");
        require(rows <= std::numeric_limits<int32_t>::max(), "add_rmsnorm: too many rows");
        auto half = [&](at::ScalarType t) { return t == type || t == at::kFloat; };
        auto check = [&](const at::Tensor* t, const char* name, at::IntArrayRef shape) {
            if (!t) return;
            beside(*t, name, device);
            shaped(*t, name, shape);
            in_rows(*t, name);
        };
        check(&weight, "weight", {dim});
        require(half(weight.scalar_type()), "weight must be of the type of x or fp32");
        check(post, "post_weight", {dim});
        check(vector, "residual_scale, if not a number,", {dim});
        require((!post || post->scalar_type() == weight.scalar_type()) && (!vector || vector->scalar_type() == weight.scalar_type()),
                "post_weight and residual_scale must be of the type of weight");
        check(residual, "residual", {rows, dim});
        require(!residual || half(residual->scalar_type()), "residual must be of the type of x or fp32");
        int64_t gate_stride = 0;                                   // (one row for all)
        if (gate) {
            require(gate->scalar_type() == type, "gate must be of the type of x");
            if (gate->dim() == 2 && gate->size(1) == dim && (gate->size(0) == 1 || (gate->size(0) == rows && gate->stride(0) == 0))) {
                beside(*gate, "gate", device);
                require(gate->stride(1) == 1, "gate must be contiguous along the last dimension");
            } else if (gate->dim() == 2) {
                check(gate, "gate", {rows, dim});
                gate_stride = row_stride(*gate);
            } else {
                check(gate, "gate, if not (rows, dim),", {dim});
            }
        }
        int act = -1;
        if (PyUnicode_Check(a[6]))
            act = PyUnicode_CompareWithASCIIString(a[6], "none") == 0 ? QA_GATE_PLAIN : PyUnicode_CompareWithASCIIString(a[6], "sigmoid") == 0 ? QA_GATE_SIGMOID
                  : PyUnicode_CompareWithASCIIString(a[6], "silu") == 0 ? QA_GATE_SILU : -1;
        supported(act >= 0, "gate_act must be none, sigmoid or silu");
        const auto out_type = dtype_or_none(a[11], "out_dtype").value_or(type);
        supported(out_type == type || out_type == at::kChar, "out_dtype must be that of x or int8");
        const bool fixed = a[12] != Py_None;
        const double out_scale = fixed ? number(a[12]) : 0.0;
        require(!fixed || out_type == at::kChar, "out_scale is for int8 output");
        require(!fixed || (static_cast<float>(out_scale) >= std::numeric_limits<float>::min() && static_cast<float>(out_scale) <= std::numeric_limits<float>::max()),
                "out_scale must be positive and no smaller than fp32's normal numbers");
        const bool dynamic = out_type == at::kChar && !fixed;
        const auto asked = dtype_or_none(a[9], "residual_dtype");
        require(!residual || !asked || *asked == residual->scalar_type(), "residual_dtype differs from the type of residual");
        const auto stream_type = residual ? residual->scalar_type() : asked.value_or(type);
        supported(half(stream_type), "the stream is of the type of x or fp32");
        require(prenorm || !given, "residual_out without prenorm");

        QaAddNormParams p = {};
        if (given) {
            check(given, "residual_out", {rows, dim});
            require(given->scalar_type() == stream_type, "residual_out must be of the type of the stream");
            // the memory between the first and the last element of each
            auto span = [](const at::Tensor& t) {
                const char* first = static_cast<const char*>(t.const_data_ptr());
                const int64_t last = t.dim() == 2 ? (t.size(0) - 1) * t.stride(0) + t.size(1) : t.size(0);
                return std::make_pair(first, first + last * t.element_size());
            };
            auto apart = [&](const at::Tensor* t, const char* name) {
                if (!t || rows == 0) return;
                if (t == residual && t->const_data_ptr() == given->const_data_ptr() && (rows == 1 || t->stride(0) == given->stride(0))) return;
                const auto [f, l] = span(*t);
                const auto [of, ol] = span(*given);
                if (l <= of || ol <= f) return;
                // rows (or one) between the rows of `given`: in its pitch, behind the columns of one and in front of the next one's
                const bool one = t->dim() == 1 || t->size(0) == 1 || t->stride(0) == 0;
                bool between = rows > 1 && (one || t->stride(0) * t->element_size() == given->stride(0) * given->element_size());
                if (between) {
                    const int64_t pitch = given->stride(0) * given->element_size(), behind = ((f - of) % pitch + pitch) % pitch;
                    between = behind >= dim * given->element_size() && behind + dim * t->element_size() <= pitch;
                }
                require(between, std::string("residual_out overlaps ") + name);
            };
            apart(&x, "x"); apart(&weight, "weight"); apart(residual, "residual"); apart(post, "post_weight"); apart(gate, "gate"); apart(vector, "residual_scale");
        }
        p.rows = static_cast<int32_t>(rows);
        p.dim = static_cast<int32_t>(dim);
        p.x_type = lm_type(type);
        p.param_type = lm_type(weight.scalar_type());
        p.residual_type = lm_type(stream_type);
        p.out_type = lm_type(out_type);
        p.gate_act = act;
        p.dynamic_scale = dynamic;
        p.eps = static_cast<float>(number(a[2]));
        p.scale = vector ? 1.0f : static_cast<float>(number(a[7]));
        p.out_scale = static_cast<float>(out_scale);
        const OnDevice on(device);
        const auto opts = at::TensorOptions().device(device);
        const at::Tensor y = at::empty({rows, dim}, opts.dtype(out_type));
        const at::Tensor v = given ? *given : prenorm ? at::empty({rows, dim}, opts.dtype(stream_type)) : at::Tensor();
        const at::Tensor scales = dynamic ? at::empty({rows}, opts.dtype(at::kFloat)) : at::Tensor();
        p.x_row_stride = row_stride(x);
        p.gate_row_stride = gate_stride;
        p.residual_row_stride = residual ? row_stride(*residual) : 0;
        p.residual_out_row_stride = v.defined() ? row_stride(v) : 0;
        p.out_row_stride = dim;
        p.x = x.const_data_ptr();
        p.weight = weight.const_data_ptr();
        p.post_weight = address(post);
        p.gate = address(gate);
        p.scale_vector = address(vector);
        p.residual = address(residual);
        p.residual_out = v.defined() ? v.data_ptr() : nullptr;
        p.out = y.data_ptr();
        p.scales = dynamic ? scales.data_ptr<float>() : nullptr;
        enqueue(g.add_rmsnorm, p, device, "add_rmsnorm");
        if (given && !given->is_inference()) given->unsafeGetTensorImpl()->bump_version();      // (as torch's own writes in place do)
        return Py_BuildValue("(NNN)", wrapped(y), given ? Py_NewRef(a[10]) : wrapped_or_none(v), wrapped_or_none(scales));
    });
}

constexpr int64_t kTogether = 1024;        // fp32 answers of one allocation, at most

// Tokens, answers and workspace of both operators, the call, and the answers as a tuple.
template <class Params>
PyObject* answer(Params& p, const at::Tensor& tokens_as_given, at::IntArrayRef shape, int64_t top, at::Device device, int64_t (*bytes)(const Params*),
                 int (*call)(const Params*, void*), const char* what) {
    beside(tokens_as_given, "tokens", device);
    require(tokens_as_given.scalar_type() == at::kInt || tokens_as_given.scalar_type() == at::kLong, "tokens must be int32 or int64");
    shaped(tokens_as_given, "tokens", shape);
    const OnDevice on(device);
    const at::Tensor tokens = tokens_as_given.is_contiguous() ? tokens_as_given : tokens_as_given.contiguous();
    const auto opts = at::TensorOptions().device(device);
    at::DimVector best(shape.begin(), shape.end());
    best.push_back(top);
    const at::Tensor top_tokens = at::empty(best, opts.dtype(at::kLong));
    // (A call on few rows takes the GPU 8 us and the host as long: there the three fp32 answers are one allocation, each on 16 bytes, and made without
    // torch's dispatch.  Above kTogether values who keeps one of them would keep the others' memory, and the time does not show.)
    const int64_t count = c10::multiply_integers(shape), places = (count + 3) / 4 * 4;
    const bool together = 2 * places + count * top <= kTogether;
    const at::Tensor memory = together ? at::empty({2 * places + count * top}, opts.dtype(at::kFloat)) : at::Tensor();
    int64_t used = 0;
    auto part = [&](at::IntArrayRef sizes) {
        if (!together) return at::empty(sizes, opts.dtype(at::kFloat));
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(memory.storage()), memory.key_set(), memory.dtype());
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        t.unsafeGetTensorImpl()->set_storage_offset(used);
        used += places;
        return t;
    };
    const at::Tensor logprobs = part(shape), entropy = part(shape), top_logprobs = part(best);
    p.top = static_cast<int32_t>(top);
    p.token_bytes = static_cast<int32_t>(tokens.element_size());
    p.tokens = tokens.const_data_ptr();
    p.logprobs = logprobs.data_ptr<float>();
    p.entropy = entropy.data_ptr<float>();
    p.top_logprobs = top_logprobs.data_ptr<float>();
    p.top_tokens = top_tokens.data_ptr<int64_t>();
    p.workspace_bytes = bytes(&p);
    const at::Tensor workspace = p.workspace_bytes ? at::empty({p.workspace_bytes}, opts.dtype(at::kByte)) : at::Tensor();
    p.workspace = p.workspace_bytes ? workspace.data_ptr() : nullptr;
    enqueue(call, p, device, what);
    return Py_BuildValue("(NNNN)", wrapped(logprobs), wrapped(entropy), wrapped(top_logprobs), wrapped(top_tokens));
}

// token_logprobs(logits, tokens, top) -> (logprobs, entropy, top_logprobs, top_tokens)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "token_logprobs takes 3 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor& logits = tensor(a[0], "logits");
        const at::Tensor& tokens = tensor(a[1], "tokens");
        const int64_t top = whole(a[2]);
        require(logits.dim() >= 1, "logits must be (..., vocab)");
        on_gpu(logits, "logits");
        require(is_float(logits.scalar_type()), "logits must be fp16, bf16 or fp32");
        const int64_t vocab = logits.size(-1);
        require(vocab >= 1, "logits without a vocabulary");
        require(top >= 0 && top <= vocab, "top must be between 0 and the vocabulary's size");
        supported(top <= 64, "token_logprobs: top up to 64");
        const auto shape = logits.sizes().slice(0, logits.dim() - 1);
        const int64_t rows = c10::multiply_integers(shape);
        require(rows <= std::numeric_limits<int32_t>::max() && vocab <= std::numeric_limits<int32_t>::max(), "token_logprobs: too many rows or too large a vocabulary");
        // (dimensions in front are rows where they lie evenly apart; else this is a copy)
        at::Tensor copy;
        if (logits.dim() != 2) {
            const OnDevice on(logits.device());
            copy = logits.reshape({rows, vocab});
        }
        const at::Tensor& flat = logits.dim() == 2 ? logits : copy;
        in_rows(flat, "logits");
        QaTokenLogprobsParams p = {};
        p.rows = static_cast<int32_t>(rows);
        p.vocab = static_cast<int32_t>(vocab);
        p.logits_type = lm_type(logits.scalar_type());
        p.row_stride = row_stride(flat);
        p.logits = flat.const_data_ptr();
        return answer(p, tokens, shape, top, logits.device(), g.token_logprobs_bytes, g.token_logprobs, "token_logprobs");
    });
}

// scaled_mm_token_logprobs(a, b, a_scales, b_scales, tokens, top, vocab) -> (logprobs, entropy, top_logprobs, top_tokens)
PyObject* scaled_mm_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "scaled_mm_token_logprobs takes 7 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor &a = tensor(args[0], "a"), &b = tensor(args[1], "b"), &a_scales = tensor(args[2], "a_scales"), &b_scales = tensor(args[3], "b_scales");
        const at::Tensor& tokens = tensor(args[4], "tokens");
        const int64_t top = whole(args[5]);
        require(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar, "a and b must be int8");
        require(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0), "shape mismatch: a (M,K) x b (K,N)");
        on_gpu(a, "a");
        const at::Device device = a.device();
        beside(b, "b", device);
        const int64_t M = a.size(0), K = a.size(1), N = b.size(1), vocab = args[6] == Py_None ? N : whole(args[6]);
        require(vocab >= 1 && vocab <= N, "vocab must be between 1 and the columns of b");
        require(K >= 1 && K % 16 == 0 && K <= 131056, "K must be a multiple of 16 up to 131056");
        require(a.stride(1) == 1 && b.stride(0) == 1, "a must be row-major and b column-major");
        const int64_t lda = M > 1 ? a.stride(0) : K, ldw = N > 1 ? b.stride(1) : K;
        require(lda % 16 == 0 && ldw % 16 == 0, "row strides of a and b must be multiples of 16");
        require(std::max({M, N, K}) <= std::numeric_limits<int32_t>::max(), "scaled_mm_token_logprobs: a size beyond 32 bits");
        auto scales = [&](const at::Tensor& t, const char* name, int64_t full) {
            beside(t, name, device);
            require(t.scalar_type() == at::kFloat && t.is_contiguous(), std::string(name) + " must be contiguous fp32");
            require(t.numel() == 1 || t.numel() == full, std::string(name) + " must have 1 or " + std::to_string(full) + " elements");
        };
        scales(a_scales, "a_scales", M);
        scales(b_scales, "b_scales", N);
        supported(top == 0 || top == 1, "scaled_mm_token_logprobs: top is 0 or 1 (more: token_logprobs of the written logits)");
        QaMmTokenLogprobsParams p = {};
        p.rows = static_cast<int32_t>(M);
        p.vocab = static_cast<int32_t>(vocab);
        p.k = static_cast<int32_t>(K);
        p.a_scale_numel = static_cast<int32_t>(a_scales.numel());
        p.w_scale_numel = static_cast<int32_t>(b_scales.numel());
        p.lda = lda;
        p.ldw = ldw;
        p.a = a.const_data_ptr<int8_t>();
        p.w = b.const_data_ptr<int8_t>();
        p.a_scale = a_scales.const_data_ptr<float>();
        p.w_scale = b_scales.const_data_ptr<float>();
        return answer(p, tokens, {M}, top, device, g.mm_token_logprobs_bytes, g.mm_token_logprobs, "scaled_mm_token_logprobs");
    });
}

// bind(addresses of the library's functions in the order of Bound, (get_device, set_device, get_stream, out-of-memory error, check))
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long f[5];
    PyObject* py[5];
    if (!PyArg_ParseTuple(args, "(KKKKK)(OOOOO)", &f[0], &f[1], &f[2], &f[3], &f[4], &py[0], &py[1], &py[2], &py[3], &py[4])) return nullptr;
    g.add_rmsnorm = reinterpret_cast<decltype(g.add_rmsnorm)>(f[0]);
    g.token_logprobs_bytes = reinterpret_cast<decltype(g.token_logprobs_bytes)>(f[1]);
    g.token_logprobs = reinterpret_cast<decltype(g.token_logprobs)>(f[2]);
    g.mm_token_logprobs_bytes = reinterpret_cast<decltype(g.mm_token_logprobs_bytes)>(f[3]);
    g.mm_token_logprobs = reinterpret_cast<decltype(g.mm_token_logprobs)>(f[4]);
    torch_side.keep(py);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* bound_only(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    if (g.add_rmsnorm) return F(self, args, n);
    PyErr_SetString(PyExc_RuntimeError, "quamba_amd._lm_host: bind() first");
    return nullptr;
}
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bound_only<F>)); }

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "Takes the library's functions."},
                         {"add_rmsnorm", fast<add_rmsnorm>(), METH_FASTCALL, "ops.add_rmsnorm"},
                         {"token_logprobs", fast<token_logprobs>(), METH_FASTCALL, "ops.token_logprobs"},
                         {"scaled_mm_token_logprobs", fast<scaled_mm_token_logprobs>(), METH_FASTCALL, "ops.scaled_mm_token_logprobs"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_lm_host", "Host side of the operators around the mixers.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__lm_host() {
    PyObject* m = PyModule_Create(&module_def);
    if (m && PyModule_AddIntConstant(m, "LM_ABI_VERSION", QA_LM_ABI_VERSION) < 0) Py_CLEAR(m);
    return m;
}
