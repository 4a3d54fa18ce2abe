// The host side of the microscaled 4-bit operators and of beam search: quamba_amd._mx_beam_host.
//
// As the operators around the mixers: each function checks its arguments, allocates outputs and workspace, fills the block of include/quamba_amd_mx.h or
// include/quamba_amd_beam.h and enqueues the call on the current stream of its tensors' device.
#include "host_common.hpp"

#include <vector>

#include "../../include/quamba_amd_beam.h"
#include "../../include/quamba_amd_mx.h"

namespace {

// What bind() was given: the library's functions.
struct Bound {
    int (*quant)(const QaMxQuantParams*, void*) = nullptr;
    int (*dequant)(const QaMxDequantParams*, void*) = nullptr;
    int64_t (*mm_bytes)(const QaMxGemmParams*) = nullptr;
    int (*mm)(const QaMxGemmParams*, void*) = nullptr;
    int64_t (*beam_bytes)(const QaBeamSearchParams*) = nullptr;
    int (*beam)(const QaBeamSearchParams*, void*) = nullptr;
    int (*reorder)(const QaReorderParams*, void*) = nullptr;
} g;

constexpr int64_t kBlock = 32, kGroup = 512, kMost = std::numeric_limits<int32_t>::max();

int64_t groups_of(int64_t k) { return (k + kGroup - 1) / kGroup; }

// (..., k) as rows, a copy where the dimensions in front do not lie evenly apart
at::Tensor as_rows(const at::Tensor& t, int64_t width) {
    if (t.dim() == 2) return t;
    const OnDevice on(t.device());
    return t.reshape({width ? t.numel() / width : c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)), width});
}
at::DimVector with_last(at::IntArrayRef shape, int64_t last) {
    at::DimVector d(shape.begin(), shape.end());
    d.back() = last;
    return d;
}

// Answers of one allocation, each on 16 bytes and made without torch's dispatch (a call on little takes the host as long as the GPU, and an allocation 1.2 us).  For
// answers of kTogether bytes in all: of larger ones who keeps one would keep the others' memory, and the time does not show.
constexpr int64_t kTogether = 8192;
class Together {
  public:
    Together(int64_t bytes, at::Device device) : memory_(at::empty({bytes}, at::TensorOptions().device(device).dtype(at::kByte))) {}
    static int64_t place(int64_t bytes) { return (bytes + 15) / 16 * 16; }
    at::Tensor next(at::IntArrayRef sizes, at::ScalarType type) {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(memory_.storage()), memory_.key_set(), c10::scalarTypeToTypeMeta(type));
        const int64_t each = static_cast<int64_t>(c10::elementSize(type));
        t.unsafeGetTensorImpl()->set_storage_offset(used_ / each);
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        used_ += place(t.numel() * each);
        return t;
    }

  private:
    at::Tensor memory_;
    int64_t used_ = 0;
};

// an operand's codes (rows, k / 2) and scales (groups, rows, 16)
struct Operand {
    int64_t rows, k, pitch, group_stride;
    const uint8_t *codes, *scales;
};
Operand operand(const at::Tensor& codes, const at::Tensor& scales, const char* name, const char* of_scales, at::Device device) {
    beside(codes, name, device);
    beside(scales, of_scales, device);
    require(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, name, " and ", of_scales, " must be uint8");
    require(codes.dim() == 2 && codes.size(1) % 16 == 0, name, " must be (rows, K / 2), K a multiple of 32");
    in_rows(codes, name);
    Operand o = {codes.size(0), 2 * codes.size(1), row_stride(codes), 0, codes.const_data_ptr<uint8_t>(), scales.const_data_ptr<uint8_t>()};
    require(std::max(o.rows, o.k) <= kMost, name, ": a size beyond 32 bits");
    shaped(scales, of_scales, {groups_of(o.k), o.rows, 16});
    o.group_stride = scales.size(0) > 1 ? scales.stride(0) : 16 * o.rows;
    require(scales.numel() == 0 || (scales.stride(2) == 1 && (o.rows == 1 || scales.stride(1) == 16) && o.group_stride >= 16 * o.rows && o.group_stride % 16 == 0),
            of_scales, " must lie as mxfp4_quant gives them: 16 bytes a row, rows next to each other");
    auto whole = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    require(codes.numel() == 0 || (whole(o.codes) && whole(o.scales) && o.pitch % 16 == 0), name, " and ", of_scales, ": rows on 16 bytes");
    return o;
}

// mxfp4_quant(x) -> (codes, scales)
PyObject* mxfp4_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 1) {
        PyErr_SetString(PyExc_TypeError, "mxfp4_quant takes 1 argument");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "x");
        require(x.dim() >= 1, "x must be (..., K)");
        on_gpu(x, "x");
        require(is_float(x.scalar_type()), "x must be fp16, bf16 or fp32");
        const int64_t k = x.size(-1);
        require(k % kBlock == 0, "K must be a multiple of 32");
        const at::Tensor flat = as_rows(x, k);
        in_rows(flat, "x");
        require(flat.size(0) <= kMost && k <= kMost, "mxfp4_quant: a size beyond 32 bits");
        const OnDevice on(x.device());
        at::Tensor codes, scales;
        const int64_t code_bytes = flat.size(0) * (k / 2), scale_bytes = groups_of(k) * flat.size(0) * 16;
        if (code_bytes + scale_bytes <= kTogether) {
            Together all(Together::place(code_bytes) + scale_bytes, x.device());
            codes = all.next(with_last(x.sizes(), k / 2), at::kByte);
            scales = all.next({groups_of(k), flat.size(0), 16}, at::kByte);
        } else {
            const auto opts = at::TensorOptions().device(x.device()).dtype(at::kByte);
            codes = at::empty(with_last(x.sizes(), k / 2), opts);
            scales = at::empty({groups_of(k), flat.size(0), 16}, opts);
        }
        QaMxQuantParams p = {};
        p.rows = static_cast<int32_t>(flat.size(0));
        p.k = static_cast<int32_t>(k);
        p.x_type = lm_type(x.scalar_type());
        p.x_row_stride = row_stride(flat);
        p.code_row_stride = k / 2;
        p.scale_group_stride = 16 * flat.size(0);
        p.x = flat.const_data_ptr();
        p.codes = codes.data_ptr<uint8_t>();
        p.scales = scales.data_ptr<uint8_t>();
        enqueue(g.quant, p, x.device(), "mxfp4_quant");
        return Py_BuildValue("(NN)", wrapped(codes), wrapped(scales));
    });
}

// mxfp4_dequant(codes, scales, dtype) -> values
PyObject* mxfp4_dequant(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "mxfp4_dequant takes 3 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor &codes = tensor(a[0], "codes"), &scales = tensor(a[1], "scales");
        const auto type = dtype_or_none(a[2], "dtype").value_or(at::kFloat);
        supported(is_float(type), "dtype must be fp16, bf16 or fp32");
        require(codes.dim() >= 1, "codes must be (..., K / 2)");
        on_gpu(codes, "codes");
        const at::Tensor flat = as_rows(codes, codes.size(-1));
        const Operand o = operand(flat, scales, "codes", "scales", codes.device());
        const OnDevice on(codes.device());
        const at::Tensor out = at::empty(with_last(codes.sizes(), o.k), at::TensorOptions().device(codes.device()).dtype(type));
        QaMxDequantParams p = {};
        p.rows = static_cast<int32_t>(o.rows);
        p.k = static_cast<int32_t>(o.k);
        p.out_type = lm_type(type);
        p.out_row_stride = o.k;
        p.code_row_stride = o.pitch;
        p.scale_group_stride = o.group_stride;
        p.codes = o.codes;
        p.scales = o.scales;
        p.out = out.data_ptr();
        enqueue(g.dequant, p, codes.device(), "mxfp4_dequant");
        return wrapped(out);
    });
}

// the product with weights, into a tensor of `shape`
PyObject* multiply(QaMxGemmParams& p, const Operand& w, at::IntArrayRef shape, at::ScalarType type, at::Device device, const char* what) {
    const OnDevice on(device);
    const auto opts = at::TensorOptions().device(device);
    const at::Tensor out = at::empty(shape, opts.dtype(type));
    p.n = static_cast<int32_t>(w.rows);
    p.k = static_cast<int32_t>(w.k);
    p.out_type = lm_type(type);
    p.ldw = w.pitch;
    p.ldd = w.rows;
    p.w_scale_group_stride = w.group_stride;
    p.w = w.codes;
    p.w_scales = w.scales;
    p.d = out.data_ptr();
    p.workspace_bytes = g.mm_bytes(&p);
    const at::Tensor workspace = p.workspace_bytes ? at::empty({p.workspace_bytes}, opts.dtype(at::kByte)) : at::Tensor();
    p.workspace = p.workspace_bytes ? workspace.data_ptr() : nullptr;
    enqueue(g.mm, p, device, what);
    return wrapped(out);
}

// mxfp4_mm(a, a_scales, w, w_scales, out_dtype) -> (M, N)
PyObject* mxfp4_mm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "mxfp4_mm takes 5 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor &a = tensor(args[0], "a"), &w = tensor(args[2], "w");
        const auto type = dtype_or_none(args[4], "out_dtype").value_or(at::kHalf);
        supported(is_float(type), "out_dtype must be fp16, bf16 or fp32");
        on_gpu(a, "a");
        const Operand of_a = operand(a, tensor(args[1], "a_scales"), "a", "a_scales", a.device()), of_w = operand(w, tensor(args[3], "w_scales"), "w", "w_scales", a.device());
        require(of_a.k == of_w.k, "a and w must have the same K");
        QaMxGemmParams p = {};
        p.m = static_cast<int32_t>(of_a.rows);
        p.a_type = QA_LM_I8;
        p.lda = of_a.pitch;
        p.a_scale_group_stride = of_a.group_stride;
        p.a = of_a.codes;
        p.a_scales = of_a.scales;
        return multiply(p, of_w, {of_a.rows, of_w.rows}, type, a.device(), "mxfp4_mm");
    });
}

// mxfp4_linear(x, w, w_scales, out_dtype) -> (..., N)
PyObject* mxfp4_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "mxfp4_linear takes 4 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor &x = tensor(args[0], "x"), &w = tensor(args[1], "w");
        require(x.dim() >= 1, "x must be (..., K)");
        on_gpu(x, "x");
        require(is_float(x.scalar_type()), "x must be fp16, bf16 or fp32");
        const auto type = dtype_or_none(args[3], "out_dtype").value_or(x.scalar_type());
        supported(is_float(type), "out_dtype must be fp16, bf16 or fp32");
        const Operand of_w = operand(w, tensor(args[2], "w_scales"), "w", "w_scales", x.device());
        require(x.size(-1) == of_w.k, "x and w must have the same K");
        const at::Tensor flat = as_rows(x, of_w.k);
        in_rows(flat, "x");
        require(flat.size(0) <= kMost, "mxfp4_linear: a size beyond 32 bits");
        QaMxGemmParams p = {};
        p.m = static_cast<int32_t>(flat.size(0));
        p.a_type = lm_type(x.scalar_type());
        p.lda = row_stride(flat);
        p.a = flat.const_data_ptr();
        return multiply(p, of_w, with_last(x.sizes(), of_w.rows), type, x.device(), "mxfp4_linear");
    });
}

// beam_search_step(logits, scores, count, done) -> (scores, tokens, parents)
PyObject* beam_search_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "beam_search_step takes 4 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor &logits = tensor(a[0], "logits"), &scores = tensor(a[1], "scores");
        const int64_t count = whole(a[2]);
        const at::Tensor* done = tensor_or_none(a[3], "done");
        require(logits.dim() == 3, "logits must be (batch, beams, vocab)");
        on_gpu(logits, "logits");
        require(is_float(logits.scalar_type()), "logits must be fp16, bf16 or fp32");
        const int64_t batch = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
        const at::Device device = logits.device();
        require(beams >= 1 && vocab >= 1, "logits without beams or a vocabulary");
        require(batch <= kMost && vocab <= kMost, "beam_search_step: a size beyond 32 bits");
        require(vocab == 1 || logits.stride(2) == 1, "logits must be contiguous along the last dimension");
        supported(beams <= 64 && vocab <= 1 << 20, "beam_search_step: up to 64 beams and 2^20 tokens");
        require(count >= 1 && count <= beams * vocab, "count must be between 1 and what the beams offer");
        supported(count <= 64, "beam_search_step: count up to 64");
        beside(scores, "scores", device);
        require(scores.scalar_type() == at::kFloat, "scores must be fp32");
        shaped(scores, "scores", {batch, beams});
        if (done) {
            beside(*done, "done", device);
            require(done->scalar_type() == at::kBool, "done must be bool");
            shaped(*done, "done", {batch, beams});
        }
        const OnDevice on(device);
        const at::Tensor own = scores.is_contiguous() ? scores : scores.contiguous(), at_end = !done || done->is_contiguous() ? (done ? *done : at::Tensor()) : done->contiguous();
        const auto opts = at::TensorOptions().device(device);
        at::Tensor best, tokens, parents;
        const int64_t places = batch * count;
        if (places * (4 + 2 * 8) <= kTogether) {
            Together all(2 * Together::place(places * 8) + places * 4, device);
            tokens = all.next({batch, count}, at::kLong);
            parents = all.next({batch, count}, at::kLong);
            best = all.next({batch, count}, at::kFloat);
        } else {
            best = at::empty({batch, count}, opts.dtype(at::kFloat));
            tokens = at::empty({batch, count}, opts.dtype(at::kLong));
            parents = at::empty({batch, count}, opts.dtype(at::kLong));
        }
        QaBeamSearchParams p = {};
        p.batch = static_cast<int32_t>(batch);
        p.beams = static_cast<int32_t>(beams);
        p.vocab = static_cast<int32_t>(vocab);
        p.logits_type = lm_type(logits.scalar_type());
        p.count = static_cast<int32_t>(count);
        p.logits_batch_stride = logits.stride(0);
        p.logits_beam_stride = logits.stride(1);
        p.logits = logits.const_data_ptr();
        p.scores = own.const_data_ptr<float>();
        p.done = at_end.defined() ? static_cast<const uint8_t*>(at_end.const_data_ptr()) : nullptr;
        p.out_scores = best.data_ptr<float>();
        p.tokens = tokens.data_ptr<int64_t>();
        p.parents = parents.data_ptr<int64_t>();
        p.workspace_bytes = g.beam_bytes(&p);
        const at::Tensor workspace = p.workspace_bytes ? at::empty({p.workspace_bytes}, opts.dtype(at::kByte)) : at::Tensor();
        p.workspace = p.workspace_bytes ? workspace.data_ptr() : nullptr;
        enqueue(g.beam, p, device, "beam_search_step");
        return Py_BuildValue("(NNN)", wrapped(best), wrapped(tokens), wrapped(parents));
    });
}

// Memory that a tensor's rows take: rows of `bytes` from `first` on, `stride` apart.
struct Rows {
    const char* first;
    int64_t count, bytes, stride;
    const char* last() const { return first + (count - 1) * stride + bytes; }
};
// whether two of them, a not behind b, have a byte in common (or may have: pitches that differ are not followed up)
bool may_share(const Rows& a, const Rows& b) {
    if (!a.bytes || !b.bytes || a.last() <= b.first) return false;
    // rows between rows: of one pitch, behind the end of one and in front of the next
    if (a.count == 1 || (b.count > 1 && a.stride != b.stride)) return true;
    const int64_t behind = (b.first - a.first) % a.stride;
    return behind < a.bytes || behind + b.bytes > a.stride;
}

// reorder_states(states, parents) -> None
PyObject* reorder_states(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "reorder_states takes 2 arguments");
        return nullptr;
    }
    return guarded([&]() -> PyObject* {
        const at::Tensor& parents = tensor(a[1], "parents");
        require(parents.dim() == 2, "parents must be (batch, beams)");
        on_gpu(parents, "parents");
        require(parents.scalar_type() == at::kInt || parents.scalar_type() == at::kLong, "parents must be int32 or int64");
        const int64_t batch = parents.size(0), beams = parents.size(1);
        const at::Device device = parents.device();
        require(beams >= 1, "parents without beams");
        supported(beams <= 64, "reorder_states: up to 64 beams");
        supported(batch <= 65535, "reorder_states: up to 65535 entries");
        const bool single = THPVariable_Check(a[0]);
        PyObject* const sequence = single ? nullptr : PySequence_Fast(a[0], "states must be a tensor or a sequence of tensors");
        if (!single && !sequence) throw Raised{};
        struct Release {
            PyObject* o;
            ~Release() { Py_XDECREF(o); }
        } release{sequence};
        const Py_ssize_t count = single ? 1 : PySequence_Fast_GET_SIZE(sequence);
        require(count <= kMost, "reorder_states: too many tensors");
        std::vector<QaStateRows> states;
        std::vector<Rows> memory;
        std::vector<at::Tensor> tensors;                                   // (held: another thread may change a list meanwhile)
        states.reserve(count);
        memory.reserve(count + 1);
        tensors.reserve(count);
        std::vector<std::pair<int64_t, int64_t>> dims;                     // (stride, size) of a row
        for (Py_ssize_t i = 0; i < count; ++i) {
            const at::Tensor& t = tensor(single ? a[0] : PySequence_Fast_GET_ITEM(sequence, i), "each of states");
            beside(t, "each of states", device);
            require(t.dim() >= 1 && t.size(0) == batch * beams, "each of states must have batch x beams rows");
            // a row in one piece, its dimensions in any order
            int64_t values = 1;
            if (t.is_contiguous()) {
                for (int64_t d = 1; d < t.dim(); ++d) values *= t.size(d);
            } else {
                dims.clear();
                for (int64_t d = 1; d < t.dim(); ++d) {
                    if (t.size(d) != 1) dims.emplace_back(t.stride(d), t.size(d));
                }
                std::sort(dims.begin(), dims.end());
                for (const auto& [stride, size] : dims) {
                    require(t.numel() == 0 || stride == values, "the rows of each of states must be in one piece");
                    values *= size;
                }
                require(t.numel() == 0 || t.size(0) <= 1 || t.stride(0) >= values, "the rows of each of states must not overlap");
            }
            if (t.numel() == 0) continue;
            const int64_t bytes = values * static_cast<int64_t>(t.element_size()), stride = t.size(0) > 1 ? t.stride(0) * static_cast<int64_t>(t.element_size()) : bytes;
            states.push_back({t.data_ptr(), bytes, stride});
            memory.push_back({static_cast<const char*>(t.const_data_ptr()), t.size(0), bytes, stride});
            tensors.push_back(t);
        }
        const OnDevice on(device);
        const at::Tensor index = parents.is_contiguous() ? parents : parents.contiguous();
        if (index.numel()) memory.push_back({static_cast<const char*>(index.const_data_ptr()), 1, index.numel() * static_cast<int64_t>(index.element_size()), 0});
        // (in the order of their first bytes, each against those that begin before its end; rows of one buffer are a few of them)
        std::sort(memory.begin(), memory.end(), [](const Rows& x, const Rows& y) { return x.first < y.first; });
        for (size_t i = 0; i < memory.size(); ++i) {
            for (size_t j = i + 1; j < memory.size() && memory[j].first < memory[i].last(); ++j)
                require(!may_share(memory[i], memory[j]), "states must not share memory with each other or with parents");
        }
        QaReorderParams p = {};
        p.batch = static_cast<int32_t>(batch);
        p.beams = static_cast<int32_t>(beams);
        p.tensors = static_cast<int32_t>(states.size());
        p.index_bytes = static_cast<int32_t>(index.element_size());
        p.states = states.data();
        p.parents = index.const_data_ptr();
        enqueue(g.reorder, p, device, "reorder_states");
        for (const at::Tensor& t : tensors) {
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();                // (as torch's own writes in place do)
        }
        return Py_NewRef(Py_None);
    });
}

// bind(addresses of the library's functions in the order of Bound, (get_device, set_device, get_stream, out-of-memory error, check))
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long f[7];
    PyObject* py[5];
    if (!PyArg_ParseTuple(args, "(KKKKKKK)(OOOOO)", &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6], &py[0], &py[1], &py[2], &py[3], &py[4])) return nullptr;
    g.quant = reinterpret_cast<decltype(g.quant)>(f[0]);
    g.dequant = reinterpret_cast<decltype(g.dequant)>(f[1]);
    g.mm_bytes = reinterpret_cast<decltype(g.mm_bytes)>(f[2]);
    g.mm = reinterpret_cast<decltype(g.mm)>(f[3]);
    g.beam_bytes = reinterpret_cast<decltype(g.beam_bytes)>(f[4]);
    g.beam = reinterpret_cast<decltype(g.beam)>(f[5]);
    g.reorder = reinterpret_cast<decltype(g.reorder)>(f[6]);
    torch_side.keep(py);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* bound_only(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    if (g.quant) return F(self, args, n);
    PyErr_SetString(PyExc_RuntimeError, "quamba_amd._mx_beam_host: bind() first");
    return nullptr;
}
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bound_only<F>)); }

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "Takes the library's functions."},
                         {"mxfp4_quant", fast<mxfp4_quant>(), METH_FASTCALL, "ops.mxfp4_quant"},
                         {"mxfp4_dequant", fast<mxfp4_dequant>(), METH_FASTCALL, "ops.mxfp4_dequant"},
                         {"mxfp4_mm", fast<mxfp4_mm>(), METH_FASTCALL, "ops.mxfp4_mm"},
                         {"mxfp4_linear", fast<mxfp4_linear>(), METH_FASTCALL, "ops.mxfp4_linear"},
                         {"beam_search_step", fast<beam_search_step>(), METH_FASTCALL, "ops.beam_search_step"},
                         {"reorder_states", fast<reorder_states>(), METH_FASTCALL, "ops.reorder_states"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_mx_beam_host", "Host side of the microscaled 4-bit operators and of beam search.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mx_beam_host() {
    PyObject* m = PyModule_Create(&module_def);
    if (m && (PyModule_AddIntConstant(m, "MX_ABI_VERSION", QA_MX_ABI_VERSION) < 0 || PyModule_AddIntConstant(m, "BEAM_ABI_VERSION", QA_BEAM_ABI_VERSION) < 0)) Py_CLEAR(m);
    return m;
}
