// What the host sides of the operators share: arguments and their checks, errors, the device and the stream of a call.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <limits>
#include <optional>
#include <string>

#include "../../include/quamba_amd_lm.h"

namespace {

// What bind() was given of the Python side of torch's runtime.
struct TorchSide {
    PyObject *get_device = nullptr, *set_device = nullptr, *get_stream = nullptr, *oom = nullptr, *check = nullptr;
    void keep(PyObject* const (&py)[5]) {
        PyObject** const kept[5] = {&get_device, &set_device, &get_stream, &oom, &check};
        for (int i = 0; i < 5; ++i) {
            PyObject* before = *kept[i];
            *kept[i] = Py_NewRef(py[i]);
            Py_XDECREF(before);
        }
    }
} torch_side;

struct Refused {
    PyObject* type;
    std::string text;
};
struct Raised {};              // a Python error is set

// (texts are put together where a check fails only: a dozen of them a call would take it a microsecond)
template <class... Parts>
[[noreturn]] void refuse(PyObject* type, const Parts&... parts) {
    std::string text;
    ((text += parts), ...);
    throw Refused{type, text};
}
template <class... Parts>
void require(bool fine, const Parts&... parts) {
    if (!fine) refuse(PyExc_RuntimeError, parts...);
}
template <class... Parts>
void supported(bool fine, const Parts&... parts) {
    if (!fine) refuse(PyExc_NotImplementedError, parts...);
}

// No C++ exception passes through the interpreter.
template <class Body>
PyObject* guarded(Body&& body) {
    try {
        return body();
    } catch (const Raised&) {
    } catch (const Refused& e) {
        PyErr_SetString(e.type, e.text.c_str());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(torch_side.oom ? torch_side.oom : PyExc_MemoryError, e.what_without_backtrace());
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// ---- arguments ----------------------------------------------------------------------------------------------------
const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, std::string(name) + " must be a tensor"};
    return THPVariable_Unpack(o);
}
const at::Tensor* tensor_or_none(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

std::optional<at::ScalarType> dtype_or_none(PyObject* o, const char* name) {
    if (o == Py_None) return std::nullopt;
    if (!THPDtype_Check(o)) throw Refused{PyExc_TypeError, std::string(name) + " must be a torch.dtype"};
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}
int64_t whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

int lm_type(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return QA_LM_F16;
        case at::kBFloat16: return QA_LM_BF16;
        case at::kFloat: return QA_LM_F32;
        case at::kChar: return QA_LM_I8;
        default: return -1;
    }
}
bool is_float(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat; }

std::string shape_text(at::IntArrayRef s) {
    std::string text = "(";
    for (size_t i = 0; i < s.size(); ++i) text += (i ? ", " : "") + std::to_string(s[i]);
    return text + (s.size() == 1 ? ",)" : ")");
}
void on_gpu(const at::Tensor& t, const char* name) { require(t.is_cuda(), name, " must be a GPU tensor (quamba_amd has no CPU path)"); }
void beside(const at::Tensor& t, const char* name, at::Device device) {
    if (t.device() != device) refuse(PyExc_RuntimeError, name, " must be on ", device.str());
}
void shaped(const at::Tensor& t, const char* name, at::IntArrayRef shape) {
    if (!t.sizes().equals(shape)) refuse(PyExc_RuntimeError, name, " must have shape ", shape_text(shape), ", not ", shape_text(t.sizes()));
}
// rows next to or apart from each other, each of them in one piece
void in_rows(const at::Tensor& t, const char* name) {
    const int64_t n = t.dim();
    require(n == 0 || t.stride(n - 1) == 1 || t.size(n - 1) <= 1, name, " must be contiguous along the last dimension");
    require(n < 2 || t.size(0) <= 1 || t.stride(0) >= t.size(1), "the rows of ", name, " must not overlap");
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
const void* address(const at::Tensor* t) { return t ? t->const_data_ptr() : nullptr; }

// ---- the call -----------------------------------------------------------------------------------------------------
// A device as the current one for as long as this stands, however the call ends.
class OnDevice {
  public:
    explicit OnDevice(at::Device device) {
        PyObject* at = PyObject_CallNoArgs(torch_side.get_device);
        if (!at) throw Raised{};
        back_ = PyLong_AsLong(at);
        Py_DECREF(at);
        if (PyErr_Occurred()) throw Raised{};
        if (back_ == device.index()) return;
        if (!set(device.index())) throw Raised{};
        moved_ = true;
    }
    ~OnDevice() {
        if (!moved_) return;
        PyObject *type, *value, *trace;
        PyErr_Fetch(&type, &value, &trace);
        if (!set(back_)) PyErr_WriteUnraisable(torch_side.set_device);
        PyErr_Restore(type, value, trace);
    }
    OnDevice(const OnDevice&) = delete;

  private:
    static bool set(long device) {
        PyObject* r = PyObject_CallFunction(torch_side.set_device, "l", device);
        Py_XDECREF(r);
        return r != nullptr;
    }
    long back_ = 0;
    bool moved_ = false;
};

template <class Params>
void enqueue(int (*call)(const Params*, void*), const Params& p, at::Device device, const char* what) {
    PyObject* stream_o = PyObject_CallFunction(torch_side.get_stream, "i", static_cast<int>(device.index()));
    if (!stream_o) throw Raised{};
    void* stream = PyLong_AsVoidPtr(stream_o);
    Py_DECREF(stream_o);
    if (PyErr_Occurred()) throw Raised{};
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = call(&p, stream);
    Py_END_ALLOW_THREADS
    if (status == QA_OK) return;
    Py_XDECREF(PyObject_CallFunction(torch_side.check, "is", status, what));        // raises
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, what);
    throw Raised{};
}

PyObject* wrapped(const at::Tensor& t) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) throw Raised{};
    return o;
}
PyObject* wrapped_or_none(const at::Tensor& t) { return t.defined() ? wrapped(t) : Py_NewRef(Py_None); }

}  // namespace
