// binding.hpp -- what the native bindings of the plans share: the operands of a
// call, their checks, the stream.
//
// A step of a decoding loop runs kernels of a few microseconds, so what is done
// for each call before the launch counts as much as they do: the checks of ten
// operands and a call of thirty arguments take 10 to 20 us in Python and 1 us
// here.  Every function takes a plan's sizes (packed 8-byte values), the stream
// (None: torch's current one) and the operands, checks the operands against the
// sizes, raises InvalidProblem as the other plans do, and returns the status of
// the one C entry point that it calls.
#pragma once

#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>

#include "baracuda_kernels.h"

namespace binding {

inline PyObject *g_invalid = nullptr;      // plans.InvalidProblem
inline PyObject *g_raw_stream = nullptr;   // device index -> the current stream's handle

struct Raised {};

[[noreturn]] inline void refuse(const char *what, const char *why) {
    PyErr_Format(g_invalid, "%s %s", what, why);
    throw Raised{};
}

// Sizes: a struct of 8-byte values, as the module's plans pack them.
template <typename Sizes>
class Operands {
public:
    Operands(PyObject *const *args, Py_ssize_t n, Py_ssize_t want) : args_(args + 2), stream_(args[1]) {
        if (n != want + 2 || !PyBytes_Check(args[0]) || PyBytes_GET_SIZE(args[0]) != (Py_ssize_t)sizeof(Sizes)) {
            PyErr_SetString(PyExc_TypeError, "a plan's sizes, a stream and its operands");
            throw Raised{};
        }
        std::memcpy(&s, PyBytes_AS_STRING(args[0]), sizeof(Sizes));
        dtype = s.element == 0 ? at::kFloat : s.element == 1 ? at::kHalf : at::kBFloat16;
    }

    bool given(int i) const { return args_[i] != Py_None; }

    const at::Tensor &tensor(int i, const char *what) {
        PyObject *o = args_[i];
        if (o == Py_None) refuse(what, "is required");
        if (!THPVariable_Check(o)) refuse(what, "must be a tensor");
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.is_cuda()) host_ = true;
        else if (device_ < 0) device_ = t.get_device();
        else if (device_ != t.get_device()) refuse(what, "must be on the GPU of the other operands");
        return t;
    }

    // A dense tensor of one dimension or two (columns < 0: one).
    template <typename P>
    P *dense(int i, const char *what, at::ScalarType type, int64_t n, int64_t columns = -1) {
        const at::Tensor &t = tensor(i, what);
        const bool shape = columns < 0 ? t.dim() == 1 && t.size(0) == n : t.dim() == 2 && t.size(0) == n && t.size(1) == columns;
        if (!shape) refuse(what, "does not have the descriptor's sizes");
        if (t.scalar_type() != type) refuse(what, "is of another type");
        if (!t.is_contiguous()) refuse(what, "must be contiguous");
        return (P *)t.data_ptr();
    }

    void *workspace(int i, size_t &bytes) {
        bytes = 0;
        if (!given(i)) return nullptr;
        const at::Tensor &t = tensor(i, "workspace");
        if (!t.is_contiguous()) refuse("workspace", "must be contiguous");
        bytes = t.nbytes();
        return t.data_ptr();
    }

    // After all operands: they are on a GPU, and this is its stream.  That GPU is
    // the current one until the call ends (a default stream's handle is null on
    // every GPU and stands for the current one's).
    void *stream() {
        if (host_ || device_ < 0) refuse("operand tensors", "must be on the GPU");
        guard_.reset_device(at::Device(at::kCUDA, (at::DeviceIndex)device_));
        PyObject *v = nullptr;
        if (stream_ == Py_None) {
            PyObject *index = PyLong_FromLong(device_);
            v = index ? PyObject_CallFunctionObjArgs(g_raw_stream, index, nullptr) : nullptr;
            Py_XDECREF(index);
        } else if (PyLong_Check(stream_)) {
            Py_INCREF(stream_);
            v = stream_;
        } else {
            v = PyObject_GetAttrString(stream_, "cuda_stream");
        }
        if (!v) throw Raised{};
        void *h = PyLong_AsVoidPtr(v);
        Py_DECREF(v);
        if (!h && PyErr_Occurred()) throw Raised{};
        return h;
    }

    Sizes s;
    at::ScalarType dtype;

protected:
    PyObject *const *args_;
    PyObject *stream_;
    int device_ = -1;
    bool host_ = false;
    c10::OptionalDeviceGuard guard_;
};

template <typename Call, int N, typename F>
PyObject *guarded(PyObject *const *args, Py_ssize_t n, F f) {
    try {
        Call c(args, n, N);
        return PyLong_FromLong(f(c));
    } catch (const Raised &) {
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown exception");
        return nullptr;
    }
}

// The exception that refusals raise, and torch's lookup of the current stream.
inline PyObject *connect(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != 2) {
        PyErr_SetString(PyExc_TypeError, "connect(exception, raw_stream)");
        return nullptr;
    }
    Py_INCREF(args[0]);
    Py_INCREF(args[1]);
    Py_XDECREF(g_invalid);
    Py_XDECREF(g_raw_stream);
    g_invalid = args[0], g_raw_stream = args[1];
    Py_RETURN_NONE;
}

#define BK_METHOD(NAME) {#NAME, (PyCFunction)(void (*)(void))NAME, METH_FASTCALL, nullptr}

}  // namespace binding
