// kv4_binding.cpp -- the plans' calls of the 4-bit cache's entry points.
//
// A step of a decoding loop runs kernels of a few microseconds, so what is done
// for each call before the launch counts as much as they do: the checks of ten
// operands and a call of thirty arguments take 10 to 20 us in Python and 1 us
// here.  Every function takes a plan's sizes (packed 8-byte values), the stream
// (None: torch's current one) and the operands, checks the operands against the
// sizes, raises InvalidProblem as the other plans do, and returns the status of
// the one C entry point that it calls.
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>

#include "baracuda_kernels.h"

namespace {

PyObject *g_invalid = nullptr;      // plans.InvalidProblem
PyObject *g_raw_stream = nullptr;   // device index -> the current stream's handle

struct Raised {};

[[noreturn]] void refuse(const char *what, const char *why) {
    PyErr_Format(g_invalid, "%s %s", what, why);
    throw Raised{};
}

// The sizes that every plan packs, in this order; what a plan has no use for is 0.
struct Sizes {
    int64_t tokens, hq, hk, D, rope, axes, interleaved, element, norm;
    double eps;
    int64_t ps, pages, seqs, max_q, max_kv, max_pages, causal, window;
    double scale;
    int64_t layers, page_bytes, rows;
};

class Call {
public:
    Call(PyObject *const *args, Py_ssize_t n, Py_ssize_t want) : args_(args + 2), stream_(args[1]) {
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

    struct Rows {
        void *p = nullptr;
        int64_t token = 0, head = 0;
    };

    // [tokens, heads, D] of the plan's element, the values of a head dense.
    Rows rows(int i, const char *what, int64_t tokens, int64_t heads, bool out) {
        const at::Tensor &t = tensor(i, what);
        if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != s.D)
            refuse(what, "must be [tokens, heads, head_dim] as in the descriptor");
        if (t.scalar_type() != dtype) refuse(what, "must be of the descriptor's element");
        if (s.D > 1 && t.stride(2) != 1) refuse(what, "must have the values of a head dense");
        const int64_t t0 = t.stride(0), t1 = t.stride(1);
        if (out && t.numel()) {   // every element in a place of its own
            const bool tokens_first = (heads <= 1 || t1 >= s.D) && (tokens <= 1 || t0 >= (heads - 1) * t1 + s.D);
            const bool heads_first = (tokens <= 1 || t0 >= s.D) && (heads <= 1 || t1 >= (tokens - 1) * t0 + s.D);
            if (!tokens_first && !heads_first) refuse(what, "must not have rows that overlap");
        }
        return Rows{t.data_ptr(), t0, t1};
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

    void *cache(int i, int64_t a, int64_t b, int64_t c, bool any_byte) {
        const at::Tensor &t = tensor(i, "cache");
        if (t.dim() != 3 || t.size(0) != a || t.size(1) != b || t.size(2) != c)
            refuse("cache", "does not have the descriptor's sizes");
        if (any_byte ? t.element_size() != 1 : t.scalar_type() != at::kByte) refuse("cache", "must be bytes");
        if (!t.is_contiguous()) refuse("cache", "must be contiguous");
        return t.data_ptr();
    }

    void *workspace(int i, size_t &bytes) {
        bytes = 0;
        if (!given(i)) return nullptr;
        const at::Tensor &t = tensor(i, "workspace");
        if (!t.is_contiguous()) refuse("workspace", "must be contiguous");
        bytes = t.nbytes();
        return t.data_ptr();
    }

    struct Rotation {
        void *q_weight = nullptr, *k_weight = nullptr;
        const int32_t *positions = nullptr, *pair_axis = nullptr;
        const float *cosine = nullptr, *sine = nullptr;
        int64_t table_rows = 0;
    };

    // q_weight, k_weight, positions, cos, sin, pair_axis from operand i on.
    Rotation rotation(int i) {
        Rotation r;
        if (s.norm) {
            r.q_weight = dense<void>(i, "q_weight", dtype, s.D);
            r.k_weight = dense<void>(i + 1, "k_weight", dtype, s.D);
        } else if (given(i) || given(i + 1)) {
            refuse("q_weight, k_weight:", "a descriptor without norm takes none");
        }
        if (!s.rope) {
            if (given(i + 2) || given(i + 3) || given(i + 4) || given(i + 5))
                refuse("positions, cos, sin, pair_axis:", "a descriptor without rope_dim takes none");
            return r;
        }
        if (s.axes == 1 && given(i + 2) && THPVariable_Check(args_[i + 2]) && THPVariable_Unpack(args_[i + 2]).dim() == 1)
            r.positions = dense<int32_t>(i + 2, "positions", at::kInt, s.tokens);
        else
            r.positions = dense<int32_t>(i + 2, "positions", at::kInt, s.axes, s.tokens);
        const at::Tensor &c = tensor(i + 3, "cos");
        if (c.dim() != 2 || c.size(0) < 1) refuse("cos", "must have a row for each position");
        r.table_rows = c.size(0);
        r.cosine = dense<float>(i + 3, "cos", at::kFloat, r.table_rows, s.rope / 2);
        r.sine = dense<float>(i + 4, "sin", at::kFloat, r.table_rows, s.rope / 2);
        if (s.axes > 1) r.pair_axis = dense<int32_t>(i + 5, "pair_axis", at::kInt, s.rope / 2);
        else if (given(i + 5)) refuse("pair_axis:", "one axis takes none");
        return r;
    }

    // After all operands: they are on a GPU, and this is its stream.
    void *stream() {
        if (host_ || device_ < 0) refuse("operand tensors", "must be on the GPU");
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

private:
    PyObject *const *args_;
    PyObject *stream_;
    int device_ = -1;
    bool host_ = false;
};

template <int N, typename F>
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

// q, k, q_out, k_out, q_weight, k_weight, positions, cos, sin, pair_axis
PyObject *qk_norm_rope(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<10>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const auto q = c.rows(0, "q", s.tokens, s.hq, false), k = c.rows(1, "k", s.tokens, s.hk, false);
        const auto qo = c.rows(2, "q_out", s.tokens, s.hq, true), ko = c.rows(3, "k_out", s.tokens, s.hk, true);
        const auto r = c.rotation(4);
        void *stream = c.stream();
        return baracuda_kernels_qk_norm_rope_gfx950_run(
            s.tokens, s.hq, s.hk, s.D, s.rope, s.axes, s.interleaved, s.element, s.eps, q.p, q.token, q.head, k.p, k.token,
            k.head, qo.p, qo.token, qo.head, ko.p, ko.token, ko.head, r.q_weight, r.k_weight, r.positions, r.cosine, r.sine,
            r.table_rows, r.pair_axis, stream);
    });
}

int64_t head_bytes(const Sizes &s) { return s.ps * (s.D + s.D / 16); }

// k, v, cache, slots, q, q_out, q_weight, k_weight, positions, cos, sin, pair_axis
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<12>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const auto k = c.rows(0, "k", s.tokens, s.hk, false), v = c.rows(1, "v", s.tokens, s.hk, false);
        void *cache = c.cache(2, s.pages, s.hk, head_bytes(s), false);
        const int64_t *slots = c.dense<int64_t>(3, "slots", at::kLong, s.tokens);
        Call::Rows q, qo;
        if (s.hq) q = c.rows(4, "q", s.tokens, s.hq, false), qo = c.rows(5, "q_out", s.tokens, s.hq, true);
        else if (c.given(4) || c.given(5)) refuse("q, q_out:", "a descriptor without query heads takes none");
        const auto r = c.rotation(6);
        void *stream = c.stream();
        return baracuda_kernels_kv4_append_gfx950_run(
            s.tokens, s.hq, s.hk, s.D, s.rope, s.axes, s.interleaved, s.element, s.eps, s.ps, s.pages, q.p, q.token, q.head,
            k.p, k.token, k.head, v.p, v.token, v.head, qo.p, qo.token, qo.head, cache, slots, r.q_weight, r.k_weight,
            r.positions, r.cosine, r.sine, r.table_rows, r.pair_axis, stream);
    });
}

// cache, slots, k_out, v_out
PyObject *read(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<4>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        void *cache = c.cache(0, s.pages, s.hk, head_bytes(s), false);
        const int64_t *slots = c.dense<int64_t>(1, "slots", at::kLong, s.tokens);
        const auto k = c.rows(2, "k_out", s.tokens, s.hk, true), v = c.rows(3, "v_out", s.tokens, s.hk, true);
        void *stream = c.stream();
        return baracuda_kernels_kv4_read_gfx950_run(s.tokens, s.hk, s.D, s.element, s.ps, s.pages, cache, slots, k.p, k.token,
                                                    k.head, v.p, v.token, v.head, stream);
    });
}

// q, cache, tables, kv_lens, out, cu_q, workspace
PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<7>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const auto q = c.rows(0, "q", s.tokens, s.hq, false);
        void *cache = c.cache(1, s.pages, s.hk, head_bytes(s), false);
        const at::Tensor &t = c.tensor(2, "tables");
        if (t.dim() != 2 || t.size(0) != s.seqs || t.size(1) != s.max_pages || t.scalar_type() != at::kInt)
            refuse("tables", "must be int32 [num_seqs, max_pages]");
        if (s.max_pages > 1 && t.stride(1) != 1) refuse("tables", "must have a sequence's pages dense");
        const int32_t *lens = c.dense<int32_t>(3, "kv_lens", at::kInt, s.seqs);
        const auto out = c.rows(4, "out", s.tokens, s.hq, true);
        const int32_t *cu = nullptr;
        if (c.given(5)) cu = c.dense<int32_t>(5, "cu_q", at::kInt, s.seqs + 1);
        else if (s.max_q != 1 || s.tokens != s.seqs) refuse("cu_q", "is required unless every sequence has one new token");
        size_t bytes;
        void *ws = c.workspace(6, bytes);
        void *stream = c.stream();
        return baracuda_kernels_kv4_attention_gfx950_run(
            s.seqs, s.tokens, s.max_q, s.max_kv, s.hq, s.hk, s.D, s.ps, s.pages, s.max_pages, s.element, s.causal, s.window,
            (float)s.scale, q.p, q.token, q.head, cache, (const int32_t *)t.data_ptr(), t.stride(0), lens, cu, out.p, out.token,
            out.head, ws, bytes, stream);
    });
}

// cache, src, dst
PyObject *pages_copy(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<3>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        void *cache = c.cache(0, s.layers, s.pages, s.page_bytes, true);
        const at::Tensor &t = c.tensor(1, "src");
        const int64_t count = t.dim() == 1 ? t.size(0) : -1;
        const int32_t *src = c.dense<int32_t>(1, "src", at::kInt, count), *dst = c.dense<int32_t>(2, "dst", at::kInt, count);
        void *stream = c.stream();
        return baracuda_kernels_kv_pages_copy_gfx950_run(s.layers, s.pages, s.page_bytes, count, cache, src, dst, stream);
    });
}

// cache, tables, lens, refs, parents, children, fresh
PyObject *pages_fork(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<7>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        void *cache = c.cache(0, s.layers, s.pages, s.page_bytes, true);
        int32_t *tables = c.dense<int32_t>(1, "tables", at::kInt, s.rows, s.max_pages);
        int32_t *lens = c.dense<int32_t>(2, "lens", at::kInt, s.rows), *refs = c.dense<int32_t>(3, "refs", at::kInt, s.pages);
        const at::Tensor &t = c.tensor(4, "parents");
        const int64_t count = t.dim() == 1 ? t.size(0) : -1;
        if (count > INT32_MAX) refuse("parents", "has more entries than there can be rows");
        const int32_t *parents = c.dense<int32_t>(4, "parents", at::kInt, count);
        const int32_t *children = c.dense<int32_t>(5, "children", at::kInt, count);
        int32_t *fresh = c.dense<int32_t>(6, "fresh", at::kInt, count);
        void *stream = c.stream();
        return baracuda_kernels_kv_pages_fork_gfx950_run(s.layers, s.pages, s.page_bytes, s.ps, s.rows, s.max_pages, count, cache,
                                                         tables, lens, refs, parents, children, fresh, stream);
    });
}

// tables, lens, refs, rows
PyObject *pages_release(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<4>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        int32_t *tables = c.dense<int32_t>(0, "tables", at::kInt, s.rows, s.max_pages);
        int32_t *lens = c.dense<int32_t>(1, "lens", at::kInt, s.rows), *refs = c.dense<int32_t>(2, "refs", at::kInt, s.pages);
        const at::Tensor &t = c.tensor(3, "rows");
        const int64_t count = t.dim() == 1 ? t.size(0) : -1;
        if (count > INT32_MAX) refuse("rows", "has more entries than there can be rows");
        const int32_t *which = c.dense<int32_t>(3, "rows", at::kInt, count);
        void *stream = c.stream();
        return baracuda_kernels_kv_pages_release_gfx950_run(s.pages, s.rows, s.max_pages, count, tables, lens, refs, which,
                                                            stream);
    });
}

// cache, tables, refs, tables_out, refs_out, remap, live, workspace
PyObject *pages_compact(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<8>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        void *cache = c.cache(0, s.layers, s.pages, s.page_bytes, true);
        const int32_t *tables = c.dense<int32_t>(1, "tables", at::kInt, s.rows, s.max_pages);
        const int32_t *refs = c.dense<int32_t>(2, "refs", at::kInt, s.pages);
        int32_t *tables_out = c.dense<int32_t>(3, "tables_out", at::kInt, s.rows, s.max_pages);
        int32_t *refs_out = c.dense<int32_t>(4, "refs_out", at::kInt, s.pages);
        int32_t *remap = c.dense<int32_t>(5, "remap", at::kInt, s.pages), *live = c.dense<int32_t>(6, "live", at::kInt, 1);
        if (refs == refs_out) refuse("refs_out", "must not be refs");
        size_t bytes;
        void *ws = c.workspace(7, bytes);
        void *stream = c.stream();
        return baracuda_kernels_kv_pages_compact_gfx950_run(s.layers, s.pages, s.page_bytes, s.ps, s.rows, s.max_pages, cache,
                                                            tables, refs, tables_out, refs_out, remap, live, ws, bytes, stream);
    });
}

// The exception that refusals raise, and torch's lookup of the current stream.
PyObject *connect(PyObject *, PyObject *const *args, Py_ssize_t n) {
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
PyMethodDef kMethods[] = {BK_METHOD(connect),       BK_METHOD(qk_norm_rope), BK_METHOD(append),
                          BK_METHOD(read),          BK_METHOD(attention),    BK_METHOD(pages_copy),
                          BK_METHOD(pages_fork),    BK_METHOD(pages_release), BK_METHOD(pages_compact),
                          {nullptr, nullptr, 0, nullptr}};
#undef BK_METHOD

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kv4", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv4() { return PyModule_Create(&kModule); }
