// w4_binding.cpp -- the plans' calls of the products with 4-bit weights.
#include "binding.hpp"

namespace {

using namespace binding;

// The sizes that every plan packs, in this order; what a plan has no use for is 0 or 1.
struct Sizes {
    int64_t element, n, k, rows, matrices, topk, gated, bytes;
};

class Call : public Operands<Sizes> {
public:
    using Operands::Operands;

    // uint8 [matrices, bytes]; one matrix also as [bytes].
    uint8_t *packed(int i) {
        const at::Tensor &t = tensor(i, "packed");
        const bool one = t.dim() == 1 && s.matrices == 1 && t.size(0) == s.bytes;
        if (!one && (t.dim() != 2 || t.size(0) != s.matrices || t.size(1) != s.bytes))
            refuse("packed", "must be [matrices, packed_bytes(n, k)]");
        if (t.scalar_type() != at::kByte) refuse("packed", "must be bytes");
        if (!t.is_contiguous()) refuse("packed", "must be contiguous");
        return (uint8_t *)t.data_ptr();
    }

    struct Matrices {
        void *p;
        int64_t matrix, row;
    };

    // [matrices, n, k] of the plan's element, or [n, k] of one matrix; rows dense.
    Matrices weights(int i) {
        const at::Tensor &t = tensor(i, "weights");
        const int64_t d = t.dim();
        if ((d != 3 && !(d == 2 && s.matrices == 1)) || (d == 3 && t.size(0) != s.matrices) || t.size(d - 2) != s.n ||
            t.size(d - 1) != s.k)
            refuse("weights", "must be [matrices, n, k] as in the descriptor");
        if (t.scalar_type() != dtype) refuse("weights", "must be of the descriptor's element");
        if (t.stride(d - 1) != 1) refuse("weights", "must have rows that are dense");
        return Matrices{t.data_ptr(), d == 3 ? t.stride(0) : 0, t.stride(d - 2)};
    }

    // uint8 [matrices, n, columns], or [n, columns] of one matrix, contiguous.
    uint8_t *bytes_of(int i, const char *what, int64_t columns) {
        const at::Tensor &t = tensor(i, what);
        const int64_t d = t.dim();
        if ((d != 3 && !(d == 2 && s.matrices == 1)) || (d == 3 && t.size(0) != s.matrices) || t.size(d - 2) != s.n ||
            t.size(d - 1) != columns)
            refuse(what, "does not have the descriptor's sizes");
        if (t.scalar_type() != at::kByte) refuse(what, "must be bytes");
        if (!t.is_contiguous()) refuse(what, "must be contiguous");
        return (uint8_t *)t.data_ptr();
    }

    struct Matrix {
        void *p;
        int64_t ld;
        bool dense;
    };

    // [rows, columns] of the plan's element, the columns dense.
    Matrix matrix(int i, const char *what, int64_t rows, int64_t columns) {
        const at::Tensor &t = tensor(i, what);
        if (t.dim() != 2 || t.size(0) != rows || t.size(1) != columns) refuse(what, "does not have the descriptor's sizes");
        if (t.scalar_type() != dtype) refuse(what, "must be of the descriptor's element");
        if (columns > 1 && t.stride(1) != 1) refuse(what, "must have rows that are dense");
        return Matrix{t.data_ptr(), t.stride(0), t.is_contiguous()};
    }

    int64_t columns() const { return s.gated ? s.n / 2 : s.n; }
};

// weights, packed
PyObject *quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<Call, 2>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const auto w = c.weights(0);
        void *packed = c.packed(1), *stream = c.stream();
        return baracuda_kernels_w4_quantize_gfx950_run(s.matrices, s.n, s.k, s.element, w.p, w.matrix, w.row, packed, stream);
    });
}

// codes, scales, packed
PyObject *pack(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<Call, 3>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const uint8_t *codes = c.bytes_of(0, "codes", s.k / 2), *scales = c.bytes_of(1, "scales", s.k / 32);
        void *packed = c.packed(2), *stream = c.stream();
        return baracuda_kernels_w4_pack_gfx950_run(s.matrices, s.n, s.k, codes, scales, packed, stream);
    });
}

// packed, weights
PyObject *read(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<Call, 2>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const void *packed = c.packed(0);
        const auto w = c.weights(1);
        void *stream = c.stream();
        return baracuda_kernels_w4_read_gfx950_run(s.matrices, s.n, s.k, s.element, packed, w.p, w.matrix, w.row, stream);
    });
}

// x, packed, out, bias, workspace
PyObject *linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<Call, 5>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const auto x = c.matrix(0, "x", s.rows, s.k);
        const void *packed = c.packed(1);
        const auto out = c.matrix(2, "out", s.rows, c.columns());
        const float *bias = c.given(3) ? c.dense<float>(3, "bias", at::kFloat, s.n) : nullptr;
        size_t bytes;
        void *ws = c.workspace(4, bytes), *stream = c.stream();
        return baracuda_kernels_w4_linear_gfx950_run(s.rows, s.n, s.k, s.element, s.gated, x.p, x.ld, packed, bias, out.p,
                                                     out.ld, ws, bytes, stream);
    });
}

// x, packed, sorted_token_ids, expert_ids, out, expert_counts, expert_offsets, bias, topk_weights, workspace
PyObject *grouped(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded<Call, 10>(args, n, [](Call &c) {
        const Sizes &s = c.s;
        const bool weighted = c.given(8);
        const auto x = c.matrix(0, "x", weighted ? s.rows : (s.rows + s.topk - 1) / s.topk, s.k);
        const void *packed = c.packed(1);
        const int32_t *order = c.dense<int32_t>(2, "sorted_token_ids", at::kInt, s.rows);
        const int32_t *ids = c.dense<int32_t>(3, "expert_ids", at::kInt, s.rows);
        const auto out = c.matrix(4, "out", s.rows, c.columns());
        if (!x.dense) refuse("x", "must be contiguous");
        if (!out.dense) refuse("out", "must be contiguous");
        int32_t *counts = c.dense<int32_t>(5, "expert_counts", at::kInt, s.matrices);
        int32_t *offsets = c.dense<int32_t>(6, "expert_offsets", at::kInt, s.matrices + 1);
        const float *bias = c.given(7) ? c.dense<float>(7, "bias", at::kFloat, s.matrices, s.n) : nullptr;
        const float *mix = weighted ? c.dense<float>(8, "topk_weights", at::kFloat, s.rows) : nullptr;
        size_t bytes;
        void *ws = c.workspace(9, bytes), *stream = c.stream();
        return baracuda_kernels_moe_w4_grouped_gfx950_run(s.matrices, s.topk, s.rows, s.n, s.k, s.element, s.gated, x.p, packed,
                                                          order, ids, mix, bias, out.p, counts, offsets, ws, bytes, stream);
    });
}

PyMethodDef kMethods[] = {BK_METHOD(connect), BK_METHOD(quantize), BK_METHOD(pack),      BK_METHOD(read),
                          BK_METHOD(linear),  BK_METHOD(grouped),  {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_w4", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__w4() { return PyModule_Create(&kModule); }
