// Short cuts for the calls of superkmeans_b200/ops.py that need no conversion: plain CUDA tensors of the right types, shapes and strides,
// no gradient to be recorded.  Such a call goes from its tensors to the C ABI without Python in between (a lookup of a few rows: 9.5 us
// through ctypes, 5 here; the kernel launch alone is 3).  Everything else - refusals, copies, gradients - is
// answered with None, and ops.py makes the call itself (a failure on the GPU is raised).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "../../include/skm_b200.h"

namespace {

constexpr int64_t kMostIds = 0x7fffffff;

// Whether the storage holds all that the tensor reaches (throws where there is none).
bool has_memory(const at::Tensor& t) {
    const int64_t numel = t.numel();
    if (numel == 0) return true;
    const c10::Storage& storage = t.storage();
    if (storage.device() != t.device() || t._is_zerotensor()) return false;
    int64_t ends = t.storage_offset() + numel;
    if (!t.is_contiguous()) {
        const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
        ends = t.storage_offset() + 1;
        for (size_t i = 0; i < sizes.size(); ++i) ends += (sizes[i] - 1) * strides[i];
    }
    return storage.nbytes() >= static_cast<size_t>(ends) * t.element_size() && storage.data() != nullptr;
}

// Nothing that a call has to refuse whatever it goes on to ask for.
bool is_ordinary(const at::Tensor& t) {
    return t.defined() && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t._fw_grad(0).defined() && has_memory(t);
}

bool plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && !t.is_neg() && is_ordinary(t);
}
bool wants_grad(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

int kind_of(at::ScalarType type) { return type == at::kFloat ? SKM_F32 : type == at::kHalf ? SKM_F16 : type == at::kBFloat16 ? SKM_BF16 : -1; }

// Rows whose values lie side by side.
struct Rows {
    at::Tensor t;
    uint64_t n = 0, d = 0, ld = 0;
    int kind = -1;

    bool take(PyObject* o, const at::Tensor* like = nullptr) {
        if (!plain(o)) return false;
        t = THPVariable_Unpack(o);
        if (t.dim() != 2 || wants_grad(t)) return false;
        if (like && t.get_device() != like->get_device()) return false;
        kind = kind_of(t.scalar_type());
        n = t.size(0);
        d = t.size(1);
        if (kind < 0 || d == 0 || (d > 1 && t.stride(1) != 1)) return false;
        ld = n > 1 ? t.stride(0) : d;
        return true;
    }
};

struct Ids {
    at::Tensor t;
    int bits = 0;

    bool take(PyObject* o, const at::Tensor* like = nullptr) {
        if (!plain(o)) return false;
        t = THPVariable_Unpack(o);
        const auto type = t.scalar_type();
        bits = type == at::kLong ? 64 : type == at::kInt || type == at::kUInt32 ? 32 : 0;
        return bits != 0 && t.is_contiguous() && t.numel() <= kMostIds && (!like || t.get_device() == like->get_device());
    }
};

// None, or contiguous floats of a shape.
struct Floats {
    at::Tensor t;

    bool take(PyObject* o, at::IntArrayRef shape, const at::Tensor& like) {
        if (o == Py_None) return true;
        if (!plain(o)) return false;
        t = THPVariable_Unpack(o);
        return t.scalar_type() == at::kFloat && t.is_contiguous() && t.sizes() == shape && t.get_device() == like.get_device() && !wants_grad(t);
    }
    const float* p() const { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
};

// Where a grouping has its rows.
struct Places {
    at::Tensor order, position, offsets;
    uint64_t n = 0, m = 1, k = 0;

    static bool take_one(PyObject* o, const at::Tensor& like, at::Tensor& t) {
        if (!plain(o)) return false;
        t = THPVariable_Unpack(o);
        return t.scalar_type() == at::kInt && t.is_contiguous() && t.get_device() == like.get_device();
    }
    bool take(PyObject* const* of, const at::Tensor& like) {   // order, position, offsets
        if (!take_one(of[0], like, order) || !take_one(of[1], like, position) || !take_one(of[2], like, offsets)) return false;
        if (position.dim() < 1 || position.dim() > 2 || offsets.dim() != 1 || offsets.size(0) < 2 || order.dim() != 1 || order.size(0) != position.numel()) return false;
        n = position.size(0);
        if (position.dim() == 2) m = position.size(1);
        k = offsets.size(0) - 1;
        return m > 0;
    }
    const uint32_t* pairs() const { return static_cast<const uint32_t*>(order.const_data_ptr()); }
    const uint32_t* positions() const { return static_cast<const uint32_t*>(position.const_data_ptr()); }
    const uint32_t* starts() const { return static_cast<const uint32_t*>(offsets.const_data_ptr()); }
};

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) { return at::empty(shape, like.options().dtype(type)); }
at::Tensor workspace(uint64_t bytes, const at::Tensor& like) { return bytes == 0 ? at::Tensor() : make({static_cast<int64_t>(bytes)}, at::kByte, like); }
void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

PyObject* none() { Py_RETURN_NONE; }
PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap(const at::Tensor& a, const at::Tensor& b) {
    PyObject* x = THPVariable_Wrap(a);
    PyObject* y = x ? THPVariable_Wrap(b) : nullptr;
    PyObject* both = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return both;
}

// What the C ABI refuses is refused again in Python, in its words; another failure (which may be told only once) is raised here.
PyObject* failed(skm_status status) {
    if (status == SKM_INVALID_ARGUMENT) return none();
    PyErr_SetString(PyExc_RuntimeError, skm_last_error(nullptr));
    return nullptr;
}

// Whether torch looks on as calls are made, some of whose ways to do so ops.py refuses.
bool is_watched() {
    return at::tracer::impl::is_dispatch_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
}

// An exception of torch's (no memory) is the caller's to meet again.
template <class F>
PyObject* shortcut(F&& f) {
    if (is_watched()) return none();
    // (no gradient is recorded here: allocations and views go straight to what makes them)
    const at::AutoDispatchBelowADInplaceOrView direct;
    try {
        return f();
    } catch (const std::exception&) {
        return none();
    }
}

// True where all arguments that are tensors are ordinary ones; ops.py says what is wrong with others
PyObject* ordinary(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        for (Py_ssize_t i = 0; i < count; ++i)
            if (THPVariable_Check(a[i]) && !is_ordinary(THPVariable_Unpack(a[i]))) return none();
        Py_RETURN_TRUE;
    });
}

// table, ids, scale, row_scales
PyObject* lookup(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Rows table;
        Ids ids;
        Floats scales;
        if (count != 4 || !table.take(a[0]) || !ids.take(a[1], &table.t) || !PyFloat_CheckExact(a[2]) || !scales.take(a[3], ids.t.sizes(), table.t)) return none();
        c10::SmallVector<int64_t, 5> shape(ids.t.sizes().begin(), ids.t.sizes().end());
        shape.push_back(static_cast<int64_t>(table.d));
        const at::Tensor out = make(shape, table.t.scalar_type(), table.t);
        const skm_status status = skm_op_lookup(table.t.get_device(), table.t.const_data_ptr(), table.ld, table.kind, table.n, table.d, ids.t.const_data_ptr(), ids.bits, ids.t.numel(),
                          static_cast<float>(PyFloat_AS_DOUBLE(a[2])), scales.p(), out.data_ptr(), stream(table.t));
        if (status != SKM_OK) return failed(status);
        return wrap(out);
    });
}

// grad, ids, n_rows, scale, row_scales (the gradient in the type of grad)
PyObject* lookup_grad(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Rows grad;
        Ids ids;
        Floats scales;
        if (count != 5 || !grad.take(a[0]) || !ids.take(a[1], &grad.t) || !PyLong_CheckExact(a[2]) || !PyFloat_CheckExact(a[3]) || !scales.take(a[4], ids.t.sizes(), grad.t)) return none();
        if (ids.t.dim() != 1 || static_cast<uint64_t>(ids.t.numel()) != grad.n) return none();
        const long long k = PyLong_AsLongLong(a[2]);
        if (k <= 0 || k >= kMostIds) {
            PyErr_Clear();
            return none();
        }
        const at::Tensor out = make({k, static_cast<int64_t>(grad.d)}, grad.t.scalar_type(), grad.t);
        const uint64_t bytes = skm_op_lookup_grad_workspace(grad.n, k, grad.d, grad.kind);
        const at::Tensor space = workspace(bytes, grad.t);
        const skm_status status = skm_op_lookup_grad(grad.t.get_device(), grad.t.const_data_ptr(), grad.ld, grad.kind, k, grad.d, ids.t.const_data_ptr(), ids.bits, grad.n,
                               static_cast<float>(PyFloat_AS_DOUBLE(a[3])), scales.p(), out.data_ptr(), grad.kind, address(space), bytes, stream(grad.t));
        if (status != SKM_OK) return failed(status);
        return wrap(out);
    });
}

// grad, table, ids, scale
PyObject* lookup_scale_grad(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Rows grad, table;
        Ids ids;
        if (count != 4 || !grad.take(a[0]) || !table.take(a[1], &grad.t) || !ids.take(a[2], &grad.t) || !PyFloat_CheckExact(a[3])) return none();
        if (table.kind != grad.kind || table.d != grad.d || table.n == 0 || ids.t.dim() != 1 || static_cast<uint64_t>(ids.t.numel()) != grad.n) return none();
        const at::Tensor out = make({static_cast<int64_t>(grad.n)}, at::kFloat, grad.t);
        const skm_status status = skm_op_lookup_scale_grad(grad.t.get_device(), grad.t.const_data_ptr(), grad.ld, table.t.const_data_ptr(), table.ld, grad.kind, table.n, grad.d, ids.t.const_data_ptr(), ids.bits,
                                     grad.n, static_cast<float>(PyFloat_AS_DOUBLE(a[3])), out.data_ptr<float>(), stream(grad.t));
        if (status != SKM_OK) return failed(status);
        return wrap(out);
    });
}

// ids, n_clusters
PyObject* group_rows(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Ids ids;
        if (count != 2 || !ids.take(a[0]) || !PyLong_CheckExact(a[1])) return none();
        const int64_t dim = ids.t.dim(), n = ids.t.numel();
        const long long k = PyLong_AsLongLong(a[1]);
        if (k <= 0 || k >= kMostIds || dim < 1 || dim > 2 || (dim == 2 && ids.t.size(1) == 0)) {
            PyErr_Clear();
            return none();
        }
        const at::Tensor whole = make({2 * n + k + 1}, at::kInt, ids.t);
        const uint64_t bytes = skm_op_group_rows_workspace(n, k);
        const at::Tensor space = workspace(bytes, ids.t);
        uint32_t* p = static_cast<uint32_t*>(whole.data_ptr());
        const skm_status status = skm_op_group_rows(ids.t.get_device(), ids.t.const_data_ptr(), ids.bits, n, k, p, p + n, p + 2 * n, address(space), bytes, stream(ids.t));
        if (status != SKM_OK) return failed(status);
        PyObject* x = THPVariable_Wrap(whole.as_strided({n}, {1}, 0));
        PyObject* y = THPVariable_Wrap(dim == 1 ? whole.as_strided({n}, {1}, n) : whole.as_strided(ids.t.sizes(), ids.t.strides(), n));
        PyObject* z = THPVariable_Wrap(whole.as_strided({k + 1}, {1}, 2 * n));
        PyObject* all = x && y && z ? PyTuple_Pack(3, x, y, z) : nullptr;
        Py_XDECREF(x);
        Py_XDECREF(y);
        Py_XDECREF(z);
        return all;
    });
}

// x, order, position, offsets
PyObject* to_clusters(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Rows x;
        Places at;
        if (count != 4 || !x.take(a[0]) || !at.take(a + 1, x.t) || x.n != at.n) return none();
        const at::Tensor out = make({static_cast<int64_t>(at.n * at.m), static_cast<int64_t>(x.d)}, x.t.scalar_type(), x.t);
        const skm_status status = skm_op_to_clusters(x.t.get_device(), x.t.const_data_ptr(), x.ld, x.kind, x.d, at.pairs(), at.positions(), at.starts(), at.k, at.n, at.m, out.data_ptr(), stream(x.t));
        if (status != SKM_OK) return failed(status);
        return wrap(out);
    });
}

// y, order, position, offsets, weights
PyObject* from_clusters(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Rows y;
        Places at;
        Floats weights;
        if (count != 5 || !y.take(a[0]) || !at.take(a + 1, y.t) || !weights.take(a[4], at.position.sizes(), y.t) || y.n != at.n * at.m) return none();
        const at::Tensor out = make({static_cast<int64_t>(at.n), static_cast<int64_t>(y.d)}, y.t.scalar_type(), y.t);
        const skm_status status = skm_op_from_clusters(y.t.get_device(), y.t.const_data_ptr(), y.ld, y.kind, y.d, at.pairs(), at.positions(), at.starts(), at.k, at.n, at.m, weights.p(), out.data_ptr(), stream(y.t));
        if (status != SKM_OK) return failed(status);
        return wrap(out);
    });
}

// grad, y, order, position, offsets, weights (both gradients)
PyObject* from_clusters_grad(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Rows grad, y;
        Places at;
        Floats weights;
        if (count != 6 || a[5] == Py_None || !grad.take(a[0]) || !y.take(a[1], &grad.t) || !at.take(a + 2, grad.t) || !weights.take(a[5], at.position.sizes(), grad.t)) return none();
        if (grad.n != at.n || y.n != at.n * at.m || y.d != grad.d || y.kind != grad.kind) return none();
        const at::Tensor grad_y = make({static_cast<int64_t>(y.n), static_cast<int64_t>(y.d)}, grad.t.scalar_type(), grad.t);
        const at::Tensor grad_weights = make(at.position.sizes(), at::kFloat, grad.t);
        const skm_status status = skm_op_from_clusters_grad(grad.t.get_device(), grad.t.const_data_ptr(), grad.ld, y.t.const_data_ptr(), y.ld, grad.kind, grad.d, at.pairs(), at.positions(), at.starts(), at.k, at.n, at.m,
                                      weights.p(), grad_y.data_ptr(), grad_weights.data_ptr<float>(), stream(grad.t));
        if (status != SKM_OK) return failed(status);
        return wrap(grad_y, grad_weights);
    });
}

// x
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        Rows x;
        if (count != 1 || !x.take(a[0])) return none();
        const int64_t n = x.n, d = x.d, pitch = (d + 15) / 16 * 16;
        const at::Tensor q = make({n, pitch}, at::kChar, x.t), scales = make({n}, at::kFloat, x.t);
        const skm_status status = skm_op_quantize_rows(x.t.get_device(), x.t.const_data_ptr(), x.ld, x.kind, n, d, static_cast<int8_t*>(q.data_ptr()), pitch, scales.data_ptr<float>(), stream(x.t));
        if (status != SKM_OK) return failed(status);
        return wrap(pitch == d ? q : q.as_strided({n, d}, {pitch, 1}, 0), scales);
    });
}

// x, x_scales, w, w_scales, offsets, dtype's number
PyObject* product_8bit(PyObject*, PyObject* const* a, Py_ssize_t count) {
    return shortcut([&]() -> PyObject* {
        if (count != 6 || !plain(a[0]) || !plain(a[2]) || a[1] == Py_None || a[3] == Py_None || !PyLong_CheckExact(a[5])) return none();
        const at::Tensor& x = THPVariable_Unpack(a[0]);
        const at::Tensor& w = THPVariable_Unpack(a[2]);
        const bool grouped = a[4] != Py_None;
        const int64_t d = x.dim() == 2 ? x.size(1) : 0, last = w.dim() - 1;
        if (x.scalar_type() != at::kChar || w.scalar_type() != at::kChar || d == 0 || last != (grouped ? 2 : 1) || w.size(last) != d || w.get_device() != x.get_device()) return none();
        if (d > 1 && (x.stride(1) != 1 || w.stride(last) != 1)) return none();
        const int64_t n = x.size(0), m = w.size(last - 1), e = grouped ? w.size(0) : 0;
        Floats x_scales, w_scales;
        if (!x_scales.take(a[1], {n}, x) || !w_scales.take(a[3], w.sizes().slice(0, last), x)) return none();
        const uint32_t* offsets = nullptr;
        if (grouped) {
            if (!plain(a[4]) || e == 0 || m == 0 || (e > 1 && m > 1 && w.stride(0) != m * w.stride(1))) return none();
            const at::Tensor& o = THPVariable_Unpack(a[4]);
            if (o.scalar_type() != at::kInt || o.dim() != 1 || o.size(0) != e + 1 || !o.is_contiguous() || o.get_device() != x.get_device()) return none();
            offsets = static_cast<const uint32_t*>(o.const_data_ptr());
        }
        const long kind = PyLong_AsLong(a[5]);
        const uint64_t ld_x = n > 1 ? x.stride(0) : d, ld_w = m > 1 ? w.stride(last - 1) : e > 1 ? w.stride(0) : d;
        const auto *px = static_cast<const int8_t*>(x.const_data_ptr()), *pw = static_cast<const int8_t*>(w.const_data_ptr());
        const at::Tensor out = make({n, m}, kind == SKM_F32 ? at::kFloat : kind == SKM_F16 ? at::kHalf : at::kBFloat16, x);
        const uint64_t bytes = skm_op_product_8bit_workspace(px, ld_x, pw, ld_w, n, m, d, e);
        const at::Tensor space = workspace(bytes, x);
        const skm_status status = skm_op_product_8bit(x.get_device(), px, ld_x, x_scales.p(), pw, ld_w, w_scales.p(), n, m, d, e, offsets, out.data_ptr(), static_cast<int>(kind), address(space), bytes,
                                stream(x));
        if (status != SKM_OK) return failed(status);
        return wrap(out);
    });
}

#define SKM_CALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {SKM_CALL(ordinary),      SKM_CALL(lookup),           SKM_CALL(lookup_grad),        SKM_CALL(lookup_scale_grad), SKM_CALL(group_rows), SKM_CALL(to_clusters),
                         SKM_CALL(from_clusters), SKM_CALL(from_clusters_grad), SKM_CALL(quantize_rows),     SKM_CALL(product_8bit), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

// `built_for` says for which torch and Python: the layouts of their objects are compiled in.
PyMODINIT_FUNC PyInit__ops_calls() {
    PyObject* made = PyModule_Create(&module);
    if (made && PyModule_AddStringConstant(made, "built_for", SKM_BUILT_FOR) < 0) {
        Py_DECREF(made);
        return nullptr;
    }
    return made;
}
