// Calls of the paged-cache operators from Python, for layouts whose checks
// have passed before.
//
// neuralzip_b200.gpu.paged checks a call's tensors in Python and makes it
// through ctypes, 15 to 35 us of host time. It then registers the call's
// layout here: types, shapes, strides, devices and sizes (no
// addresses, no contents), with the part of the C struct that they fix. A
// call of a known layout only allocates its outputs, fills in the addresses
// and enqueues, in 4.4 to 7 us. Everything else returns None, and the caller takes the
// checking path, which also words the errors.

#include "nz_b200.h"

#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <string>
#include <unordered_map>

namespace {

using Call = int (*)(const void*, void*);

constexpr size_t kMostLayouts = 4096;

struct Layout {
    std::string tail;       // the struct behind its addresses
    int64_t workspace = 0;  // bytes
    float scale = 0.0f;
};

// One operator: its C entry point and its known layouts.
struct Operator {
    Call call = nullptr;
    std::unordered_map<std::string, Layout> layouts;
};
Operator g_operators[4];
enum { kReserve, kRelease, kRotary, kAttention };

// A call's tensors, and the key of its layout.
struct Arguments {
    std::string key;
    bool good = true;

    void number(int64_t x) { key.append(reinterpret_cast<const char*>(&x), sizeof(x)); }
    // A tensor, or null for None. Anything else is for the checking path.
    const at::Tensor* tensor(PyObject* object) {
        if (object == Py_None) {
            number(-1);
            return nullptr;
        }
        if (!THPVariable_CheckExact(object)) {
            good = false;
            return nullptr;
        }
        const at::Tensor& t = THPVariable_Unpack(object);
        if (!t.is_cuda()) {
            good = false;
            return nullptr;
        }
        number(static_cast<int64_t>(t.scalar_type()) << 32 | t.device().index() << 8 | t.dim());
        key.append(reinterpret_cast<const char*>(t.sizes().data()), t.dim() * sizeof(int64_t));
        key.append(reinterpret_cast<const char*>(t.strides().data()), t.dim() * sizeof(int64_t));
        return &t;
    }
    void whole(PyObject* object) {
        if (object == Py_None) return number(-1);
        if (!PyLong_CheckExact(object)) {
            good = false;
            return;
        }
        int overflow = 0;
        const int64_t x = PyLong_AsLongLongAndOverflow(object, &overflow);
        if (overflow || x < 0) good = false;
        number(x);
    }
    void flag(PyObject* object) { number(PyObject_IsTrue(object) == 1); }
    const Layout* find(int op) const {
        if (!good) return nullptr;
        const auto it = g_operators[op].layouts.find(key);
        return it == g_operators[op].layouts.end() ? nullptr : &it->second;
    }
};

uint64_t address(const at::Tensor* t) { return t ? reinterpret_cast<uint64_t>(t->data_ptr()) : 0U; }

// Of either mode: the forward one has a single level, and no_grad does not turn it off.
bool needs_gradient(std::initializer_list<const at::Tensor*> tensors) {
    const bool backward = c10::GradMode::is_enabled();
    for (const at::Tensor* t : tensors)
        if (t && ((backward && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
    return false;
}

// Tells autograd of tensors written in place, so that a backward pass that
// saved one is refused.
void wrote(std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* t : tensors)
        if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// A number that float holds; false (and no Python error) otherwise.
bool number(PyObject* object, float* out) {
    const double x = PyFloat_AsDouble(object);
    if (x == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    *out = static_cast<float>(x);
    return std::isfinite(*out) || !std::isfinite(x);
}

// The call itself: the addresses, then the layout's tail, then `more`.
int enqueue(int op, const Layout& layout, const uint64_t* addresses, size_t count, const void* more, size_t more_size,
            const at::Tensor& on) {
    alignas(8) char args[512];
    const size_t size = count * sizeof(uint64_t) + layout.tail.size() + more_size;
    if (size > sizeof(args)) return NZ_ERUNTIME;
    std::memcpy(args, addresses, count * sizeof(uint64_t));
    std::memcpy(args + count * sizeof(uint64_t), layout.tail.data(), layout.tail.size());
    std::memcpy(args + count * sizeof(uint64_t) + layout.tail.size(), more, more_size);
    const c10::cuda::CUDAGuard guard(on.device());
    return g_operators[op].call(args, c10::cuda::getCurrentCUDAStream(on.device().index()).stream());
}

// A status for the caller to raise.
PyObject* failed(int status) { return PyLong_FromLong(status); }

at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }

// Elements [first, first + size) of a fresh vector, as a tensor of its own
// over the same memory.
at::Tensor part(const at::Tensor& whole, int64_t first, int64_t size) {
    auto impl = whole.unsafeGetTensorImpl()->shallow_copy_and_detach(c10::VariableVersion(0), true);
    const int64_t sizes[] = {size}, strides[] = {1};
    impl->set_sizes_and_strides(at::IntArrayRef(sizes), at::IntArrayRef(strides), first);
    return at::Tensor(std::move(impl));
}

// A tuple of new references; null when one of them is.
PyObject* tuple_of(std::initializer_list<PyObject*> items) {
    PyObject* result = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
    bool good = result != nullptr;
    Py_ssize_t i = 0;
    for (PyObject* item : items) {
        good = good && item;
        if (result && item) PyTuple_SET_ITEM(result, i++, item);
        else Py_XDECREF(item);
    }
    if (!good) Py_CLEAR(result);
    return result;
}

// Everything behind a Python entry point: C++ exceptions become Python's.
template <typename Body>
PyObject* guarded(Body body) {
    try {
        return body();
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

struct ReserveArguments : Arguments {
    const at::Tensor *lengths, *new_tokens, *table, *free_pages, *used, *lengths_out, *used_out;
    int64_t rows = 0;

    // lengths, new_tokens, block_table, free_pages, used, page_size, rows, row_stride, lengths_out, used_out
    explicit ReserveArguments(PyObject* const* a) {
        lengths = tensor(a[0]), new_tokens = tensor(a[1]), table = tensor(a[2]), free_pages = tensor(a[3]), used = tensor(a[4]);
        whole(a[5]), whole(a[6]), whole(a[7]);
        lengths_out = tensor(a[8]), used_out = tensor(a[9]);
        if (good) rows = a[6] == Py_None ? 0 : PyLong_AsLongLong(a[6]);
    }
};

bool overlaps_in_part(const at::Tensor* out, const at::Tensor& source) {
    if (!out) return false;
    const int64_t apart = static_cast<int64_t>(address(out)) - static_cast<int64_t>(address(&source));
    return apart != 0 && std::llabs(apart) < 4 * source.numel();
}

PyObject* reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 10) Py_RETURN_NONE;
        const ReserveArguments args(a);
        const Layout* layout = args.find(kReserve);
        if (!layout || overlaps_in_part(args.lengths_out, *args.lengths)) Py_RETURN_NONE;
        const int64_t requests = args.lengths->numel(), rows = args.rows;
        const at::Tensor out = fresh({2 * rows + 2 * requests + 3}, at::kInt, *args.lengths);
        const at::Tensor positions = part(out, 0, rows), slots = part(out, rows, rows);
        const at::Tensor offsets = part(out, 2 * rows, requests + 1), refused = part(out, 2 * rows + requests + 1, 1);
        const at::Tensor lengths_out = args.lengths_out ? *args.lengths_out : part(out, 2 * rows + requests + 2, requests);
        const at::Tensor used_out = args.used_out ? *args.used_out : part(out, 2 * rows + 2 * requests + 2, 1);
        const uint64_t addresses[] = {address(args.lengths), address(args.new_tokens), address(args.table),
                                      address(args.free_pages), address(args.used), address(&positions), address(&slots),
                                      address(&offsets), address(&lengths_out), address(&used_out), address(&refused)};
        const int status = enqueue(kReserve, *layout, addresses, 11, nullptr, 0, *args.lengths);
        if (status) return failed(status);
        wrote({args.table, args.lengths_out, args.used_out});
        return tuple_of({THPVariable_Wrap(positions), THPVariable_Wrap(slots), THPVariable_Wrap(offsets),
                         args.lengths_out ? Py_NewRef(a[8]) : THPVariable_Wrap(lengths_out),
                         args.used_out ? Py_NewRef(a[9]) : THPVariable_Wrap(used_out), THPVariable_Wrap(refused)});
    });
}

struct ReleaseArguments : Arguments {
    const at::Tensor *lengths, *done, *table, *free_pages, *used, *lengths_out, *used_out;

    // lengths, done, block_table, free_pages, used, page_size, lengths_out, used_out
    explicit ReleaseArguments(PyObject* const* a) {
        lengths = tensor(a[0]), done = tensor(a[1]), table = tensor(a[2]), free_pages = tensor(a[3]), used = tensor(a[4]);
        whole(a[5]);
        lengths_out = tensor(a[6]), used_out = tensor(a[7]);
    }
};

PyObject* release(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 8) Py_RETURN_NONE;
        const ReleaseArguments args(a);
        const Layout* layout = args.find(kRelease);
        if (!layout || overlaps_in_part(args.lengths_out, *args.lengths)) Py_RETURN_NONE;
        const at::Tensor lengths_out = args.lengths_out ? *args.lengths_out : fresh_like(*args.lengths);
        const at::Tensor used_out = args.used_out ? *args.used_out : fresh_like(*args.used);
        const uint64_t addresses[] = {address(args.lengths),    address(args.done), address(args.table),
                                      address(args.free_pages), address(args.used), address(&lengths_out),
                                      address(&used_out)};
        const int status = enqueue(kRelease, *layout, addresses, 7, nullptr, 0, *args.lengths);
        if (status) return failed(status);
        wrote({args.free_pages, args.lengths_out, args.used_out});
        return tuple_of({args.lengths_out ? Py_NewRef(a[6]) : THPVariable_Wrap(lengths_out),
                         args.used_out ? Py_NewRef(a[7]) : THPVariable_Wrap(used_out)});
    });
}

struct RotaryArguments : Arguments {
    const at::Tensor *query, *key_, *value, *positions, *slots, *rotary, *key_pages, *value_pages, *query_norm, *key_norm,
        *query_out, *key_out;

    // query, key, value, positions, slots, rotary, key_pages, value_pages, interleaved, query_norm, key_norm,
    // query_out, key_out, eps
    explicit RotaryArguments(PyObject* const* a) {
        query = tensor(a[0]), key_ = tensor(a[1]), value = tensor(a[2]), positions = tensor(a[3]), slots = tensor(a[4]);
        rotary = tensor(a[5]), key_pages = tensor(a[6]), value_pages = tensor(a[7]);
        flag(a[8]);
        query_norm = tensor(a[9]), key_norm = tensor(a[10]), query_out = tensor(a[11]), key_out = tensor(a[12]);
    }
};

PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 14) Py_RETURN_NONE;
        const RotaryArguments args(a);
        const Layout* layout = args.find(kRotary);
        float eps[2] = {0.0f, 0.0f};
        if (!layout || !number(a[13], eps) ||
            needs_gradient({args.query, args.key_, args.value, args.rotary, args.query_norm, args.key_norm, args.key_pages,
                            args.value_pages, args.query_out, args.key_out}))
            Py_RETURN_NONE;
        const at::Tensor out = args.query_out ? *args.query_out : fresh_like(*args.query);
        const uint64_t addresses[] = {address(args.query),      address(args.key_),      address(args.value),
                                      address(&out),            address(args.key_out),   address(args.key_pages),
                                      address(args.value_pages), address(args.positions), address(args.slots),
                                      address(args.rotary),     address(args.query_norm), address(args.key_norm)};
        const int status = enqueue(kRotary, *layout, addresses, 12, eps, sizeof(eps), *args.query);
        if (status) return failed(status);
        wrote({args.key_pages, args.value_pages, args.query_out, args.key_out});
        return args.query_out ? Py_NewRef(a[11]) : THPVariable_Wrap(out);
    });
}

struct AttentionArguments : Arguments {
    const at::Tensor *query, *key_pages, *value_pages, *table, *lengths, *out;

    // query, key_pages, value_pages, block_table, lengths, window, out, scale, return_lse
    explicit AttentionArguments(PyObject* const* a) {
        query = tensor(a[0]), key_pages = tensor(a[1]), value_pages = tensor(a[2]), table = tensor(a[3]), lengths = tensor(a[4]);
        whole(a[5]);
        out = tensor(a[6]);
    }
};

PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 9) Py_RETURN_NONE;
        const AttentionArguments args(a);
        const Layout* layout = args.find(kAttention);
        if (!layout || ((address(args.key_pages) | address(args.value_pages)) & 15U) ||
            needs_gradient({args.query, args.key_pages, args.value_pages, args.out}))
            Py_RETURN_NONE;
        float scale = layout->scale;
        if (a[7] != Py_None && !number(a[7], &scale)) Py_RETURN_NONE;
        const int return_lse = PyObject_IsTrue(a[8]);
        if (return_lse < 0) return nullptr;
        const at::Tensor out = args.out ? *args.out : fresh_like(*args.query);
        at::Tensor lse, workspace;
        if (return_lse)
            lse = fresh({args.query->size(0), args.query->size(1)}, at::kFloat, *args.query);
        if (layout->workspace) workspace = fresh({layout->workspace}, at::kByte, *args.query);
        const uint64_t addresses[] = {address(args.query),   address(args.key_pages), address(args.value_pages),
                                      address(args.table),   address(args.lengths),   address(&out),
                                      return_lse ? address(&lse) : 0U, layout->workspace ? address(&workspace) : 0U};
        const int status = enqueue(kAttention, *layout, addresses, 8, &scale, sizeof(scale), *args.query);
        if (status) return failed(status);
        wrote({args.out});
        PyObject* first = args.out ? Py_NewRef(a[6]) : THPVariable_Wrap(out);
        return return_lse ? tuple_of({first, THPVariable_Wrap(lse)}) : first;
    });
}

// remember(operator, arguments of its call, tail bytes, workspace bytes, default scale)
PyObject* remember(PyObject*, PyObject* arguments) {
    return guarded([&]() -> PyObject* {
        int op = 0;
        PyObject* call = nullptr;
        const char* tail = nullptr;
        Py_ssize_t size = 0;
        long long workspace = 0;
        double scale = 0.0;
        if (!PyArg_ParseTuple(arguments, "iO!y#Ld", &op, &PyTuple_Type, &call, &tail, &size, &workspace, &scale)) return nullptr;
        PyObject* const* a = &PyTuple_GET_ITEM(call, 0);
        const Py_ssize_t wanted[] = {10, 8, 14, 9};
        if (op < 0 || op > 3 || PyTuple_GET_SIZE(call) != wanted[op]) {
            PyErr_SetString(PyExc_ValueError, "No such call.");
            return nullptr;
        }
        const Arguments found = op == kReserve   ? static_cast<const Arguments&>(ReserveArguments(a))
                                : op == kRelease ? static_cast<const Arguments&>(ReleaseArguments(a))
                                : op == kRotary  ? static_cast<const Arguments&>(RotaryArguments(a))
                                                 : static_cast<const Arguments&>(AttentionArguments(a));
        if (found.good) {
            auto& layouts = g_operators[op].layouts;
            if (layouts.size() >= kMostLayouts) layouts.clear();
            Layout layout;
            layout.tail.assign(tail, static_cast<size_t>(size));
            layout.workspace = workspace;
            layout.scale = static_cast<float>(scale);
            layouts[found.key] = layout;
        }
        Py_RETURN_NONE;
    });
}

// bind(addresses of nz_pages_reserve, nz_pages_release, nz_rotary_store, nz_paged_attention)
PyObject* bind(PyObject*, PyObject* arguments) {
    unsigned long long at[4];
    if (!PyArg_ParseTuple(arguments, "KKKK", &at[0], &at[1], &at[2], &at[3])) return nullptr;
    for (int i = 0; i < 4; ++i) {
        g_operators[i].call = reinterpret_cast<Call>(at[i]);
        g_operators[i].layouts.clear();
    }
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"remember", remember, METH_VARARGS, nullptr},
    {"reserve", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(reserve)), METH_FASTCALL, nullptr},
    {"release", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(release)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "nz_paged_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_nz_paged_torch() { return PyModule_Create(&g_module); }
