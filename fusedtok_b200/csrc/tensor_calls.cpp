// The plain calls of a decode loop on an 8-bit cache, from Python to the C ABI in one step: a CPython module
// (fusedtok_b200/_tensors.so) over torch's C++ tensors.
//
// A decode step makes a few of these calls per layer, and the checks, the allocations and the argument conversion of the
// Python wrappers cost more than the launches (8 - 15 us a call, of which the launches are 2.5 - 5). Each function here
// looks at the operands of one call; if they are what the operator takes as they stand (CUDA tensors of the right types,
// contiguous, on the current device, shapes that agree) it allocates the results, calls the C ABI on the current stream
// and returns them. In every other case it returns None and has done nothing: the wrapper then finds out what is wrong, or
// converts what may be converted, and launches through ctypes. Nothing else is reached only from here: with this module
// missing every call takes the wrapper's way.
//
// The module is not linked to the library: bind() gets the addresses of the entry points that ctypes has loaded, so both
// call the same build.

#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>
#include <ATen/ops/empty.h>

#include "../../include/fusedtok_b200.h"

namespace {

decltype(&fusedtok_last_error) last_error = nullptr;
decltype(&fusedtok_attention_decode_paged_q8_workspace) decode_workspace = nullptr;
decltype(&fusedtok_attention_decode_paged_q8_launch) decode_launch = nullptr;
decltype(&fusedtok_kv_append_paged_q8_launch) append_launch = nullptr;
decltype(&fusedtok_block_table_extend_launch) extend_launch = nullptr;
decltype(&fusedtok_block_table_trim_launch) trim_launch = nullptr;
PyObject* step_type = nullptr;                 // BlockTableStep

// The tensor behind a Python object, or null.
const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// Operands of one call: `ok` while all are contiguous CUDA tensors with the types asked for on the current device.
struct Operands {
    bool ok = true;
    int device = -1;
    const at::Tensor* take(PyObject* o, at::ScalarType type, int64_t dims) {
        const at::Tensor* t = tensor_of(o);
        if (!t || !t->is_cuda() || t->scalar_type() != type || t->dim() != dims || !t->is_contiguous()) {
            ok = false;
            return nullptr;
        }
        if (device < 0) {
            device = t->get_device();
            if (device != c10::cuda::current_device()) ok = false;
        } else if (t->get_device() != device) {
            ok = false;
        }
        return t;
    }
    uintptr_t stream() const { return reinterpret_cast<uintptr_t>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream()); }
};
int storage_code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }
int code_type(at::ScalarType t) { return t == at::kChar ? 0 : t == at::kFloat8_e4m3fn ? 1 : -1; }
bool fits_int(int64_t x) { return x <= 0x7fffffff; }
template <typename T> T* data(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

// Other Python threads run while a call allocates and launches: a launch waits where the stream's queue is full, which may
// be until one of them has done its part. Nothing of Python's may be touched meanwhile.
struct Unlocked {
    PyThreadState* const state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked&) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject* declined() { Py_RETURN_NONE; }
PyObject* failed(int rc) {
    PyErr_SetString(rc == FUSEDTOK_INVALID_ARGUMENT ? PyExc_ValueError : PyExc_RuntimeError, last_error());
    return nullptr;
}
// A Python int within [lo, 2^31), or -1.
int64_t whole(PyObject* o, int64_t lo) {
    if (!PyLong_Check(o)) return -1;
    int overflow = 0;
    const long long x = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow || x < lo || x > 0x7fffffff ? -1 : x;
}

// The pools and scales of an 8-bit cache whose types and shapes agree.
struct Cache {
    const at::Tensor *k = nullptr, *v = nullptr, *scales = nullptr;
    int store = -1;
    int64_t blocks = 0, heads = 0, page = 0, dim = 0;
    bool take(Operands& in, PyObject* k_pool, PyObject* v_pool, PyObject* kv_scales) {
        const at::Tensor* t = tensor_of(k_pool);
        if (!t || (store = code_type(t->scalar_type())) < 0) return false;
        k = in.take(k_pool, t->scalar_type(), 4);
        v = in.take(v_pool, t->scalar_type(), 4);
        scales = in.take(kv_scales, at::kFloat, 3);
        if (!in.ok) return false;
        blocks = k->size(0);
        heads = k->size(1);
        page = k->size(2);
        dim = k->size(3);
        return v->sizes() == k->sizes() && scales->size(0) == blocks && scales->size(1) == heads && scales->size(2) == 2 &&
               page >= 1 && fits_int(heads) && fits_int(page) && fits_int(dim);
    }
};

PyObject* attention_decode_paged_q8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !decode_launch) return declined();
    const at::Tensor* first = tensor_of(args[0]);
    const int dtype = first ? storage_code(first->scalar_type()) : -1;
    if (dtype < 0) return declined();
    Operands in;
    Cache cache;
    const at::Tensor* q = in.take(args[0], first->scalar_type(), 3);
    if (!cache.take(in, args[1], args[2], args[3])) return declined();
    const at::Tensor* table = in.take(args[4], at::kInt, 2);
    const at::Tensor* lens = args[5] == Py_None ? nullptr : in.take(args[5], at::kInt, 1);
    if (!in.ok) return declined();
    const int64_t b = q->size(0), hq = q->size(1), d = q->size(2), width = table->size(1);
    if (b < 1 || d != cache.dim || cache.heads < 1 || hq < 1 || hq % cache.heads || table->size(0) != b || !fits_int(b) ||
        !fits_int(hq) || !fits_int(width) || (lens && lens->size(0) != b))
        return declined();
    at::Tensor out;
    int rc = 0;
    {
        Unlocked other_threads;
        const long long need = decode_workspace(dtype, (int)b, (int)hq, (int)cache.heads, (int)cache.page, (int)width, (int)d);
        if (need < 0) {
            rc = (int)-need;
        } else {
            out = at::empty(q->sizes(), q->options());
            at::Tensor scratch = at::empty({(need + 3) / 4}, cache.scales->options());
            rc = decode_launch(dtype, cache.store, q->data_ptr(), cache.k->data_ptr(), cache.v->data_ptr(), data<float>(*cache.scales),
                               data<int>(*table), lens ? data<int>(*lens) : nullptr, out.data_ptr(), scratch.data_ptr(), need,
                               (int)b, (int)hq, (int)cache.heads, (int)cache.page, (int)width, cache.blocks, (int)d, in.stream());
        }
    }
    if (rc) return failed(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// True: done.
PyObject* kv_append_paged_q8(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !append_launch) return declined();
    const at::Tensor* first = tensor_of(args[3]);
    const int dtype = first ? storage_code(first->scalar_type()) : -1;
    if (dtype < 0) return declined();
    Operands in;
    Cache cache;
    if (!cache.take(in, args[0], args[1], args[2])) return declined();
    const at::Tensor* k_new = in.take(args[3], first->scalar_type(), 3);
    const at::Tensor* v_new = in.take(args[4], first->scalar_type(), 3);
    const at::Tensor* slots = in.take(args[5], at::kInt, 1);
    if (!in.ok) return declined();
    const int64_t tokens = k_new->size(0);
    if (tokens < 1 || !fits_int(tokens) || v_new->sizes() != k_new->sizes() || k_new->size(1) != cache.heads ||
        k_new->size(2) != cache.dim || slots->size(0) != tokens)
        return declined();
    int rc = 0;
    {
        Unlocked other_threads;
        rc = append_launch(dtype, cache.store, k_new->data_ptr(), v_new->data_ptr(), data<int>(*slots), cache.k->data_ptr(),
                           cache.v->data_ptr(), data<float>(*cache.scales), (int)tokens, (int)cache.heads, (int)cache.dim,
                           (int)cache.page, cache.blocks, in.stream());
    }
    if (rc) return failed(rc);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// Operands common to the block table calls.
struct Table {
    const at::Tensor *table = nullptr, *lens = nullptr, *change = nullptr, *free_blocks = nullptr, *free_count = nullptr;
    int64_t b = 0, width = 0, page = -1;
    bool take(Operands& in, PyObject* const* args) {
        table = in.take(args[0], at::kInt, 2);
        lens = in.take(args[1], at::kInt, 1);
        change = in.take(args[2], at::kInt, 1);
        free_blocks = in.take(args[3], at::kInt, 1);
        free_count = in.take(args[4], at::kInt, 1);
        page = whole(args[5], 1);
        if (!in.ok || page < 1) return false;
        b = table->size(0);
        width = table->size(1);
        return lens->size(0) == b && change->size(0) == b && free_count->size(0) == 1 && fits_int(b) && fits_int(width) &&
               fits_int(free_blocks->size(0));
    }
};

PyObject* block_table_extend(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !extend_launch) return declined();
    Operands in;
    Table t;
    const int64_t tokens = whole(args[6], 0);
    if (tokens < 0 || !t.take(in, args)) return declined();
    at::Tensor made[4];
    int rc = 0;
    {
        Unlocked other_threads;
        const auto options = t.lens->options();
        const int64_t sizes[4] = {tokens, t.b + 1, t.b, 1};
        for (int i = 0; i < 4; ++i) made[i] = at::empty({sizes[i]}, options);
        rc = extend_launch(data<int>(*t.table), data<int>(*t.lens), data<int>(*t.change), data<int>(*t.free_blocks),
                           data<int>(*t.free_count), data<int>(made[0]), data<int>(made[1]), data<int>(made[2]), data<int>(made[3]),
                           (int)t.b, (int)t.width, (int)t.page, (int)t.free_blocks->size(0), (int)tokens, in.stream());
    }
    if (rc) return failed(rc);
    PyObject* results[4] = {nullptr, nullptr, nullptr, nullptr};
    PyObject* step = nullptr;
    bool all = true;
    for (int i = 0; i < 4 && all; ++i) all = (results[i] = THPVariable_Wrap(std::move(made[i]))) != nullptr;
    if (all) step = PyObject_Vectorcall(step_type, results, 4, nullptr);
    for (PyObject* r : results) Py_XDECREF(r);
    return step;
    END_HANDLE_TH_ERRORS
}

PyObject* block_table_trim(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !trim_launch) return declined();
    Operands in;
    Table t;
    if (!t.take(in, args)) return declined();
    at::Tensor lens, count;
    int rc = 0;
    {
        Unlocked other_threads;
        lens = at::empty({t.b}, t.lens->options());
        count = at::empty({1}, t.lens->options());
        rc = trim_launch(data<int>(*t.table), data<int>(*t.lens), data<int>(*t.change), data<int>(*t.free_blocks),
                         data<int>(*t.free_count), data<int>(lens), data<int>(count), (int)t.b, (int)t.width, (int)t.page,
                         (int)t.free_blocks->size(0), in.stream());
    }
    if (rc) return failed(rc);
    PyObject* a = THPVariable_Wrap(std::move(lens));
    PyObject* c = a ? THPVariable_Wrap(std::move(count)) : nullptr;
    PyObject* both = c ? PyTuple_Pack(2, a, c) : nullptr;
    Py_XDECREF(a);
    Py_XDECREF(c);
    return both;
    END_HANDLE_TH_ERRORS
}

// bind(address of each entry point below, BlockTableStep)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "bind: six addresses and the type of a step are expected");
        return nullptr;
    }
    void* at[6];
    for (int i = 0; i < 6; ++i) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (!at[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
            return nullptr;
        }
    }
    last_error = reinterpret_cast<decltype(last_error)>(at[0]);
    decode_workspace = reinterpret_cast<decltype(decode_workspace)>(at[1]);
    decode_launch = reinterpret_cast<decltype(decode_launch)>(at[2]);
    append_launch = reinterpret_cast<decltype(append_launch)>(at[3]);
    extend_launch = reinterpret_cast<decltype(extend_launch)>(at[4]);
    trim_launch = reinterpret_cast<decltype(trim_launch)>(at[5]);
    Py_XDECREF(step_type);
    Py_INCREF(args[6]);
    step_type = args[6];
    Py_RETURN_NONE;
}

#define FTK_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FTK_METHOD(attention_decode_paged_q8), FTK_METHOD(kv_append_paged_q8), FTK_METHOD(block_table_extend),
                         FTK_METHOD(block_table_trim), FTK_METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);      // whose classes it was built for
    return m;
}
