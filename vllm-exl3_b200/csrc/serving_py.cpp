// serving_py.cpp -- the short way from Python into the serving entries.
//
// The operators run for a few microseconds, and a call from Python spends
// three times that on attribute lookups, a ctypes call and views.  Each
// function here takes the tensors as they are, looks whether everything is as
// the kernels want it, allocates the outputs and makes the C call of
// include/exl3_b200.h.  Where anything is not (a wrong type, a layout that
// needs a copy, tensors on another than the current device), it does nothing
// and returns None: the Python function then goes its own way, which refuses
// or copies, and is complete without this file.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/grad_mode.h>
#include <cmath>
#include <exception>
#include <map>
#include <utility>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/exl3_b200.h"

namespace {

struct Entries {
    int (*plan)(const exl3_kv_plan_args*, void*) = nullptr;
    int (*append)(const exl3_kv_append_args*, void*) = nullptr;
    int (*attend)(const exl3_kv_attend_args*, void*) = nullptr;
    size_t (*attend_bytes)(int, int, int, int, int, int64_t) = nullptr;
    int (*logprobs)(const exl3_token_logprobs_args*, void*) = nullptr;
    size_t (*logprobs_bytes)(int64_t, int64_t, int, int) = nullptr;
    uint64_t (*capture_id)(void*) = nullptr;
} entry;
PyObject* workspace_of = nullptr;  // (device index, stream, bytes, capture) -> (address, bytes)
PyObject* check = nullptr;         // (status, operator's name): raises

// Raised by the helpers below when the short way is not open.
struct NotHere {};

const at::Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) throw NotHere();
    return THPVariable_Unpack(o);
}

void want(bool ok) {
    if (!ok) throw NotHere();
}

bool plain_i32(const at::Tensor& t, int64_t dims, const c10::Device& dev) {
    return t.scalar_type() == at::kInt && t.dim() == dims && t.is_contiguous() && t.device() == dev;
}

int64_t whole(PyObject* o) {
    want(PyLong_Check(o));
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw NotHere();
    }
    return v;
}

// autograd wants to know of it
bool recorded(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

struct PyFailed {};

bool truth(PyObject* o) {  // as Python's `if`
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PyFailed();
    return v != 0;
}

c10::Device current(const at::Tensor& t) {
    const c10::Device dev = t.device();
    want(dev.is_cuda() && dev.index() == c10::cuda::current_device());
    return dev;
}

struct Space {
    void* at;
    int64_t bytes;
};

// Eager calls' workspaces, asked for before: they stay for the life of the process (0.5 us a call)
std::map<std::pair<int, cudaStream_t>, Space> known;

Space workspace(const c10::Device& dev, cudaStream_t stream, size_t need) {
    const unsigned long long capture = entry.capture_id(stream);
    const std::pair<int, cudaStream_t> where(dev.index(), stream);
    if (capture == 0) {
        const auto k = known.find(where);
        if (k != known.end() && size_t(k->second.bytes) >= need) return k->second;
    }
    PyObject* r = PyObject_CallFunction(workspace_of, "iLnK", int(dev.index()), (long long)(intptr_t)stream, Py_ssize_t(need), capture);
    if (!r) throw PyFailed();
    Space s{PyLong_AsVoidPtr(PyTuple_GET_ITEM(r, 0)), PyLong_AsLongLong(PyTuple_GET_ITEM(r, 1))};
    Py_DECREF(r);
    if (capture == 0) known[where] = s;
    return s;
}

void checked(int rc, const char* who) {
    if (rc == EXL3_OK) return;
    if (rc == EXL3_ERR_ARG) throw NotHere();  // nothing was launched: the long way says what is wrong
    PyObject* r = PyObject_CallFunction(check, "is", rc, who);
    Py_XDECREF(r);
    if (!r) throw PyFailed();
}

// A part of a flat tensor
at::Tensor part(const at::Tensor& t, int64_t from, int64_t n) { return t.narrow(0, from, n); }

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

struct Cache {
    int64_t code, pages, heads, page, dim;
    c10::Device dev;
};

Cache cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs) {
    const c10::Device dev = current(k);
    const bool e4m3 = k.scalar_type() == at::kFloat8_e4m3fn;
    want((e4m3 || k.scalar_type() == at::kChar) && v.scalar_type() == k.scalar_type() && k.dim() == 4 &&
         v.sizes() == k.sizes() && k.size(1) > 0 && k.is_contiguous() && v.is_contiguous() && v.device() == dev);
    for (const at::Tensor* s : {&ks, &vs})
        want(s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == k.size(0) && s->size(1) == k.size(1) &&
             s->is_contiguous() && s->device() == dev);
    return Cache{e4m3 ? EXL3_KV_E4M3 : EXL3_KV_INT8, k.size(0), k.size(1), k.size(2), k.size(3), dev};
}

int64_t row_type(const at::Tensor& t) {
    want(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16);
    return t.scalar_type() == at::kHalf ? EXL3_DT_F16 : EXL3_DT_BF16;
}

// rows as the kernels read them: values side by side, rows at multiples of 16 bytes
bool rows_ready(const at::Tensor& t) {
    return t.dim() == 3 && t.stride(2) == 1 && ((t.stride(0) | t.stride(1)) & 7) == 0 &&
           (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

template <class T>
T* data(const at::Tensor& t) {
    return static_cast<T*>(t.data_ptr());
}

PyObject* plan_(PyObject* const* a) {
    const at::Tensor &lens = tensor(a[0]), &fresh = tensor(a[1]), &table = tensor(a[2]), &free_pages = tensor(a[3]), &cursor = tensor(a[4]);
    const int64_t page = whole(a[5]), n = whole(a[6]);
    const c10::Device dev = current(lens);
    const int64_t B = lens.numel();
    want(plain_i32(lens, 1, dev) && plain_i32(fresh, 1, dev) && plain_i32(free_pages, 1, dev) && plain_i32(cursor, 1, dev) &&
         plain_i32(table, 2, dev) && fresh.numel() == B && table.size(0) == B && cursor.numel() == 1 && n >= 0);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index());
    const Space ws = workspace(dev, stream, 0);
    const at::Tensor ints = at::empty({n + 2 * B + 2}, lens.options()), slots = at::empty({n}, lens.options().dtype(at::kLong));
    int32_t* at = data<int32_t>(ints);
    exl3_kv_plan_args c{};
    c.lens = data<int32_t>(lens), c.new_tokens = data<int32_t>(fresh), c.requests = B, c.block_table = data<int32_t>(table);
    c.width = table.size(1), c.free_pages = data<int32_t>(free_pages), c.n_free = free_pages.numel();
    c.cursor = data<int32_t>(cursor), c.page = page, c.n_tokens = n, c.positions = at, c.kv_lens = at + n;
    c.cu_tokens = at + n + B, c.cursor_out = at + n + 2 * B + 1, c.slots = data<int64_t>(slots);
    c.status = static_cast<int*>(ws.at);
    checked(entry.plan(&c, stream), "kv_plan");
    PyObject* out = PyTuple_New(5);
    if (!out) throw PyFailed();
    PyTuple_SET_ITEM(out, 0, wrap(part(ints, n, B)));
    PyTuple_SET_ITEM(out, 1, wrap(part(ints, n + B, B + 1)));
    PyTuple_SET_ITEM(out, 2, wrap(part(ints, 0, n)));
    PyTuple_SET_ITEM(out, 3, wrap(slots));
    PyTuple_SET_ITEM(out, 4, wrap(part(ints, n + 2 * B + 1, 1)));
    return out;
}

PyObject* append_(PyObject* const* a) {
    const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &slots = tensor(a[2]);
    const at::Tensor &kc = tensor(a[3]), &vc = tensor(a[4]), &ks = tensor(a[5]), &vs = tensor(a[6]);
    const Cache m = cache(kc, vc, ks, vs);
    const int64_t n = slots.numel();
    want(rows_ready(k) && rows_ready(v) && k.scalar_type() == v.scalar_type() && k.size(0) == n && k.size(1) == m.heads &&
         k.size(2) == m.dim && v.sizes() == k.sizes() && k.device() == m.dev && v.device() == m.dev &&
         slots.device() == m.dev && slots.scalar_type() == at::kLong && slots.is_contiguous());
    exl3_kv_append_args c{};
    c.x_dtype = row_type(k);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(m.dev.index());
    const Space ws = workspace(m.dev, stream, 0);
    c.k = k.data_ptr(), c.k_tok_stride = k.stride(0), c.k_head_stride = k.stride(1);
    c.v = v.data_ptr(), c.v_tok_stride = v.stride(0), c.v_head_stride = v.stride(1);
    c.slots = data<int64_t>(slots), c.tokens = n, c.k_cache = kc.data_ptr(), c.v_cache = vc.data_ptr();
    c.k_scale = data<float>(ks), c.v_scale = data<float>(vs), c.code = m.code, c.pages = m.pages, c.kv_heads = m.heads;
    c.page = m.page, c.dim = m.dim, c.status = static_cast<int*>(ws.at);
    checked(entry.append(&c, stream), "kv_append");
    Py_RETURN_TRUE;
}

PyObject* attend_(PyObject* const* a) {
    const at::Tensor &q = tensor(a[0]), &kc = tensor(a[1]), &vc = tensor(a[2]), &ks = tensor(a[3]), &vs = tensor(a[4]);
    const at::Tensor &table = tensor(a[5]), &lens = tensor(a[6]);
    const bool has_cu = a[7] != Py_None;
    const int64_t max_new = whole(a[8]), window = whole(a[10]);
    const Cache m = cache(kc, vc, ks, vs);
    const int64_t B = lens.numel();
    want(!recorded(q));
    want(rows_ready(q) && q.device() == m.dev && q.size(2) == m.dim && q.size(1) > 0 && q.size(1) % m.heads == 0 &&
         plain_i32(table, 2, m.dev) && plain_i32(lens, 1, m.dev) && table.size(0) == B && max_new >= 1 &&
         max_new <= INT32_MAX && window >= 0);
    exl3_kv_attend_args c{};
    if (has_cu) {
        const at::Tensor& cu = tensor(a[7]);
        want(plain_i32(cu, 1, m.dev) && cu.numel() == B + 1);
        c.cu_tokens = data<int32_t>(cu);
    } else {
        want(q.size(0) == B && max_new == 1);
    }
    c.scale = a[9] == Py_None ? 1.0 / std::sqrt(double(m.dim)) : PyFloat_AsDouble(a[9]);
    if (c.scale == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw NotHere();
    }
    c.x_dtype = row_type(q);
    const int64_t rows = q.size(0), heads = q.size(1);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(m.dev.index());
    const Space ws = workspace(m.dev, stream, entry.attend_bytes(int(heads), int(m.heads), int(m.dim), int(max_new), int(B), rows));
    const at::Tensor out = at::empty(q.sizes(), q.options());
    at::Tensor lse;
    if (truth(a[11])) {
        lse = at::empty({rows, heads}, q.options().dtype(at::kFloat));
        c.lse = data<float>(lse);
    }
    c.q = q.data_ptr(), c.q_tok_stride = q.stride(0), c.q_head_stride = q.stride(1), c.q_rows = rows, c.heads = heads;
    c.k_cache = kc.data_ptr(), c.v_cache = vc.data_ptr(), c.k_scale = data<float>(ks), c.v_scale = data<float>(vs);
    c.code = m.code, c.pages = m.pages, c.kv_heads = m.heads, c.page = m.page, c.dim = m.dim;
    c.block_table = data<int32_t>(table), c.width = table.size(1), c.requests = B, c.kv_lens = data<int32_t>(lens);
    c.max_new = max_new, c.window = window, c.out = out.data_ptr(), c.workspace = ws.at, c.workspace_bytes = ws.bytes;
    checked(entry.attend(&c, stream), "kv_attend");
    if (!lse.defined()) return wrap(out);
    PyObject* both = PyTuple_New(2);
    if (!both) throw PyFailed();
    PyTuple_SET_ITEM(both, 0, wrap(out));
    PyTuple_SET_ITEM(both, 1, wrap(lse));
    return both;
}

PyObject* logprobs_(PyObject* const* a) {
    const at::Tensor &x = tensor(a[0]), &tok = tensor(a[1]);
    const int64_t top = whole(a[2]);
    const c10::Device dev = current(x);
    want(!recorded(x));
    exl3_token_logprobs_args c{};
    const auto kind = x.scalar_type();
    want(kind == at::kFloat || kind == at::kHalf || kind == at::kBFloat16);
    c.x_dtype = kind == at::kFloat ? EXL3_DT_F32 : kind == at::kHalf ? EXL3_DT_F16 : EXL3_DT_BF16;
    want(x.dim() == 2 && tok.dim() == 1 && tok.device() == dev && tok.is_contiguous() &&
         (tok.scalar_type() == at::kLong || tok.scalar_type() == at::kInt));
    const int64_t rows = x.size(0), vocab = x.size(1);
    want(tok.size(0) == rows && rows > 0 && x.stride(1) == 1 && (rows == 1 || x.stride(0) >= vocab) && top >= 0 &&
         top <= EXL3_LOGPROBS_MAX_TOP && top <= vocab);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index());
    const Space ws = workspace(dev, stream, entry.logprobs_bytes(rows, vocab, int(top), int(c.x_dtype)));
    const auto f = x.options().dtype(at::kFloat), i = x.options().dtype(at::kInt);
    const at::Tensor two = at::empty({2 * rows}, f), rank = at::empty({rows}, i);
    const at::Tensor vals = at::empty({rows, top}, f), ids = at::empty({rows, top}, i);
    c.logits = x.data_ptr(), c.rows = rows, c.row_stride = x.stride(0), c.vocab = vocab, c.tokens = tok.data_ptr();
    c.ids_dtype = tok.scalar_type() == at::kLong ? EXL3_DT_I64 : EXL3_DT_I32, c.top = top;
    c.logprob = data<float>(two), c.entropy = data<float>(two) + rows, c.rank = data<int32_t>(rank);
    c.top_logprobs = top ? data<float>(vals) : nullptr, c.top_ids = top ? data<int32_t>(ids) : nullptr;
    c.workspace = ws.at, c.workspace_bytes = ws.bytes;
    checked(entry.logprobs(&c, stream), "token_logprobs");
    PyObject* out = PyTuple_New(5);
    if (!out) throw PyFailed();
    PyTuple_SET_ITEM(out, 0, wrap(part(two, 0, rows)));
    PyTuple_SET_ITEM(out, 1, wrap(part(two, rows, rows)));
    PyTuple_SET_ITEM(out, 2, wrap(rank));
    PyTuple_SET_ITEM(out, 3, wrap(vals));
    PyTuple_SET_ITEM(out, 4, wrap(ids));
    return out;
}

// No C++ exception leaves an entry.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", N, n);
        return nullptr;
    }
    if (!entry.plan) Py_RETURN_NONE;
    try {
        at::AutoDispatchBelowADInplaceOrView plain;  // nothing here is differentiated
        return F(args);
    } catch (const NotHere&) {
        Py_RETURN_NONE;
    } catch (const PyFailed&) {
        return nullptr;
    } catch (const std::exception&) {  // of the allocator, before anything is launched: the long way raises torch's own
        if (PyErr_Occurred()) return nullptr;
        Py_RETURN_NONE;
    }
}

// setup(plan, append, attend, attend_bytes, logprobs, logprobs_bytes, capture_id, workspace_of, check): addresses of the C entries
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 9) {
        PyErr_SetString(PyExc_TypeError, "9 arguments expected");
        return nullptr;
    }
    void* p[7];
    for (int i = 0; i < 7; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    Py_INCREF(a[7]);
    Py_INCREF(a[8]);
    workspace_of = a[7], check = a[8];
    entry.capture_id = reinterpret_cast<decltype(entry.capture_id)>(p[6]);
    entry.append = reinterpret_cast<decltype(entry.append)>(p[1]);
    entry.attend = reinterpret_cast<decltype(entry.attend)>(p[2]);
    entry.attend_bytes = reinterpret_cast<decltype(entry.attend_bytes)>(p[3]);
    entry.logprobs = reinterpret_cast<decltype(entry.logprobs)>(p[4]);
    entry.logprobs_bytes = reinterpret_cast<decltype(entry.logprobs_bytes)>(p[5]);
    entry.plan = reinterpret_cast<decltype(entry.plan)>(p[0]);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"setup", FAST(setup)},
                         {"kv_plan", FAST((call<plan_, 7>))},
                         {"kv_append", FAST((call<append_, 7>))},
                         {"kv_attend", FAST((call<attend_, 12>))},
                         {"token_logprobs", FAST((call<logprobs_, 3>))},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving_py", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__serving_py() { return PyModule_Create(&module); }
