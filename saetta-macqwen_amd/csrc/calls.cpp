// The calls that a program makes per chunk and per token, from Python without ctypes: the tensors' checks and pointers, the
// current stream and the call of the C ABI in one step.  A small launch is 2.7 us of the host in the HIP runtime; a call through
// ctypes, with its checks in Python, was 2 to 3.5 us more.  (Host code only: the kernels are the library's, which is
// loaded from the path that `setup` was given when the first call needs it.)
#include <Python.h>

#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>

#include "../../include/saetta_hip.h"

namespace {

struct Library {
    bool loaded;
    decltype(&saetta_last_error) last_error;
    decltype(&saetta_to_half) to_half;
    decltype(&saetta_kv_quantize) kv_quantize;
    decltype(&saetta_attn_prefill) attn_prefill;
    decltype(&saetta_attn_prefill_quant) attn_prefill_quant;
    decltype(&saetta_token_params_set) token_params_set;
    decltype(&saetta_plan_run) plan_run;
    decltype(&saetta_paged_tables) paged_tables;
    decltype(&saetta_paged_store) paged_store;
    decltype(&saetta_paged_gather) paged_gather;
    decltype(&saetta_paged_split) paged_split;
    decltype(&saetta_paged_attn) paged_attn;
};

// What a copy of the package has set up (`setup`), kept with its module.
struct State {
    PyObject *error, *flash_params, *path;  // SaettaError, FlashParamsC, the library's path
    Library lib;
};
State &state_of(PyObject *module) { return *static_cast<State *>(PyModule_GetState(module)); }

// A Python exception is set.
struct Raised {};

[[noreturn]] void raise(PyObject *type, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    PyErr_FormatV(type, fmt, ap);
    va_end(ap);
    throw Raised{};
}

// (the GIL is held: one thread at a time gets here)
const Library &library(State &st) {
    Library &lib = st.lib;
    if (!lib.loaded) {
        if (!st.path) raise(PyExc_RuntimeError, "_saetta_calls: not set up");
        const char *path = PyUnicode_AsUTF8(st.path);
        if (!path) throw Raised{};
        void *h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
        if (!h) raise(st.error, "%s is missing: run __graft_entry__.build() (make -C csrc): %s", path, dlerror());
        auto find = [&](auto &f, const char *name) {
            f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(h, name));
            if (!f) raise(st.error, "%s has no %s", path, name);
        };
        find(lib.last_error, "saetta_last_error"), find(lib.to_half, "saetta_to_half"), find(lib.kv_quantize, "saetta_kv_quantize");
        find(lib.attn_prefill, "saetta_attn_prefill"), find(lib.attn_prefill_quant, "saetta_attn_prefill_quant");
        find(lib.token_params_set, "saetta_token_params_set"), find(lib.plan_run, "saetta_plan_run");
        find(lib.paged_tables, "saetta_paged_tables"), find(lib.paged_store, "saetta_paged_store"), find(lib.paged_gather, "saetta_paged_gather");
        find(lib.paged_split, "saetta_paged_split"), find(lib.paged_attn, "saetta_paged_attn");
        lib.loaded = true;
    }
    return lib;
}

// A contiguous tensor of `dtype` on the GPU.
const at::Tensor &need(PyObject *o, at::ScalarType dtype, const char *what) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.scalar_type() == dtype && t.is_cuda() && t.is_contiguous()) return t;
    }
    raise(PyExc_TypeError, "%s: expected a contiguous torch.%s tensor on the GPU", what,
          dtype == at::kFloat ? "float32" : dtype == at::kHalf ? "float16" : "uint8");
}
template <class T>
T *pointer(const at::Tensor &t) {
    return static_cast<T *>(t.data_ptr());
}
// A tensor that a kernel can reach.
template <class T>
T *pointer_of(PyObject *o, const char *what) {
    if (THPVariable_Check(o)) {
        const at::Tensor &t = THPVariable_Unpack(o);
        if (t.is_cuda() || t.is_pinned()) return pointer<T>(t);
    }
    raise(PyExc_TypeError, "%s: expected a tensor on the GPU or in pinned memory", what);
}

long long integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}
uint32_t u32(PyObject *o) { return uint32_t(PyLong_AsUnsignedLongMask(o)); }

// None: torch's current stream of the current device.
saetta_stream_t stream_of(PyObject *o) {
    if (o == Py_None) return reinterpret_cast<saetta_stream_t>(c10::hip::getCurrentHIPStream().stream());
    void *p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw Raised{};
    return reinterpret_cast<saetta_stream_t>(p);
}

saetta_flash_params flash_params(const State &st, PyObject *o, const char *what) {
    const int is = st.flash_params ? PyObject_IsInstance(o, st.flash_params) : 0;
    if (is < 0) throw Raised{};
    if (!is) raise(PyExc_TypeError, "%s: expected FlashParams", what);
    Py_buffer b;
    if (PyObject_GetBuffer(o, &b, PyBUF_SIMPLE)) throw Raised{};
    saetta_flash_params p;
    const bool fits = size_t(b.len) >= sizeof p;
    if (fits) memcpy(&p, b.buf, sizeof p);
    PyBuffer_Release(&b);
    if (!fits) raise(PyExc_TypeError, "%s: expected FlashParams", what);
    return p;
}

// Calls the library with the GIL released, as ctypes does (a launch waits where the queue is full).
template <class F>
PyObject *call(const char *what, const State &st, F f) {
    PyThreadState *thread = PyEval_SaveThread();
    const int rc = f();
    PyEval_RestoreThread(thread);
    if (rc) raise(st.error, "%s: %s (code %d)", what, st.lib.last_error(), rc);
    Py_RETURN_NONE;
}

template <class F>
PyObject *guarded(Py_ssize_t n, Py_ssize_t wanted, const char *what, F f) {
    try {
        if (n != wanted) raise(PyExc_TypeError, "%s takes %zd arguments (%zd given)", what, wanted, n);
        return f();
    } catch (const Raised &) {
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_Format(PyExc_RuntimeError, "%s: unknown error", what);
        return nullptr;
    }
}

// setup(path, SaettaError, FlashParamsC)
PyObject *setup(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 3, "setup", [&]() -> PyObject * {
        State &st = state_of(module);
        Py_INCREF(a[0]), Py_INCREF(a[1]), Py_INCREF(a[2]);
        Py_XSETREF(st.path, a[0]);
        Py_XSETREF(st.error, a[1]);
        Py_XSETREF(st.flash_params, a[2]);
        Py_RETURN_NONE;
    });
}

// to_half(x, out, stream)
PyObject *to_half(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 3, "to_half", [&] {
        const at::Tensor &x = need(a[0], at::kFloat, "to_half x"), &out = need(a[1], at::kHalf, "to_half out");
        if (out.numel() < x.numel()) raise(PyExc_ValueError, "to_half: out does not hold x's values");
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[2]);
        const float *from = pointer<float>(x);
        uint16_t *to = pointer<uint16_t>(out);
        const size_t count = size_t(x.numel());
        return call("to_half", st, [&] { return lib.to_half(s, from, to, count); });
    });
}

// kv_encode(bits, per_token, capacity, data, scales, biases, x, pos, tokens, stream)
PyObject *kv_encode(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 10, "kv_encode", [&] {
        const long long per_token = integer(a[1]), capacity = integer(a[2]), pos = integer(a[7]), tokens = integer(a[8]);
        const bool fit = tokens >= 0 && tokens <= capacity && pos >= 0 && pos <= capacity - tokens;
        if (!fit) raise(PyExc_ValueError, "QuantRows.encode: tokens do not fit");
        const at::Tensor &x = need(a[6], at::kFloat, "QuantRows.encode x");
        if (x.numel() < tokens * per_token * SAETTA_QUANT_GROUP) raise(PyExc_ValueError, "QuantRows.encode: tokens do not fit");
        const saetta_quant_rows rows{pointer_of<uint32_t>(a[3], "QuantRows.encode data"), pointer_of<uint16_t>(a[4], "QuantRows.encode scales"),
                                     pointer_of<uint16_t>(a[5], "QuantRows.encode biases")};
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[9]);
        const saetta_kv_quant_params p{uint32_t(per_token * tokens), uint32_t(per_token)};
        const int bits = int(integer(a[0]));
        const float *from = pointer<float>(x);
        return call("kv_quantize", st, [&] { return lib.kv_quantize(s, bits, from, rows, p, nullptr, uint32_t(pos)); });
    });
}

// prefill(kernel, q, keys, values, q_and_gate, out, p, workspace, stream)
PyObject *prefill(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 9, "prefill", [&] {
        State &st = state_of(module);
        const saetta_flash_params p = flash_params(st, a[6], "prefill attention");
        if (p.heads != p.kv_heads * SAETTA_GQA_GROUP) raise(PyExc_ValueError, "%S needs 8 q heads per kv head", a[0]);
        const at::Tensor &q = need(a[1], at::kHalf, "q"), &keys = need(a[2], at::kHalf, "keys"), &values = need(a[3], at::kHalf, "values"),
                         &qg = need(a[4], at::kFloat, "q_and_gate"), &out = need(a[5], at::kFloat, "out"), &ws = need(a[7], at::kByte, "workspace");
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[8]);
        const uint16_t *q_ptr = pointer<uint16_t>(q), *k = pointer<uint16_t>(keys), *v = pointer<uint16_t>(values);
        const float *g = pointer<float>(qg);
        float *o = pointer<float>(out);
        void *w = ws.data_ptr();
        const size_t bytes = size_t(ws.numel());
        return call("attn_prefill", st, [&] { return lib.attn_prefill(s, q_ptr, k, v, g, o, p, w, bytes); });
    });
}

// prefill_quant(bits, q, keys' data, scales, biases, values' data, scales, biases, q_and_gate, out, p, workspace, stream)
PyObject *prefill_quant(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 13, "prefill_quant", [&] {
        State &st = state_of(module);
        const saetta_flash_params p = flash_params(st, a[10], "prefill attention");
        if (p.heads != p.kv_heads * SAETTA_GQA_GROUP) raise(PyExc_ValueError, "prefill attention needs 8 q heads per kv head");
        const at::Tensor &q = need(a[1], at::kHalf, "q"), &qg = need(a[8], at::kFloat, "q_and_gate"), &out = need(a[9], at::kFloat, "out"),
                         &ws = need(a[11], at::kByte, "workspace");
        const saetta_quant_rows keys{pointer_of<uint32_t>(a[2], "keys"), pointer_of<uint16_t>(a[3], "keys"), pointer_of<uint16_t>(a[4], "keys")},
            values{pointer_of<uint32_t>(a[5], "values"), pointer_of<uint16_t>(a[6], "values"), pointer_of<uint16_t>(a[7], "values")};
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[12]);
        const int bits = int(integer(a[0]));
        const uint16_t *q_ptr = pointer<uint16_t>(q);
        const float *g = pointer<float>(qg);
        float *o = pointer<float>(out);
        void *w = ws.data_ptr();
        const size_t bytes = size_t(ws.numel());
        return call("attn_prefill_quant", st, [&] { return lib.attn_prefill_quant(s, bits, q_ptr, keys, values, g, o, p, w, bytes); });
    });
}

// token_params_set(params, token, position, kv_len, pad)
PyObject *token_params_set(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, "token_params_set", [&] {
        saetta_token_params *to = pointer_of<saetta_token_params>(a[0], "token_params_set params");
        const saetta_token_params value{u32(a[1]), u32(a[2]), u32(a[3]), u32(a[4])};
        if (PyErr_Occurred()) throw Raised{};
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(Py_None);
        return call("token_params_set", st, [&] { return lib.token_params_set(s, to, value); });
    });
}

// plan_run(the plan's address, stream)
PyObject *plan_run(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 2, "plan_run", [&] {
        const saetta_plan *plan = static_cast<const saetta_plan *>(PyLong_AsVoidPtr(a[0]));
        if (!plan && PyErr_Occurred()) throw Raised{};
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[1]);
        return call("plan_run", st, [&] { return lib.plan_run(s, plan); });
    });
}

// ---- a cache in blocks ------------------------------------------------------------------------------------------------
// The objects of host.py hand their buffers and sizes over as one tuple, made once; what changes from call to call is checked here.

PyObject *item(PyObject *tuple, Py_ssize_t i, Py_ssize_t n, const char *what) {
    if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != n) raise(PyExc_TypeError, "%s: expected a tuple of %zd", what, n);
    return PyTuple_GET_ITEM(tuple, i);
}
// Sizes that the library takes in 32 bits.
void fits32(long long n, const char *what) {
    if (n > 0xffffffffll) raise(PyExc_ValueError, "%s: %lld of them (fewer than 2^32)", what, n);
}
// A contiguous tensor of `dtype` on the current device.
const at::Tensor &here(PyObject *o, at::ScalarType dtype, const char *what) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s: expected a tensor", what);
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.scalar_type() != dtype || !t.is_cuda() || !t.is_contiguous())
        raise(PyExc_TypeError, "%s: expected a contiguous torch.%s tensor on the GPU", what, dtype == at::kInt ? "int32" : "uint8");
    if (t.get_device() != c10::hip::current_device())
        raise(PyExc_ValueError, "%s is on cuda:%d, the current device is cuda:%d", what, int(t.get_device()), int(c10::hip::current_device()));
    return t;
}
int type_of(const at::Tensor &t, bool floats, const char *what) {
    if (t.scalar_type() == at::kHalf) return SAETTA_F16;
    if (t.scalar_type() == at::kBFloat16) return SAETTA_BF16;
    if (t.scalar_type() == at::kFloat && floats) return SAETTA_F32;
    raise(PyExc_TypeError, "%s: expected a tensor of %storch.float16 or torch.bfloat16 on the GPU", what, floats ? "torch.float32, " : "");
}
// [tokens, heads, 256] with rows that are contiguous.
struct Rows {
    saetta_strided_rows rows;
    long long tokens;
    int type;
};
Rows rows_of(PyObject *o, long long heads, bool floats, const char *what) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s: expected a tensor", what);
    const at::Tensor &t = THPVariable_Unpack(o);
    const int type = type_of(t, floats, what);
    if (!t.is_cuda()) raise(PyExc_TypeError, "%s: expected a tensor on the GPU", what);
    if (t.get_device() != c10::hip::current_device())
        raise(PyExc_ValueError, "%s is on cuda:%d, the current device is cuda:%d", what, int(t.get_device()), int(c10::hip::current_device()));
    if (t.dim() != 3 || t.size(1) != heads || t.size(2) != SAETTA_HEAD_DIM || t.stride(2) != 1)
        raise(PyExc_ValueError, "%s: expected [tokens, %lld, %d] with contiguous rows", what, heads, SAETTA_HEAD_DIM);
    // (a dim of one has whatever stride torch left there)
    return {{t.data_ptr(), uint64_t(t.size(0) > 1 ? t.stride(0) : 0), uint64_t(heads > 1 ? t.stride(1) : 0)}, t.size(0), type};
}
// (keys, values, key_scales, value_scales, blocks, block_tokens, kv_heads)
saetta_paged_cache paged_cache(PyObject *o) {
    auto codes = [&](Py_ssize_t i) { return pointer<uint8_t>(here(item(o, i, 7, "paged cache"), at::kByte, "paged cache")); };
    return {codes(0), codes(1), codes(2), codes(3), u32(item(o, 4, 7, "paged cache")), u32(item(o, 5, 7, "paged cache")), u32(item(o, 6, 7, "paged cache"))};
}
// (query_starts, kv_lens, block_table, requests, max_blocks, block_tokens)
saetta_paged_batch paged_batch(PyObject *o) {
    auto ints = [&](Py_ssize_t i) { return pointer<uint32_t>(here(item(o, i, 6, "paged batch"), at::kInt, "paged batch")); };
    return {ints(0), ints(1), reinterpret_cast<const int32_t *>(ints(2)), u32(item(o, 3, 6, "paged batch")), u32(item(o, 4, 6, "paged batch")),
            u32(item(o, 5, 6, "paged batch"))};
}
// (heads, kv_heads, tokens, rows, scale)
saetta_paged_attn_params paged_params(PyObject *o) {
    const double scale = PyFloat_AsDouble(item(o, 4, 5, "paged attention"));
    if (scale == -1.0 && PyErr_Occurred()) throw Raised{};
    return {u32(item(o, 0, 5, "paged attention")), u32(item(o, 1, 5, "paged attention")), u32(item(o, 2, 5, "paged attention")),
            u32(item(o, 3, 5, "paged attention")), float(scale)};
}

// paged_tables(context_lens, new_lens, (the nine tensors of PagedTables.tensors), (requests, max_blocks, block_tokens, blocks, tokens), stream)
PyObject *paged_tables(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, "paged_tables", [&] {
        const saetta_paged_tables_params p{u32(item(a[3], 0, 5, "PagedTables")), u32(item(a[3], 1, 5, "PagedTables")), u32(item(a[3], 2, 5, "PagedTables")),
                                           u32(item(a[3], 3, 5, "PagedTables")), u32(item(a[3], 4, 5, "PagedTables"))};
        if (PyErr_Occurred()) throw Raised{};
        const at::Tensor &context = here(a[0], at::kInt, "PagedTables context_lens"), &fresh = here(a[1], at::kInt, "PagedTables new_lens");
        if (context.numel() != p.requests || fresh.numel() != p.requests)
            raise(PyExc_ValueError, "PagedTables: context_lens and new_lens must be of %u requests", p.requests);
        auto ints = [&](Py_ssize_t i) { return pointer<int32_t>(here(item(a[2], i, 9, "PagedTables"), at::kInt, "PagedTables")); };
        auto lengths = [&](Py_ssize_t i) { return reinterpret_cast<uint32_t *>(ints(i)); };
        const saetta_paged_state state{ints(0), lengths(1), ints(2), lengths(3)};
        const saetta_paged_step step{lengths(4), lengths(5), ints(6), ints(7), lengths(8)};
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[4]);
        const uint32_t *c = pointer<uint32_t>(context), *f = pointer<uint32_t>(fresh);
        return call("paged_tables", st, [&] { return lib.paged_tables(s, c, f, state, step, p); });
    });
}

// paged_store(k, v, slots, cache, stream)
PyObject *paged_store(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, "paged_store", [&] {
        const saetta_paged_cache cache = paged_cache(a[3]);
        if (PyErr_Occurred()) throw Raised{};
        const Rows k = rows_of(a[0], cache.kv_heads, true, "PagedCache k"), v = rows_of(a[1], cache.kv_heads, true, "PagedCache v");
        const at::Tensor &slots = here(a[2], at::kInt, "PagedCache slots");
        if (k.type != v.type || k.tokens != v.tokens || slots.numel() != k.tokens)
            raise(PyExc_ValueError, "PagedCache: k, v and slots must be of as many tokens, k and v of one type");
        fits32(k.tokens, "PagedCache slots");
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[4]);
        const int32_t *at = pointer<int32_t>(slots);
        return call("paged_store", st, [&] { return lib.paged_store(s, k.type, k.rows, v.rows, at, cache, uint32_t(k.tokens)); });
    });
}

// paged_gather(slots, keys or None, values or None, cache, stream)
PyObject *paged_gather(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, "paged_gather", [&] {
        const saetta_paged_cache cache = paged_cache(a[3]);
        if (PyErr_Occurred()) throw Raised{};
        const at::Tensor &slots = here(a[0], at::kInt, "PagedCache slots");
        int type = -1;
        void *to[2] = {nullptr, nullptr};
        for (int i = 0; i < 2; i++) {
            if (a[1 + i] == Py_None) continue;
            if (!THPVariable_Check(a[1 + i])) raise(PyExc_TypeError, "PagedCache: keys and values must be tensors");
            const at::Tensor &t = THPVariable_Unpack(a[1 + i]);
            const int is = type_of(t, true, "PagedCache keys and values");
            if (!t.is_cuda() || !t.is_contiguous()) raise(PyExc_TypeError, "PagedCache keys and values: expected contiguous tensors on the GPU");
            if (t.get_device() != c10::hip::current_device())
                raise(PyExc_ValueError, "PagedCache keys and values: on cuda:%d, the current device is cuda:%d", int(t.get_device()), int(c10::hip::current_device()));
            if (type >= 0 && is != type) raise(PyExc_ValueError, "PagedCache: keys and values of one type");
            if (t.numel() < slots.numel() * int64_t(cache.kv_heads) * SAETTA_HEAD_DIM) raise(PyExc_ValueError, "PagedCache: keys and values do not hold the slots' rows");
            type = is, to[i] = t.data_ptr();
        }
        if (type < 0) raise(PyExc_ValueError, "PagedCache: keys or values or both");
        fits32(slots.numel(), "PagedCache slots");
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[4]);
        const int32_t *at = pointer<int32_t>(slots);
        const uint32_t tokens = uint32_t(slots.numel());
        return call("paged_gather", st, [&] { return lib.paged_gather(s, type, cache, at, to[0], to[1], tokens); });
    });
}

// paged_split(batch, params, split, stream)
PyObject *paged_split(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 4, "paged_split", [&] {
        const saetta_paged_batch batch = paged_batch(a[0]);
        const saetta_paged_attn_params p = paged_params(a[1]);
        if (PyErr_Occurred()) throw Raised{};
        void *split = here(a[2], at::kByte, "paged attention").data_ptr();
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[3]);
        return call("paged_split", st, [&] { return lib.paged_split(s, batch, p, split); });
    });
}

// paged_attn(q, gate or None, out, cache, batch, params, split, workspace, stream)
PyObject *paged_attn(PyObject *module, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 9, "paged_attn", [&] {
        const saetta_paged_cache cache = paged_cache(a[3]);
        const saetta_paged_batch batch = paged_batch(a[4]);
        const saetta_paged_attn_params p = paged_params(a[5]);
        if (PyErr_Occurred()) throw Raised{};
        const Rows q = rows_of(a[0], p.heads, false, "q"), out = rows_of(a[2], p.heads, false, "out");
        Rows gate{{nullptr, 0, 0}, q.tokens, q.type};
        if (a[1] != Py_None) gate = rows_of(a[1], p.heads, false, "gate");
        for (const Rows *r : {&q, static_cast<const Rows *>(&gate), &out})
            if (r->type != q.type || r->tokens < p.tokens) raise(PyExc_ValueError, "paged attention: q, gate and out must be of one type and of %u tokens", p.tokens);
        if ((out.tokens > 1 && out.rows.token_stride == 0) || (p.heads > 1 && out.rows.head_stride == 0))
            raise(PyExc_ValueError, "paged attention: out's rows must lie apart");
        void *split = here(a[6], at::kByte, "paged attention").data_ptr();
        const at::Tensor &ws = here(a[7], at::kByte, "paged attention");
        void *workspace = ws.data_ptr();
        const size_t bytes = size_t(ws.numel());
        State &st = state_of(module);
        const Library &lib = library(st);
        const saetta_stream_t s = stream_of(a[8]);
        return call("paged_attn", st, [&] { return lib.paged_attn(s, q.type, q.rows, cache, batch, split, gate.rows, out.rows, p, workspace, bytes); });
    });
}

#define FUNCTION(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FUNCTION(setup), FUNCTION(to_half), FUNCTION(kv_encode), FUNCTION(prefill), FUNCTION(prefill_quant),
                           FUNCTION(token_params_set), FUNCTION(plan_run), FUNCTION(paged_tables), FUNCTION(paged_store), FUNCTION(paged_gather),
                           FUNCTION(paged_split), FUNCTION(paged_attn), {nullptr, nullptr, 0, nullptr}};
#undef FUNCTION

int traverse(PyObject *module, visitproc visit, void *arg) {
    const State &st = state_of(module);
    Py_VISIT(st.path);
    Py_VISIT(st.error);
    Py_VISIT(st.flash_params);
    return 0;
}
int clear(PyObject *module) {
    State &st = state_of(module);
    Py_CLEAR(st.path);
    Py_CLEAR(st.error);
    Py_CLEAR(st.flash_params);
    return 0;
}
// (a state per module object: a process may hold more than one copy of the package)
PyModuleDef_Slot g_slots[] = {{0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_saetta_calls", nullptr, sizeof(State), g_methods, g_slots, traverse, clear, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__saetta_calls() { return PyModuleDef_Init(&g_module); }
