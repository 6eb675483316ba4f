// Python binding of the KV-cache operators (and of assign_block_ids): tensors -> descriptors -> phase 1 -> workspace ->
// phase 2 in one native call, on the tensors' device and torch's current stream.  A decode step makes several of these
// calls per layer, and building a dozen descriptors through ctypes costs more host time than the kernels take.
// The C-ABI is reached through addresses that the package hands over (bind), so this module uses the library that the
// package has loaded.  Checks of operands are phase 1's; here only what descriptors cannot show: the devices.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cstring>
#include <optional>
#include <string>

#include "../../include/acl_shim.h"

namespace {

PyObject* g_error = nullptr;   // custom_ops._abi.AclError

// Entry points, in the order in which bind() takes them.
struct Api {
    aclTensor* (*create)(const int64_t*, uint64_t, aclDataType, const int64_t*, int64_t, aclFormat, const int64_t*, uint64_t, void*);
    aclnnStatus (*destroy)(const aclTensor*);
    aclTensorList* (*create_list)(const aclTensor* const*, uint64_t);
    aclnnStatus (*destroy_list)(const aclTensorList*);
    const char* (*message)();
    void *append_ws, *append, *gather_ws, *gather, *attention_ws, *attention, *assign_ws, *assign;
} g_api;
using Exec = aclnnStatus (*)(void*, uint64_t, aclOpExecutor*, aclrtStream);
using Desc = const aclTensor*;

struct Failure { std::string text; bool type_error; };
[[noreturn]] void raise(const std::string& text) { throw Failure{text, false}; }

aclDataType acl_type(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return ACL_FLOAT;
        case at::kHalf: return ACL_FLOAT16;
        case at::kBFloat16: return ACL_BF16;
        case at::kChar: return ACL_INT8;
        case at::kByte: return ACL_UINT8;
        case at::kShort: return ACL_INT16;
        case at::kInt: return ACL_INT32;
        case at::kLong: return ACL_INT64;
        case at::kDouble: return ACL_DOUBLE;
        case at::kBool: return ACL_BOOL;
        default: raise(std::string("Unsupported tensor dtype ") + c10::toString(t));
    }
}

// The tensors of one call.  None and tensors without elements are absent operands (a null descriptor).
class Call {
public:
    explicit Call(const char* what) : what_(what) {}
    ~Call() {
        for (int i = 0; i < n_; ++i) g_api.destroy(descs_[i]);
        if (list_) g_api.destroy_list(list_);
    }
    static const at::Tensor* tensor(PyObject* o, const char* name) {
        if (o == nullptr || o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) throw Failure{std::string(name) + " must be a tensor", true};
        return &THPVariable_Unpack(o);
    }
    // notes the operand's device; all of them have to agree
    const at::Tensor* take(PyObject* o, const char* name) {
        const at::Tensor* t = tensor(o, name);
        if (t && t->numel() > 0) {
            if (!t->is_cuda()) raise("custom_ops operands must live on the GPU (there is no CPU implementation)");
            if (!device_) device_ = t->device();
            else if (*device_ != t->device())
                raise(std::string(what_) + ": operands on several devices (" + device_->str() + ", " + t->device().str() + ")");
        }
        return t;
    }
    Desc desc(const at::Tensor* t) {
        if (!t || t->numel() == 0) return nullptr;
        Desc d = raw(*t);
        descs_[n_++] = d;
        return d;
    }
    Desc desc(PyObject* o, const char* name) { return desc(take(o, name)); }
    aclTensorList* list_of(const at::Tensor* t) {
        if (!t || t->numel() == 0) return nullptr;
        Desc d = raw(*t);
        return list_ = g_api.create_list(&d, 1);      // owns the descriptor
    }
    at::Device device() const {
        if (!device_) raise(std::string(what_) + ": no operand holds any element");
        return *device_;
    }
    void fail(aclnnStatus s, const char* phase) const {
        const char* m = g_api.message();
        raise(std::string(what_) + phase + " failed: " + std::to_string(s) + ": " + (m ? m : ""));
    }
    // phase 2 on the current stream of the operands' device (which the caller has made current), with a workspace of the
    // caching allocator: it belongs to that stream, so it may be freed as soon as the launch is enqueued
    void run(aclnnStatus planned, uint64_t ws_bytes, aclOpExecutor* e, void* exec) const {
        if (planned != ACLNN_SUCCESS) fail(planned, "GetWorkspaceSize");
        at::Tensor ws;
        if (ws_bytes > 0) ws = at::empty({(int64_t)ws_bytes}, at::TensorOptions().dtype(at::kByte).device(device()));
        const auto stream = c10::hip::getCurrentHIPStream(device().index());
        const aclnnStatus s = ((Exec)exec)(ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, e, (aclrtStream)stream.stream());
        if (s != ACLNN_SUCCESS) fail(s, "");
    }

private:
    Desc raw(const at::Tensor& t) {
        const auto sz = t.sizes(), st = t.strides();
        Desc d = g_api.create(sz.data(), sz.size(), acl_type(t.scalar_type()), st.data(), 0, ACL_FORMAT_ND, sz.data(), sz.size(),
                              t.data_ptr());
        if (!d) raise("out of host memory");
        return d;
    }
    const char* what_;
    std::optional<at::Device> device_;
    std::array<Desc, 24> descs_{};
    int n_ = 0;
    aclTensorList* list_ = nullptr;
};

// A call without rows launches nothing, so phase 1 does not see its operands: those that go by rows must have none either
// (an output would come back unwritten).
void no_rows(const at::Tensor* t, const char* name) {
    if (t && t->numel() > 0) raise(std::string("no rows to work on, but ") + name + " holds elements");
}

// Whether two tensors' elements lie in a common range of memory.
bool overlap(const at::Tensor& a, const at::Tensor& b) {
    auto end = [](const at::Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return (const char*)t.data_ptr() + (last + 1) * t.element_size();
    };
    if (a.numel() == 0 || b.numel() == 0) return false;
    return (const char*)a.data_ptr() < end(b) && (const char*)b.data_ptr() < end(a);
}

int64_t integer(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Failure{std::string(name) + " must be an integer", true};
    }
    return v;
}
double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Failure{std::string(name) + " must be a number", true};
    }
    return v;
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F&& f) {
    if (n != want) return PyErr_Format(PyExc_TypeError, "%zd arguments, expected %zd", n, want);
    try {
        return f();
    } catch (const Failure& e) {
        PyErr_SetString(e.type_error ? PyExc_TypeError : (g_error ? g_error : PyExc_RuntimeError), e.text.c_str());
    } catch (const c10::OutOfMemoryError& e) {
        PyErr_SetString(PyExc_MemoryError, e.what());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// append(key, value, key_cache, value_cache, block_table, seq_len, query, query_out, query_start, cos_sin, positions,
//        antiquant_scale, antiquant_offset, key_params, value_params, block_size, interleaved, antiquant_mode)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 18, [&]() -> PyObject* {
        Call c("aclnnAppendKvCache");
        const at::Tensor *key = c.take(a[0], "key"), *query = c.take(a[6], "query"), *given = c.take(a[7], "query_out");
        if (!key) throw Failure{"key must be a tensor", true};
        if (!query && given) raise("append_kv_cache: query_out given without query");
        at::Tensor out;
        if (given) out = *given;
        else if (query) out = at::empty(query->sizes(), query->options());
        auto result = [&]() -> PyObject* {
            if (!query) Py_RETURN_NONE;
            if (given) { Py_INCREF(a[7]); return a[7]; }
            return THPVariable_Wrap(out);
        };
        if (key->dim() == 3 && key->size(0) == 0) {
            no_rows(c.take(a[1], "value"), "value");
            no_rows(query, "query");
            no_rows(given, "query_out");
            return result();
        }
        const Desc kd = c.desc(key), vd = c.desc(a[1], "value"), kc = c.desc(a[2], "key_cache"), vc = c.desc(a[3], "value_cache"),
                   bt = c.desc(a[4], "block_table"), sl = c.desc(a[5], "seq_len"), qd = c.desc(query), qs = c.desc(a[8], "query_start"),
                   cs = c.desc(a[9], "cos_sin"), ps = c.desc(a[10], "positions"), sc = c.desc(a[11], "antiquant_scale"),
                   of = c.desc(a[12], "antiquant_offset"), kp = c.desc(a[13], "key_params"), vp = c.desc(a[14], "value_params"),
                   od = out.defined() ? c.desc(&out) : nullptr;
        const int64_t bs = integer(a[15], "block_size"), inter = integer(a[16], "interleaved"), mode = integer(a[17], "antiquant_mode");
        const c10::DeviceGuard guard(c.device());
        using Plan = aclnnStatus (*)(Desc, Desc, Desc, Desc, Desc, Desc, Desc, Desc, Desc, Desc, int64_t, int64_t, int64_t, int64_t, Desc,
                                     Desc, Desc, Desc, Desc, uint64_t*, aclOpExecutor**);
        uint64_t ws = 0;
        aclOpExecutor* e = nullptr;
        const aclnnStatus s = ((Plan)g_api.append_ws)(kd, vd, qd, cs, ps, bt, sl, qs, sc, of, bs, inter, mode, given ? 0 : 1, kc, vc, kp,
                                                      vp, od, &ws, &e);
        c.run(s, ws, e, g_api.append);
        return result();
    });
}

// gather(key_cache, value_cache, key_params, value_params, block_table, seq_len, query_start, antiquant_scale,
//        antiquant_offset, key_out, value_out, block_size, antiquant_mode, tokens, heads, head_dim, bfloat16) -> (key, value)
// key_out None: new tensors [tokens, heads, head_dim] in float16 or bfloat16, whose rows in no sequence are zeros.
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 17, [&]() -> PyObject* {
        Call c("aclnnGatherKvCache");
        static const char* const names[9] = {"key_cache", "value_cache", "key_params", "value_params", "block_table", "seq_len",
                                             "query_start", "antiquant_scale", "antiquant_offset"};
        const int64_t bs = integer(a[11], "block_size"), mode = integer(a[12], "antiquant_mode"), T = integer(a[13], "num_tokens"),
                      heads = integer(a[14], "num_key_value_heads"), D = integer(a[15], "head dim"), bf16 = integer(a[16], "bfloat16");
        const at::Tensor *cache = c.take(a[0], names[0]), *ko = c.take(a[9], "key_out"), *vo = c.take(a[10], "value_out");
        const bool own = ko == nullptr;
        at::Tensor k, v;
        if (own) {
            if (!cache) throw Failure{"key_cache must be a tensor", true};
            if (T < 0 || heads < 0 || D < 0) raise("gather_kv_cache: a negative number of tokens, heads or channels");
            const auto opts = cache->options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
            k = at::empty({T, heads, D}, opts);
            v = at::empty({T, heads, D}, opts);
        } else {
            k = *ko;
            v = *vo;
        }
        auto result = [&]() -> PyObject* {
            PyObject *pk = own ? THPVariable_Wrap(k) : a[9], *pv = own ? THPVariable_Wrap(v) : a[10];
            if (!own) { Py_INCREF(pk); Py_INCREF(pv); }
            PyObject* both = PyTuple_Pack(2, pk, pv);
            Py_DECREF(pk);
            Py_DECREF(pv);
            return both;
        };
        if (k.dim() >= 1 && k.size(0) == 0) {
            no_rows(&v, "value_out");
            return result();
        }
        if (!own && overlap(k, v)) raise("gather_kv_cache: key_out and value_out must not overlap");
        Desc d[9];
        for (int i = 0; i < 9; ++i) d[i] = c.desc(a[i], names[i]);
        const Desc kd = c.desc(&k), vd = c.desc(&v);
        const c10::DeviceGuard guard(c.device());
        using Plan = aclnnStatus (*)(Desc, Desc, Desc, Desc, Desc, Desc, Desc, Desc, Desc, int64_t, int64_t, int64_t, Desc, Desc, uint64_t*,
                                     aclOpExecutor**);
        uint64_t ws = 0;
        aclOpExecutor* e = nullptr;
        const aclnnStatus s = ((Plan)g_api.gather_ws)(d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7], d[8], bs, mode, own ? 1 : 0, kd, vd, &ws, &e);
        c.run(s, ws, e, g_api.gather);
        return result();
    });
}

// attention(query, key_cache, value_cache, key_params, value_params, block_table, seq_len, query_start, block_position, out,
//           softmax_lse, scale_value, num_key_value_heads, block_size, max_query_len (< 0: all rows), causal, float32_out)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 17, [&]() -> PyObject* {
        Call c("aclnnPagedAttentionInt4");
        const at::Tensor *query = c.take(a[0], "query"), *given = c.take(a[9], "out");
        if (!query) throw Failure{"query must be a tensor", true};
        const double scale = number(a[11], "scale_value");
        const int64_t heads = integer(a[12], "num_key_value_heads"), bs = integer(a[13], "block_size"), most = integer(a[14], "max_query_len"),
                      causal = integer(a[15], "causal"), f32 = integer(a[16], "float32 output");
        at::Tensor out = given ? *given : at::empty(query->sizes(), f32 ? query->options().dtype(at::kFloat) : query->options());
        auto result = [&]() -> PyObject* {
            if (given) { Py_INCREF(a[9]); return a[9]; }
            return THPVariable_Wrap(out);
        };
        if (query->dim() == 3 && query->size(0) == 0) {
            no_rows(&out, "out");
            no_rows(c.take(a[10], "softmax_lse"), "softmax_lse");
            return result();
        }
        // (query itself is fine: the rows of a work item have been read by all that share it before the last of them writes)
        if (given && overlap(*query, out) &&
            !(query->data_ptr() == out.data_ptr() && query->scalar_type() == out.scalar_type() && query->is_contiguous()))
            raise("paged_attention_int4: out must be query itself or not overlap it");
        static const char* const names[9] = {"query", "key_cache", "value_cache", "key_params", "value_params", "block_table", "seq_len",
                                             "query_start", "block_position"};
        Desc d[9];
        for (int i = 0; i < 9; ++i) d[i] = c.desc(a[i], names[i]);
        const Desc lse = c.desc(a[10], "softmax_lse"), od = c.desc(&out);
        const c10::DeviceGuard guard(c.device());
        using Plan = aclnnStatus (*)(Desc, Desc, Desc, Desc, Desc, Desc, Desc, Desc, Desc, double, int64_t, int64_t, int64_t, int64_t, int64_t,
                                     Desc, Desc, uint64_t*, aclOpExecutor**);
        uint64_t ws = 0;
        aclOpExecutor* e = nullptr;
        const aclnnStatus s = ((Plan)g_api.attention_ws)(d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7], d[8], scale, heads, bs,
                                                         most < 0 ? query->size(0) : most, causal, given ? 0 : 1, od, lse, &ws, &e);
        c.run(s, ws, e, g_api.attention);
        return result();
    });
}

// assign(key, block_table, seq_len, first_new_page, l1_cent, antiquant_scale, antiquant_offset, block_ids, block_size,
//        max_new_pages)
PyObject* assign(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject* {
        Call c("aclnnAssignBlockIds");
        aclTensorList* key = c.list_of(c.take(a[0], "key"));
        static const char* const names[8] = {"key", "block_table", "seq_len", "first_new_page", "l1_cent", "antiquant_scale",
                                             "antiquant_offset", "block_ids"};
        Desc d[8];
        for (int i = 1; i < 8; ++i) d[i] = c.desc(a[i], names[i]);
        const int64_t bs = integer(a[8], "block_size"), most = integer(a[9], "max_new_pages");
        const c10::DeviceGuard guard(c.device());
        using Plan = aclnnStatus (*)(const aclTensorList*, Desc, Desc, Desc, Desc, Desc, Desc, int64_t, int64_t, Desc, uint64_t*, aclOpExecutor**);
        uint64_t ws = 0;
        aclOpExecutor* e = nullptr;
        const aclnnStatus s = ((Plan)g_api.assign_ws)(key, d[1], d[2], d[3], d[4], d[5], d[6], bs, most, d[7], &ws, &e);
        c.run(s, ws, e, g_api.assign);
        Py_RETURN_NONE;
    });
}

// bind(AclError, address, ...): the entry points of the loaded library, in the order of Api
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    constexpr Py_ssize_t want = 1 + sizeof(Api) / sizeof(void*);
    if (n != want) return PyErr_Format(PyExc_TypeError, "bind: %zd arguments, expected %zd", n, want);
    void* addr[sizeof(Api) / sizeof(void*)];
    for (Py_ssize_t i = 1; i < n; ++i) {
        addr[i - 1] = PyLong_AsVoidPtr(a[i]);
        if (addr[i - 1] == nullptr) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null entry point");
            return nullptr;
        }
    }
    memcpy(&g_api, addr, sizeof(addr));
    Py_XDECREF(g_error);
    g_error = a[0];
    Py_INCREF(g_error);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", (PyCFunction)(void (*)())append, METH_FASTCALL, nullptr},
    {"gather", (PyCFunction)(void (*)())gather, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)())attention, METH_FASTCALL, nullptr},
    {"assign", (PyCFunction)(void (*)())assign, METH_FASTCALL, nullptr},
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_binding() { return PyModule_Create(&module); }
