// calls.cpp -- the per-token calls of zkie_b200/decode.py as a CPython
// extension (zkie_b200/_calls.so): argument checks, output allocation and the
// call of the C entry point.  A step of generation makes some eighty of these
// calls, each of a few microseconds on the device; in Python with ctypes the
// checks and the conversion of 18 to 28 arguments took 5 to 9 us of a call.
// The C functions are libzkie_b200.so's own (include/zkie2.h).
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <sstream>
#include <string>

#include "../../include/zkie2.h"

namespace {

// thrown where a Python error has been set
struct Refused {};

[[noreturn]] void refuse(const std::string& what) {
    PyErr_SetString(PyExc_ValueError, what.c_str());
    throw Refused{};
}

std::string said(const at::Tensor& t) {
    std::ostringstream s;
    s << t.scalar_type() << " " << t.sizes() << " with strides " << t.strides() << " on " << t.device();
    return s.str();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + ": a tensor on the current CUDA device is wanted, not " +
                                      Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

// the tensor that the call's device is taken from
int device_of(const at::Tensor& t, const char* name) {
    if (!t.is_cuda() || t.get_device() != c10::cuda::current_device())
        refuse(std::string(name) + ": a tensor on the current CUDA device is wanted, not " + said(t));
    return t.get_device();
}

// a matrix of field elements with rows of `cols` numbers of unit stride that do not overlap
struct Rows {
    const uint64_t* data = nullptr;
    int64_t n = 0, stride = 0;
};
Rows rows(const at::Tensor& t, const char* name, int64_t cols, int dev) {
    if (t.scalar_type() != at::kUInt64 || !t.is_cuda() || t.get_device() != dev || t.dim() != 2 || t.size(1) != cols ||
        (cols > 1 && t.size(0) > 0 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < cols))
        refuse(std::string(name) + ": a uint64 matrix of " + std::to_string(cols) +
               " columns on the call's device, unit stride within its rows, is wanted, not " + said(t));
    return {static_cast<const uint64_t*>(t.data_ptr()), t.size(0), t.stride(0)};
}

// a contiguous tensor of a type (and a shape)
template <typename T>
T* flat(const at::Tensor& t, const char* name, at::ScalarType type, int dev, at::IntArrayRef shape) {
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != dev || !t.is_contiguous() || t.sizes() != shape) {
        std::ostringstream s;
        s << name << ": a contiguous " << type << " tensor " << shape << " on the call's device is wanted, not " << said(t);
        refuse(s.str());
    }
    return static_cast<T*>(t.data_ptr());
}
// a table of field elements: its length is what it is
const uint64_t* table_of(const at::Tensor& t, const char* name, int dev) {
    if (t.numel() == 0) refuse(std::string(name) + ": an empty table");
    return flat<uint64_t>(t, name, at::kUInt64, dev, {t.numel()});
}

int64_t number(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused{};
    return v;
}
// What a handle holds: its tensors and sizes.  Addresses are taken from the tensors at the call,
// so that a handle that was copied or restored works on its own memory and one whose tensors were
// given other memory is not read past its end.
struct Handle {
    PyObject* items;
    const char* name;
    int dev;
    Handle(PyObject* o, Py_ssize_t size, const char* what, int on) : items(o), name(what), dev(on) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != size) refuse(std::string(what) + ": a handle of zkie_b200.decode is wanted");
    }
    PyObject* at(int i) const { return PyTuple_GET_ITEM(items, i); }
    int64_t size(int i) const { return number(at(i)); }
    template <typename T>
    T* memory(PyObject* o, const char* what, at::ScalarType type, int64_t numel) const {
        const at::Tensor& t = tensor(o, what);
        if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != dev || !t.is_contiguous() || t.numel() != numel)
            refuse(std::string(name) + ": " + what + " is not the memory of " + std::to_string(numel) +
                   " numbers on the call's device that it was, but " + said(t));
        return static_cast<T*>(t.data_ptr());
    }
    template <typename T>
    T* memory(int i, const char* what, at::ScalarType type, int64_t numel) const {
        return memory<T>(at(i), what, type, numel);
    }
};
// a shift of a rounding division
uint32_t shift_of(PyObject* o, const char* name) {
    const int64_t v = number(o);
    if (v < 0 || v > 62) refuse(std::string(name) + ": a shift 0 .. 62 is wanted");
    return (uint32_t)v;
}
struct Scale {
    int64_t factor;
    uint32_t shift;
};
Scale scale(PyObject* o, const char* name) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) refuse(std::string(name) + ": (factor, shift) is wanted");
    return {number(PyTuple_GET_ITEM(o, 0)), shift_of(PyTuple_GET_ITEM(o, 1), name)};
}

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, int dev) {
    return at::Tensor(at::detail::empty_cuda(shape, type, at::Device(at::kCUDA, (at::DeviceIndex)dev), std::nullopt));
}
at::Tensor output(PyObject* o, at::IntArrayRef shape, int dev) {
    if (o == Py_None) return make(shape, at::kUInt64, dev);
    const at::Tensor& t = tensor(o, "out");
    flat<uint64_t>(t, "out", at::kUInt64, dev, shape);
    return t;
}
// What a call writes -- an output that is given, a cache -- shares no memory with anything that its
// blocks read (or write) at different times; the residual may be the output itself, each number being
// read by the thread that writes it.
struct Apart {
    const char *begin = nullptr, *end = nullptr;  // none where the call makes its output
    const char* what;
    explicit Apart(const at::Tensor& out, const char* name) : what(name) {
        if (out.numel() == 0) return;
        begin = static_cast<const char*>(out.data_ptr());
        end = begin + out.nbytes();
    }
    Apart(PyObject* given, const at::Tensor& out) : what("out") {
        if (given != Py_None) *this = Apart(out, "out");
    }
    void from(const void* data, int64_t bytes, const char* name) const {
        const char* b = static_cast<const char*>(data);
        if (begin && b && bytes > 0 && begin < b + bytes && b < end) refuse(std::string(what) + " shares memory with " + name);
    }
    void from(const at::Tensor& t, const char* name) const {
        if (begin && t.numel()) from(t.data_ptr(), (int64_t)t.nbytes(), name);
    }
    void from(const Rows& in, int64_t cols, const char* name, bool same = false) const {
        if (!begin || in.n == 0 || (same && reinterpret_cast<const char*>(in.data) == begin && (in.n == 1 || in.stride == cols))) return;
        from(in.data, 8 * ((in.n - 1) * in.stride + cols), name);
    }
};
uint32_t* word(PyObject* o, int dev) {
    const at::Tensor& t = tensor(o, "err");
    if (t.numel() != 1) refuse("err: one int32 word is wanted, not " + said(t));
    return reinterpret_cast<uint32_t*>(flat<int32_t>(t, "err", at::kInt, dev, t.sizes()));
}
zkie_stream_t stream(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

void done(int rc, const char* what) {
    if (rc) {
        PyErr_Format(PyExc_RuntimeError, "%s failed with CUDA error %d", what, rc);
        throw Refused{};
    }
}

// what torch itself throws -- an output that finds no memory -- is raised as torch raises it
template <typename F>
PyObject* guarded(F f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// project(x, (packed, k, n, group, segment, experts), shift, bias, table, offset, residual, out, err)
PyObject* project(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 9) refuse("project: 9 arguments");
        const at::Tensor& x = tensor(a[0], "x");
        const int dev = device_of(x, "x");
        const Handle w(a[1], 6, "QuantWeight", dev);
        const int64_t k = w.size(1), n = w.size(2), segment = w.size(4), experts = w.size(5);
        const uint32_t group = (uint32_t)w.size(3);
        const Rows in = rows(x, "x", k, dev);
        if (experts != 1) refuse("project: one weight (no stack of experts) is wanted");
        const auto* packed = reinterpret_cast<const uint32_t*>(
            w.memory<int32_t>(0, "packed", at::kInt, (int64_t)zkie2_q4_words(1, k, n, group, segment)));
        if (in.n > 65535) refuse("project: at most 65535 rows are wanted");
        const uint32_t shift = shift_of(a[2], "project");
        const uint64_t* bias = a[3] == Py_None ? nullptr : flat<uint64_t>(tensor(a[3], "bias"), "bias", at::kUInt64, dev, {n});
        const uint64_t* table = nullptr;
        int64_t table_len = 0, offset = 0;
        if (a[4] != Py_None) {
            const at::Tensor& t = tensor(a[4], "table");
            table = table_of(t, "table", dev);
            table_len = t.numel();
            offset = a[5] == Py_None ? table_len / 2 : number(a[5]);
        }
        Rows residual;
        if (a[6] != Py_None) {
            residual = rows(tensor(a[6], "residual"), "residual", n, dev);
            if (residual.n != in.n)
                refuse("residual: " + std::to_string(residual.n) + " rows, " + std::to_string(in.n) + " are wanted");
        }
        const at::Tensor out = output(a[7], {in.n, n}, dev);
        const Apart apart(a[7], out);
        apart.from(in, k, "x");
        apart.from(residual, n, "the residual (and is not it)", true);
        apart.from(bias, 8 * n, "the bias");
        apart.from(table, 8 * table_len, "the table");
        apart.from(tensor(w.at(0), "packed"), "the weight");
        apart.from(tensor(a[8], "err"), "the error word");
        done(zkie2_q4_project(in.data, in.stride, in.n, packed, k, n, group, segment, shift, bias, table, table_len,
                              offset, residual.data, residual.stride, static_cast<uint64_t*>(out.data_ptr()),
                              word(a[8], dev), stream(dev)), "zkie2_q4_project");
        return THPVariable_Wrap(out);
    });
}

// attend(q, (k, v, lens, batch, heads, dk, dv, capacity), table, k, v, q_scale, k_scale, score_scale, offset,
//        out_shift, out, err)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 12) refuse("attend: 12 arguments");
        const at::Tensor& q = tensor(a[0], "q");
        const int dev = device_of(q, "q");
        const Handle c(a[1], 8, "KvCache", dev);
        const int64_t batch = c.size(3), heads = c.size(4), dk = c.size(5), dv = c.size(6), cap = c.size(7);
        auto* ck = c.memory<int32_t>(0, "k", at::kInt, batch * heads * cap * dk);
        auto* cv = c.memory<int32_t>(1, "v", at::kInt, batch * heads * cap * dv);
        const auto* lens = c.memory<int32_t>(2, "lens", at::kInt, batch);
        const int64_t cols = q.dim() == 2 ? q.size(1) : 0;
        if (cols == 0 || cols % (heads * dk) || cols / dk > 65535)
            refuse("q: a row per sequence of a multiple of " + std::to_string(heads * dk) + " columns is wanted, not " + said(q));
        const Rows in = rows(q, "q", cols, dev);
        if (in.n != batch || (a[3] == Py_None) != (a[4] == Py_None))
            refuse("attend: a row per sequence, and k and v together, are wanted");
        Rows k, v;
        if (a[3] != Py_None) {
            k = rows(tensor(a[3], "k"), "k", heads * dk, dev);
            v = rows(tensor(a[4], "v"), "v", heads * dv, dev);
            if (k.n != batch || v.n != batch) refuse("attend: a row of k and v per sequence is wanted");
        }
        const at::Tensor& t = tensor(a[2], "table");
        const uint64_t* table = table_of(t, "table", dev);
        const Scale qs = scale(a[5], "q_scale"), ks = scale(a[6], "k_scale"), ss = scale(a[7], "score_scale");
        const int64_t offset = a[8] == Py_None ? t.numel() : number(a[8]);
        const uint32_t out_shift = shift_of(a[9], "out_shift");
        const at::Tensor out = output(a[10], {batch, cols / dk * dv}, dev);
        const Apart apart(a[10], out);
        apart.from(in, cols, "q");
        apart.from(k, heads * dk, "k");
        apart.from(v, heads * dv, "v");
        apart.from(t, "the table");
        for (int i = 0; apart.begin && i < 3; i++) apart.from(tensor(c.at(i), "cache"), "the cache");
        apart.from(tensor(a[11], "err"), "the error word");
        for (int i = 0; i < 2 && k.data; i++) {  // the new token is stored while other blocks read
            const Apart cache(tensor(c.at(i), "cache"), "the cache");
            cache.from(in, cols, "q");
            cache.from(k, heads * dk, "k");
            cache.from(v, heads * dv, "v");
            cache.from(t, "the table");
        }
        done(zkie2_kv_attend(in.data, in.stride, cols / dk, qs.factor, qs.shift, k.data, k.stride, v.data, v.stride, ks.factor,
                             ks.shift, ck, cv, lens, batch, heads, dk, dv, cap, ss.factor, ss.shift, table, t.numel(), offset,
                             out_shift, static_cast<uint64_t*>(out.data_ptr()), word(a[11], dev), stream(dev)),
             "zkie2_kv_attend");
        return THPVariable_Wrap(out);
    });
}

// moe(x, (h, experts, top_k, f, shared_f, group, shift, router, gate and up, down, the shared experts' same, exp, silu),
//     residual, out, err) -> (out, gate)
PyObject* moe(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 5) refuse("moe: 5 arguments");
        const at::Tensor& x = tensor(a[0], "x");
        const int dev = device_of(x, "x");
        const Handle b(a[1], 14, "MoeBlock", dev);
        const int64_t h = b.size(0), experts = b.size(1), top_k = b.size(2), f = b.size(3), shared_f = b.size(4);
        const uint32_t group = (uint32_t)b.size(5);
        const Rows in = rows(x, "x", h, dev);
        if (in.n > 65535) refuse("MoeBlock: at most 65535 rows are wanted");
        const auto* router = reinterpret_cast<const uint32_t*>(
            b.memory<int32_t>(7, "router", at::kInt, (int64_t)zkie2_moe_router_words(h, experts)));
        const int64_t pairs = (h + 31) / 32 * 32;  // columns of the down weights' pairs of tiles
        const int64_t words[4] = {2 * (int64_t)zkie2_q4_words(experts, h, f, group, 0), (int64_t)zkie2_q4_words(experts, f, pairs, group, 0),
                                  2 * (int64_t)zkie2_q4_words(1, h, shared_f, group, 0), (int64_t)zkie2_q4_words(1, shared_f, pairs, group, 0)};
        const uint32_t* weights[4];
        for (int i = 0; i < 4; i++)
            weights[i] = reinterpret_cast<const uint32_t*>(b.memory<int32_t>(8 + i, "packed", at::kInt, words[i]));
        const at::Tensor &exp = tensor(b.at(12), "exp_table"), &silu = tensor(b.at(13), "silu_table");
        const uint64_t *exp_table = table_of(exp, "exp_table", dev), *silu_table = table_of(silu, "silu_table", dev);
        Rows residual;
        if (a[2] != Py_None) {
            residual = rows(tensor(a[2], "residual"), "residual", h, dev);
            if (residual.n != in.n)
                refuse("residual: " + std::to_string(residual.n) + " rows, " + std::to_string(in.n) + " are wanted");
        }
        const at::Tensor out = output(a[3], {in.n, h}, dev), gate = make({in.n, experts}, at::kUInt64, dev);
        const Apart apart(a[3], out);
        apart.from(in, h, "x");
        apart.from(residual, h, "the residual (and is not it)", true);
        for (int i = 7; apart.begin && i < 14; i++) apart.from(tensor(b.at(i), "MoeBlock"), "the block's weights and tables");
        apart.from(tensor(a[4], "err"), "the error word");
        // this call's own: calls on other streams may run beside it
        const uint64_t elems = zkie2_moe_rows_scratch_elems(in.n, h, experts, top_k, f, shared_f, group);
        const at::Tensor scratch = make({(int64_t)elems + 1}, at::kLong, dev);
        done(zkie2_moe_rows(in.data, in.stride, in.n, h, experts, top_k, f, shared_f, group, router, weights, exp_table,
                            exp.numel(), silu_table, silu.numel(), (uint32_t)b.size(6), residual.data, residual.stride,
                            static_cast<uint64_t*>(out.data_ptr()),
                            static_cast<uint64_t*>(gate.data_ptr()), word(a[4], dev), static_cast<uint64_t*>(scratch.data_ptr()),
                            stream(dev)), "zkie2_moe_rows");
        return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(gate));
    });
}

// choose(logits, history, history_lens, (pos, neg), presence, frequency, bias, allowed, mask_value, out, err) -> (token, out)
PyObject* choose(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return guarded([&]() -> PyObject* {
        if (n_args != 11) refuse("choose: 11 arguments");
        const at::Tensor& x = tensor(a[0], "logits");
        const int dev = device_of(x, "logits");
        if (x.dim() != 2 || x.size(1) == 0 || x.size(0) > 65535 || x.size(1) > 0x7FFFFFFF)
            refuse("logits: at most 65535 rows of a vocabulary are wanted, not " + said(x));
        const int64_t b = x.size(0), v = x.size(1), words = (v + 31) / 32;
        const auto* logits = flat<uint64_t>(x, "logits", at::kUInt64, dev, {b, v});
        const int32_t *history = nullptr, *lens = nullptr;
        int64_t tokens = 0;
        if (a[1] != Py_None) {
            const at::Tensor& t = tensor(a[1], "history");
            if (t.dim() != 2 || t.size(0) != b) refuse("history: " + std::to_string(b) + " rows of tokens are wanted, not " + said(t));
            tokens = t.size(1);
            history = flat<int32_t>(t, "history", at::kInt, dev, {b, tokens});
            if (a[2] != Py_None) lens = flat<int32_t>(tensor(a[2], "history_lens"), "history_lens", at::kInt, dev, {b});
            if (tokens == 0) history = lens = nullptr;  // an empty tensor has no address
        } else if (a[2] != Py_None) {
            refuse("choose_token: history_lens without a history");
        }
        if (!PyTuple_Check(a[3]) || PyTuple_GET_SIZE(a[3]) != 2) refuse("repeat: two factors are wanted");
        const uint64_t* bias = nullptr;
        int64_t bias_stride = 0, allowed_stride = 0;
        if (a[6] != Py_None) {
            const at::Tensor& t = tensor(a[6], "bias");
            bias_stride = t.dim() == 1 ? 0 : v;
            bias = bias_stride ? flat<uint64_t>(t, "bias", at::kUInt64, dev, {b, v}) : flat<uint64_t>(t, "bias", at::kUInt64, dev, {v});
        }
        const uint32_t* allowed = nullptr;
        if (a[7] != Py_None) {
            const at::Tensor& t = tensor(a[7], "allowed");
            allowed_stride = t.dim() == 1 ? 0 : words;
            allowed = reinterpret_cast<const uint32_t*>(allowed_stride ? flat<int32_t>(t, "allowed", at::kInt, dev, {b, words})
                                                                       : flat<int32_t>(t, "allowed", at::kInt, dev, {words}));
        }
        const at::Tensor out = output(a[9], {b, v}, dev), token = make({b}, at::kUInt32, dev);
        const Apart apart(a[9], out);
        apart.from(x, "the logits");
        apart.from(bias, 8 * v * (bias_stride ? b : 1), "the bias");
        apart.from(allowed, 4 * words * (allowed_stride ? b : 1), "the mask");
        apart.from(history, 4 * b * tokens, "the history");
        apart.from(lens, 4 * b, "the history's lengths");
        apart.from(tensor(a[10], "err"), "the error word");
        done(zkie2_choose_token(logits, b, v, history, tokens, lens, number(PyTuple_GET_ITEM(a[3], 0)),
                                number(PyTuple_GET_ITEM(a[3], 1)), number(a[4]), number(a[5]), bias, bias_stride, allowed,
                                allowed_stride, number(a[8]), static_cast<uint64_t*>(out.data_ptr()),
                                static_cast<uint32_t*>(token.data_ptr()), word(a[10], dev), stream(dev)), "zkie2_choose_token");
        return Py_BuildValue("(NN)", THPVariable_Wrap(token), THPVariable_Wrap(out));
    });
}

PyMethodDef methods[] = {
    {"project", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(project)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {"moe", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(moe)), METH_FASTCALL, nullptr},
    {"choose", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(choose)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
