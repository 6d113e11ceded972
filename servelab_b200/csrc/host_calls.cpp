// The host side of a call whose kernel takes few microseconds: checks of the arguments and the structure that the kernel gets.
//
// The attention over a cache is handed nine to eleven tensors.  Asked in Python for types, shapes, strides, devices and
// addresses, they cost 9 us a call before the launch itself, more than the kernel of a small step takes (5.7 us); here less
// than one.  Each operator has one function that checks and returns its structure as bytes with the tensors' device, and a
// launch function that calls a kernel's C entry with it.  Errors are KernelError.  Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "cache_args.h"

namespace {

PyObject* kernel_error = nullptr;

struct Refused {
    std::string why;
};
struct PythonError {};                           // (is set already)

std::string shape_of(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}
[[noreturn]] void refuse(const std::string& why) { throw Refused{why}; }

// The call's arguments in their order.
class Arguments {
public:
    Arguments(PyObject* const* args, Py_ssize_t n, Py_ssize_t wanted) : args_(args) {
        if (n != wanted) refuse(std::to_string(n) + " arguments, not " + std::to_string(wanted));
    }
    const char* text() {
        const char* s = PyUnicode_AsUTF8(args_[at_++]);
        if (s == nullptr) throw PythonError{};
        return s;
    }
    long long number() {
        const long long x = PyLong_AsLongLong(args_[at_++]);
        if (x == -1 && PyErr_Occurred()) throw PythonError{};
        return x;
    }
    int size(const char* name) {                 // a number that a kernel takes as an int
        const long long x = number();
        if (x < -0x7fffffffll || x > 0x7fffffffll) refuse(std::string(name) + " of " + std::to_string(x));
        return (int)x;
    }
    double real() {
        const double x = PyFloat_AsDouble(args_[at_++]);
        if (x == -1.0 && PyErr_Occurred()) throw PythonError{};
        return x;
    }
    const at::Tensor* tensor_or_none(const char* name) {
        PyObject* o = args_[at_++];
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) refuse(std::string(name) + " is no tensor");
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.layout() != at::kStrided) refuse(std::string(name) + " is not strided");
        return &t;
    }
    const at::Tensor& tensor(const char* name) {
        const at::Tensor* t = tensor_or_none(name);
        if (t == nullptr) refuse(std::string(name) + " is missing");
        return *t;
    }

private:
    PyObject* const* args_;
    int at_ = 0;
};

template <typename T> T* address(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T> T* address(const at::Tensor* t) { return t == nullptr ? nullptr : static_cast<T*>(t->data_ptr()); }

int in_int(int64_t n, const char* name) {
    if (n > 0x7fffffffll) refuse(std::string(name) + " of " + std::to_string(n));
    return (int)n;
}
void check_rows(const at::Tensor& t, const char* name) {
    if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) refuse(std::string(name) + " must be float32 or bfloat16");
}
void check_ints(const at::Tensor* t, const char* name) {
    if (t != nullptr && (t->scalar_type() != at::kInt || !t->is_contiguous())) refuse(std::string(name) + " must be a contiguous int32 tensor");
}
// All on one CUDA device (the caller compares it with the current one: a launch goes to that one's stream).
int device_of(const at::Tensor& first, std::initializer_list<const at::Tensor*> others) {
    if (!first.is_cuda()) refuse("a tensor on the CPU: there is no CPU path");
    const int here = first.get_device();
    for (const at::Tensor* t : others)
        if (t != nullptr && (!t->is_cuda() || t->get_device() != here))
            refuse("tensors on " + t->device().str() + " and cuda:" + std::to_string(here));
    return here;
}

// A layer's caches [pages, kv heads, page size, head size], whose scales [pages, kv heads, page size] are float32 and exist
// exactly for 8-bit kinds: the kind.
int cache_kind(const at::Tensor& rows, const at::Tensor& k, const at::Tensor& v, const at::Tensor* ks, const at::Tensor* vs, int kv_heads,
               int page, int dim) {
    const auto type = k.scalar_type();
    const int kind = type == rows.scalar_type() ? CACHE_PLAIN : type == at::kChar ? CACHE_INT8 : type == at::kFloat8_e4m3fn ? CACHE_E4M3 : -1;
    if (kind < 0 || v.scalar_type() != type)
        refuse(std::string("caches of ") + c10::toString(type) + " and " + c10::toString(v.scalar_type()) + " beside " +
               c10::toString(rows.scalar_type()) + " rows: the rows' type, int8 or float8_e4m3fn, both alike");
    if (k.dim() != 4 || v.sizes() != k.sizes() || k.size(1) != kv_heads || k.size(2) != page || k.size(3) != dim)
        refuse("caches of shapes " + shape_of(k) + " and " + shape_of(v) + ", not [pages, " + std::to_string(kv_heads) + ", " +
               std::to_string(page) + ", " + std::to_string(dim) + "]");
    if (!k.is_contiguous() || !v.is_contiguous()) refuse("the caches must be contiguous");
    if (kind != CACHE_PLAIN) {
        for (const at::Tensor* s : {ks, vs})
            if (s == nullptr || s->scalar_type() != at::kFloat || s->sizes() != k.sizes().slice(0, 3) || !s->is_contiguous())
                refuse("an 8-bit cache needs contiguous float32 scales [pages, kv heads, page size]");
    } else if (ks != nullptr || vs != nullptr) {
        refuse("a cache in the compute type has no scales");
    }
    return kind;
}

// What an operator raises: "<operator>: <why>"
template <typename F> PyObject* guarded(PyObject* const* args, Py_ssize_t n, F f) {
    const char* what = n > 0 && PyUnicode_Check(args[0]) ? PyUnicode_AsUTF8(args[0]) : "a call";
    try {
        return f();
    } catch (const Refused& r) {
        PyErr_SetString(kernel_error, (std::string(what) + ": " + r.why).c_str());
    } catch (const PythonError&) {
    } catch (const std::exception& e) {
        PyErr_SetString(kernel_error, (std::string(what) + ": " + e.what()).c_str());
    }
    return nullptr;
}
template <typename A> PyObject* as_bytes(const A& a) { return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&a), sizeof(A)); }
template <typename A> A from_bytes(PyObject* o) {
    if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) != (Py_ssize_t)sizeof(A)) refuse("no arguments of a kernel");
    A a;
    memcpy(&a, PyBytes_AS_STRING(o), sizeof(A));
    return a;
}

// write_args(what, qkv, bias, positions, slots, seq_of_token, block_table, page size, inv_freq, rotary_dim, q_out, k_cache, v_cache,
// k_scale, v_scale, heads, kv heads, head size, angles in 64 bits) -> (structure, device)
PyObject* write_args(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded(args, n, [&]() -> PyObject* {
        Arguments in(args, n, 19);
        in.text();
        const at::Tensor &qkv = in.tensor("qkv"), *bias = in.tensor_or_none("bias"), &pos = in.tensor("positions"),
                         *slots = in.tensor_or_none("slots"), &seq = in.tensor("seq_of_token"), &table = in.tensor("block_table");
        const int page = in.size("page size");
        const at::Tensor* inv_freq = in.tensor_or_none("inv_freq");
        const int rot = in.size("rotary size");
        const at::Tensor &q_out = in.tensor("q_out"), &k = in.tensor("k_cache"), &v = in.tensor("v_cache"),
                         *ks = in.tensor_or_none("k_scale"), *vs = in.tensor_or_none("v_scale");
        const int H = in.size("heads"), Hkv = in.size("kv heads"), D = in.size("head size"), exact = in.size("exact_angles");
        check_rows(qkv, "qkv");
        const int kind = cache_kind(qkv, k, v, ks, vs, Hkv, page, D);
        const int64_t width = ((int64_t)H + 2 * (int64_t)Hkv) * D;
        if (qkv.dim() != 2 || qkv.size(1) != width || q_out.dim() != 2 || q_out.size(0) != qkv.size(0) || q_out.size(1) != (int64_t)H * D ||
            q_out.scalar_type() != qkv.scalar_type())
            refuse("rows of " + shape_of(qkv) + " into queries of " + shape_of(q_out));
        const int64_t T = qkv.size(0);
        if (T > 0 && (qkv.stride(1) != 1 || q_out.stride(1) != 1)) refuse("rows whose elements are not neighbours");
        check_ints(&pos, "positions");
        check_ints(slots, "slots");
        check_ints(&seq, "seq_of_token");
        check_ints(&table, "block_table");
        if (pos.numel() < T || seq.numel() < T || (slots != nullptr && slots->numel() < T) || table.dim() != 2)
            refuse("positions, slots and requests of every token, and a table [requests, pages]");
        if (bias != nullptr && (bias->scalar_type() != at::kFloat || bias->numel() != width || !bias->is_contiguous()))
            refuse("a float32 bias of " + std::to_string(width) + " elements");
        if (inv_freq != nullptr && (inv_freq->scalar_type() != at::kFloat || 2 * inv_freq->numel() < rot || !inv_freq->is_contiguous()))
            refuse("float32 frequencies, one for each pair of rotary elements");
        const int device = device_of(qkv, {bias, &pos, slots, &seq, &table, inv_freq, &q_out, &k, &v, ks, vs});
        CacheWriteArgs a{};
        a.qkv = address<void>(qkv); a.ld = qkv.stride(0);
        a.bias = address<float>(bias);
        a.pos = address<int>(pos); a.slots = address<int>(slots);
        a.seq = address<int>(seq); a.table = address<int>(table);
        a.max_pages = in_int(table.size(1), "a table's width"); a.num_seqs = in_int(table.size(0), "requests");
        a.ps = page; a.num_pages = in_int(k.size(0), "pages");
        a.inv_freq = address<float>(inv_freq); a.rot = inv_freq != nullptr ? rot : 0;
        a.q_out = address<void>(q_out); a.ldq = q_out.stride(0);
        a.k = address<void>(k); a.v = address<void>(v); a.ks = address<float>(ks); a.vs = address<float>(vs);
        a.T = in_int(T, "tokens"); a.H = H; a.Hkv = Hkv; a.D = D; a.kind = kind; a.exact = exact != 0;
        return Py_BuildValue("(Ni)", as_bytes(a), device);
    });
}

// read_args(what, k_cache, v_cache, k_scale, v_scale, block_table, first, cu_rows, page size, k_out, v_out) -> (structure, device)
PyObject* read_args(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded(args, n, [&]() -> PyObject* {
        Arguments in(args, n, 11);
        in.text();
        const at::Tensor &k = in.tensor("k_cache"), &v = in.tensor("v_cache"), *ks = in.tensor_or_none("k_scale"),
                         *vs = in.tensor_or_none("v_scale"), &table = in.tensor("block_table"), &first = in.tensor("first"),
                         &cu = in.tensor("cu_rows");
        const int page = in.size("page size");
        const at::Tensor &k_out = in.tensor("k_out"), &v_out = in.tensor("v_out");
        if (k_out.dim() != 3 || k_out.sizes() != v_out.sizes() || v_out.scalar_type() != k_out.scalar_type())
            refuse("outputs of " + shape_of(k_out) + " and " + shape_of(v_out) + ": [rows, kv heads, head size], both alike");
        check_rows(k_out, "k_out");
        const int64_t rows = k_out.size(0);
        const int Hkv = in_int(k_out.size(1), "kv heads"), D = in_int(k_out.size(2), "head size");
        const int kind = cache_kind(k_out, k, v, ks, vs, Hkv, page, D);
        for (const at::Tensor* t : {&k_out, &v_out})
            if (rows > 0 && (t->stride(2) != 1 || t->stride(1) != D)) refuse("output rows whose heads are not neighbours");
        check_ints(&table, "block_table");
        check_ints(&first, "first");
        check_ints(&cu, "cu_rows");
        if (table.dim() != 2 || first.numel() < table.size(0) || cu.numel() < table.size(0) + 1)
            refuse("a table [requests, pages], first [requests] and cu_rows [requests + 1]");
        const int device = device_of(k, {&v, ks, vs, &table, &first, &cu, &k_out, &v_out});
        CacheReadArgs a{};
        a.k = address<void>(k); a.v = address<void>(v); a.ks = address<float>(ks); a.vs = address<float>(vs);
        a.table = address<int>(table);
        a.max_pages = in_int(table.size(1), "a table's width"); a.num_seqs = in_int(table.size(0), "requests");
        a.ps = page; a.num_pages = in_int(k.size(0), "pages");
        a.first = address<int>(first); a.cu = address<int>(cu);
        a.k_out = address<void>(k_out); a.v_out = address<void>(v_out); a.ldk = k_out.stride(0); a.ldv = v_out.stride(0);
        a.rows = in_int(rows, "rows"); a.Hkv = Hkv; a.D = D; a.kind = kind;
        return Py_BuildValue("(Ni)", as_bytes(a), device);
    });
}

// attention_args(what, largest head size, q, k_cache, v_cache, k_scale, v_scale, out, table, cu_q, ctx_len, mask, positions, heads,
// kv heads, head size, page size, scale, window, longest_q, longest_context) -> (structure, device, tokens, requests, whether
// the tensor-core kernels take the type, head size and alignment, kind of cache); None: nothing to do
PyObject* attention_args(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded(args, n, [&]() -> PyObject* {
        Arguments in(args, n, 21);
        in.text();
        const int most = in.size("head size");
        const at::Tensor &q = in.tensor("q"), &k = in.tensor("k_cache"), &v = in.tensor("v_cache"), *ks = in.tensor_or_none("k_scale"),
                         *vs = in.tensor_or_none("v_scale"), &out = in.tensor("out"), &table = in.tensor("table"), &cu = in.tensor("cu_q"),
                         &ctx = in.tensor("ctx_len"), *mask = in.tensor_or_none("mask"), *pos = in.tensor_or_none("positions");
        const int H = in.size("heads"), Hkv = in.size("kv heads"), D = in.size("head size"), page = in.size("page size");
        const double scale = in.real();
        const int window = in.size("window"), longest_q = in.size("longest_q"), longest_context = in.size("longest_context");
        if (D < 1 || D > most) refuse("head sizes 1.." + std::to_string(most) + ", got " + std::to_string(D));
        check_rows(q, "q");
        if (H < 1 || Hkv < 1 || H % Hkv) refuse(std::to_string(H) + " heads are no multiple of " + std::to_string(Hkv) + " kv heads");
        if (q.dim() != 2 || q.size(1) != (int64_t)H * D || out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type())
            refuse("queries " + shape_of(q) + " and results " + shape_of(out) + ", both [tokens, " + std::to_string((int64_t)H * D) +
                   "] of one type");
        const int kind = cache_kind(q, k, v, ks, vs, Hkv, page, D);
        check_ints(&table, "table");
        check_ints(&cu, "cu_q");
        check_ints(&ctx, "ctx_len");
        check_ints(mask, "mask");
        check_ints(pos, "positions");
        const int64_t T = q.size(0), S = cu.numel() - 1;
        if (S < 0 || table.dim() != 2 || table.size(0) < S || ctx.numel() < S)
            refuse("a table [requests, pages], cu_q [requests + 1] and ctx_len [requests]");
        if (!(scale > 0) || window < 0 || longest_q < 0 || longest_context < 0)
            refuse("scale " + std::to_string(scale) + " must be positive, window, longest_q and longest_context not negative");
        const int device = device_of(q, {&k, &v, ks, vs, &out, &table, &cu, &ctx, mask, pos});
        if (T == 0 || S == 0) Py_RETURN_NONE;
        if (q.stride(1) != 1 || out.stride(1) != 1) refuse("rows whose elements are not neighbours");
        CacheAttnArgs a{};
        a.q = address<void>(q); a.ldq = q.stride(0);
        a.out = address<void>(out); a.ldo = out.stride(0);
        a.k = address<void>(k); a.v = address<void>(v); a.ks = address<float>(ks); a.vs = address<float>(vs);
        a.table = address<int>(table); a.max_pages = in_int(table.size(1), "a table's width");
        a.cu_q = address<int>(cu); a.ctx_len = address<int>(ctx);
        a.mask = address<int>(mask); a.mask_words = mask != nullptr ? in_int(mask->size(1), "mask words") : 0;
        a.pos = address<int>(pos);
        a.parts = 1;
        a.T = in_int(T, "tokens"); a.S = in_int(S, "requests"); a.H = H; a.Hkv = Hkv; a.D = D; a.ps = page;
        a.num_pages = in_int(k.size(0), "pages"); a.kind = kind; a.window = window;
        a.scale = (float)scale;
        a.tiles = 1; a.cluster = 1;
        const bool fast = q.scalar_type() == at::kBFloat16 && (D == 64 || D == 128) && a.ldq % 8 == 0 && a.ldo % 8 == 0 &&
                          (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0;
        return Py_BuildValue("(NiiiOi)", as_bytes(a), device, a.T, a.S, fast ? Py_True : Py_False, kind);
    });
}

// launch(what, entry's address, structure, stream) -> the entry's code: of the write and read kernels
PyObject* launch(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded(args, n, [&]() -> PyObject* {
        Arguments in(args, n, 4);
        if (!PyBytes_Check(args[2]) || (PyBytes_GET_SIZE(args[2]) != (Py_ssize_t)sizeof(CacheWriteArgs) &&
                                        PyBytes_GET_SIZE(args[2]) != (Py_ssize_t)sizeof(CacheReadArgs)))
            refuse("no arguments of a kernel");
        in.text();
        const long long entry = in.number();
        const char* bytes = PyBytes_AS_STRING(args[2]);
        void* stream = reinterpret_cast<void*>(PyLong_AsUnsignedLongLong(args[3]));
        if (PyErr_Occurred()) throw PythonError{};
        return PyLong_FromLong(reinterpret_cast<int (*)(const void*, void*)>(entry)(bytes, stream));
    });
}

// launch_attention(what, entry's address, structure, stream, parts, units with one more, address of their sums, of their references,
// tiles, cluster, rows a block: 0 where the entry does not take them) -> the entry's code
PyObject* launch_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded(args, n, [&]() -> PyObject* {
        Arguments in(args, n, 11);
        in.text();
        const long long entry = in.number();
        CacheAttnArgs a = from_bytes<CacheAttnArgs>(args[2]);
        Arguments rest(args + 3, n - 3, 8);
        void* stream = reinterpret_cast<void*>(rest.number());
        a.parts = rest.size("parts");
        a.more = rest.size("units");
        a.part_o = reinterpret_cast<float*>(rest.number());
        a.part_ml = reinterpret_cast<float*>(rest.number());
        a.tiles = rest.size("tiles");
        a.cluster = rest.size("cluster");
        const int block = rest.size("rows a block");
        if (block > 0) return PyLong_FromLong(reinterpret_cast<int (*)(const void*, int, void*)>(entry)(&a, block, stream));
        return PyLong_FromLong(reinterpret_cast<int (*)(const void*, void*)>(entry)(&a, stream));
    });
}

// use_error(class): what the functions raise
PyObject* use_error(PyObject*, PyObject* error) {
    Py_INCREF(error);
    Py_XSETREF(kernel_error, error);
    Py_RETURN_NONE;
}

#define SLB_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {
    {"write_args", SLB_FAST(write_args), "checks cache_write's arguments"},
    {"read_args", SLB_FAST(read_args), "checks cache_read's arguments"},
    {"attention_args", SLB_FAST(attention_args), "checks the arguments of an attention over a cache"},
    {"launch", SLB_FAST(launch), "calls a kernel's entry"},
    {"launch_attention", SLB_FAST(launch_attention), "calls an attention kernel's entry"},
    {"use_error", use_error, METH_O, "the class of the errors"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "slb_host", "Checks and launches in native code.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_slb_host(void) { return PyModule_Create(&module); }
