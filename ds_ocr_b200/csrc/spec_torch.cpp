// spec_torch.cpp — the Python module ds_ocr_b200._spec: the speculative-
// decoding entry points of the C ABI (ds_cuda_tree_*, ds_cuda_token_probs_dev)
// on torch tensors. It checks the tensors, allocates outputs and the workspace,
// fills the descriptor and enqueues the call on torch's current stream. In
// Python a dozen tensors' types, shapes, strides and addresses cost 12 us a
// call, more than the kernels of a small step; here all of it is 3 us.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "ds_cuda.h"

namespace {

// Raised as ValueError (a bad tensor) or DsCudaError (a negative status).
struct Bad : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Failed : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python error is already set

PyObject *g_error = nullptr;  // DsCudaError

// The C ABI's entry points, of the library that the contexts come from (this
// module is not linked to one: there may be several).
#define ENTRIES(X)                                                                                                      \
    X(last_error) X(tree_attention_workspace) X(tree_attention_dev) X(tree_mask_dev) X(token_probs_dev) X(tree_verify_dev) \
        X(tree_verify_greedy_dev) X(tree_commit_dev)
#define X(f) decltype(&ds_cuda_##f) f;
struct {
    bool bound;
    ENTRIES(X)
} abi;
#undef X

std::string text(c10::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + ")";
}

struct Call {
    ds_cuda_ctx_t *ctx;
    c10::DeviceIndex device;
    c10::TensorOptions options;

    Call(PyObject *const *args, Py_ssize_t n, Py_ssize_t want) {
        if (!abi.bound) throw Failed("the module is not bound to the library");
        if (n != want) throw Bad("expected " + std::to_string(want) + " arguments");
        ctx = static_cast<ds_cuda_ctx_t *>(PyLong_AsVoidPtr(args[0]));
        device = static_cast<c10::DeviceIndex>(PyLong_AsLong(args[1]));
        if (PyErr_Occurred()) throw Raised();
        options = c10::TensorOptions().device(c10::Device(c10::DeviceType::CUDA, device));
    }
    // torch's default stream is the legacy stream (handle 0), which the C ABI
    // would take for the context's own
    void *stream() const {
        cudaStream_t s = c10::cuda::getCurrentCUDAStream(device).stream();
        return s ? s : cudaStreamLegacy;
    }
    void check(int rc, const char *what) const {
        if (rc < 0) throw Failed(std::string(what) + " failed (" + std::to_string(rc) + "): " + abi.last_error(ctx));
    }

    const at::Tensor &tensor(const char *name, PyObject *o) const {
        if (!THPVariable_Check(o)) throw Bad(std::string(name) + ": expected a tensor");
        return THPVariable_Unpack(o);
    }
    // A tensor of this shape and type on the device, its last dimension contiguous.
    const at::Tensor &strided(const char *name, PyObject *o, c10::IntArrayRef shape, at::ScalarType type) const {
        const at::Tensor &t = tensor(name, o);
        if (t.scalar_type() != type || t.sizes() != shape || t.layout() != at::kStrided || !t.is_cuda() ||
            t.device().index() != device)
            throw Bad(std::string(name) + ": expected " + c10::toString(type) + " " + text(shape) + " on cuda:" +
                      std::to_string(device) + ", got " + c10::toString(t.scalar_type()) + " " + text(t.sizes()) + " on " +
                      t.device().str());
        if (t.stride(-1) != 1 && t.size(-1) > 1) throw Bad(std::string(name) + ": the last dimension must be contiguous");
        return t;
    }
    const at::Tensor &whole(const char *name, PyObject *o, c10::IntArrayRef shape, at::ScalarType type) const {
        const at::Tensor &t = strided(name, o, shape, type);
        if (!t.is_contiguous()) throw Bad(std::string(name) + ": must be contiguous");
        return t;
    }
    template <class T> T *ptr(const char *name, PyObject *o, c10::IntArrayRef shape, at::ScalarType type) const {
        return static_cast<T *>(whole(name, o, shape, type).data_ptr());
    }
    template <class T> T *maybe(const char *name, PyObject *o, c10::IntArrayRef shape, at::ScalarType type) const {
        return o == Py_None ? nullptr : ptr<T>(name, o, shape, type);
    }
    static void strides(const at::Tensor &t, int64_t *s, int n) {
        for (int i = 0; i < n; i++) s[i] = t.stride(i);
    }
};

// A size for the C ABI, whose sizes are ints.
int size(const char *name, int64_t n) {
    if (n > INT32_MAX) throw Bad(std::string(name) + ": " + std::to_string(n) + " (at most 2^31 - 1)");
    return (int)n;
}

int spec_type(const char *name, at::ScalarType t) {
    if (t == at::kBFloat16) return DS_CUDA_SPEC_BF16;
    if (t == at::kHalf) return DS_CUDA_SPEC_F16;
    if (t == at::kFloat) return DS_CUDA_SPEC_F32;
    throw Bad(std::string(name) + ": unsupported dtype " + c10::toString(t));
}

// One tensor, or with F32 queries its BF16 plane and optional lo plane.
struct Planes {
    PyObject *hi, *lo = nullptr;
    Planes(const char *name, PyObject *o, bool pair) : hi(o) {
        if (THPVariable_Check(o)) return;
        if (!PyTuple_Check(o) && !PyList_Check(o)) throw Bad(std::string(name) + ": expected a tensor or its planes");
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
        if (n < 1 || n > (pair ? 2 : 1))
            throw Bad(std::string(name) + ": " + std::to_string(n) + " planes" +
                      (pair ? " (at most 2)" : " (a second plane goes with float32 queries)"));
        hi = PySequence_Fast_GET_ITEM(o, 0);
        if (n == 2) lo = PySequence_Fast_GET_ITEM(o, 1);
    }
};

PyObject *tree_attention(PyObject *const *x, Py_ssize_t n_args) {
    const Call c(x, n_args, 13);
    const at::Tensor &q0 = c.tensor("q", x[2]);
    if (q0.dim() != 4) throw Bad("q: expected [batch x n_nodes x n_heads x head_dim]");
    const at::ScalarType type = q0.scalar_type();
    ds_cuda_tree_attention_t d = {};
    d.type = spec_type("q", type);
    const bool pair = d.type == DS_CUDA_SPEC_F32;
    const at::ScalarType rows = pair ? at::kBFloat16 : type;
    const int64_t b = q0.size(0), n = q0.size(1), heads = q0.size(2), hd = q0.size(3);
    const Planes k("k", x[3], pair), v("v", x[4], pair), tk("tree_k", x[5], pair), tv("tree_v", x[6], pair);
    const at::Tensor &k0 = c.tensor("k", k.hi);
    if (k0.dim() != 4) throw Bad("k: expected [batch x n_kv_heads x kv_max x head_dim]");
    const int64_t kv = k0.size(1), cap = k0.size(2);
    const int64_t shape[4] = {b, n, heads, hd}, cache[4] = {b, kv, cap, hd}, tree[4] = {b, kv, n, hd};
    d.batch = size("batch", b), d.n_nodes = size("n_nodes", n), d.n_heads = size("n_heads", heads);
    d.n_kv_heads = size("n_kv_heads", kv), d.head_dim = size("head_dim", hd), d.kv_max = size("kv_max", cap);
    d.scale = x[10] == Py_None ? 1.f / std::sqrt((float)hd) : (float)PyFloat_AsDouble(x[10]);
    if (PyErr_Occurred()) throw Raised();
    const at::Tensor &q = c.strided("q", x[2], shape, type);
    d.q = q.data_ptr();
    c.strides(q, d.q_stride, 3);
    auto side = [&](const char *name, const Planes &p, c10::IntArrayRef s, const void *&hi, const void *&lo, int64_t *st) {
        const at::Tensor &t = c.strided(name, p.hi, s, rows);
        hi = t.data_ptr();
        c.strides(t, st, 3);
        if (!p.lo) return;
        const at::Tensor &u = c.strided(name, p.lo, s, rows);
        for (int i = 0; i < 3; i++)  // (the stride of a dimension of one element is never used)
            if (t.size(i) > 1 && u.stride(i) != t.stride(i)) throw Bad(std::string(name) + ": the planes must have the same strides");
        lo = u.data_ptr();
    };
    side("k", k, cache, d.k, d.k_lo, d.k_stride);
    side("v", v, cache, d.v, d.v_lo, d.v_stride);
    side("tree_k", tk, tree, d.tree_k, d.tree_k_lo, d.tree_k_stride);
    side("tree_v", tv, tree, d.tree_v, d.tree_v_lo, d.tree_v_stride);
    d.lens = c.ptr<int>("lens", x[7], {b}, at::kInt);
    d.mask = c.ptr<uint64_t>("mask", x[8], {b, n, (n + 63) / 64}, at::kLong);
    d.nodes = c.maybe<int>("counts", x[9], {b}, at::kInt);
    d.lse = c.maybe<float>("lse", x[12], {b, n, heads}, at::kFloat);
    const at::Tensor out = x[11] == Py_None ? at::empty(shape, c.options.dtype(type)) : c.strided("out", x[11], shape, type);
    d.out = out.data_ptr();
    c.strides(out, d.out_stride, 3);
    at::Tensor ws;
    d.workspace_bytes = abi.tree_attention_workspace(c.ctx, &d);
    if (d.workspace_bytes) {
        ws = at::empty({(int64_t)d.workspace_bytes}, c.options.dtype(at::kByte));
        d.workspace = ws.data_ptr();
    }
    c.check(abi.tree_attention_dev(c.ctx, &d, c.stream()), "tree_attention");
    return THPVariable_Wrap(out);
}

PyObject *tree_mask(PyObject *const *x, Py_ssize_t n_args) {
    const Call c(x, n_args, 4);
    const at::Tensor &p = c.tensor("parents", x[2]);
    if (p.dim() != 2) throw Bad("parents: expected [batch x n_nodes]");
    const int64_t b = size("batch", p.size(0)), n = size("n_nodes", p.size(1));
    const int *parents = c.ptr<int>("parents", x[2], {b, n}, at::kInt), *nodes = c.maybe<int>("counts", x[3], {b}, at::kInt);
    const at::Tensor mask = at::empty({b, n, (n + 63) / 64}, c.options.dtype(at::kLong)), depth = at::empty({b, n}, c.options.dtype(at::kInt));
    c.check(abi.tree_mask_dev(c.ctx, parents, nodes, (int)b, (int)n, static_cast<uint64_t *>(mask.data_ptr()),
                                  static_cast<int *>(depth.data_ptr()), c.stream()), "tree_mask");
    return Py_BuildValue("(NN)", THPVariable_Wrap(mask), THPVariable_Wrap(depth));
}

PyObject *token_probs(PyObject *const *x, Py_ssize_t n_args) {
    const Call c(x, n_args, 5);
    const at::Tensor &l = c.tensor("logits", x[2]);
    if (l.dim() != 2) throw Bad("logits: expected [rows x vocab]");
    const int64_t shape[2] = {size("rows", l.size(0)), size("vocab", l.size(1))};
    const int type = spec_type("logits", l.scalar_type());
    c.strided("logits", x[2], shape, l.scalar_type());
    const float *temp = c.maybe<float>("temperature", x[3], {shape[0]}, at::kFloat);
    const at::Tensor out = x[4] == Py_None ? at::empty(shape, c.options.dtype(at::kFloat)) : c.whole("out", x[4], shape, at::kFloat);
    c.check(abi.token_probs_dev(c.ctx, type, l.data_ptr(), (int)shape[0], (int)shape[1], l.stride(0), temp,
                                    static_cast<float *>(out.data_ptr()), c.stream()), "token_probs");
    return THPVariable_Wrap(out);
}

// path [b x n], accepted [b], token [b]
struct Results {
    at::Tensor path, both, accepted, token;
    Results(const Call &c, int64_t b, int64_t n)
        : path(at::empty({b, n}, c.options.dtype(at::kInt))), both(at::empty({2, b}, c.options.dtype(at::kInt))),
          accepted(both.select(0, 0)), token(both.select(0, 1)) {}
    static int *p(const at::Tensor &t) { return static_cast<int *>(t.data_ptr()); }
    PyObject *wrap() const { return Py_BuildValue("(NNN)", THPVariable_Wrap(path), THPVariable_Wrap(accepted), THPVariable_Wrap(token)); }
};

PyObject *verify(PyObject *const *x, Py_ssize_t n_args) {
    const Call c(x, n_args, 9);
    const at::Tensor &t0 = c.tensor("tokens", x[2]), &p0 = c.tensor("target", x[4]);
    if (t0.dim() != 2) throw Bad("tokens: expected [batch x n_nodes]");
    if (p0.dim() != 3) throw Bad("target: expected [batch x n_nodes x vocab]");
    const int64_t b = t0.size(0), n = t0.size(1), vocab = p0.size(2), shape[3] = {b, n, vocab};
    ds_cuda_tree_verify_t d = {};
    d.batch = size("batch", b), d.n_nodes = size("n_nodes", n), d.vocab = size("vocab", vocab);
    d.tokens = c.ptr<int>("tokens", x[2], {b, n}, at::kInt);
    d.parents = c.ptr<int>("parents", x[3], {b, n}, at::kInt);
    auto probs = [&](const char *name, PyObject *o, const float *&p, int64_t *st) {
        const at::Tensor &t = c.strided(name, o, shape, at::kFloat);
        p = static_cast<const float *>(t.data_ptr());
        c.strides(t, st, 2);
    };
    probs("target", x[4], d.target, d.target_stride);
    if (x[5] != Py_None) probs("draft", x[5], d.draft, d.draft_stride);
    d.accept_u = c.ptr<float>("accept_u", x[6], {b, n}, at::kFloat);
    d.sample_u = c.ptr<float>("sample_u", x[7], {b}, at::kFloat);
    d.nodes = c.maybe<int>("counts", x[8], {b}, at::kInt);
    const Results r(c, b, n);
    d.path = r.p(r.path), d.accepted = r.p(r.accepted), d.token = r.p(r.token);
    c.check(abi.tree_verify_dev(c.ctx, &d, c.stream()), "tree_verify");
    return r.wrap();
}

PyObject *verify_greedy(PyObject *const *x, Py_ssize_t n_args) {
    const Call c(x, n_args, 6);
    const at::Tensor &t0 = c.tensor("tokens", x[2]);
    if (t0.dim() != 2) throw Bad("tokens: expected [batch x n_nodes]");
    const int64_t b = size("batch", t0.size(0)), n = size("n_nodes", t0.size(1));
    const int *tokens = c.ptr<int>("tokens", x[2], {b, n}, at::kInt), *parents = c.ptr<int>("parents", x[3], {b, n}, at::kInt);
    const int *want = c.ptr<int>("target_tokens", x[4], {b, n}, at::kInt), *nodes = c.maybe<int>("counts", x[5], {b}, at::kInt);
    const Results r(c, b, n);
    c.check(abi.tree_verify_greedy_dev(c.ctx, tokens, parents, nodes, want, (int)b, (int)n, r.p(r.path), r.p(r.accepted),
                                           r.p(r.token), c.stream()), "tree_verify_greedy");
    return r.wrap();
}

PyObject *commit(PyObject *const *x, Py_ssize_t n_args) {
    const Call c(x, n_args, 7);
    for (int i = 2; i < 4; i++)
        if (!PyTuple_Check(x[i]) && !PyList_Check(x[i])) throw Bad("commit: expected a list of caches and a list of trees");
    const Py_ssize_t m = PySequence_Fast_GET_SIZE(x[2]);
    if (m < 1 || m > 8 || PySequence_Fast_GET_SIZE(x[3]) != m)
        throw Bad("commit: " + std::to_string(m) + " caches and " + std::to_string(PySequence_Fast_GET_SIZE(x[3])) + " trees (1 to 8 pairs)");
    const at::Tensor &first = c.tensor("cache", PySequence_Fast_GET_ITEM(x[2], 0)), &path = c.tensor("path", x[5]);
    if (first.dim() != 5 || first.element_size() != 2)
        throw Bad("caches: expected 16-bit [layers x batch x n_kv_heads x kv_max x head_dim]");
    if (path.dim() != 2) throw Bad("path: expected [batch x n_nodes]");
    const int64_t b = path.size(0), n = path.size(1), layers = first.size(0), kv = first.size(2), cap = first.size(3), hd = first.size(4);
    const int64_t cache[5] = {layers, b, kv, cap, hd}, tree[5] = {layers, b, kv, n, hd};
    ds_cuda_tree_commit_t d = {};
    d.n_tensors = (int)m, d.layers = size("layers", layers), d.batch = size("batch", b), d.n_nodes = size("n_nodes", n);
    d.n_kv_heads = size("n_kv_heads", kv), d.head_dim = size("head_dim", hd), d.kv_max = size("kv_max", cap);
    for (Py_ssize_t i = 0; i < m; i++) {
        const at::Tensor &t = c.strided("cache", PySequence_Fast_GET_ITEM(x[2], i), cache, first.scalar_type());
        const at::Tensor &u = c.strided("tree", PySequence_Fast_GET_ITEM(x[3], i), tree, first.scalar_type());
        d.cache[i] = t.data_ptr();
        d.tree[i] = u.data_ptr();
        c.strides(t, d.cache_stride[i], 4);
        c.strides(u, d.tree_stride[i], 4);
    }
    d.lens = c.ptr<int>("lens", x[4], {b}, at::kInt);
    d.path = c.ptr<int>("path", x[5], {b, n}, at::kInt);
    d.accepted = c.ptr<int>("accepted", x[6], {b}, at::kInt);
    const at::Tensor lens = at::empty({b}, c.options.dtype(at::kInt));
    d.new_lens = static_cast<int *>(lens.data_ptr());
    c.check(abi.tree_commit_dev(c.ctx, &d, c.stream()), "tree_commit");
    return THPVariable_Wrap(lens);
}

template <PyObject *(*F)(PyObject *const *, Py_ssize_t)> PyObject *guarded(PyObject *, PyObject *const *args, Py_ssize_t n) {
    try {
        return F(args, n);
    } catch (const Raised &) {
    } catch (const Bad &e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const Failed &e) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, e.what());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// bind({"ds_cuda_...": address}): every entry of the list, or KeyError.
PyObject *bind(PyObject *, PyObject *table) {
    abi.bound = false;
    auto find = [&](const char *name) {
        PyObject *p = PyMapping_GetItemString(table, name);
        void *at = p ? PyLong_AsVoidPtr(p) : nullptr;
        Py_XDECREF(p);
        return at;
    };
#define X(f) \
    if (!(abi.f = reinterpret_cast<decltype(abi.f)>(find("ds_cuda_" #f)))) return nullptr;
    ENTRIES(X)
#undef X
    abi.bound = true;
    Py_RETURN_NONE;
}

PyObject *set_error(PyObject *, PyObject *type) {
    Py_INCREF(type);
    Py_XDECREF(g_error);
    g_error = type;
    Py_RETURN_NONE;
}

#define ENTRY(f) {#f, (PyCFunction)(void (*)(void))guarded<f>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(tree_attention), ENTRY(tree_mask), ENTRY(token_probs), ENTRY(verify), ENTRY(verify_greedy),
                         ENTRY(commit), {"bind", bind, METH_O, nullptr}, {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_spec", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__spec() { return PyModule_Create(&module); }
