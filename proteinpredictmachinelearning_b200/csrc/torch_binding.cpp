// torch_binding.cpp -- host side of the entries that a serving program calls many times for a token (8-bit Linears, norm and
// rotation of queries and keys), as a CPython module over the C ABI: checks of the tensors, new results and workspaces from torch's
// allocator on the current stream, one call into libppml_b200.so.  Done in Python, the same checks and the argument conversion of
// ctypes take 7 to 14 us a call, several times what the kernels take for one token.
//
// Wrong tensors raise ValueError, a status of the library RuntimeError, an allocation that fails torch.OutOfMemoryError; no C++ exception
// leaves a function.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <climits>
#include <cstring>
#include <stdexcept>
#include <string>

#include "../../include/ppml_b200.h"

namespace {

struct Refused : std::invalid_argument { using std::invalid_argument::invalid_argument; };

[[noreturn]] void refuse(const char* name, const std::string& want) { throw Refused(std::string(name) + ": " + want); }
[[noreturn]] void refuse(const char* name, const at::Tensor& t, const std::string& want) {
    refuse(name, c10::str(want, " wanted, got ", t.sizes(), " of ", t.scalar_type(), " on ", t.device(), " with strides ", t.strides()));
}
void check(int rc, const char* what) {
    if (rc != 0) throw std::runtime_error(std::string(what) + " failed with status " + std::to_string(rc));
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(name, "a tensor is wanted");
    return THPVariable_Unpack(o);
}
const at::Tensor* optional_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int integer(PyObject* o, const char* name) {
    const long v = PyLong_AsLong(o);
    if ((v == -1 && PyErr_Occurred()) || v < INT_MIN || v > INT_MAX) { PyErr_Clear(); refuse(name, "an integer is wanted"); }
    return static_cast<int>(v);
}
// index of a word in a list
template <size_t N> int word(PyObject* o, const char* const (&words)[N], const char* name) {
    const char* s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    std::string all;
    for (size_t i = 0; i < N; ++i) {
        if (s && std::strcmp(s, words[i]) == 0) return static_cast<int>(i);
        all += std::string(i ? ", " : "") + words[i];
    }
    PyErr_Clear();
    refuse(name, "one of " + all + " is wanted");
}
constexpr const char* kActs[] = {"none", "sigmoid", "silu", "gelu", "tanh", "relu"};
constexpr const char* kNorms[] = {"none", "rms", "layer"};

int type_code(at::ScalarType t) {
    return t == at::kFloat ? PPML_B200_TYPE_F32 : t == at::kHalf ? PPML_B200_TYPE_F16 : t == at::kBFloat16 ? PPML_B200_TYPE_BF16 : -1;
}

// The row pitch of an [M, K] matrix of that type and device whose rows are contiguous and lie apart.
int64_t pitch(const at::Tensor& t, at::ScalarType type, int64_t M, int64_t K, c10::Device dev, const char* name) {
    if (t.dim() == 2 && t.scalar_type() == type && t.device() == dev && t.size(0) == M && t.size(1) == K && (K <= 1 || t.stride(1) == 1)) {
        const int64_t s = t.stride(0);
        if (s >= K) return s;
        if (M <= 1) return K;
    }
    refuse(name, t, c10::str("[", M, ", ", K, "] of ", type, " on ", dev, ", rows contiguous and apart,"));
}
const float* vec(const at::Tensor* t, int64_t n, c10::Device dev, const char* name) {
    if (!t) return nullptr;
    if (t->dim() == 1 && t->size(0) == n && t->scalar_type() == at::kFloat && t->device() == dev && (n <= 1 || t->stride(0) == 1))
        return static_cast<const float*>(t->data_ptr());
    refuse(name, *t, c10::str(n, " contiguous fp32 values on ", dev));
}
int extent(int64_t n, const char* name) {
    if (n > INT_MAX) refuse(name, "an extent beyond 32 bits");
    return static_cast<int>(n);
}
// torch's CUDA allocation without its dispatcher (0.6 us less a tensor)
at::Tensor fresh(at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type, c10::Device dev) {
    return at::Tensor(at::detail::empty_strided_cuda(sizes, strides, type, dev));
}
void* stream_of(c10::Device dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// What a function makes: tensors that may also be the caller's own.
PyObject* give(const at::Tensor& t, PyObject* own) { return own && own != Py_None ? Py_NewRef(own) : THPVariable_Wrap(t); }

// ---- 8-bit Linears ----
const at::Tensor& activations(PyObject* o) {
    const at::Tensor& x = tensor(o, "x");
    if (x.dim() != 2 || !x.is_cuda() || type_code(x.scalar_type()) < 0) refuse("x", x, "a matrix of fp32, fp16 or bf16 on the GPU");
    return x;
}

// quantize_tokens_i8(x, q | None, scale | None) -> (q, scale)
PyObject* quantize_tokens_i8(PyObject* const* a) {
    const at::Tensor& x = activations(a[0]);
    const int64_t M = x.size(0), K = x.size(1);
    const c10::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t ld = pitch(x, x.scalar_type(), M, K, dev, "x");
    const at::Tensor* own_q = optional_tensor(a[1], "q");
    const at::Tensor* own_s = optional_tensor(a[2], "scale");
    const at::Tensor q = own_q ? *own_q : fresh({M, K}, {(K + 15) / 16 * 16, 1}, at::kChar, dev), s = own_s ? *own_s : fresh({M}, {1}, at::kFloat, dev);
    check(ppml_b200_quantize_tokens_i8(x.data_ptr(), type_code(x.scalar_type()), ld, static_cast<int8_t*>(q.data_ptr()), pitch(q, at::kChar, M, K, dev, "q"),
                                       const_cast<float*>(vec(&s, M, dev, "scale")), M, extent(K, "x"), stream_of(dev)), "quantize_tokens_i8");
    PyObject* two = PyTuple_New(2);
    if (!two) return nullptr;
    PyTuple_SET_ITEM(two, 0, give(q, a[1])); PyTuple_SET_ITEM(two, 1, give(s, a[2]));
    return two;
}

// What both products take: W, w_scale, bias | None, gate | None, act, dtype | None, path, out | None from a[0].
struct Product {
    const at::Tensor* W; const at::Tensor* gate;
    at::Tensor out;
    const float* w_scale; const float* bias;
    int64_t ldb, ldc, ld_gate;
    int M, K, N, c_type, act, path;
    Product(PyObject* const* a, int64_t M_, int64_t K_, c10::Device dev, at::ScalarType type) {
        W = &tensor(a[0], "W");
        if (W->dim() != 2) refuse("W", *W, "[N, K]");
        const int64_t n = W->size(0);
        act = word(a[4], kActs, "act");
        const at::Tensor* own = optional_tensor(a[7], "out");
        if (own) type = own->scalar_type();
        else if (a[5] != Py_None) {
            if (!THPDtype_Check(a[5])) refuse("dtype", "a type is wanted");
            type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
        }
        c_type = type_code(type);
        if (c_type < 0) refuse("dtype", "fp32, fp16 or bf16 is wanted");
        path = integer(a[6], "path");
        ldb = pitch(*W, at::kChar, n, K_, dev, "W");
        w_scale = vec(&tensor(a[1], "w_scale"), n, dev, "w_scale");
        bias = vec(optional_tensor(a[2], "bias"), n, dev, "bias");
        gate = optional_tensor(a[3], "gate");
        ld_gate = gate ? pitch(*gate, type, M_, n, dev, "gate") : 0;
        if (own) { out = *own; ldc = pitch(out, type, M_, n, dev, "out"); }
        else { out = fresh({M_, n}, {n, 1}, type, dev); ldc = n; }
        M = extent(M_, "x"); K = extent(K_, "x"); N = extent(n, "W");
    }
    const void* gate_ptr() const { return gate ? gate->data_ptr() : nullptr; }
    const int8_t* w_ptr() const { return static_cast<const int8_t*>(W->data_ptr()); }
};

// mul_mat_i8(A, a_scale, W, w_scale, bias, gate, act, dtype, path, out) -> out
PyObject* mul_mat_i8(PyObject* const* a) {
    const at::Tensor& A = tensor(a[0], "A");
    if (A.dim() != 2 || !A.is_cuda() || A.scalar_type() != at::kChar) refuse("A", A, "an int8 matrix on the GPU");
    const int64_t M = A.size(0), K = A.size(1);
    const c10::Device dev = A.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t lda = pitch(A, at::kChar, M, K, dev, "A");
    const float* a_scale = vec(&tensor(a[1], "a_scale"), M, dev, "a_scale");
    const Product p(a + 2, M, K, dev, at::kFloat);
    check(ppml_b200_mul_mat_i8(static_cast<const int8_t*>(A.data_ptr()), lda, a_scale, p.w_ptr(), p.ldb, p.w_scale, p.out.data_ptr(), p.ldc, p.c_type,
                               p.M, p.K, p.N, p.bias, p.gate_ptr(), p.ld_gate, p.act, p.path, stream_of(dev)), "mul_mat_i8");
    return give(p.out, a[9]);
}

// Whether the memory from the first to the last element of two matrices has a byte in common.
bool ranges_meet(const at::Tensor& a, int64_t pitch_a, const at::Tensor& b, int64_t pitch_b) {
    auto bytes = [](const at::Tensor& t, int64_t p) { return static_cast<uintptr_t>(((t.size(0) - 1) * p + t.size(1)) * t.element_size()); };
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.data_ptr()), b0 = reinterpret_cast<uintptr_t>(b.data_ptr());
    return a0 < b0 + bytes(b, pitch_b) && b0 < a0 + bytes(a, pitch_a);
}

// linear_i8(x, W, w_scale, bias, gate, act, dtype, path, out) -> out
PyObject* linear_i8(PyObject* const* a) {
    const at::Tensor& x = activations(a[0]);
    const int64_t M = x.size(0), K = x.size(1);
    const c10::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t ld = pitch(x, x.scalar_type(), M, K, dev, "x");
    const Product p(a + 1, M, K, dev, x.scalar_type());
    const int64_t need = ppml_b200_linear_i8_workspace(M, p.K);
    at::Tensor ws;
    if (need) ws = fresh({need}, {1}, at::kByte, dev);
    // An `out` around x itself: the one kernel for a few tokens reads x until its end, so the integers are made first.
    if (!need && M > 0 && a[8] != Py_None && p.path != PPML_B200_PATH_UMMA && ranges_meet(x, ld, p.out, p.ldc)) {
        const int64_t row = (K + 15) / 16 * 16;
        ws = fresh({M * row}, {1}, at::kChar, dev);
        const at::Tensor scale = fresh({M}, {1}, at::kFloat, dev);
        int8_t* q = static_cast<int8_t*>(ws.data_ptr());
        float* s = static_cast<float*>(scale.data_ptr());
        check(ppml_b200_quantize_tokens_i8(x.data_ptr(), type_code(x.scalar_type()), ld, q, row, s, M, p.K, stream_of(dev)), "linear_i8");
        check(ppml_b200_mul_mat_i8(q, row, s, p.w_ptr(), p.ldb, p.w_scale, p.out.data_ptr(), p.ldc, p.c_type, p.M, p.K, p.N, p.bias, p.gate_ptr(), p.ld_gate,
                                   p.act, p.path, stream_of(dev)), "linear_i8");
        return give(p.out, a[8]);
    }
    check(ppml_b200_linear_i8(x.data_ptr(), type_code(x.scalar_type()), ld, p.w_ptr(), p.ldb, p.w_scale, p.out.data_ptr(), p.ldc, p.c_type, p.M, p.K, p.N,
                              p.bias, p.gate_ptr(), p.ld_gate, p.act, p.path, need ? ws.data_ptr() : nullptr, need, stream_of(dev)), "linear_i8");
    return give(p.out, a[8]);
}

// ---- norm and rotation ----
// The view of a tensor with the shape, type and device of `like` [B, L, h, d], contiguous d and any other strides.
ppml_b200_heads heads(const at::Tensor& t, const at::Tensor& like, const char* name) {
    if (t.dim() != 4 || t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type() || t.device() != like.device() ||
        (t.stride(3) != 1 && t.size(3) > 1))
        refuse(name, t, c10::str(like.sizes(), " of ", like.scalar_type(), " on ", like.device(), " with a contiguous head dim"));
    return ppml_b200_heads{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
struct OptionalHeads {
    ppml_b200_heads v{};
    bool is = false;
    OptionalHeads(const at::Tensor* t, const at::Tensor* like, const char* name) : is(t != nullptr) {
        if ((t == nullptr) != (like == nullptr)) refuse(name, "missing, or without its input");
        if (t) v = heads(*t, *like, name);
    }
    const ppml_b200_heads* ptr() const { return is ? &v : nullptr; }
};

// Q | None, K | None, q_weight | None, k_weight | None, norm, eps, cos | None, sin | None, positions | None, interleaved
struct QkArgs {
    const at::Tensor* Q; const at::Tensor* K; const at::Tensor* any;
    ppml_b200_qk_cfg cfg{};
    const float* qw; const float* kw; const float* cos = nullptr; const float* sin = nullptr;
    const int32_t* pos = nullptr;
    c10::Device dev = c10::Device(c10::kCPU);
    explicit QkArgs(PyObject* const* a) {
        Q = optional_tensor(a[0], "Q"); K = optional_tensor(a[1], "K");
        any = Q ? Q : K;
        if (!any) refuse("Q", "Q, K or both are wanted");
        if (any->dim() != 4 || !any->is_cuda() || type_code(any->scalar_type()) < 0)
            refuse(Q ? "Q" : "K", *any, "[B, L, heads, d] of fp32, fp16 or bf16 on the GPU");
        dev = any->device();
        const int64_t B = any->size(0), L = any->size(1), d = any->size(3);
        if (Q && K && (K->dim() != 4 || K->size(0) != B || K->size(1) != L || K->size(3) != d || K->scalar_type() != Q->scalar_type() || K->device() != dev))
            refuse("K", *K, c10::str("[", B, ", ", L, ", heads, ", d, "] of ", Q->scalar_type(), " on ", dev));
        cfg.B = extent(B, "Q"); cfg.L = extent(L, "Q"); cfg.d = extent(d, "Q");
        cfg.hq = Q ? extent(Q->size(2), "Q") : 0; cfg.hk = K ? extent(K->size(2), "K") : 0;
        cfg.type = type_code(any->scalar_type());
        cfg.norm = word(a[4], kNorms, "norm");
        cfg.eps = static_cast<float>(PyFloat_AsDouble(a[5]));
        if (PyErr_Occurred()) { PyErr_Clear(); refuse("eps", "a number is wanted"); }
        qw = vec(optional_tensor(a[2], "q_weight"), d, dev, "q_weight");
        kw = vec(optional_tensor(a[3], "k_weight"), d, dev, "k_weight");
        const at::Tensor* c = optional_tensor(a[6], "cos");
        const at::Tensor* s = optional_tensor(a[7], "sin");
        if (c || s) {
            if (!c || !s) refuse("cos", "cos and sin come together");
            for (const at::Tensor* t : {c, s})
                if (t->dim() != 2 || t->sizes() != c->sizes() || t->scalar_type() != at::kFloat || t->device() != dev || !t->is_contiguous())
                    refuse("cos, sin", *t, c10::str("[rows, rot / 2], contiguous fp32 on ", dev));
            cfg.table_rows = extent(c->size(0), "cos");
            cfg.rot = extent(2 * c->size(1), "cos");
            if (cfg.rot) { cos = static_cast<const float*>(c->data_ptr()); sin = static_cast<const float*>(s->data_ptr()); }
        }
        if (const at::Tensor* p = optional_tensor(a[8], "positions")) {
            const int64_t n = p->dim();
            if (p->scalar_type() != at::kInt || p->device() != dev || !(n == 1 || (n == 2 && p->size(0) == B)) || p->size(n - 1) != L ||
                (L > 1 && p->stride(n - 1) != 1))
                refuse("positions", *p, c10::str("[", L, "] or [", B, ", ", L, "] int32 on ", dev, " with contiguous rows"));
            cfg.pos_b = n == 2 ? p->stride(0) : 0;
            pos = static_cast<const int32_t*>(p->data_ptr());
        }
        const int truth = PyObject_IsTrue(a[9]);
        if (truth < 0) { PyErr_Clear(); refuse("interleaved", "a truth value is wanted"); }
        cfg.interleaved = truth;
    }
};
// a new [B, L, h, d] like t, or the caller's own
at::Tensor result(const at::Tensor* t, PyObject* own, const char* name) {
    if (own != Py_None) return tensor(own, name);
    if (!t) return at::Tensor();
    const int64_t L = t->size(1), h = t->size(2), d = t->size(3);
    return fresh(t->sizes(), {L * h * d, h * d, d, 1}, t->scalar_type(), t->device());
}
const at::Tensor* maybe(const at::Tensor& t) { return t.defined() ? &t : nullptr; }
PyObject* give_or_none(const at::Tensor& t, PyObject* own) { return t.defined() ? give(t, own) : Py_NewRef(Py_None); }

// qk_norm_rope(<QkArgs>, out Q | None, out K | None) -> (Q', K')
PyObject* qk_norm_rope(PyObject* const* a) {
    const QkArgs q(a);
    const c10::cuda::CUDAGuard guard(q.dev);
    const at::Tensor Qo = result(q.Q, a[10], "out[0]"), Ko = result(q.K, a[11], "out[1]");
    const OptionalHeads vq(q.Q, q.Q, "Q"), vk(q.K, q.K, "K"), vqo(maybe(Qo), q.Q, "out[0]"), vko(maybe(Ko), q.K, "out[1]");
    check(ppml_b200_qk_norm_rope(&q.cfg, vq.ptr(), vk.ptr(), q.qw, q.kw, q.cos, q.sin, q.pos, vqo.ptr(), vko.ptr(), stream_of(q.dev)), "qk_norm_rope");
    PyObject* two = PyTuple_New(2);
    if (!two) return nullptr;
    PyTuple_SET_ITEM(two, 0, give_or_none(Qo, a[10])); PyTuple_SET_ITEM(two, 1, give_or_none(Ko, a[11]));
    return two;
}

// qk_norm_rope_backward(<QkArgs>, dQo | None, dKo | None, dQ | None, dK | None) -> (dQ, dK, dq_weight, dk_weight)
PyObject* qk_norm_rope_backward(PyObject* const* a) {
    const QkArgs q(a);
    const c10::cuda::CUDAGuard guard(q.dev);
    const at::Tensor dQ = result(q.Q, a[12], "dQ"), dK = result(q.K, a[13], "dK");
    const OptionalHeads vq(q.Q, q.Q, "Q"), vk(q.K, q.K, "K"), vqo(optional_tensor(a[10], "dQo"), q.Q, "dQo"), vko(optional_tensor(a[11], "dKo"), q.K, "dKo"),
        vdq(maybe(dQ), q.Q, "dQ"), vdk(maybe(dK), q.K, "dK");
    at::Tensor dqw, dkw, ws;
    if (q.qw) dqw = fresh({q.cfg.d}, {1}, at::kFloat, q.dev);
    if (q.kw) dkw = fresh({q.cfg.d}, {1}, at::kFloat, q.dev);
    const int64_t need = q.qw || q.kw ? ppml_b200_qk_norm_rope_backward_workspace(&q.cfg) : 0;
    if (need) ws = fresh({need}, {1}, at::kByte, q.dev);
    auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    check(ppml_b200_qk_norm_rope_backward(&q.cfg, vq.ptr(), vk.ptr(), q.qw, q.kw, q.cos, q.sin, q.pos, vqo.ptr(), vko.ptr(), vdq.ptr(), vdk.ptr(),
                                          static_cast<float*>(ptr(dqw)), static_cast<float*>(ptr(dkw)), ptr(ws), need, stream_of(q.dev)),
          "qk_norm_rope_backward");
    PyObject* four = PyTuple_New(4);
    if (!four) return nullptr;
    PyTuple_SET_ITEM(four, 0, give_or_none(dQ, a[12])); PyTuple_SET_ITEM(four, 1, give_or_none(dK, a[13]));
    PyTuple_SET_ITEM(four, 2, give_or_none(dqw, Py_None)); PyTuple_SET_ITEM(four, 3, give_or_none(dkw, Py_None));
    return four;
}

// torch's own class, which programs catch to go on with less; RuntimeError, its base, where it cannot be had
void set_out_of_memory(const char* what) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (!type) PyErr_Clear();
    PyErr_SetString(type ? type : PyExc_RuntimeError, what);
    Py_XDECREF(type);
    Py_XDECREF(torch);
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    try {
        if (n != N) refuse("arguments", std::to_string(N) + " are wanted");
        return F(args);
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        set_out_of_memory(e.what_without_backtrace());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N> PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<quantize_tokens_i8, 3>("quantize_tokens_i8"), method<mul_mat_i8, 10>("mul_mat_i8"), method<linear_i8, 9>("linear_i8"),
                         method<qk_norm_rope, 12>("qk_norm_rope"), method<qk_norm_rope_backward, 14>("qk_norm_rope_backward"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ppml_b200_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ppml_b200_torch(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", PPML_TORCH_VERSION) != 0) { Py_DECREF(m); return nullptr; }
    return m;
}
