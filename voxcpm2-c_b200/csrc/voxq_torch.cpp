// voxq_torch.cpp -- the batched operators' calls on torch tensors, for voxq/batched.py.
//
// A small step's kernel takes 2 to 3 microseconds on the device and its C call as much on the host; checking a dozen
// tensors and packing a descriptor from Python took 8 more.  Here that is 1 to 2.  The functions take positional
// arguments from batched.py's wrappers (which document them), check them, make missing outputs on the current stream and
// call libvoxq's entry points, whose addresses `bind` gets from the ctypes binding.  A tensor that does not fit raises
// ValueError; a code from the library raises VoxqError.  A call's tensors are on one GPU, which is made the current one for
// it: kernels, plans and the library's status word belong to the current device, the stream to the tensors'.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "voxq.h"

namespace {

struct {
    VoxCPMError (*rope_append)(const voxq_rope*, void*);
    VoxCPMError (*paged_attention)(const voxq_paged_attn*, void*);
    size_t (*paged_workspace)(const voxq_paged_attn*);
    VoxCPMError (*lora)(const voxq_lora*, void*);
    VoxCPMError (*norm_residual)(const voxq_norm*, void*);
    PyObject* error;  // voxq.VoxqError
} g;

// Thrown after a Python error has been set.
struct Raised {};

[[noreturn]] void refuse(const char* what) {
    PyErr_SetString(PyExc_ValueError, what);
    throw Raised{};
}
void need(bool ok, const char* what) {
    if (!ok) refuse(what);
}
void done(VoxCPMError code, const char* what) {
    if (code == VOXCPM_SUCCESS) return;
    PyObject* e = PyObject_CallFunction(g.error, "is", (int)code, what);
    if (e) {
        PyErr_SetObject(g.error, e);
        Py_DECREF(e);
    }
    throw Raised{};
}

const at::Tensor* tensor(PyObject* o, const char* what) {
    if (o == Py_None) return nullptr;
    need(THPVariable_Check(o), what);
    return &THPVariable_Unpack(o);
}
const at::Tensor& present(PyObject* o, const char* what) {
    const at::Tensor* t = tensor(o, what);
    if (!t) refuse(what);
    return *t;
}
int code_of(at::ScalarType t) {
    return t == at::kFloat ? VOXQ_F32 : t == at::kHalf ? VOXQ_F16 : t == at::kBFloat16 ? VOXQ_BF16 : -1;
}
// rows of a last dimension that is contiguous, on the GPU
bool rows_ok(const at::Tensor& t, int64_t dims) {
    return t.dim() == dims && t.is_cuda() && (t.stride(-1) == 1 || t.size(-1) <= 1);
}
// tensors (or nullptr) on the device of `like`
void beside(const at::Tensor& like, std::initializer_list<const at::Tensor*> others) {
    for (const at::Tensor* t : others) need(!t || t->device() == like.device(), "all tensors of a call are needed on one GPU");
}
// a contiguous device vector of n values
const void* vec(const at::Tensor& t, int64_t n, at::ScalarType type, const char* what) {
    need(t.scalar_type() == type && t.numel() == n && t.is_cuda() && t.is_contiguous(), what);
    return t.const_data_ptr();
}
int64_t as_int(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}
int as_i32(PyObject* o, const char* what) {
    const int64_t v = as_int(o);
    need(v >= INT32_MIN && v <= INT32_MAX, what);
    return (int)v;
}
bool as_bool(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised{};
    return v != 0;
}
float as_float(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return (float)v;
}
int i32(int64_t v) {
    need(v <= INT32_MAX, "a dimension is past 2^31");
    return (int)v;
}
void* stream_of(const at::Tensor& like) { return (void*)c10::cuda::getCurrentCUDAStream(like.get_device()).stream(); }

// Makes a tensor's GPU the current one.  (It mostly is, and a guard asks three times.)
struct Here {
    c10::cuda::OptionalCUDAGuard guard;
    explicit Here(const at::Tensor& like) {
        if (like.get_device() != c10::cuda::current_device()) guard.set_device(like.device());
    }
};

// Memory of the current stream, contiguous, without the dispatcher's half microsecond a tensor.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

template <typename F>
PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F f) {
    if (have != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments are needed", want);
        return nullptr;
    }
    try {
        return f();
    } catch (const Raised&) {
    } catch (const std::exception& e) {  // out of memory and the like, from torch
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

void caches(const at::Tensor& k, const at::Tensor& v, int64_t head_dim) {
    need(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.strides() == k.strides() && k.is_cuda() &&
             v.is_cuda() && k.stride(3) == 1 && k.size(3) == head_dim,
         "caches: two [pages, page_size, kv_heads, head_dim] CUDA tensors of one type and layout, contiguous along head_dim, are needed");
}

// q k v freqs positions slots cache_k cache_v q_out interleaved
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&] {
        const at::Tensor &q = present(a[0], "q: a tensor is needed"), &k = present(a[1], "k: a tensor is needed"), &v = present(a[2], "v: a tensor is needed");
        const at::Tensor *freqs = tensor(a[3], "freqs: a tensor is needed"), &slots = present(a[5], "slots: a tensor is needed");
        const at::Tensor &ck = present(a[6], "cache_k: a tensor is needed"), &cv = present(a[7], "cache_v: a tensor is needed"), *given = tensor(a[8], "q_out: a tensor is needed");
        const at::Tensor* positions = freqs ? &present(a[4], "positions: a tensor is needed") : nullptr;
        need(rows_ok(q, 3) && rows_ok(k, 3) && rows_ok(v, 3), "q, k, v: 3-dimensional CUDA tensors with a contiguous last dimension are needed");
        beside(q, {&k, &v, freqs, positions, &slots, &ck, &cv, given});
        const int64_t T = q.size(0), H = q.size(1), D = q.size(2), KVH = k.size(1);
        need(v.sizes() == k.sizes() && k.size(0) == T && k.size(2) == D && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
             "q [T, heads, D] and k, v [T, kv_heads, D] of one type are needed");
        caches(ck, cv, D);
        need(ck.size(2) == KVH, "the caches' kv_heads differ from k's");
        const Here here(q);
        at::Tensor out = given ? *given : fresh(q.sizes(), ck.scalar_type(), q);
        need(rows_ok(out, 3) && out.sizes() == q.sizes() && out.scalar_type() == ck.scalar_type(), "q_out: q's shape and the caches' type, on the GPU");
        voxq_rope d{};
        if (freqs) {
            need(freqs->dim() == 3 && freqs->size(2) == 2, "freqs: [n_pos, rot / 2, 2]");
            d.freqs = (const float*)vec(*freqs, freqs->numel(), at::kFloat, "freqs: a contiguous fp32 CUDA tensor is needed");
            d.positions = (const int32_t*)vec(*positions, T, at::kInt, "positions: a contiguous CUDA vector of int32, one per token");
            d.n_pos = i32(freqs->size(0));
            d.rot_dim = i32(2 * freqs->size(1));
        }
        d.q = q.const_data_ptr();
        d.k = k.const_data_ptr();
        d.v = v.const_data_ptr();
        d.q_stride = q.stride(0);
        d.q_head_stride = q.stride(1);
        d.k_stride = k.stride(0);
        d.k_head_stride = k.stride(1);
        d.v_stride = v.stride(0);
        d.v_head_stride = v.stride(1);
        d.q_out = out.data_ptr();
        d.qo_stride = out.stride(0);
        d.qo_head_stride = out.stride(1);
        d.cache_k = ck.data_ptr();
        d.cache_v = cv.data_ptr();
        d.page_stride = ck.stride(0);
        d.row_stride = ck.stride(1);
        d.head_stride = ck.stride(2);
        d.slots = (const int64_t*)vec(slots, T, at::kLong, "slots: a contiguous CUDA vector of int64, one per token");
        d.tokens = i32(T);
        d.heads = i32(H);
        d.kv_heads = i32(KVH);
        d.head_dim = i32(D);
        d.interleaved = as_bool(a[9]);
        d.pages = i32(ck.size(0));
        d.page_size = i32(ck.size(1));
        d.in_dtype = code_of(q.scalar_type());
        d.cache_dtype = code_of(ck.scalar_type());
        done(g.rope_append(&d, stream_of(q)), "voxq_rope_append");
        return THPVariable_Wrap(std::move(out));
    });
}

// q cache_k cache_v block_table cu_q kv_len max_q max_kv causal scale out
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 11, [&]() -> PyObject* {
        const at::Tensor &q = present(a[0], "q: a tensor is needed"), &ck = present(a[1], "cache_k: a tensor is needed"), &cv = present(a[2], "cache_v: a tensor is needed");
        const at::Tensor &bt = present(a[3], "block_table: a tensor is needed"), &cu = present(a[4], "cu_q: a tensor is needed"), &kv = present(a[5], "kv_len: a tensor is needed");
        const at::Tensor* given = tensor(a[10], "out: a tensor is needed");
        need(rows_ok(q, 3), "q: a 3-dimensional CUDA tensor with a contiguous last dimension is needed");
        beside(q, {&ck, &cv, &bt, &cu, &kv, given});
        caches(ck, cv, q.size(2));
        const int64_t B = kv.numel();
        need(rows_ok(bt, 2) && bt.size(0) == B && bt.scalar_type() == at::kInt && ck.scalar_type() == q.scalar_type(),
             "caches of q's type and an int32 block_table [batch, width] on the GPU are needed");
        voxq_paged_attn d{};
        d.max_q = as_i32(a[6], "max_q is past 2^31");
        d.max_kv = as_i32(a[7], "max_kv is past 2^31");
        need(d.max_kv <= bt.size(1) * ck.size(1), "max_kv is more than the block table's pages hold");
        const Here here(q);
        at::Tensor out = given ? *given : fresh(q.sizes(), q.scalar_type(), q);
        need(rows_ok(out, 3) && out.sizes() == q.sizes(), "out: q's shape, contiguous along head_dim, on the GPU");
        d.q = q.const_data_ptr();
        d.q_stride = q.stride(0);
        d.q_head_stride = q.stride(1);
        d.out = out.data_ptr();
        d.o_stride = out.stride(0);
        d.o_head_stride = out.stride(1);
        d.k = ck.const_data_ptr();
        d.v = cv.const_data_ptr();
        d.page_stride = ck.stride(0);
        d.row_stride = ck.stride(1);
        d.head_stride = ck.stride(2);
        d.block_table = bt.const_data_ptr<int32_t>();
        d.table_stride = bt.stride(0);
        d.cu_q = (const int32_t*)vec(cu, B + 1, at::kInt, "cu_q: a contiguous CUDA vector of int32, one more than sequences");
        d.kv_len = (const int32_t*)vec(kv, B, at::kInt, "kv_len: a contiguous CUDA vector of int32, one per sequence");
        d.batch = i32(B);
        d.heads = i32(q.size(1));
        d.kv_heads = i32(ck.size(2));
        d.head_dim = i32(q.size(2));
        d.pages = i32(ck.size(0));
        d.page_size = i32(ck.size(1));
        d.total_q = i32(q.size(0));
        d.dtype = code_of(q.scalar_type());
        d.out_dtype = code_of(out.scalar_type());
        d.causal = as_bool(a[8]);
        d.scale = as_float(a[9]);
        const size_t bytes = g.paged_workspace(&d);
        at::Tensor ws;
        if (bytes) {
            ws = fresh({(int64_t)bytes}, at::kByte, q);
            d.workspace = ws.data_ptr();
            d.workspace_bytes = bytes;
        }
        done(g.paged_attention(&d, stream_of(q)), "voxq_paged_attention");
        return THPVariable_Wrap(std::move(out));
    });
}

// x a b cu adapter scale base out ranks
PyObject* lora(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded(n, 9, [&] {
        const at::Tensor &x = present(o[0], "x: a tensor is needed"), &a = present(o[1], "a: a tensor is needed"), &b = present(o[2], "b: a tensor is needed");
        const at::Tensor &cu = present(o[3], "cu: a tensor is needed"), &who = present(o[4], "adapter: a tensor is needed"), &scale = present(o[5], "scale: a tensor is needed");
        const at::Tensor *base = tensor(o[6], "base: a tensor is needed"), *given = tensor(o[7], "out: a tensor is needed"), *ranks = tensor(o[8], "ranks: a tensor is needed");
        need(rows_ok(x, 2), "x: a 2-dimensional CUDA tensor with a contiguous last dimension is needed");
        beside(x, {&a, &b, &cu, &who, &scale, base, given, ranks});
        need(a.dim() == 3 && b.dim() == 3 && a.size(2) == x.size(1) && b.size(0) == a.size(0) && b.size(2) == a.size(1) &&
                 a.scalar_type() == b.scalar_type() && a.is_contiguous() && b.is_contiguous() && a.is_cuda() && b.is_cuda(),
             "contiguous CUDA a [adapters, rank, K] and b [adapters, N, rank] of one type are needed");
        const int64_t M = x.size(0), N = b.size(1), B = who.numel(), nA = a.size(0);
        auto fits = [&](const at::Tensor& t) { return rows_ok(t, 2) && t.size(0) == M && t.size(1) == N && t.scalar_type() == x.scalar_type(); };
        need(!base || fits(*base), "base: [rows, N] of x's type, contiguous along N, on the GPU");
        const Here here(x);
        at::Tensor out = given ? *given : fresh({M, N}, x.scalar_type(), x);
        need(fits(out), "out: [rows, N] of x's type, contiguous along N, on the GPU");
        voxq_lora d{};
        d.x = x.const_data_ptr();
        d.ldx = x.stride(0);
        if (base) {
            d.base = base->const_data_ptr();
            d.ldb = base->stride(0);
        }
        d.out = out.data_ptr();
        d.ldo = out.stride(0);
        d.a = a.const_data_ptr();
        d.b = b.const_data_ptr();
        d.cu = (const int32_t*)vec(cu, B + 1, at::kInt, "cu: a contiguous CUDA vector of int32, one more than requests");
        d.adapter = (const int32_t*)vec(who, B, at::kInt, "adapter: a contiguous CUDA vector of int32, one per request");
        if (ranks) d.ranks = (const int32_t*)vec(*ranks, nA, at::kInt, "ranks: a contiguous CUDA vector of int32, one per adapter");
        d.scale = (const float*)vec(scale, nA, at::kFloat, "scale: a contiguous CUDA vector of fp32, one per adapter");
        d.rows = i32(M);
        d.batch = i32(B);
        d.K = i32(x.size(1));
        d.N = i32(N);
        d.rank = i32(a.size(1));
        d.adapters = i32(nA);
        d.dtype = code_of(x.scalar_type());
        d.w_dtype = code_of(a.scalar_type());
        done(g.lora(&d, stream_of(x)), "voxq_lora_forward");
        return THPVariable_Wrap(std::move(out));
    });
}

// y x w_pre w_post gate gate_index alpha eps h_out n_out
PyObject* norm_residual(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject* {
        const at::Tensor &y = present(a[0], "y: a tensor is needed"), &x = present(a[1], "x: a tensor is needed");
        const at::Tensor *w_pre = tensor(a[2], "w_pre: a tensor is needed"), *w_post = tensor(a[3], "w_post: a tensor is needed");
        const at::Tensor *gate = tensor(a[4], "gate: a tensor is needed"), *index = tensor(a[5], "gate_index: a tensor is needed");
        const at::Tensor *h_given = tensor(a[8], "h_out: a tensor is needed"), *n_given = tensor(a[9], "n_out: a tensor is needed");
        need(rows_ok(y, 2), "y: a 2-dimensional CUDA tensor with a contiguous last dimension is needed");
        beside(y, {&x, w_pre, w_post, gate, index, h_given, n_given});
        auto fits = [&](const at::Tensor& t) { return rows_ok(t, 2) && t.sizes() == y.sizes() && t.scalar_type() == y.scalar_type(); };
        need(fits(x), "y and x: [rows, D] of one type, contiguous along D, on the GPU");
        need(w_pre || !n_given, "n_out needs w_pre");
        const int64_t M = y.size(0), D = y.size(1);
        const Here here(y);
        voxq_norm d{};
        if (gate) {
            need(rows_ok(*gate, 2) && gate->size(1) == D && gate->scalar_type() == y.scalar_type(),
                 "gate: [gate_rows, D] of y's type, contiguous along D, on the GPU");
            d.gate = gate->const_data_ptr();
            d.ldg = gate->stride(0);
            d.gate_rows = i32(gate->size(0));
            if (index) d.gate_index = (const int32_t*)vec(*index, M, at::kInt, "gate_index: a contiguous CUDA vector of int32, one per row");
        }
        if (w_post) d.w_post = (const float*)vec(*w_post, D, at::kFloat, "w_post: a contiguous CUDA vector of D fp32");
        if (w_pre) d.w_pre = (const float*)vec(*w_pre, D, at::kFloat, "w_pre: a contiguous CUDA vector of D fp32");
        at::Tensor h = h_given ? *h_given : fresh(y.sizes(), y.scalar_type(), y), nn;
        need(fits(h), "h_out: [rows, D] of y's type, contiguous along D, on the GPU");
        if (w_pre) {
            nn = n_given ? *n_given : fresh(y.sizes(), y.scalar_type(), y);
            need(fits(nn), "n_out: [rows, D] of y's type, contiguous along D, on the GPU");
            d.n_out = nn.data_ptr();
            d.ldn = nn.stride(0);
        }
        d.y = y.const_data_ptr();
        d.x = x.const_data_ptr();
        d.ldy = y.stride(0);
        d.ldx = x.stride(0);
        d.h_out = h.data_ptr();
        d.ldh = h.stride(0);
        d.rows = i32(M);
        d.D = i32(D);
        d.dtype = code_of(y.scalar_type());
        d.alpha = as_float(a[6]);
        d.eps = as_float(a[7]);
        done(g.norm_residual(&d, stream_of(y)), "voxq_norm_residual");
        PyObject* hp = THPVariable_Wrap(std::move(h));
        PyObject* np = w_pre ? THPVariable_Wrap(std::move(nn)) : Py_NewRef(Py_None);
        PyObject* r = hp && np ? PyTuple_Pack(2, hp, np) : nullptr;
        Py_XDECREF(hp);
        Py_XDECREF(np);
        return r;
    });
}

// addresses of rope_append, paged_attention, its workspace function, lora_forward, norm_residual; VoxqError
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 6, [&]() -> PyObject* {
        g.rope_append = (decltype(g.rope_append))(uintptr_t)as_int(a[0]);
        g.paged_attention = (decltype(g.paged_attention))(uintptr_t)as_int(a[1]);
        g.paged_workspace = (decltype(g.paged_workspace))(uintptr_t)as_int(a[2]);
        g.lora = (decltype(g.lora))(uintptr_t)as_int(a[3]);
        g.norm_residual = (decltype(g.norm_residual))(uintptr_t)as_int(a[4]);
        Py_XSETREF(g.error, Py_NewRef(a[5]));
        Py_RETURN_NONE;
    });
}

#define VOXQ_FAST(f) (PyCFunction)(void (*)(void)) f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", VOXQ_FAST(bind)}, {"rope_append", VOXQ_FAST(rope_append)}, {"paged_attention", VOXQ_FAST(paged_attention)},
                         {"lora", VOXQ_FAST(lora)}, {"norm_residual", VOXQ_FAST(norm_residual)}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch(void) { return PyModule_Create(&module); }
