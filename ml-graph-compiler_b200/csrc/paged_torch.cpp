// Python binding of the paged-cache operators for torch tensors (module _mgc_paged): the checks that
// need types, shapes and devices, the output tensors, the current stream, then the C entry points.
// The same checks in Python took 10 us a call, four times what a small call takes on the GPU.
//
// The entry points and exception types are handed over once by mgc_cuda.paged (bind), so this file
// links against torch only.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <initializer_list>
#include <sstream>
#include <string>

#include "mgc_cuda.h"

namespace {

int (*append_fn)(const mgc_cuda_kv_append_args *, void *) = nullptr;
int (*attend_fn)(const mgc_cuda_paged_attention_args *, void *) = nullptr;
int64_t (*workspace_fn)(const mgc_cuda_paged_attention_args *) = nullptr;
int (*append_heads_fn)(const mgc_cuda_kv_append_heads_args *, void *) = nullptr;
int (*read_fn)(const mgc_cuda_kv_read_args *, void *) = nullptr;
int (*attend_quantized_fn)(const mgc_cuda_paged_attention_quantized_args *, void *) = nullptr;
int64_t (*quantized_workspace_fn)(const mgc_cuda_paged_attention_quantized_args *) = nullptr;
const char *(*error_fn)() = nullptr;
PyObject *graph_error = nullptr, *codegen_error = nullptr;

// What a call cannot take: becomes GraphError.
struct Refused {
    std::string text;
};

std::string shape_of(const at::Tensor &t) {
    std::ostringstream s;
    s << t.sizes();
    return s.str();
}

[[noreturn]] void refuse(const char *what, const std::string &why) { throw Refused{std::string(what) + ": " + why}; }

const at::Tensor *tensor(PyObject *o, const char *what, const char *name, bool optional = false) {
    if (o == Py_None && optional) return nullptr;
    if (!THPVariable_Check(o)) refuse(what, std::string(name) + " is not a torch tensor");
    return &THPVariable_Unpack(o);
}

int64_t dtype_of(at::ScalarType t) {
    switch (t) {
    case at::kFloat: return MGC_F32;
    case at::kHalf: return MGC_F16;
    case at::kBFloat16: return MGC_BF16;
    default: return -1;
    }
}

// There is no backward pass: an operand that a gradient is recorded for is refused.
void no_gradient(const char *what, std::initializer_list<const at::Tensor *> operands) {
    if (!at::GradMode::is_enabled()) return;
    for (const at::Tensor *t : operands)
        if (t && t->defined() && t->requires_grad()) refuse(what, "an operand requires a gradient, which the call cannot record (torch.no_grad(), or detach it)");
}

// The kernels wrote t: autograd's saved copies of it are out of date.
void written(const at::Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A truth value.
bool truth(PyObject *o, const char *what, const char *name) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        refuse(what, std::string(name) + " has no truth value");
    }
    return v != 0;
}

// A whole number.
int64_t whole(PyObject *o, const char *what, const char *name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(what, std::string(name) + " is not a whole number");
    }
    return v;
}

// A cache operand: a tensor of pages, or the tuple (codes, scales, bits).
struct Pages {
    const at::Tensor *values = nullptr, *scales = nullptr;
    int64_t bits = 0;
};
Pages pages_of(PyObject *o, const char *what, const char *name) {
    Pages g;
    if (!PyTuple_Check(o)) {
        g.values = tensor(o, what, name);
        return g;
    }
    if (PyTuple_GET_SIZE(o) != 3) refuse(what, std::string(name) + ": quantised pages are (codes, scales, bits)");
    g.values = tensor(PyTuple_GET_ITEM(o, 0), what, name);
    g.scales = tensor(PyTuple_GET_ITEM(o, 1), what, name);
    g.bits = whole(PyTuple_GET_ITEM(o, 2), what, "the bits of quantised pages");
    if (g.bits != 4 && g.bits != 8) refuse(what, std::string(name) + ": pages of " + std::to_string(g.bits) + " bits (4 or 8)");
    return g;
}

// The pages of quantised caches and their scales.
void fill_quantized(mgc_cuda_paged &p, mgc_cuda_quantized &z, const char *what, const Pages &k, const Pages &v) {
    const at::Tensor &c = *k.values, &s = *k.scales;
    if (c.scalar_type() != at::kByte || v.values->scalar_type() != at::kByte || s.scalar_type() != at::kHalf ||
        v.scales->scalar_type() != at::kHalf)
        refuse(what, "quantised pages are uint8 codes and float16 scales");
    if (c.dim() != 4 || v.values->sizes() != c.sizes() || v.values->strides() != c.strides() || v.bits != k.bits || (c.size(3) * 8) % k.bits)
        refuse(what, "codes " + shape_of(c) + " and " + shape_of(*v.values) +
                         ": two [pages, page_size, kv_heads, head_dim * bits / 8] of the same bits and strides");
    if (s.dim() != 5 || v.scales->sizes() != s.sizes() || v.scales->strides() != s.strides() || s.size(0) != c.size(0) ||
        s.size(1) != c.size(1) || s.size(2) != c.size(2) || s.size(4) != 2)
        refuse(what, "scales " + shape_of(s) + " and " + shape_of(*v.scales) +
                         ": two [pages, page_size, kv_heads, groups, 2] of the same strides");
    if ((c.stride(3) != 1 && c.size(3) > 1) || s.stride(4) != 1 || (s.stride(3) != 2 && s.size(3) > 1) || s.stride(0) % 2 ||
        s.stride(1) % 2 || s.stride(2) % 2)
        refuse(what, "the codes or the scales of a row are not contiguous");
    if (s.device() != c.device() || v.scales->device() != c.device()) refuse(what, "the tensors are on several devices");
    p.head_dim = c.size(3) * 8 / k.bits;
    if (s.size(3) < 1 || p.head_dim % s.size(3))
        refuse(what, std::to_string(s.size(3)) + " groups of " + std::to_string(p.head_dim) + " channels");
    z.bits = k.bits;
    z.group = p.head_dim / s.size(3);
    z.k_scales = s.data_ptr();
    z.v_scales = v.scales->data_ptr();
    z.page_stride = s.stride(0) / 2;
    z.token_stride = s.stride(1) / 2;
    z.head_stride = s.stride(2) / 2;
}

// The first six operands of every call and the status word. `dtype`: the call's type where pages are
// quantised, which plain ones have themselves.
void fill(mgc_cuda_paged &p, mgc_cuda_quantized &z, const char *what, PyObject *const *a, PyObject *status, int64_t tokens, int64_t dtype) {
    const Pages kp = pages_of(a[0], what, "k_cache"), vp = pages_of(a[1], what, "v_cache");
    if (!kp.scales != !vp.scales) refuse(what, "one cache is quantised and the other is not");
    const at::Tensor &k = *kp.values, &v = *vp.values, &table = *tensor(a[2], what, "block_table"),
                     &lens = *tensor(a[3], what, "kv_lens"), &starts = *tensor(a[4], what, "q_starts");
    const auto device = k.device();
    if (!k.is_cuda()) refuse(what, "the cache is on " + device.str());
    if (kp.scales) {
        p.dtype = dtype;
        fill_quantized(p, z, what, kp, vp);
    } else {
        p.dtype = dtype_of(k.scalar_type());
        if (p.dtype < 0 || v.scalar_type() != k.scalar_type())
            refuse(what, "pages of both caches are float32, float16 or bfloat16");
        if (k.dim() != 4 || v.sizes() != k.sizes() || v.strides() != k.strides())
            refuse(what, "caches " + shape_of(k) + " and " + shape_of(v) + ": two [pages, page_size, kv_heads, head_dim] of the same strides");
        if (k.stride(3) != 1 && k.size(3) > 1) refuse(what, "the cache's channels are not contiguous");
        p.head_dim = k.size(3);
    }
    if (table.scalar_type() != at::kInt || lens.scalar_type() != at::kInt || starts.scalar_type() != at::kInt)
        refuse(what, "block_table, kv_lens and q_starts are int32");
    const int64_t batch = lens.dim() == 1 ? lens.size(0) : -1;
    if (batch < 0 || table.dim() != 2 || starts.dim() != 1 || table.size(0) != batch || starts.size(0) != batch + 1 ||
        (table.stride(1) != 1 && table.size(1) > 1) || (lens.stride(0) != 1 && batch > 1) || (starts.stride(0) != 1 && batch > 0))
        refuse(what, "block_table " + shape_of(table) + ", kv_lens " + shape_of(lens) + ", q_starts " + shape_of(starts) +
                         ": [batch, n], [batch], [batch + 1], contiguous rows");
    if (v.device() != device || table.device() != device || lens.device() != device || starts.device() != device)
        refuse(what, "the tensors are on several devices");
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.pages = k.size(0);
    p.page_size = k.size(1);
    p.kv_heads = k.size(2);
    p.page_stride = k.stride(0);
    p.token_stride = k.stride(1);
    p.head_stride = k.stride(2);
    p.block_table = static_cast<const int32_t *>(table.data_ptr());
    p.table_stride = table.stride(0);
    p.table_pages = table.size(1);
    p.kv_lens = static_cast<const int32_t *>(lens.data_ptr());
    p.q_starts = static_cast<const int32_t *>(starts.data_ptr());
    p.batch = batch;
    p.tokens = tokens;
    p.status_dev = nullptr;
    if (const at::Tensor *s = tensor(status, what, "status", true)) {
        if (s->scalar_type() != at::kInt || s->numel() != 1 || s->device() != device)
            refuse(what, "status is one int32 on the cache's device");
        p.status_dev = static_cast<int32_t *>(s->data_ptr());
    }
}

// A packed [tokens, heads, head_dim] operand.
void rows(const char *what, const char *name, const at::Tensor &t, int64_t tokens, int64_t heads, int64_t dim,
          at::Device device, int64_t &token_stride, int64_t &head_stride) {
    if (t.dim() != 3 || t.size(0) != tokens || (heads > 0 && t.size(1) != heads) || t.size(2) != dim)
        refuse(what, std::string(name) + " " + shape_of(t) + ": [" + std::to_string(tokens) + ", " +
                         (heads > 0 ? std::to_string(heads) : std::string("heads")) + ", " + std::to_string(dim) + "]");
    if (t.device() != device) refuse(what, std::string(name) + " is on " + t.device().str() + ", the cache on " + device.str());
    if (t.stride(2) != 1 && dim > 1) refuse(what, std::string(name) + "'s channels are not contiguous");
    token_stride = t.stride(0);
    head_stride = t.stride(1);
}

void check(int status, const char *what) {
    if (status != 0) throw std::runtime_error(std::string(what) + " failed with status " + std::to_string(status) + ": " + error_fn());
}

// Runs `call`, turning C++ exceptions into Python ones.
template <typename F> PyObject *guarded(F call) {
    try {
        return call();
    } catch (const Refused &e) {
        PyErr_SetString(graph_error, e.text.c_str());
    } catch (const std::exception &e) {
        PyErr_SetString(codegen_error, e.what());
    } catch (...) {
        PyErr_SetString(codegen_error, "unknown C++ exception");
    }
    return nullptr;
}

// (k, v, k_cache, v_cache, block_table, kv_lens, q_starts, q, cos, sin, interleaved, q_out, status, q_norm,
// k_norm, eps)
PyObject *kv_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const char *what = "kv_append";
        if (n != 16 || !append_fn) refuse(what, "not bound, or 16 arguments expected");
        const at::Tensor &k = *tensor(a[0], what, "k"), &v = *tensor(a[1], what, "v");
        if (k.dim() != 3) refuse(what, "k " + shape_of(k) + ": [tokens, kv_heads, head_dim]");
        const int64_t tokens = k.size(0);
        mgc_cuda_kv_append_heads_args y{};
        mgc_cuda_kv_append_args &x = y.append;
        x.src_dtype = dtype_of(k.scalar_type());
        fill(x.paged, y.quantized, what, a + 2, a[12], tokens, x.src_dtype);
        const Pages k_pages = pages_of(a[2], what, "k_cache"), v_pages = pages_of(a[3], what, "v_cache");
        const at::Tensor &cache = *k_pages.values;
        // queries come back in the cache's type, from quantised pages' call in their own
        const auto out_type = k_pages.scales ? k.scalar_type() : cache.scalar_type();
        const auto device = cache.device();
        const int64_t dim = x.paged.head_dim;
        const at::Tensor *q = tensor(a[7], what, "q", true), *cos = tensor(a[8], what, "cos", true),
                         *sin = tensor(a[9], what, "sin", true);
        if (x.src_dtype < 0 || v.scalar_type() != k.scalar_type() || (q && q->scalar_type() != k.scalar_type()))
            refuse(what, "q, k and v are of one type, float32, float16 or bfloat16");
        rows(what, "k", k, tokens, x.paged.kv_heads, dim, device, x.k_token_stride, x.k_head_stride);
        rows(what, "v", v, tokens, x.paged.kv_heads, dim, device, x.v_token_stride, x.v_head_stride);
        x.k = k.data_ptr();
        x.v = v.data_ptr();
        at::Tensor out;
        if (q) {
            rows(what, "q", *q, tokens, 0, dim, device, x.q_token_stride, x.q_head_stride);
            x.q_heads = q->size(1);
            x.q = q->data_ptr();
            if (const at::Tensor *given = tensor(a[11], what, "q_out", true)) out = *given;
            else out = at::empty({tokens, x.q_heads, dim}, cache.options().dtype(out_type).requires_grad(false));
            if (out.scalar_type() != out_type) refuse(what, k_pages.scales ? "q_out is of q's type" : "q_out is of the cache's type");
            rows(what, "q_out", out, tokens, x.q_heads, dim, device, x.qo_token_stride, x.qo_head_stride);
            x.q_out = out.data_ptr();
        }
        const bool interleaved = truth(a[10], what, "interleaved");
        if (!cos != !sin) refuse(what, "cos and sin come together");
        if (cos) {
            if (cos->dim() != 2 || sin->sizes() != cos->sizes() || cos->scalar_type() != at::kFloat ||
                sin->scalar_type() != at::kFloat || cos->strides() != sin->strides() || (cos->stride(1) != 1 && cos->size(1) > 1) ||
                cos->device() != device || sin->device() != device)
                refuse(what, "cos " + shape_of(*cos) + " and sin " + shape_of(*sin) +
                                 ": float32 [positions, rot / 2] on the cache's device, of the same strides");
            x.cos = static_cast<const float *>(cos->data_ptr());
            x.sin = static_cast<const float *>(sin->data_ptr());
            x.table_row = cos->stride(0);
            x.positions = cos->size(0);
            x.rot = 2 * cos->size(1);
            x.interleaved = interleaved;
        }
        const at::Tensor *q_norm = tensor(a[13], what, "q_norm", true), *k_norm = tensor(a[14], what, "k_norm", true);
        for (const at::Tensor *w : {q_norm, k_norm})
            if (w && (w->dim() != 1 || w->size(0) != dim || w->scalar_type() != at::kFloat || (w->stride(0) != 1 && dim > 1) || w->device() != device))
                refuse(what, "norm weights " + shape_of(*w) + ": float32 [" + std::to_string(dim) + "] on the cache's device");
        if (q_norm && !q) refuse(what, "q_norm without q");
        y.q_norm = q_norm ? static_cast<const float *>(q_norm->data_ptr()) : nullptr;
        y.k_norm = k_norm ? static_cast<const float *>(k_norm->data_ptr()) : nullptr;
        y.eps = PyFloat_AsDouble(a[15]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            refuse(what, "eps is a number");
        }
        no_gradient(what, {&k, &v, &cache, v_pages.values, k_pages.scales, v_pages.scales, q, cos, sin, q_norm, k_norm, &out});
        const c10::cuda::CUDAGuard guard(device);
        if (q && x.paged.batch == 0) out.copy_(*q);  // no sequence: the call itself does nothing
        void *stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        int status;
        Py_BEGIN_ALLOW_THREADS;
        status = k_pages.scales || q_norm || k_norm ? append_heads_fn(&y, stream) : append_fn(&x, stream);
        Py_END_ALLOW_THREADS;
        check(status, what);
        for (const at::Tensor *w : {k_pages.values, v_pages.values, k_pages.scales, v_pages.scales})
            if (w) written(*w);
        if (!q) Py_RETURN_NONE;
        if (a[11] != Py_None) written(out);
        return THPVariable_Wrap(std::move(out));
    });
}

// (q, k_cache, v_cache, block_table, kv_lens, q_starts, max_q, max_kv, scale, causal, window, out, status)
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const char *what = "paged_attention";
        if (n != 13 || !attend_fn) refuse(what, "not bound, or 13 arguments expected");
        const at::Tensor &q = *tensor(a[0], what, "q");
        if (q.dim() != 3) refuse(what, "q " + shape_of(q) + ": [tokens, heads, head_dim]");
        const int64_t tokens = q.size(0);
        mgc_cuda_paged_attention_quantized_args y{};
        mgc_cuda_paged_attention_args &x = y.attention;
        fill(x.paged, y.quantized, what, a + 1, a[12], tokens, dtype_of(q.scalar_type()));
        const Pages k_pages = pages_of(a[1], what, "k_cache"), v_pages = pages_of(a[2], what, "v_cache");
        const at::Tensor &cache = *k_pages.values;
        const bool codes = k_pages.scales;
        const auto device = cache.device();
        const int64_t dim = x.paged.head_dim;
        if (codes ? x.paged.dtype < 0 : q.scalar_type() != cache.scalar_type())
            refuse(what, codes ? "q is float32, float16 or bfloat16" : "q is not of the cache's type");
        rows(what, "q", q, tokens, 0, dim, device, x.q_token_stride, x.q_head_stride);
        x.q_heads = q.size(1);
        x.q = q.data_ptr();
        at::Tensor out;
        if (const at::Tensor *given = tensor(a[11], what, "out", true)) out = *given;
        else out = at::empty({tokens, x.q_heads, dim}, cache.options().dtype(q.scalar_type()).requires_grad(false));
        if (out.scalar_type() != q.scalar_type()) refuse(what, "out is of q's type");
        rows(what, "out", out, tokens, x.q_heads, dim, device, x.o_token_stride, x.o_head_stride);
        x.out = out.data_ptr();
        x.max_q = a[6] == Py_None ? tokens : whole(a[6], what, "max_q");
        x.max_kv = a[7] == Py_None ? x.paged.table_pages * x.paged.page_size : whole(a[7], what, "max_kv");
        x.scale = a[8] == Py_None ? 1.0 / std::sqrt((double)dim) : PyFloat_AsDouble(a[8]);
        if (PyErr_Occurred()) {
            PyErr_Clear();
            refuse(what, "scale is a number");
        }
        x.causal = truth(a[9], what, "causal");
        x.window = a[10] == Py_None ? 0 : whole(a[10], what, "window");
        no_gradient(what, {&q, &cache, v_pages.values, k_pages.scales, v_pages.scales, &out});
        const c10::cuda::CUDAGuard guard(device);
        if (x.paged.batch == 0) out.zero_();  // no sequence: the call itself does nothing
        void *stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        // partial results of keys that are shared out, from torch's stream-ordered allocator: the
        // block returns to this stream's pool after the call
        at::Tensor space;
        x.workspace_bytes = codes ? quantized_workspace_fn(&y) : workspace_fn(&x);
        if (x.workspace_bytes < 0) throw std::runtime_error(std::string(what) + ": " + error_fn());
        if (x.workspace_bytes > 0) {
            space = at::empty({x.workspace_bytes}, cache.options().dtype(at::kByte).requires_grad(false));
            x.workspace = space.data_ptr();
        }
        int status;
        Py_BEGIN_ALLOW_THREADS;
        status = codes ? attend_quantized_fn(&y, stream) : attend_fn(&x, stream);
        Py_END_ALLOW_THREADS;
        check(status, what);
        if (a[11] != Py_None) written(out);
        return THPVariable_Wrap(std::move(out));
    });
}

// (k_cache, v_cache, block_table, kv_lens, q_starts, rows, dtype, k_out, v_out, status)
PyObject *kv_read(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        const char *what = "kv_read";
        if (n != 10 || !read_fn) refuse(what, "not bound, or 10 arguments expected");
        const int64_t tokens = whole(a[5], what, "rows");
        if (tokens < 0) refuse(what, "a negative number of rows");
        if (!THPDtype_Check(a[6])) refuse(what, "dtype is not a torch type");
        const auto type = reinterpret_cast<THPDtype *>(a[6])->scalar_type;
        if (dtype_of(type) < 0) refuse(what, "dtype is float32, float16 or bfloat16");
        mgc_cuda_kv_read_args x{};
        fill(x.paged, x.quantized, what, a, a[9], tokens, dtype_of(type));
        const Pages k_pages = pages_of(a[0], what, "k_cache"), v_pages = pages_of(a[1], what, "v_cache");
        if (!k_pages.scales) refuse(what, "the cache is not quantised");
        const at::Tensor &cache = *k_pages.values;
        const auto device = cache.device();
        const c10::cuda::CUDAGuard guard(device);
        auto output = [&](PyObject *o, const char *name, void *&at, int64_t &token_stride, int64_t &head_stride) {
            at::Tensor out;
            if (const at::Tensor *given = tensor(o, what, name, true)) out = *given;
            else out = at::empty({tokens, x.paged.kv_heads, x.paged.head_dim}, cache.options().dtype(type).requires_grad(false));
            if (out.scalar_type() != type) refuse(what, std::string(name) + " is not of dtype");
            rows(what, name, out, tokens, x.paged.kv_heads, x.paged.head_dim, device, token_stride, head_stride);
            at = out.data_ptr();
            return out;
        };
        at::Tensor k = output(a[7], "k_out", x.k_out, x.k_token_stride, x.k_head_stride);
        at::Tensor v = output(a[8], "v_out", x.v_out, x.v_token_stride, x.v_head_stride);
        no_gradient(what, {&cache, v_pages.values, k_pages.scales, v_pages.scales, &k, &v});
        if (x.paged.batch == 0) {  // no sequence: the call itself does nothing
            k.zero_();
            v.zero_();
        }
        void *stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
        int status;
        Py_BEGIN_ALLOW_THREADS;
        status = read_fn(&x, stream);
        Py_END_ALLOW_THREADS;
        check(status, what);
        if (a[7] != Py_None) written(k);
        if (a[8] != Py_None) written(v);
        PyObject *pair = PyTuple_New(2);
        if (!pair) return nullptr;
        PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(k)));
        PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(v)));
        return pair;
    });
}

// (address of mgc_cuda_kv_append, _paged_attention, _paged_attention_workspace, _last_error, _kv_append_heads, _kv_read,
// _paged_attention_quantized, _paged_attention_quantized_workspace, GraphError, CodegenError)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 10) {
        PyErr_SetString(PyExc_TypeError, "bind: 10 arguments expected");
        return nullptr;
    }
    void *address[8];
    for (int i = 0; i < 8; ++i) {
        address[i] = PyLong_AsVoidPtr(a[i]);
        if (!address[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: NULL entry point");
            return nullptr;
        }
    }
    append_fn = reinterpret_cast<decltype(append_fn)>(address[0]);
    attend_fn = reinterpret_cast<decltype(attend_fn)>(address[1]);
    workspace_fn = reinterpret_cast<decltype(workspace_fn)>(address[2]);
    error_fn = reinterpret_cast<decltype(error_fn)>(address[3]);
    append_heads_fn = reinterpret_cast<decltype(append_heads_fn)>(address[4]);
    read_fn = reinterpret_cast<decltype(read_fn)>(address[5]);
    attend_quantized_fn = reinterpret_cast<decltype(attend_quantized_fn)>(address[6]);
    quantized_workspace_fn = reinterpret_cast<decltype(quantized_workspace_fn)>(address[7]);
    Py_INCREF(a[8]);
    Py_INCREF(a[9]);
    graph_error = a[8];
    codegen_error = a[9];
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(kv_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(paged_attention)), METH_FASTCALL, nullptr},
    {"kv_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(kv_read)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mgc_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mgc_paged(void) { return PyModule_Create(&module); }
