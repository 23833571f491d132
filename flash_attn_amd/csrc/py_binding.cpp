// Native front end of the Python binding: flash_attn_amd._native.
//
// flash_forward / flash_forward_splitkv of binding.py hand their arguments to the functions forward and splitkv below, which fill
// flash_params, allocate the results and call the C ABI (the launch path of the reference's main(), src/main.cu:109-192), and so do
// flash_rotary, flash_append_paged and flash_forward_paged of paged.py.
//
// What bounds a small call is this code: filling the struct field by field through ctypes, five data_ptr() calls, two
// torch.empty() and torch.cuda.current_stream() took 13-15 us of host time per flash_forward and 18-19 us per
// flash_forward_splitkv, where the kernel of a small problem (B1 H2 N128 d64) runs for 4.6 us.
//
// Anything out of the ordinary -- an argument of another type, shapes or dtypes that do not fit, a workspace that is too
// small, a program that wants to see its allocations -- returns NotImplemented with nothing allocated or launched; binding.py then takes its own path, which raises the
// errors (and serves the debug outputs).  Of the calls of paged.py it also leaves those on another stream or device than the current one
// and those that need a derivative; the others took 15 us (rotary) to 29 us (paged forward in splits) each through ctypes.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <ATen/Context.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <cmath>
#include <initializer_list>

#include "flash_attn_mi355.h"
#include "split_counters.h"

namespace {

typedef int (*launch_fn)(const flash_params*, void*);
typedef int (*resolve_fn)(const flash_params*);
launch_fn g_forward = nullptr, g_splitkv = nullptr;
resolve_fn g_resolve = nullptr;
PyObject* g_error = nullptr;  // binding.FlashError(code, where)

PyObject* not_implemented() { Py_RETURN_NOTIMPLEMENTED; }

// an ordinary tensor (no subclass with behaviour of its own), or nullptr
const at::Tensor* tensor_of(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool fp16_on_gpu(const at::Tensor& t) { return t.scalar_type() == at::kHalf && t.is_cuda() && t.dim() == 4 && t.is_contiguous(); }

enum Parsed { kOk, kPython, kRaised };

// an exact int that fits the C int; anything else is left to binding.py
bool small_int(PyObject* o, int* out)
{
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    const long v = PyLong_AsLongAndOverflow(o, &over);
    if (over != 0 || v < INT32_MIN || v > INT32_MAX) return false;
    *out = (int)v;
    return true;
}

bool real(PyObject* o, float* out)
{
    if (PyFloat_CheckExact(o)) {
        *out = (float)PyFloat_AS_DOUBLE(o);
        return true;
    }
    if (!PyLong_CheckExact(o)) return false;
    const double v = PyLong_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    *out = (float)v;
    return true;
}

bool optional_tensor(PyObject* o, const at::Tensor** t)
{
    *t = nullptr;
    return o == Py_None || (*t = tensor_of(o)) != nullptr;
}

// What the table of split_counters.h asks for.  A region is 16 KiB of the stream's own pool, kept until the process ends, at
// most 1 MiB per device.  (All of this runs with the interpreter lock held.)
struct TorchRuntime {
    int current_device() const
    {
        int d = -1;
        return hipGetDevice(&d) == hipSuccess ? d : -1;
    }
    bool capturing(void* stream) const
    {
        hipStreamCaptureStatus c;
        return hipStreamIsCapturing(static_cast<hipStream_t>(stream), &c) != hipSuccess || c != hipStreamCaptureStatusNone;
    }
    uint32_t* allocate(size_t words, void* stream) const
    {
        try {
            return static_cast<uint32_t*>(
                c10::hip::HIPCachingAllocator::raw_alloc_with_stream(words * sizeof(uint32_t), static_cast<hipStream_t>(stream)));
        } catch (const c10::Error&) {
            return nullptr;
        }
    }
    void release(uint32_t* p) const { c10::hip::HIPCachingAllocator::raw_delete(p); }
    bool clear(uint32_t* p, size_t words, void* stream) const
    {
        return hipMemsetAsync(p, 0, words * sizeof(uint32_t), static_cast<hipStream_t>(stream)) == hipSuccess;
    }
};
uint32_t* counters_of(at::Device device, void* stream, bool pooled)
{
    static auto* table = new fa::CounterTable<TorchRuntime>;  // (never freed: outlives the runtime's own end)
    TorchRuntime rt;
    return table->of(rt, device.index(), stream, pooled);
}

struct Call {
    flash_params p{};
    const at::Tensor* q = nullptr;
    const at::Tensor *out = nullptr, *lse = nullptr;
    void* stream = nullptr;
    bool pooled_stream = false;  // one of torch's own
};

// Results and workspace come from the allocator directly: through the dispatcher each takes 0.2 us more (B1 H2 N128 d64, whose
// call is bound by its host time: 5.07 against 5.47 us).  Who would notice gets torch.empty() instead: dispatch modes (fake tensors, tracers, memory accounting), and the
// deterministic mode that fills new memory.
bool allocates_plainly()
{
    return !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
           !(at::globalContext().deterministicAlgorithms() && at::globalContext().deterministicFillUninitializedMemory());
}

// Arguments that both entry points share: q, k, v and the array (softmax_scale, causal, window, alibi_slopes, dropout_p,
// seed, offset, stream, out, lse).
Parsed parse(PyObject* const* qkv, PyObject* const* a, Call* c)
{
    if (!allocates_plainly()) return kPython;
    const at::Tensor *q = tensor_of(qkv[0]), *k = tensor_of(qkv[1]), *v = tensor_of(qkv[2]), *slopes;
    if (!q || !k || !v || !fp16_on_gpu(*q) || !fp16_on_gpu(*k) || !fp16_on_gpu(*v)) return kPython;
    const auto qs = q->sizes(), ks = k->sizes();
    if (ks[0] != qs[0] || ks[1] < 1 || qs[1] % ks[1] != 0 || ks[3] != qs[3] || v->sizes() != ks) return kPython;
    for (int i = 0; i < 4; ++i)
        if (qs[i] > INT32_MAX || ks[i] > INT32_MAX) return kPython;
    flash_params& p = c->p;
    p.B = (int)qs[0], p.H = (int)qs[1], p.Nq = (int)qs[2], p.d = (int)qs[3], p.H_kv = (int)ks[1], p.Nk = (int)ks[2];
    if (a[0] == Py_None) p.softmax_scale = (float)std::pow((double)p.d, -0.5);
    else if (!real(a[0], &p.softmax_scale)) return kPython;
    const int causal = PyObject_IsTrue(a[1]);
    if (causal < 0) return kRaised;
    p.is_causal = causal;
    if (!PyTuple_CheckExact(a[2]) || PyTuple_GET_SIZE(a[2]) != 2 || !small_int(PyTuple_GET_ITEM(a[2], 0), &p.window_left) ||
        !small_int(PyTuple_GET_ITEM(a[2], 1), &p.window_right))
        return kPython;
    if (!optional_tensor(a[3], &slopes)) return kPython;
    if (!real(a[4], &p.dropout_p) || !PyLong_CheckExact(a[5]) || !PyLong_CheckExact(a[6])) return kPython;
    p.seed = PyLong_AsUnsignedLongLongMask(a[5]);
    p.offset = PyLong_AsUnsignedLongLongMask(a[6]);
    if (!optional_tensor(a[8], &c->out) || !optional_tensor(a[9], &c->lse)) return kPython;
    if (a[7] == Py_None) {
        const auto current = c10::hip::getCurrentHIPStream();
        c->stream = current.stream();
        c->pooled_stream = (current.id() & 1) != 0;  // (the id of a stream from outside is its handle, an aligned pointer)
    } else {
        PyObject* h = PyObject_GetAttrString(a[7], "cuda_stream");
        if (!h) return kRaised;
        c->stream = PyLong_AsVoidPtr(h);
        Py_DECREF(h);
        if (PyErr_Occurred()) return kRaised;
        if (PyObject* id = PyObject_GetAttrString(a[7], "stream_id")) {
            c->pooled_stream = PyLong_Check(id) && (PyLong_AsUnsignedLongLongMask(id) & 1) != 0;
            Py_DECREF(id);
        } else {
            PyErr_Clear();
        }
    }
    p.Q = q->data_ptr(), p.K = k->data_ptr(), p.V = v->data_ptr();
    p.alibi_slopes = slopes ? static_cast<const float*>(slopes->data_ptr()) : nullptr;
    c->q = q;
    return kOk;
}

at::Tensor empty_like_q(const Call& c, at::IntArrayRef size, at::ScalarType type)
{
    return at::detail::empty_cuda(size, type, c.q->device(), std::nullopt);
}

PyObject* raise(int code, const char* where)
{
    PyObject* e = PyObject_CallFunction(g_error, "is", code, where);
    if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    return nullptr;
}

// allocates what the caller has not brought, launches, returns (O, LSE)
PyObject* launch(launch_fn fn, const char* where, Call* c)
{
    flash_params& p = c->p;
    const at::Tensor o = c->out ? *c->out : empty_like_q(*c, c->q->sizes(), at::kHalf);
    const at::Tensor l = c->lse ? *c->lse : empty_like_q(*c, {p.B, p.H, p.Nq}, at::kFloat);
    p.O = o.data_ptr();
    p.LSE = static_cast<float*>(l.data_ptr());
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(&p, c->stream);
    Py_END_ALLOW_THREADS
    if (rc != FLASH_OK) return raise(rc, where);
    PyObject* res = PyTuple_New(2);
    if (!res) return nullptr;
    PyTuple_SET_ITEM(res, 0, THPVariable_Wrap(o));
    PyTuple_SET_ITEM(res, 1, THPVariable_Wrap(l));
    return res;
}

// A C++ exception (an allocation that does not fit) becomes the Python exception that torch.empty would have raised.
template <typename F>
PyObject* guarded(F f)
{
    HANDLE_TH_ERRORS
    return f();
    END_HANDLE_TH_ERRORS
}

// forward(q, k, v, softmax_scale, causal, window, alibi_slopes, dropout_p, seed, offset, stream, out, lse)
PyObject* forward(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject* {
        if (n != 13 || !g_forward) return not_implemented();
        Call c;
        const Parsed r = parse(args, args + 3, &c);
        if (r != kOk) return r == kPython ? not_implemented() : nullptr;
        c.p.num_splits = 1;
        return launch(g_forward, "flash_forward", &c);
    });
}

// splitkv(q, k, v, num_splits, workspace, softmax_scale, causal, window, alibi_slopes, dropout_p, seed, offset, stream,
// out, lse)
PyObject* splitkv(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject* {
        if (n != 15 || !g_splitkv) return not_implemented();
        Call c;
        int splits;
        if (!small_int(args[3], &splits)) return not_implemented();
        const Parsed r = parse(args, args + 5, &c);
        if (r != kOk) return r == kPython ? not_implemented() : nullptr;
        flash_params& p = c.p;
        p.num_splits = splits;
        const int S = g_resolve(&p);
        if (S < 0) return raise(S, "flash_splitkv_resolve_splits");
        p.num_splits = S;  // (the launch need not work it out again)
        const int64_t rows = S > 1 ? (int64_t)p.B * p.H * S * p.Nq : 0;
        at::Tensor own;  // workspace of this call, both parts in one allocation
        if (args[4] != Py_None) {
            if (!PyTuple_CheckExact(args[4]) || PyTuple_GET_SIZE(args[4]) != 2) return not_implemented();
            const at::Tensor *wo = tensor_of(PyTuple_GET_ITEM(args[4], 0)), *wl = tensor_of(PyTuple_GET_ITEM(args[4], 1));
            for (const at::Tensor* t : {wo, wl})
                if (!t || t->scalar_type() != at::kFloat || !t->is_cuda() || !t->is_contiguous()) return not_implemented();
            if (wo->numel() < rows * p.d || wl->numel() < rows) return not_implemented();
            p.O_partial = static_cast<float*>(wo->data_ptr());
            p.LSE_partial = static_cast<float*>(wl->data_ptr());
        } else if (rows) {
            const int64_t o_floats = (rows * p.d + 63) & ~(int64_t)63;  // the second part on a 256-byte boundary
            own = empty_like_q(c, {o_floats + rows}, at::kFloat);
            p.O_partial = static_cast<float*>(own.data_ptr());
            p.LSE_partial = p.O_partial + o_floats;
        }
        if (S > 1 && (c.stream == nullptr || c.pooled_stream)) {
            p.split_counters = counters_of(c.q->device(), c.stream, c.pooled_stream);
            p.split_counters_len = p.split_counters ? fa::kCountersPerStream : 0;
        }
        return launch(g_splitkv, "flash_forward_splitkv", &c);
    });
}

// ---- paged.py

typedef int (*rotary_fn)(const flash_rotary_params*, void*);
typedef int (*paged_fn)(const flash_paged_params*, void*);
typedef int (*paged_resolve_fn)(const flash_paged_params*);
rotary_fn g_rotary = nullptr;
paged_fn g_append = nullptr, g_paged = nullptr;
paged_resolve_fn g_paged_resolve = nullptr;

int dtype_of(const at::Tensor& t)
{
    switch (t.scalar_type()) {
        case at::kHalf: return FLASH_FP16;
        case at::kBFloat16: return FLASH_BF16;
        case at::kFloat: return FLASH_FP32;
        default: return -1;
    }
}
bool unit_stride(const at::Tensor& t) { return t.dim() > 0 && (t.size(-1) <= 1 || t.stride(-1) == 1); }
bool fits_int(const at::Tensor& t)
{
    for (const auto n : t.sizes())
        if (n > INT32_MAX) return false;
    return true;
}
// on the GPU that is current, whose current stream the call goes to
bool is_here(const at::Tensor& t) { return t.is_cuda() && t.device().index() == c10::hip::current_device(); }
at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef size, at::ScalarType type) { return at::detail::empty_cuda(size, type, like.device(), std::nullopt); }
// whether results would be detached from one of them without a word, of its gradient or of a forward-mode derivative (paged.py refuses it, or works
// out the gradient)
bool wants_derivative(std::initializer_list<const at::Tensor*> tensors)
{
    const bool grad = at::GradMode::is_enabled();
    for (const at::Tensor* t : tensors)
        if (t && ((grad && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
    return false;
}
// Tells autograd that the caller's tensors have been written, so that a backward pass that has saved one of them notices.
void written(std::initializer_list<const at::Tensor*> tensors)
{
    for (const at::Tensor* t : tensors)
        if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
bool positions_ok(const at::Tensor& t) { return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && unit_stride(t) && is_here(t); }
bool frequencies_ok(const at::Tensor& f, int64_t d)
{
    return f.scalar_type() == at::kFloat && f.dim() == 1 && f.is_contiguous() && f.numel() >= 1 && f.numel() <= d / 2 && is_here(f);
}

// rotary(x, positions, inv_freq, interleaved, factor, inverse, out)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject* {
        if (n != 7 || !g_rotary || !allocates_plainly()) return not_implemented();
        const at::Tensor *x = tensor_of(args[0]), *pos = tensor_of(args[1]), *f = tensor_of(args[2]), *out;
        if (!x || !pos || !f || !optional_tensor(args[6], &out)) return not_implemented();
        flash_rotary_params p{};
        if (!real(args[4], &p.factor) || !PyBool_Check(args[3]) || !PyBool_Check(args[5])) return not_implemented();
        p.interleaved = args[3] == Py_True, p.inverse = args[5] == Py_True;
        const int64_t dims = x->dim();
        if ((dims != 3 && dims != 4) || (p.dtype = dtype_of(*x)) < 0 || !unit_stride(*x) || !fits_int(*x) || !is_here(*x)) return not_implemented();
        if (wants_derivative({x, f, out})) return not_implemented();
        const bool tokens = dims == 3;
        p.B = tokens ? 1 : (int)x->size(0), p.H = (int)x->size(1), p.N = (int)x->size(tokens ? 0 : 2), p.d = (int)x->size(-1);
        if (!positions_ok(*pos) || !frequencies_ok(*f, p.d)) return not_implemented();
        if (!(pos->dim() == 1 && pos->size(0) == p.N) && !(pos->dim() == 2 && !tokens && pos->size(0) == p.B && pos->size(1) == p.N)) return not_implemented();
        at::Tensor y;
        if (out) {
            if (out->sizes() != x->sizes() || out->scalar_type() != x->scalar_type() || !unit_stride(*out) || !is_here(*out)) return not_implemented();
            y = *out;
        } else {  // (in x's order of dimensions, where x is dense; paged.py sees to the others)
            if (!x->is_non_overlapping_and_dense()) return not_implemented();
            y = at::detail::empty_strided_cuda(x->sizes(), x->strides(), x->scalar_type(), x->device());
        }
        auto strides = [&](const at::Tensor& t, int64_t& b, int64_t& h, int64_t& r) { b = tokens ? 0 : t.stride(0), h = t.stride(1), r = t.stride(tokens ? 0 : 2); };
        strides(*x, p.x_batch, p.x_head, p.x_row);
        strides(y, p.y_batch, p.y_head, p.y_row);
        p.X = x->data_ptr(), p.Y = y.data_ptr(), p.rot = 2 * (int)f->numel();
        p.positions = pos->data_ptr(), p.positions_64 = pos->scalar_type() == at::kLong, p.positions_batch = pos->dim() == 2 ? pos->stride(0) : 0;
        p.inv_freq = static_cast<const float*>(f->data_ptr());
        void* const stream = c10::hip::getCurrentHIPStream().stream();
        const int rc = g_rotary(&p, stream);
        if (rc != FLASH_OK) return raise(rc, "flash_rotary");
        written({out});
        return THPVariable_Wrap(y);
    });
}

// Caches and index tensors: args = (k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q)
bool parse_cache(PyObject* const* args, flash_paged_params& p)
{
    const at::Tensor* t[5];
    for (int i = 0; i < 5; ++i)
        if (!(t[i] = tensor_of(args[i])) || !is_here(*t[i]) || !fits_int(*t[i])) return false;
    const at::Tensor &k = *t[0], &v = *t[1], &table = *t[2], &lens = *t[3], &cu = *t[4];
    p.dtype = dtype_of(k);
    if ((p.dtype != FLASH_FP16 && p.dtype != FLASH_BF16) || v.scalar_type() != k.scalar_type() || k.dim() != 4 || v.sizes() != k.sizes()) return false;
    if (k.stride(3) != 1 || v.stride(3) != 1) return false;
    for (int i = 2; i < 5; ++i)
        if (t[i]->scalar_type() != at::kInt || t[i]->dim() != (i == 2 ? 2 : 1) || !unit_stride(*t[i])) return false;
    const int64_t B = lens.size(0);
    if (table.size(0) != B || cu.size(0) != B + 1) return false;
    p.K_cache = k.data_ptr(), p.V_cache = v.data_ptr();
    p.block_table = static_cast<const int32_t*>(table.data_ptr()), p.seqlens_k = static_cast<const int32_t*>(lens.data_ptr());
    p.cu_seqlens_q = static_cast<const int32_t*>(cu.data_ptr());
    p.num_pages = (int)k.size(0), p.H_kv = (int)k.size(1), p.page_size = (int)k.size(2), p.d = (int)k.size(3), p.B = (int)B, p.max_pages = (int)table.size(1);
    p.kc_page = k.stride(0), p.kc_head = k.stride(1), p.kc_row = k.stride(2);
    p.vc_page = v.stride(0), p.vc_head = v.stride(1), p.vc_row = v.stride(2);
    p.block_table_stride = table.stride(0);
    p.window_left = p.window_right = -1;
    return true;
}
// rows [T, heads, d] of the cache's type
bool rows_ok(const at::Tensor& t, int64_t T, int64_t heads, const flash_paged_params& p)
{
    return is_here(t) && t.dim() == 3 && t.size(0) == T && t.size(1) == heads && t.size(2) == p.d && dtype_of(t) == p.dtype && t.stride(2) == 1;
}

// append(k, v, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, q, inv_freq, interleaved, factor, positions, out)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject* {
        if (n != 13 || !g_append || !allocates_plainly()) return not_implemented();
        const at::Tensor *k = tensor_of(args[0]), *v = tensor_of(args[1]), *q, *f, *pos, *out;
        flash_paged_params p{};
        if (!k || !v || !parse_cache(args + 2, p) || !optional_tensor(args[7], &q) || !optional_tensor(args[8], &f) || !optional_tensor(args[11], &pos) ||
            !optional_tensor(args[12], &out) || !PyBool_Check(args[9]) || !real(args[10], &p.factor))
            return not_implemented();
        if (wants_derivative({k, v, tensor_of(args[2]), tensor_of(args[3]), q, f, out})) return not_implemented();
        if ((q && !f) || (out && !q) || (pos && !f) || k->dim() != 3 || (q && q->dim() != 3) || k->size(0) > INT32_MAX) return not_implemented();
        const int64_t T = k->size(0), H = q ? q->size(1) : p.H_kv;
        if (H > INT32_MAX || !rows_ok(*k, T, p.H_kv, p) || !rows_ok(*v, T, p.H_kv, p) || (q && !rows_ok(*q, T, H, p)) || (out && !rows_ok(*out, T, H, p))) return not_implemented();
        if (f && !frequencies_ok(*f, p.d)) return not_implemented();
        if (pos && (!positions_ok(*pos) || pos->dim() != 1 || pos->size(0) != T)) return not_implemented();
        p.total_q = (int)T, p.H = (int)H;
        p.K = k->data_ptr(), p.V = v->data_ptr(), p.k_token = k->stride(0), p.k_head = k->stride(1), p.v_token = v->stride(0), p.v_head = v->stride(1);
        if (f) p.inv_freq = static_cast<const float*>(f->data_ptr()), p.rot = 2 * (int)f->numel(), p.interleaved = args[9] == Py_True;
        if (pos) p.positions = pos->data_ptr(), p.positions_64 = pos->scalar_type() == at::kLong;
        at::Tensor y;
        if (q) {
            y = out ? *out : empty_on(*q, q->sizes(), q->scalar_type());
            p.Q = q->data_ptr(), p.O = y.data_ptr(), p.q_token = q->stride(0), p.q_head = q->stride(1), p.o_token = y.stride(0), p.o_head = y.stride(1);
        }
        const int rc = g_append(&p, c10::hip::getCurrentHIPStream().stream());
        if (rc != FLASH_OK) return raise(rc, "flash_append_paged");
        written({tensor_of(args[2]), tensor_of(args[3]), out});
        if (q) return THPVariable_Wrap(y);
        Py_RETURN_NONE;
    });
}

// paged(q, k_cache, v_cache, block_table, seqlens_k, cu_seqlens_q, max_seqlen_q, max_seqlen_k, softmax_scale, causal, window, num_splits, workspace, out, lse)
PyObject* paged(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject* {
        if (n != 15 || !g_paged || !allocates_plainly()) return not_implemented();
        const at::Tensor *q = tensor_of(args[0]), *out, *lse;
        flash_paged_params p{};
        if (!q || !parse_cache(args + 1, p) || !optional_tensor(args[13], &out) || !optional_tensor(args[14], &lse)) return not_implemented();
        if (wants_derivative({q, tensor_of(args[1]), tensor_of(args[2]), out, lse})) return not_implemented();
        if (!small_int(args[6], &p.max_seqlen_q) || !small_int(args[7], &p.max_seqlen_k) || !PyBool_Check(args[9]) || !small_int(args[11], &p.num_splits)) return not_implemented();
        if (args[8] == Py_None) p.softmax_scale = (float)std::pow((double)p.d, -0.5);
        else if (!real(args[8], &p.softmax_scale)) return not_implemented();
        if (!PyTuple_CheckExact(args[10]) || PyTuple_GET_SIZE(args[10]) != 2 || !small_int(PyTuple_GET_ITEM(args[10], 0), &p.window_left) ||
            !small_int(PyTuple_GET_ITEM(args[10], 1), &p.window_right))
            return not_implemented();
        p.is_causal = args[9] == Py_True;
        if (q->dim() != 3 || !fits_int(*q)) return not_implemented();
        const int64_t T = q->size(0), H = q->size(1), d = p.d;
        if (p.H_kv < 1 || H < 1 || H % p.H_kv != 0 || !rows_ok(*q, T, H, p) || (out && !rows_ok(*out, T, H, p))) return not_implemented();
        if (lse && (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != T || lse->size(1) != H || !lse->is_contiguous() || !is_here(*lse)))
            return not_implemented();
        p.total_q = (int)T, p.H = (int)H;
        const int S = g_paged_resolve(&p);
        if (S < 0) return raise(S, "flash_forward_paged_resolve_splits");
        const int64_t rows = S > 1 ? T * H * S : 0;
        at::Tensor own;  // workspace of this call, both parts in one allocation
        const at::Tensor *wo = nullptr, *wl = nullptr;
        if (args[12] != Py_None) {
            if (!PyTuple_CheckExact(args[12]) || PyTuple_GET_SIZE(args[12]) != 2) return not_implemented();
            wo = tensor_of(PyTuple_GET_ITEM(args[12], 0)), wl = tensor_of(PyTuple_GET_ITEM(args[12], 1));
            for (const at::Tensor* t : {wo, wl})
                if (!t || t->scalar_type() != at::kFloat || !is_here(*t) || !t->is_contiguous()) return not_implemented();
            if (wo->numel() < rows * d || wl->numel() < rows) return not_implemented();
            p.O_partial = static_cast<float*>(wo->data_ptr()), p.LSE_partial = static_cast<float*>(wl->data_ptr());
        } else if (rows) {
            const int64_t o_floats = (rows * d + 63) & ~(int64_t)63;
            own = empty_on(*q, {o_floats + rows}, at::kFloat);
            p.O_partial = static_cast<float*>(own.data_ptr()), p.LSE_partial = p.O_partial + o_floats;
        }
        const at::Tensor o = out ? *out : empty_on(*q, q->sizes(), q->scalar_type());
        const at::Tensor l = lse ? *lse : empty_on(*q, {T, H}, at::kFloat);
        p.Q = q->data_ptr(), p.O = o.data_ptr(), p.LSE = static_cast<float*>(l.data_ptr());
        p.q_token = q->stride(0), p.q_head = q->stride(1), p.o_token = o.stride(0), p.o_head = o.stride(1);
        const int rc = g_paged(&p, c10::hip::getCurrentHIPStream().stream());
        if (rc != FLASH_OK) return raise(rc, "flash_forward_paged");
        written({out, lse, wo, wl});
        PyObject* res = PyTuple_New(2);
        if (!res) return nullptr;
        PyTuple_SET_ITEM(res, 0, THPVariable_Wrap(o));
        PyTuple_SET_ITEM(res, 1, THPVariable_Wrap(l));
        return res;
    });
}

// bind_paged(addresses of flash_rotary, flash_append_paged, flash_forward_paged, flash_forward_paged_resolve_splits), behind bind()
PyObject* bind_paged(PyObject*, PyObject* args)
{
    unsigned long long r, a, f, s;
    if (!PyArg_ParseTuple(args, "KKKK", &r, &a, &f, &s)) return nullptr;
    g_rotary = reinterpret_cast<rotary_fn>(r);
    g_append = reinterpret_cast<paged_fn>(a);
    g_paged = reinterpret_cast<paged_fn>(f);
    g_paged_resolve = reinterpret_cast<paged_resolve_fn>(s);
    Py_RETURN_NONE;
}

// bind(addresses of flash_forward, flash_forward_splitkv, flash_splitkv_resolve_splits, FlashError): the library that
// binding.lib() has loaded
PyObject* bind(PyObject*, PyObject* args)
{
    unsigned long long f, s, r;
    PyObject* e;
    if (!PyArg_ParseTuple(args, "KKKO", &f, &s, &r, &e)) return nullptr;
    g_forward = reinterpret_cast<launch_fn>(f);
    g_splitkv = reinterpret_cast<launch_fn>(s);
    g_resolve = reinterpret_cast<resolve_fn>(r);
    Py_INCREF(e);
    Py_XSETREF(g_error, e);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
    {"splitkv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(splitkv)), METH_FASTCALL, nullptr},
    {"bind_paged", bind_paged, METH_VARARGS, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void)
{
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
