// The operators' Python calls on torch tensors, without an interpreter's overhead: checks, outputs from torch's allocator, the
// current stream, the C-ABI call (include/ygg_b200.h), and the gradient of token_logprobs as a node of torch's autograd.
//
// Each call takes the plain case (what a loop passes: tensors of the right types and layouts on one device) and returns None
// for any other; the Python side then checks, converts, and calls again. A call costs the host 5 to 8 us this way, most of
// it the launch; through ctypes and Python it was 15 to 17 us, more than most of the kernels take.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>

#include "ygg_b200.h"

namespace {

using at::Tensor;

PyObject *g_check;   // yggdrasil_b200._native.check: raises YggError for a code

// The library's codes as exceptions; a C++ exception that HANDLE_TH_ERRORS turns into the Python one already set.
void raise_for(int code, const char *what) {
    if (code == YGG_OK) return;
    PyGILState_STATE gil = PyGILState_Ensure();
    PyObject *r = PyObject_CallFunction(g_check, "is", code, what);
    Py_XDECREF(r);
    python_error e;
    e.persist();
    PyGILState_Release(gil);
    throw e;
}

int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return YGG_DTYPE_FLOAT;
        case at::kHalf: return YGG_DTYPE_HALF;
        case at::kBFloat16: return YGG_DTYPE_BFLOAT;
        default: return -1;
    }
}

void *stream_of(c10::DeviceIndex device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

Tensor empty(at::IntArrayRef size, at::ScalarType dtype, const at::Device &device) {
    return Tensor(at::detail::empty_cuda(size, dtype, device, std::nullopt));
}

const Tensor *cuda_tensor(PyObject *o) {
    if (!THPVariable_Check(o)) return nullptr;
    const Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() ? &t : nullptr;
}

// A contiguous row of n values of a type on a device (n < 0: any number).
bool is_row(const Tensor &t, at::ScalarType type, int64_t n, const at::Device &device) {
    return t.scalar_type() == type && t.dim() == 1 && (n < 0 || t.size(0) == n) && t.is_contiguous() &&
           t.device() == device;
}

// Whether a forward-mode derivative comes with it (the dual of a tangent), which no kernel here carries on.
bool has_tangent(const Tensor &t) {
    return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined();
}

// Whether a derivative is asked for through it, of either kind.
bool tracked(const Tensor &t) { return (t.requires_grad() && at::GradMode::is_enabled()) || has_tangent(t); }

PyObject *wrap(const Tensor &t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }

// ------------------------------------------------------------------------------------------------ token_logprobs

struct Logprobs { Tensor logprob, entropy, lse, ids, tops; };

Logprobs logprobs(const Tensor &x, const Tensor &tokens, int64_t top, float *stats) {
    const int64_t rows = x.size(0), vocab = x.size(1);
    const at::Device device = x.device();
    Logprobs o;
    o.logprob = empty({rows}, at::kFloat, device);
    o.entropy = empty({rows}, at::kFloat, device);
    o.lse = empty({rows}, at::kFloat, device);
    if (top) {
        o.ids = empty({rows, top}, at::kInt, device);
        o.tops = empty({rows, top}, at::kFloat, device);
    }
    raise_for(ygg_token_logprobs(device.index(), dtype_of(x.scalar_type()), rows, vocab, x.data_ptr(), x.stride(0),
                                 tokens.data_ptr(), (int)tokens.element_size(), (int)top, (float *)o.logprob.data_ptr(),
                                 (float *)o.entropy.data_ptr(), (float *)o.lse.data_ptr(),
                                 top ? (int32_t *)o.ids.data_ptr() : nullptr, top ? (float *)o.tops.data_ptr() : nullptr,
                                 stats, stream_of(device.index())),
              "ygg_token_logprobs");
    return o;
}

// A gradient that arrives, as the kernel reads it: it may be expanded (a sum's) or of another type.
Tensor arrived(const Tensor &g) {
    return !g.defined() || (g.scalar_type() == at::kFloat && g.is_contiguous()) ? g : g.to(at::kFloat).contiguous();
}

struct LogprobsNode : torch::autograd::Function<LogprobsNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x,
                                                  const Tensor &tokens, int64_t top) {
        const Tensor stats = empty({x.size(0), 4}, at::kFloat, x.device());
        const Logprobs o = logprobs(x, tokens, top, (float *)stats.data_ptr());
        ctx->save_for_backward({x, tokens, stats, o.ids});
        ctx->saved_data["top"] = top;
        ctx->set_materialize_grads(false);
        if (!top) return {o.logprob, o.entropy, o.lse};
        ctx->mark_non_differentiable({o.ids});
        return {o.logprob, o.entropy, o.lse, o.tops, o.ids};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                   torch::autograd::variable_list arriving) {
        TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled() && std::none_of(arriving.begin(), arriving.end(), has_tangent),
                                    "token_logprobs has no second derivative");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &tokens = saved[1], &stats = saved[2], &ids = saved[3];
        const int64_t top = ctx->saved_data["top"].toInt(), rows = x.size(0), vocab = x.size(1), step = x.stride(0);
        const c10::cuda::CUDAGuard on(x.device());
        // rows that lie to the 16-byte boundary as the logits' do move 16 bytes at a time
        const int64_t per = 16 / x.element_size(), wide = step % per == 0 ? (vocab + per - 1) / per * per : vocab;
        Tensor grad = empty({rows, wide}, x.scalar_type(), x.device());
        if (wide != vocab) grad = grad.narrow(1, 0, vocab);
        Tensor g[4];
        const void *at[4];
        for (size_t i = 0; i < 4; i++) {
            if (i < arriving.size()) g[i] = arrived(arriving[i]);
            at[i] = g[i].defined() ? g[i].data_ptr() : nullptr;
        }
        raise_for(ygg_token_logprobs_backward(
                      x.get_device(), dtype_of(x.scalar_type()), rows, vocab, x.data_ptr(), step, tokens.data_ptr(),
                      (int)tokens.element_size(), (int)top, top ? (const int32_t *)ids.data_ptr() : nullptr,
                      (const float *)stats.data_ptr(), (const float *)at[0], (const float *)at[1], (const float *)at[2],
                      (const float *)at[3], grad.data_ptr(), wide, stream_of(x.get_device())),
                  "ygg_token_logprobs_backward");
        return {grad, Tensor(), Tensor()};
    }
};

// (logits, tokens, top) -> (logprob, entropy, lse, top_ids, top_logprobs), or None
PyObject *py_token_logprobs(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3 || !PyLong_Check(args[2])) Py_RETURN_NONE;
    const Tensor *x = cuda_tensor(args[0]), *t = cuda_tensor(args[1]);
    const int64_t top = PyLong_AsLongLong(args[2]);
    if (top == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (!x || !t || dtype_of(x->scalar_type()) < 0 || x->dim() != 2 || x->size(1) < 1 ||
        (x->size(1) > 1 && x->stride(1) != 1) || top < 0 || top > std::min<int64_t>(x->size(1), YGG_TOP_MAX) ||
        (t->scalar_type() != at::kInt && t->scalar_type() != at::kLong) || t->dim() != 1 || t->size(0) != x->size(0) ||
        !t->is_contiguous() || t->device() != x->device())
        Py_RETURN_NONE;
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(*x), "token_logprobs has no forward-mode derivative");
    const c10::cuda::CUDAGuard on(x->device());
    Logprobs o;
    if (x->requires_grad() && at::GradMode::is_enabled()) {
        const auto out = LogprobsNode::apply(*x, *t, top);
        o = {out[0], out[1], out[2], top ? out[4] : Tensor(), top ? out[3] : Tensor()};
    } else {
        o = logprobs(*x, *t, top, nullptr);
    }
    PyObject *r = PyTuple_New(5);
    if (!r) throw python_error();
    PyTuple_SET_ITEM(r, 0, wrap(o.logprob));
    PyTuple_SET_ITEM(r, 1, wrap(o.entropy));
    PyTuple_SET_ITEM(r, 2, wrap(o.lse));
    PyTuple_SET_ITEM(r, 3, wrap(o.ids));
    PyTuple_SET_ITEM(r, 4, wrap(o.tops));
    return r;
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ int8_linear

bool aligned_rows(const Tensor &t) {   // (rows, K) bytes, rows a multiple of 16 bytes apart
    return t.stride(1) == 1 && t.stride(0) % 16 == 0 && t.stride(0) >= t.size(1) && (uintptr_t)t.data_ptr() % 16 == 0;
}

struct Weights {
    const Tensor *w, *scale, *bias;   // bias: null for none
};

// The weights as the kernels read them: (weight, scale, bias or None).
std::optional<Weights> weights_of(PyObject *const *args, int64_t k, const at::Device &device) {
    Weights r{cuda_tensor(args[0]), cuda_tensor(args[1]), args[2] == Py_None ? nullptr : cuda_tensor(args[2])};
    if (!r.w || !r.scale || (args[2] != Py_None && !r.bias) || r.w->scalar_type() != at::kChar || r.w->dim() != 2 ||
        r.w->size(1) != k || r.w->size(0) < 1 || r.w->device() != device || !aligned_rows(*r.w))
        return std::nullopt;
    const int64_t n = r.w->size(0);
    if (!is_row(*r.scale, at::kFloat, n, device) || (r.bias && !is_row(*r.bias, at::kFloat, n, device)) ||
        tracked(*r.scale) || (r.bias && tracked(*r.bias)))
        return std::nullopt;
    return r;
}

// The type asked for, `other` where it is None; -1 for one that is not ours.
int type_asked(PyObject *o, at::ScalarType other, at::ScalarType &type) {
    if (o == Py_None) type = other;
    else if (THPDtype_Check(o)) type = ((THPDtype *)o)->scalar_type;
    else return -1;
    return dtype_of(type);
}

bool rows_ok(const Tensor &x) {
    return dtype_of(x.scalar_type()) >= 0 && x.dim() == 2 && x.size(1) >= 1 && x.size(1) <= YGG_LINEAR_MAX_K &&
           (x.size(1) == 1 || x.stride(1) == 1) && !tracked(x);
}

// (x, weight, scale, bias or None, out_dtype or None) -> y, or None
PyObject *py_int8_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *x = n == 5 ? cuda_tensor(args[0]) : nullptr;
    if (!x || !rows_ok(*x)) Py_RETURN_NONE;
    at::ScalarType type = at::kFloat;
    const int out_dtype = type_asked(args[4], x->scalar_type(), type);
    const int64_t rows = x->size(0), k = x->size(1);
    const at::Device device = x->device();
    const auto w = weights_of(args + 1, k, device);
    if (!w || out_dtype < 0) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard on(device);
    const int64_t channels = w->w->size(0);
    Tensor out = empty({rows, channels}, type, device);
    const int64_t bytes = (int64_t)ygg_linear_workspace(rows, k);
    const Tensor room = empty({bytes}, at::kByte, device);
    raise_for(ygg_linear(device.index(), dtype_of(x->scalar_type()), rows, k, channels, x->data_ptr(), x->stride(0),
                         (const int8_t *)w->w->data_ptr(), w->w->stride(0), (const float *)w->scale->data_ptr(),
                         w->bias ? (const float *)w->bias->data_ptr() : nullptr, out_dtype, out.data_ptr(), channels,
                         room.data_ptr(), (size_t)bytes, stream_of(device.index())),
              "ygg_linear");
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// (codes, row_scale, weight, scale, bias or None, out_dtype or None) -> y, or None
PyObject *py_int8_linear_rows(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *c = n == 6 ? cuda_tensor(args[0]) : nullptr, *s = n == 6 ? cuda_tensor(args[1]) : nullptr;
    if (!c || !s || c->scalar_type() != at::kChar || c->dim() != 2 || c->size(1) < 1 || c->size(1) > YGG_LINEAR_MAX_K ||
        !aligned_rows(*c) || !is_row(*s, at::kFloat, c->size(0), c->device()) || tracked(*s))
        Py_RETURN_NONE;
    at::ScalarType type = at::kFloat;
    const int out_dtype = type_asked(args[5], at::kFloat, type);
    const int64_t rows = c->size(0), k = c->size(1);
    const at::Device device = c->device();
    const auto w = weights_of(args + 2, k, device);
    if (!w || out_dtype < 0) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard on(device);
    const int64_t channels = w->w->size(0);
    Tensor out = empty({rows, channels}, type, device);
    raise_for(ygg_linear_quantized(device.index(), rows, k, channels, (const int8_t *)c->data_ptr(), c->stride(0),
                                   (const float *)s->data_ptr(), (const int8_t *)w->w->data_ptr(), w->w->stride(0),
                                   (const float *)w->scale->data_ptr(),
                                   w->bias ? (const float *)w->bias->data_ptr() : nullptr, out_dtype, out.data_ptr(),
                                   channels, stream_of(device.index())),
              "ygg_linear_quantized");
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// (x,) -> (codes, scale), or None
PyObject *py_quantize_rows(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const Tensor *x = n == 1 ? cuda_tensor(args[0]) : nullptr;
    if (!x || !rows_ok(*x)) Py_RETURN_NONE;
    const int64_t rows = x->size(0), k = x->size(1), padded = (k + 15) / 16 * 16;
    const at::Device device = x->device();
    const c10::cuda::CUDAGuard on(device);
    Tensor codes = empty({rows, padded}, at::kChar, device);
    const Tensor scale = empty({rows}, at::kFloat, device);
    raise_for(ygg_quantize_rows(device.index(), dtype_of(x->scalar_type()), rows, k, x->data_ptr(), x->stride(0),
                                (int8_t *)codes.data_ptr(), padded, (float *)scale.data_ptr(), stream_of(device.index())),
              "ygg_quantize_rows");
    if (padded != k) codes = codes.narrow(1, 0, k);
    PyObject *r = PyTuple_New(2);
    if (!r) throw python_error();
    PyTuple_SET_ITEM(r, 0, wrap(codes));
    PyTuple_SET_ITEM(r, 1, wrap(scale));
    return r;
    END_HANDLE_TH_ERRORS
}

// (tensor,) -> whether a derivative is asked for through it
PyObject *py_tracked(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n == 1 && THPVariable_Check(args[0]) && tracked(THPVariable_Unpack(args[0]))) Py_RETURN_TRUE;
    Py_RETURN_FALSE;
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ StateCache

struct Cache {
    ygg_cache_t c;
    Tensor pages, table, length, refs;   // kept alive
};
constexpr const char *kCache = "yggdrasil_b200.cache";

void refuse_derivatives(const Tensor &t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!tracked(t), "a cache carries no gradient: use detach() or torch.no_grad()");
}

Cache *cache_of(PyObject *o) {
    Cache *c = (Cache *)PyCapsule_GetPointer(o, kCache);
    if (!c) throw python_error();
    return c;
}

// (pages, table, length, refs, address of the status words, address of the barrier's word) -> a cache, or None
PyObject *py_cache(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) Py_RETURN_NONE;
    const Tensor *t[4];
    for (int i = 0; i < 4; i++)
        if (!(t[i] = cuda_tensor(args[i])) || !t[i]->is_contiguous() || t[i]->numel() == 0 ||
            t[i]->device() != t[0]->device() || (i && t[i]->scalar_type() != at::kInt))
            Py_RETURN_NONE;
    const Tensor &pages = *t[0], &table = *t[1];
    if (pages.dim() < 2 || table.dim() != 2 || t[2]->dim() != 1 || t[2]->size(0) != table.size(0) || t[3]->dim() != 1 ||
        t[3]->size(0) != pages.size(0))
        Py_RETURN_NONE;
    refuse_derivatives(pages);
    void *status = PyLong_AsVoidPtr(args[4]), *sync = PyLong_AsVoidPtr(args[5]);
    if (PyErr_Occurred()) throw python_error();
    const int64_t count = pages.size(0);
    Cache *c = new Cache{{pages.data_ptr(), count, pages.numel() / count * pages.element_size(),
                          (int32_t *)table.data_ptr(), table.size(0), (int32_t)table.size(1), (int32_t *)t[2]->data_ptr(),
                          (int32_t *)t[3]->data_ptr(), (int32_t *)status, (uint64_t *)sync},
                         pages, table, *t[2], *t[3]};
    PyObject *r = PyCapsule_New(c, kCache, [](PyObject *o) { delete (Cache *)PyCapsule_GetPointer(o, kCache); });
    if (!r) {
        delete c;
        throw python_error();
    }
    return r;
    END_HANDLE_TH_ERRORS
}

// Indices as the kernels read them.
const Tensor *ids_of(PyObject *o, const Cache &c) {
    const Tensor *t = cuda_tensor(o);
    return t && is_row(*t, at::kInt, -1, c.pages.device()) ? t : nullptr;
}

// (cache, parents, children or None, depth or None) -> True, or None
PyObject *py_cache_fork(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) Py_RETURN_NONE;
    const Cache &c = *cache_of(args[0]);
    const Tensor *list[3];
    for (int i = 0; i < 3; i++) {
        list[i] = args[i + 1] == Py_None ? nullptr : ids_of(args[i + 1], c);
        if (!list[i] && (i == 0 || args[i + 1] != Py_None)) Py_RETURN_NONE;
        if (list[i] && list[i]->size(0) != list[0]->size(0)) Py_RETURN_NONE;
    }
    const at::Device device = c.pages.device();
    const c10::cuda::CUDAGuard on(device);
    const int64_t count = list[0]->size(0), bytes = (int64_t)ygg_cache_workspace(&c.c, count);
    const Tensor room = empty({bytes}, at::kByte, device);
    const auto at = [&](int i) { return list[i] ? (const int32_t *)list[i]->data_ptr() : nullptr; };
    raise_for(ygg_cache_fork(device.index(), &c.c, count, at(0), at(1), at(2), room.data_ptr(), (size_t)bytes,
                             stream_of(device.index())),
              "ygg_cache_fork");
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (cache, streams) -> True, or None
PyObject *py_cache_free(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2) Py_RETURN_NONE;
    const Cache &c = *cache_of(args[0]);
    const Tensor *s = ids_of(args[1], c);
    if (!s) Py_RETURN_NONE;
    const at::Device device = c.pages.device();
    raise_for(ygg_cache_free(device.index(), &c.c, s->size(0), (const int32_t *)s->data_ptr(), stream_of(device.index())),
              "ygg_cache_free");
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (cache,) -> the number of live pages, a tensor ()
PyObject *py_cache_compact(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 1) Py_RETURN_NONE;
    const Cache &c = *cache_of(args[0]);
    const at::Device device = c.pages.device();
    const c10::cuda::CUDAGuard on(device);
    const int64_t bytes = (int64_t)ygg_cache_workspace(&c.c, 0);
    const Tensor live = empty({}, at::kInt, device), room = empty({bytes}, at::kByte, device);
    raise_for(ygg_cache_compact(device.index(), &c.c, (int32_t *)live.data_ptr(), room.data_ptr(), (size_t)bytes,
                                stream_of(device.index())),
              "ygg_cache_compact");
    return wrap(live);
    END_HANDLE_TH_ERRORS
}

// (cache, streams) -> their live states, or None
PyObject *py_cache_read(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2) Py_RETURN_NONE;
    const Cache &c = *cache_of(args[0]);
    const Tensor *s = ids_of(args[1], c);
    if (!s) Py_RETURN_NONE;
    const at::Device device = c.pages.device();
    const c10::cuda::CUDAGuard on(device);
    std::vector<int64_t> size(c.pages.sizes().begin(), c.pages.sizes().end());
    size[0] = s->size(0);
    const Tensor batch = empty(size, c.pages.scalar_type(), device);
    raise_for(ygg_cache_read(device.index(), &c.c, size[0], (const int32_t *)s->data_ptr(), batch.data_ptr(),
                             stream_of(device.index())),
              "ygg_cache_read");
    return wrap(batch);
    END_HANDLE_TH_ERRORS
}

// (cache, streams, batch) -> True, or None
PyObject *py_cache_write(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) Py_RETURN_NONE;
    const Cache &c = *cache_of(args[0]);
    const Tensor *s = ids_of(args[1], c), *b = cuda_tensor(args[2]);
    if (!s || !b || !b->is_contiguous() || b->scalar_type() != c.pages.scalar_type() || b->device() != c.pages.device() ||
        b->dim() != c.pages.dim() || b->size(0) != s->size(0) || b->sizes().slice(1) != c.pages.sizes().slice(1))
        Py_RETURN_NONE;
    refuse_derivatives(*b);
    const at::Device device = c.pages.device();
    raise_for(ygg_cache_write(device.index(), &c.c, s->size(0), (const int32_t *)s->data_ptr(), b->data_ptr(),
                              stream_of(device.index())),
              "ygg_cache_write");
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// (cache, source pages, target pages) -> True, or None
PyObject *py_cache_copy(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) Py_RETURN_NONE;
    const Cache &c = *cache_of(args[0]);
    const Tensor *a = ids_of(args[1], c), *b = ids_of(args[2], c);
    if (!a || !b || a->size(0) != b->size(0)) Py_RETURN_NONE;
    const at::Device device = c.pages.device();
    raise_for(ygg_cache_copy(device.index(), &c.c, a->size(0), (const int32_t *)a->data_ptr(),
                             (const int32_t *)b->data_ptr(), stream_of(device.index())),
              "ygg_cache_copy");
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

#define CALL(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {CALL(token_logprobs), CALL(int8_linear), CALL(int8_linear_rows), CALL(quantize_rows),
                           CALL(tracked),        CALL(cache),       CALL(cache_fork),       CALL(cache_free),
                           CALL(cache_compact),  CALL(cache_read),  CALL(cache_write),      CALL(cache_copy),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() {
    PyObject *native = PyImport_ImportModule("yggdrasil_b200._native");
    if (!native) return nullptr;
    g_check = PyObject_GetAttrString(native, "check");
    Py_DECREF(native);
    return g_check ? PyModule_Create(&g_module) : nullptr;
}
