// The Python binding's call path in C++ (module mx230_amd._binding): the
// argument checks, output allocation and marshalling of the entry points a
// program calls once per layer or token, which in Python cost more than the
// short launches they enqueue. Each function takes the common case only
// (plain torch tensors on the GPU, torch's current stream) and returns
// NotImplemented for anything else, valid or not; mx230_amd/__init__.py then
// takes its own path, which accepts the rest or raises. A non-zero status of
// the C ABI comes back as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <optional>

#include "../../include/mxfa.h"

namespace {

// The C ABI, from the libmxfa the package has loaded (bind()).
struct {
    decltype(&mxfa_run_flash_lse) flash_lse;
    decltype(&mxfa_run_bwd_ws) bwd_ws;
    decltype(&mxfa_bwd_workspace_bytes) bwd_workspace_bytes;
    decltype(&mxfa_run_prefill) prefill;
    decltype(&mxfa_run_prefill_ws) prefill_ws;
    decltype(&mxfa_run_prefill_paged) prefill_paged;
    decltype(&mxfa_run_prefill_paged_ws) prefill_paged_ws;
    decltype(&mxfa_run_rotary) rotary;
    decltype(&mxfa_run_cache_append) cache_append;
    decltype(&mxfa_run_prefill_batch) prefill_batch;
    decltype(&mxfa_prefill_batch_workspace_bytes) prefill_batch_workspace_bytes;
    decltype(&mxfa_run_pages_free) pages_free;
    decltype(&mxfa_run_pages_fork) pages_fork;
    decltype(&mxfa_run_pages_compact) pages_compact;
    decltype(&mxfa_run_pages_copy) pages_copy;
    decltype(&mxfa_mx_block_bytes) mx_block_bytes;
    decltype(&mxfa_run_cache_append_mx) cache_append_mx;
    decltype(&mxfa_run_cache_read_mx) cache_read_mx;
    decltype(&mxfa_run_prefill_batch_mx) prefill_batch_mx;
    decltype(&mxfa_prefill_batch_mx_workspace_bytes) prefill_batch_mx_workspace_bytes;
} abi;

PyObject *other() { Py_RETURN_NOTIMPLEMENTED; }

// The tensor of a plain torch.Tensor (or Parameter) with its own GPU storage;
// null for subclasses, functorch and Python-dispatch tensors, views with lazy
// conjugation or negation, and other devices or layouts.
const at::Tensor *plain(PyObject *o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    using K = c10::DispatchKey;
    static const c10::DispatchKeySet special({K::Python, K::PythonTLSSnapshot, K::FuncTorchGradWrapper,
                                              K::FuncTorchBatched, K::Functionalize, K::Conjugate, K::Negative,
                                              K::ZeroTensor, K::BatchedNestedTensor});
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() ||
        t.key_set().has_any(special) || t.unsafeGetTensorImpl()->is_python_dispatch() ||
        t.unsafeGetTensorImpl()->has_symbolic_sizes_strides())
        return nullptr;
    return &t;
}

// [N, d] or [B, H, N, d], contiguous.
bool dims(const at::Tensor &t, int64_t (&n)[4]) {
    if ((t.dim() != 2 && t.dim() != 4) || !t.is_contiguous()) return false;
    for (int i = 0; i < 4; ++i) n[i] = t.dim() == 4 ? t.size(i) : i < 2 ? 1 : t.size(i - 2);
    for (int64_t x : n) {
        if (x < 1 || x > INT32_MAX) return false;
    }
    return true;
}
bool same(const int64_t (&a)[4], const int64_t (&b)[4]) {
    return a[0] == b[0] && a[1] == b[1] && a[2] == b[2] && a[3] == b[3];
}

bool is_mxfa_type(const at::Tensor &t) {
    return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat;
}

void *current_stream() { return c10::hip::getCurrentHIPStream().stream(); }

bool number(PyObject *o, double *v) {
    if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
    *v = PyFloat_AsDouble(o);
    return !PyErr_Occurred() || (PyErr_Clear(), false);
}
bool integer(PyObject *o, int *v) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    const long x = PyLong_AsLongAndOverflow(o, &over);
    if (over != 0 || x < INT32_MIN || x > INT32_MAX) return false;
    *v = (int)x;
    return true;
}

// The shape of q, k, v (all of one type, K and V alike).
bool shape_of(const at::Tensor *q, const at::Tensor *k, const at::Tensor *v, PyObject *causal, PyObject *scale,
              mxfa_shape *s) {
    int64_t nq[4], nk[4], nv[4];
    double sc;
    if (!q || !k || !v || !is_mxfa_type(*q) || k->scalar_type() != q->scalar_type() ||
        v->scalar_type() != q->scalar_type() || !dims(*q, nq) || !dims(*k, nk) || !dims(*v, nv) || !same(nk, nv) ||
        nk[0] != nq[0] || nk[2] != nq[2] || nk[3] != nq[3] || !PyBool_Check(causal) || !number(scale, &sc))
        return false;
    *s = mxfa_shape{(int)nq[0], (int)nq[1], (int)nk[1], (int)nq[2], (int)nq[3], causal == Py_True,
                    q->scalar_type() == at::kBFloat16 ? MXFA_BF16 : MXFA_F32, (float)sc};
    return true;
}

PyObject *status(int rc) { return PyLong_FromLong(rc); }

// Runs f; a C++ exception becomes the Python one torch gives it (its
// OutOfMemoryError among them).
template <class F>
PyObject *guarded(F f) {
    HANDLE_TH_ERRORS
    return f();
    END_HANDLE_TH_ERRORS
}

// attention_fwd(q, k, v, causal, scale) -> (o, lse)
PyObject *attention_fwd(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 5 || abi.flash_lse == nullptr) return other();
    return guarded([&]() -> PyObject * {
        const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]);
        mxfa_shape s;
        if (!shape_of(q, k, v, a[3], a[4], &s)) return other();
        at::Tensor o = at::empty_like(*q), lse = at::empty({s.B, s.Hq, s.N}, q->options().dtype(at::kFloat));
        void *stream = current_stream();
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = abi.flash_lse(&s, q->data_ptr(), k->data_ptr(), v->data_ptr(), o.data_ptr(),
                           static_cast<float *>(lse.data_ptr()), stream);
        Py_END_ALLOW_THREADS;
        if (rc != 0) return status(rc);
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(o)), THPVariable_Wrap(std::move(lse)));
    });
}

// attention_bwd(q, k, v, o, lse, do, causal, scale) -> (dq, dk, dv)
PyObject *attention_bwd(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 8 || abi.bwd_ws == nullptr) return other();
    return guarded([&]() -> PyObject * {
        const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *o = plain(a[3]), *lse = plain(a[4]),
                         *g = plain(a[5]);
        mxfa_shape s;
        if (!o || !lse || !g || !shape_of(q, k, v, a[6], a[7], &s)) return other();
        const int64_t nq[4] = {s.B, s.Hq, s.N, s.d};
        int64_t no[4], ng[4];
        if (o->scalar_type() != q->scalar_type() || g->scalar_type() != q->scalar_type() || !dims(*o, no) ||
            !dims(*g, ng) || !same(no, nq) || !same(ng, nq) || lse->scalar_type() != at::kFloat ||
            !lse->is_contiguous() || lse->numel() != (int64_t)s.B * s.Hq * s.N)
            return other();
        at::Tensor delta = at::empty({s.B, s.Hq, s.N}, q->options().dtype(at::kFloat));
        at::Tensor dq = at::empty_like(*q), dk = at::empty_like(*k), dv = at::empty_like(*v), ws;
        const size_t nws = abi.bwd_workspace_bytes(&s);
        if (nws > 0) ws = at::empty({(int64_t)nws}, q->options().dtype(at::kByte));
        void *stream = current_stream(), *wp = nws > 0 ? ws.data_ptr() : nullptr;
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = abi.bwd_ws(&s, q->data_ptr(), k->data_ptr(), v->data_ptr(), o->data_ptr(), g->data_ptr(),
                        static_cast<const float *>(lse->data_ptr()), static_cast<float *>(delta.data_ptr()),
                        dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), wp, nws, stream);
        Py_END_ALLOW_THREADS;
        if (rc != 0) return status(rc);
        return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(dq)), THPVariable_Wrap(std::move(dk)),
                             THPVariable_Wrap(std::move(dv)));
    });
}

// A 2-D tensor of contiguous rows, at least `rows` x `cols`: its row stride.
bool rows_of(const at::Tensor *t, at::ScalarType type, int64_t rows, int64_t cols, int *stride) {
    if (!t || t->scalar_type() != type || t->dim() != 2 || (t->size(1) > 1 && t->stride(1) != 1) ||
        t->size(0) < rows || t->size(1) < cols)
        return false;
    const int64_t s = t->size(0) > 1 ? t->stride(0) : std::max(t->size(1), cols);
    if (s < 0 || s > INT32_MAX) return false;
    *stride = (int)s;
    return true;
}

// prefill(q, kcache, vcache, out, table or None, block_size, pos0, n_head,
// n_kv_head, head_dim, scale, split, workspace): the launch's status (the
// workspace given where split)
PyObject *prefill(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 13 || abi.prefill == nullptr) return other();
    return guarded([&]() -> PyObject * {
        const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *out = plain(a[3]);
        const bool paged = a[4] != Py_None, split = a[11] == Py_True;
        const at::Tensor *table = paged ? plain(a[4]) : nullptr, *ws = split ? plain(a[12]) : nullptr;
        int block = 0, pos0, heads, kv_heads, hd, qs, ks, vs, os;
        double sc;
        if (!q || !is_mxfa_type(*q) || q->dim() != 2 || (paged && !table) || (split && !ws) ||
            (paged && (!integer(a[5], &block) || block < 1)) || !integer(a[6], &pos0) || !integer(a[7], &heads) ||
            !integer(a[8], &kv_heads) || !integer(a[9], &hd) || !number(a[10], &sc) || !PyBool_Check(a[11]) ||
            pos0 < 0 || heads < 1 || kv_heads < 1 || hd < 1 || q->size(0) < 1 || q->size(0) > INT32_MAX)
            return other();
        const int64_t n_tok = q->size(0), seen = pos0 + n_tok, crows = paged ? 1 : seen;
        if (!rows_of(q, q->scalar_type(), 1, (int64_t)heads * hd, &qs) ||
            !rows_of(k, q->scalar_type(), crows, (int64_t)kv_heads * hd, &ks) ||
            !rows_of(v, q->scalar_type(), crows, (int64_t)kv_heads * hd, &vs) || ks != vs ||
            !rows_of(out, q->scalar_type(), n_tok, (int64_t)heads * hd, &os))
            return other();
        if (paged && (table->scalar_type() != at::kInt || table->dim() != 1 || table->stride(0) != 1 ||
                      table->numel() < (seen + block - 1) / block))
            return other();
        if (split && !ws->is_contiguous()) return other();
        const mxfa_prefill_shape s{(int)n_tok, heads, kv_heads, hd, pos0, qs, ks, os,
                                   q->scalar_type() == at::kBFloat16 ? MXFA_BF16 : MXFA_F32, (float)sc};
        const void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr();
        const int *tp = paged ? static_cast<const int *>(table->data_ptr()) : nullptr;
        void *op = out->data_ptr(), *wp = split ? ws->data_ptr() : nullptr, *stream = current_stream();
        const size_t nws = split ? (size_t)ws->numel() * ws->element_size() : 0;
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        if (paged) {
            rc = split ? abi.prefill_paged_ws(&s, qp, kp, vp, op, tp, block, wp, nws, stream)
                       : abi.prefill_paged(&s, qp, kp, vp, op, tp, block, stream);
        } else {
            rc = split ? abi.prefill_ws(&s, qp, kp, vp, op, wp, nws, stream) : abi.prefill(&s, qp, kp, vp, op, stream);
        }
        Py_END_ALLOW_THREADS;
        return status(rc);
    });
}

// ---- rotary positions, a batch over a paged cache, the pages

// On the calling thread's current device, whose stream the call takes.
bool here(const at::Tensor *t) { return t != nullptr && t->get_device() == c10::hip::current_device(); }

bool flag(PyObject *o, int *v) {
    if (!PyBool_Check(o)) return false;
    *v = o == Py_True;
    return true;
}

// A contiguous vector of at least n elements of the type.
bool vec(const at::Tensor *t, at::ScalarType type, int64_t n) {
    return here(t) && t->scalar_type() == type && t->dim() == 1 && (t->numel() < 2 || t->stride(0) == 1) &&
           t->numel() >= n && t->numel() <= INT32_MAX;
}
const int *ints(const at::Tensor *t) { return static_cast<const int *>(t->data_ptr()); }
int *ints_out(const at::Tensor *t) { return static_cast<int *>(t->data_ptr()); }

// [B, H, N, d], or [N, H, d] as B = 1: sizes, and strides of the first three.
bool heads(const at::Tensor *t, at::ScalarType type, int64_t (&n)[4], long long (&s)[3]) {
    if (!here(t) || t->scalar_type() != type || (t->dim() != 3 && t->dim() != 4)) return false;
    const bool b = t->dim() == 4;
    n[0] = b ? t->size(0) : 1;
    n[1] = t->size(1);
    n[2] = b ? t->size(2) : t->size(0);
    n[3] = t->size(-1);
    s[0] = b ? t->stride(0) : 0;
    s[1] = t->stride(1);
    s[2] = b ? t->stride(2) : t->stride(0);
    for (int64_t x : n) {
        if (x < 1 || x > INT32_MAX) return false;
    }
    return n[3] == 1 || t->stride(-1) == 1;
}

// The shape of a rotary call over checked tensors (k and ko null: Q alone).
struct RotaryArgs {
    const at::Tensor *q, *k, *qo, *ko, *f, *pos;
    bool shape(mxfa_rotary_shape *s) const {
        int64_t nq[4], nk[4], no[4];
        long long sq[3], sk[3] = {0, 0, 0}, so[3], sko[3] = {0, 0, 0};
        if (!q || !is_mxfa_type(*q) || !heads(q, q->scalar_type(), nq, sq) || !heads(qo, q->scalar_type(), no, so) ||
            !same(nq, no))
            return false;
        if (k != nullptr && (!heads(k, q->scalar_type(), nk, sk) || !heads(ko, q->scalar_type(), no, sko) ||
                             !same(nk, no) || nk[0] != nq[0] || nk[2] != nq[2] || nk[3] != nq[3]))
            return false;
        if (!vec(f, at::kDouble, 1) || 2 * f->numel() > nq[3]) return false;
        if (pos != nullptr) {
            if (!here(pos) || pos->scalar_type() != at::kInt || pos->dim() < 1 || pos->dim() > 2 ||
                pos->size(-1) != nq[2] || (nq[2] > 1 && pos->stride(-1) != 1) ||
                (pos->dim() == 2 && pos->size(0) != nq[0]))
                return false;
            s->pos_bs = pos->dim() == 2 ? pos->stride(0) : 0;
        }
        s->B = (int)nq[0];
        s->Hq = (int)nq[1];
        s->Hkv = k != nullptr ? (int)nk[1] : 0;
        s->N = (int)nq[2];
        s->head_dim = (int)nq[3];
        s->rotary_dim = 2 * (int)f->numel();
        s->dtype = q->scalar_type() == at::kBFloat16 ? MXFA_BF16 : MXFA_F32;
        s->q_bs = sq[0], s->q_hs = sq[1], s->q_ts = sq[2];
        s->k_bs = sk[0], s->k_hs = sk[1], s->k_ts = sk[2];
        s->qo_bs = so[0], s->qo_hs = so[1], s->qo_ts = so[2];
        s->ko_bs = sko[0], s->ko_hs = sko[1], s->ko_ts = sko[2];
        return true;
    }
    int run(const mxfa_rotary_shape &s) const {
        return abi.rotary(&s, q->data_ptr(), k ? k->data_ptr() : nullptr, qo->data_ptr(), ko ? ko->data_ptr() : nullptr,
                          pos ? ints(pos) : nullptr, static_cast<const double *>(f->data_ptr()), current_stream());
    }
};

// rotary(q, k, q_out, k_out, frequencies, positions, pos0, interleaved, factor, inverse): the status
PyObject *rotary(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 10 || abi.rotary == nullptr) return other();
    return guarded([&]() -> PyObject * {
        const bool two = a[1] != Py_None, given = a[5] != Py_None;
        const RotaryArgs r{plain(a[0]), two ? plain(a[1]) : nullptr, plain(a[2]), two ? plain(a[3]) : nullptr,
                           plain(a[4]), given ? plain(a[5]) : nullptr};
        mxfa_rotary_shape s{};
        double factor;
        if ((two && !r.k) || (!two && a[3] != Py_None) || (given && !r.pos) || !r.shape(&s) || !integer(a[6], &s.pos0) ||
            !flag(a[7], &s.interleaved) || !number(a[8], &factor) || !flag(a[9], &s.inverse))
            return other();
        s.factor = (float)factor;
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = r.run(s);
        Py_END_ALLOW_THREADS;
        return status(rc);
    });
}

// Rows as the kernels take them: contiguous, starting on 16 bytes.
at::Tensor rows16(const at::Tensor &x) {
    const int64_t es = (int64_t)x.element_size();
    bool good = (x.size(-1) < 2 || x.stride(-1) == 1) && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) good = good && (x.size(i) < 2 || x.stride(i) * es % 16 == 0);
    return good ? x : x.clone(at::MemoryFormat::Contiguous);  // (contiguous() leaves where it begins)
}

// Q and K turned, in new tensors.
struct RotaryOptions {
    int64_t pos0;
    bool interleaved;
    double factor;
    bool inverse;
};
torch::autograd::variable_list turned(const at::Tensor &q0, const at::Tensor &k0, const at::Tensor &f,
                                      const at::Tensor *pos, const RotaryOptions &o) {
    const at::Tensor q = rows16(q0), k = rows16(k0);
    at::Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    const RotaryArgs r{&q, &k, &qo, &ko, &f, pos};
    mxfa_rotary_shape s{};
    TORCH_CHECK_VALUE(r.shape(&s), "rotary_embedding: tensors that do not fit together or are on another device");
    s.pos0 = (int)o.pos0;
    s.interleaved = o.interleaved;
    s.factor = (float)o.factor;
    s.inverse = o.inverse;
    const int rc = r.run(s);
    TORCH_CHECK(rc == 0, "rotary_embedding: mxfa_run_rotary returned ", rc);
    return {qo, ko};
}

// The differentiable rotation (autograd.rotary_embedding): its gradient is the
// transposed rotation of the outputs' gradients, itself such a node where a
// graph of it is asked for.
struct RotaryNode : torch::autograd::Function<RotaryNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const at::Tensor &q,
                                                  const at::Tensor &k, const at::Tensor &f,
                                                  const std::optional<at::Tensor> &pos,
                                                  int64_t pos0, bool interleaved, double factor, bool inverse) {
        ctx->save_for_backward({f, pos ? *pos : at::Tensor()});
        ctx->saved_data["options"] = std::make_tuple(pos0, interleaved, factor, inverse);
        return turned(q, k, f, pos ? &*pos : nullptr, RotaryOptions{pos0, interleaved, factor, inverse});
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                   torch::autograd::variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const auto o = ctx->saved_data["options"].toTuple();
        const auto &e = o->elements();
        const RotaryOptions back{e[0].toInt(), e[1].toBool(), e[2].toDouble(), !e[3].toBool()};
        const bool given = saved[1].defined();
        torch::autograd::variable_list out;
        if (c10::GradMode::is_enabled()) {
            std::optional<at::Tensor> pos;
            if (given) pos = saved[1];
            out = apply(g[0], g[1], saved[0], pos, back.pos0, back.interleaved, back.factor, back.inverse);
        } else {
            out = turned(g[0], g[1], saved[0], given ? &saved[1] : nullptr, back);
        }
        const at::Tensor none;
        return {out[0], out[1], none, none, none, none, none, none};
    }
};

// rotary_embedding(q, k, frequencies, positions or None, pos0, interleaved, factor) -> (q, k) turned
PyObject *rotary_embedding(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 7 || abi.rotary == nullptr) return other();
    return guarded([&]() -> PyObject * {
        const bool given = a[3] != Py_None;
        const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *f = plain(a[2]), *pos = given ? plain(a[3]) : nullptr;
        int pos0, interleaved;
        double factor;
        // (strides are put right in forward)
        if (!q || !k || !f || (given && !pos) || f->requires_grad() || !is_mxfa_type(*q) || q->dim() != 4 ||
            k->dim() != 4 || q->numel() == 0 || k->numel() == 0 || !integer(a[4], &pos0) || !flag(a[5], &interleaved) ||
            !number(a[6], &factor))
            return other();
        const at::Tensor &qq = *q, &kk = *k;
        if (!here(q) || !here(k) || kk.scalar_type() != qq.scalar_type() || qq.size(0) != kk.size(0) ||
            qq.size(2) != kk.size(2) || qq.size(3) != kk.size(3) || !vec(f, at::kDouble, 1) ||
            2 * f->numel() > qq.size(3) || qq.size(3) % 8 != 0 || qq.size(3) > 256 ||
            pos0 + qq.size(2) > INT32_MAX)
            return other();
        std::optional<at::Tensor> at_pos;
        if (given) at_pos = *pos;
        auto out = RotaryNode::apply(qq, kk, *f, at_pos, (int64_t)pos0, interleaved != 0, factor, false);
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out[0])), THPVariable_Wrap(std::move(out[1])));
    });
}

// A 2-D int32 table of contiguous rows for n sequences.
bool table_of(const at::Tensor *t, int64_t n, int *wide, int *stride) {
    if (!here(t) || t->scalar_type() != at::kInt || t->dim() != 2 || t->size(0) != n || t->size(1) < 1 ||
        t->size(1) > INT32_MAX || (t->size(1) > 1 && t->stride(1) != 1))
        return false;
    const int64_t s = n > 1 ? t->stride(0) : t->size(1);
    if (s < 0 || s > INT32_MAX) return false;
    *wide = (int)t->size(1);
    *stride = (int)s;
    return true;
}

// The tensors and shape that the append and the attention of a batch share.
struct Batch {
    const at::Tensor *q, *k, *v, *o, *table, *cu_q, *lens;
    mxfa_batch_shape s;
    bool read(PyObject *q_, PyObject *k_, PyObject *v_, PyObject *o_, PyObject *table_, PyObject *block, PyObject *cu_,
              PyObject *lens_, PyObject *heads_, PyObject *kv_heads, PyObject *head_dim, int kv_in_q, int bits = 0) {
        q = plain(q_), k = plain(k_), v = plain(v_), o = plain(o_), table = plain(table_), cu_q = plain(cu_);
        lens = plain(lens_);
        s = mxfa_batch_shape{};
        int ks, vs;
        if (!here(q) || !is_mxfa_type(*q) || q->dim() != 2 || !here(k) || !here(v) || !here(o) ||
            !integer(block, &s.block_size) || !integer(heads_, &s.n_head) || !integer(kv_heads, &s.n_kv_head) ||
            !integer(head_dim, &s.head_dim) || s.block_size < 1 || s.n_head < 1 || s.n_kv_head < 1 ||
            s.head_dim < 1 || q->size(0) < 1 || q->size(0) > INT32_MAX)
            return false;
        const at::ScalarType t = q->scalar_type();
        const int64_t d = s.head_dim, kw = s.n_kv_head * d;
        // a cache row in q's type; a block of bytes
        const at::ScalarType kt = bits ? at::kByte : t;
        const int64_t least = bits ? 1 : s.block_size;
        const int64_t wide = bits ? (int64_t)abi.mx_block_bytes(s.block_size, s.n_kv_head, s.head_dim, bits) : kw;
        if (wide < 1 || !rows_of(q, t, 1, (s.n_head + kv_in_q * (int64_t)s.n_kv_head) * d, &s.q_stride) ||
            !rows_of(k, kt, least, wide, &ks) || !rows_of(v, kt, least, wide, &vs) || ks != vs ||
            k->size(0) != v->size(0) || !rows_of(o, t, q->size(0), s.n_head * d, &s.out_stride) ||
            !vec(lens, at::kInt, 1) || !vec(cu_q, at::kInt, lens->numel() + 1) ||
            !table_of(table, lens->numel(), &s.max_blocks, &s.table_stride) ||
            k->size(0) / least > INT32_MAX)
            return false;
        s.n_tok = (int)q->size(0);
        s.n_seq = (int)lens->numel();
        s.max_q = 1;
        s.n_blocks = (int)(k->size(0) / least);
        s.kv_stride = ks;
        s.dtype = t == at::kBFloat16 ? MXFA_BF16 : MXFA_F32;
        return true;
    }
};

// `bits` of a microscaled cache, where a call is of one.
bool mx_bits(PyObject *o, int *bits) { return integer(o, bits) && (*bits == 8 || *bits == 4); }

// The append into either cache (R: its rotation), bits from *more.
template <class R, class Run>
PyObject *append_to(PyObject *const *a, PyObject *more, Run run) {
    return guarded([&]() -> PyObject * {
        Batch b;
        R r{};
        double factor;
        int bits = 0;
        if (more != nullptr && !mx_bits(more, &bits)) return other();
        const bool turned = a[11] != Py_None;
        const at::Tensor *f = turned ? plain(a[11]) : nullptr;
        if (!b.read(a[0], a[2], a[3], a[1], a[4], a[5], a[6], a[7], a[8], a[9], a[10], 2, bits) ||
            !flag(a[12], &r.interleaved) || !number(a[13], &factor) ||
            (turned && (!vec(f, at::kDouble, 1) || 2 * f->numel() > b.s.head_dim)))
            return other();
        r.factor = (decltype(r.factor))factor;
        if (turned) {
            r.rotary_dim = 2 * (int)f->numel();
            r.frequencies = static_cast<const double *>(f->data_ptr());
        }
        const void *q = b.q->data_ptr();
        void *o = b.o->data_ptr(), *k = b.k->data_ptr(), *v = b.v->data_ptr(), *stream = current_stream();
        const int *table = ints(b.table), *cu = ints(b.cu_q), *lens = ints(b.lens);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = run(&b.s, bits, &r, q, o, k, v, table, cu, lens, stream);
        Py_END_ALLOW_THREADS;
        return status(rc);
    });
}

// cache_append(qkv, q_out, kcache, vcache, table, block_size, cu_q, lens, n_head, n_kv_head,
// head_dim, frequencies or None, interleaved, factor): the status
PyObject *cache_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 14 || abi.cache_append == nullptr) return other();
    return append_to<mxfa_append_rotary>(a, nullptr, [](const mxfa_batch_shape *s, int, auto... x) {
        return abi.cache_append(s, x...);
    });
}
// cache_append_mx(the same, bits)
PyObject *cache_append_mx(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 15 || abi.cache_append_mx == nullptr) return other();
    return append_to<mxfa_append_rotary_mx>(a, a[14], [](auto... x) { return abi.cache_append_mx(x...); });
}

// cache_read_mx(kcache, vcache, k_out, v_out, table, block_size, cu_q, lens, n_kv_head, head_dim,
// bits): the status
PyObject *cache_read_mx(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 11 || abi.cache_read_mx == nullptr) return other();
    return guarded([&]() -> PyObject * {
        Batch b;
        int bits, vs;
        const at::Tensor *v_out = plain(a[3]);
        // (k_out in the place of q too: its rows are the batch's)
        if (!mx_bits(a[10], &bits) || !b.read(a[2], a[0], a[1], a[2], a[4], a[5], a[6], a[7], a[8], a[8], a[9], 0, bits) ||
            !here(v_out) || !rows_of(v_out, b.o->scalar_type(), b.s.n_tok, (int64_t)b.s.n_kv_head * b.s.head_dim, &vs) ||
            v_out->size(0) != b.s.n_tok || (b.s.n_tok > 1 && vs != b.s.out_stride))
            return other();
        const void *k = b.k->data_ptr(), *v = b.v->data_ptr();
        void *ko = b.o->data_ptr(), *vo = v_out->data_ptr(), *stream = current_stream();
        const int *table = ints(b.table), *cu = ints(b.cu_q), *lens = ints(b.lens);
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = abi.cache_read_mx(&b.s, bits, k, v, ko, vo, table, cu, lens, stream);
        Py_END_ALLOW_THREADS;
        return status(rc);
    });
}

// The attention over either cache, bits from *more.
PyObject *attend(PyObject *const *a, PyObject *more) {
    return guarded([&]() -> PyObject * {
        Batch b;
        double sc;
        int bits = 0;
        if (more != nullptr && !mx_bits(more, &bits)) return other();
        const bool want_lse = a[13] != Py_None, given = a[14] != Py_None;
        const at::Tensor *lse = want_lse ? plain(a[13]) : nullptr, *ws = given ? plain(a[14]) : nullptr;
        if (!b.read(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[9], a[10], a[11], 0, bits) ||
            !integer(a[8], &b.s.max_q) || !number(a[12], &sc) || (given && (!here(ws) || !ws->is_contiguous())) ||
            (want_lse && (!here(lse) || lse->scalar_type() != at::kFloat || lse->dim() != 2 ||
                          !lse->is_contiguous() || lse->size(0) != b.s.n_tok || lse->size(1) != b.s.n_head)))
            return other();
        b.s.scale = (float)sc;
        const size_t need = bits ? abi.prefill_batch_mx_workspace_bytes(&b.s, bits) : abi.prefill_batch_workspace_bytes(&b.s);
        at::Tensor own;
        if (!given) {
            if (need == 0) return other();  // a shape it does not take
            own = at::empty({(int64_t)need}, b.q->options().dtype(at::kByte));
            ws = &own;
        }
        const void *q = b.q->data_ptr(), *k = b.k->data_ptr(), *v = b.v->data_ptr();
        void *o = b.o->data_ptr(), *wp = ws->data_ptr(), *stream = current_stream();
        float *lp = want_lse ? static_cast<float *>(lse->data_ptr()) : nullptr;
        const int *table = ints(b.table), *cu = ints(b.cu_q), *lens = ints(b.lens);
        const size_t bytes = (size_t)ws->numel() * ws->element_size();
        int rc;
        Py_BEGIN_ALLOW_THREADS;
        rc = bits ? abi.prefill_batch_mx(&b.s, bits, q, k, v, o, lp, table, cu, lens, wp, bytes, stream)
                  : abi.prefill_batch(&b.s, q, k, v, o, lp, table, cu, lens, wp, bytes, stream);
        Py_END_ALLOW_THREADS;
        if (rc != 0) return status(rc);
        if (!given) return THPVariable_Wrap(std::move(own));
        Py_INCREF(a[14]);
        return a[14];
    });
}
// prefill_batch(q, kcache, vcache, out, table, block_size, cu_q, lens, max_q, n_head, n_kv_head,
// head_dim, scale, lse or None, workspace or None): the workspace, or the status
PyObject *prefill_batch(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return n != 15 || abi.prefill_batch == nullptr ? other() : attend(a, nullptr);
}
// prefill_batch_mx(the same, bits)
PyObject *prefill_batch_mx(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return n != 16 || abi.prefill_batch_mx == nullptr ? other() : attend(a, a[15]);
}

// The tables of the pages' calls: block_table, block_size, lens, refs.
struct Pages {
    const at::Tensor *table, *lens, *refs;
    mxfa_pages_shape s;
    bool read(PyObject *const *a) {
        table = plain(a[0]), lens = plain(a[2]), refs = plain(a[3]);
        s = mxfa_pages_shape{};
        if (!vec(lens, at::kInt, 1) || !vec(refs, at::kInt, 1) || !integer(a[1], &s.block_size) ||
            !table_of(table, lens->numel(), &s.max_blocks, &s.table_stride))
            return false;
        s.n_seq = (int)lens->numel();
        s.n_blocks = (int)refs->numel();
        return true;
    }
};
bool pairs_of(const at::Tensor *t, int64_t n) {
    return here(t) && t->scalar_type() == at::kInt && t->dim() == 2 && t->size(1) == 2 && t->size(0) >= n &&
           t->size(0) <= INT32_MAX && t->is_contiguous();
}

// pages_free(table, block_size, lens, refs, rows)
PyObject *pages_free(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 5 || abi.pages_free == nullptr) return other();
    return guarded([&]() -> PyObject * {
        Pages p;
        const at::Tensor *rows = plain(a[4]);
        if (!p.read(a) || !vec(rows, at::kInt, 1)) return other();
        return status(abi.pages_free(&p.s, ints_out(p.table), ints_out(p.lens), ints_out(p.refs), ints(rows),
                                     (int)rows->numel(), current_stream()));
    });
}

// pages_fork(table, block_size, lens, refs, parents, children, pairs, status, counts)
PyObject *pages_fork(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 9 || abi.pages_fork == nullptr) return other();
    return guarded([&]() -> PyObject * {
        Pages p;
        const at::Tensor *pa = plain(a[4]), *ch = plain(a[5]), *pairs = plain(a[6]), *st = plain(a[7]), *ct = plain(a[8]);
        if (!p.read(a) || !vec(pa, at::kInt, 1) || !vec(ch, at::kInt, 1) || ch->numel() != pa->numel() ||
            !pairs_of(pairs, pa->numel()) || !vec(st, at::kInt, pa->numel()) || !vec(ct, at::kInt, 2))
            return other();
        return status(abi.pages_fork(&p.s, ints_out(p.table), ints_out(p.lens), ints_out(p.refs), ints(pa), ints(ch),
                                     (int)pa->numel(), ints_out(pairs), ints_out(st), ints_out(ct), current_stream()));
    });
}

// pages_compact(table, block_size, lens, refs, new_table, new_refs, pairs, counts)
PyObject *pages_compact(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 8 || abi.pages_compact == nullptr) return other();
    return guarded([&]() -> PyObject * {
        Pages p;
        const at::Tensor *nt = plain(a[4]), *nr = plain(a[5]), *pairs = plain(a[6]), *ct = plain(a[7]);
        int wide, stride;
        if (!p.read(a) || !table_of(nt, p.s.n_seq, &wide, &stride) || wide != p.s.max_blocks ||
            !vec(nr, at::kInt, p.s.n_blocks) || !pairs_of(pairs, std::max(1, p.s.n_blocks / 2)) ||
            !vec(ct, at::kInt, 2))
            return other();
        return status(abi.pages_compact(&p.s, ints(p.table), ints(p.lens), ints(p.refs), ints_out(nt), stride,
                                        ints_out(nr), ints_out(pairs), ints_out(ct), current_stream()));
    });
}

// pages_copy(pools, block_size, pairs, count or None)
PyObject *pages_copy(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 4 || abi.pages_copy == nullptr) return other();
    return guarded([&]() -> PyObject * {
        const bool counted = a[3] != Py_None;
        const at::Tensor *x = plain(a[0]), *pairs = plain(a[2]), *ct = counted ? plain(a[3]) : nullptr;
        int block;
        if (!here(x) || (x->dim() != 2 && x->dim() != 3) || x->numel() == 0 || !integer(a[1], &block) || block < 1 ||
            x->size(-2) < block || (x->size(-1) > 1 && x->stride(-1) != 1) ||
            (x->size(-2) > 1 && x->stride(-2) != x->size(-1)) || !pairs_of(pairs, 0) ||
            (counted && !vec(ct, at::kInt, 1)) || x->size(-2) / block > INT32_MAX || x->size(0) > INT32_MAX)
            return other();
        const long long es = (long long)x->element_size();
        const bool many = x->dim() == 3;
        return status(abi.pages_copy(x->data_ptr(), many ? (int)x->size(0) : 1, many ? x->stride(0) * es : 0,
                                     (int)(x->size(-2) / block), block * x->size(-1) * es, ints(pairs),
                                     (int)pairs->size(0), counted ? ints(ct) : nullptr, current_stream()));
    });
}

// bind(addresses of the ABI functions, in the order of `abi`)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    constexpr int kCount = 20;
    if (n != kCount) {
        PyErr_Format(PyExc_TypeError, "bind: %d addresses expected", kCount);
        return nullptr;
    }
    void *f[kCount];
    for (int i = 0; i < kCount; ++i) {
        f[i] = PyLong_AsVoidPtr(a[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    abi.flash_lse = reinterpret_cast<decltype(abi.flash_lse)>(f[0]);
    abi.bwd_ws = reinterpret_cast<decltype(abi.bwd_ws)>(f[1]);
    abi.bwd_workspace_bytes = reinterpret_cast<decltype(abi.bwd_workspace_bytes)>(f[2]);
    abi.prefill = reinterpret_cast<decltype(abi.prefill)>(f[3]);
    abi.prefill_ws = reinterpret_cast<decltype(abi.prefill_ws)>(f[4]);
    abi.prefill_paged = reinterpret_cast<decltype(abi.prefill_paged)>(f[5]);
    abi.prefill_paged_ws = reinterpret_cast<decltype(abi.prefill_paged_ws)>(f[6]);
    abi.rotary = reinterpret_cast<decltype(abi.rotary)>(f[7]);
    abi.cache_append = reinterpret_cast<decltype(abi.cache_append)>(f[8]);
    abi.prefill_batch = reinterpret_cast<decltype(abi.prefill_batch)>(f[9]);
    abi.prefill_batch_workspace_bytes = reinterpret_cast<decltype(abi.prefill_batch_workspace_bytes)>(f[10]);
    abi.pages_free = reinterpret_cast<decltype(abi.pages_free)>(f[11]);
    abi.pages_fork = reinterpret_cast<decltype(abi.pages_fork)>(f[12]);
    abi.pages_compact = reinterpret_cast<decltype(abi.pages_compact)>(f[13]);
    abi.pages_copy = reinterpret_cast<decltype(abi.pages_copy)>(f[14]);
    abi.mx_block_bytes = reinterpret_cast<decltype(abi.mx_block_bytes)>(f[15]);
    abi.cache_append_mx = reinterpret_cast<decltype(abi.cache_append_mx)>(f[16]);
    abi.cache_read_mx = reinterpret_cast<decltype(abi.cache_read_mx)>(f[17]);
    abi.prefill_batch_mx = reinterpret_cast<decltype(abi.prefill_batch_mx)>(f[18]);
    abi.prefill_batch_mx_workspace_bytes = reinterpret_cast<decltype(abi.prefill_batch_mx_workspace_bytes)>(f[19]);
    Py_RETURN_NONE;
}

#define MXFA_METHOD(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(NAME)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MXFA_METHOD(bind), MXFA_METHOD(attention_fwd), MXFA_METHOD(attention_bwd),
                         MXFA_METHOD(prefill), MXFA_METHOD(rotary), MXFA_METHOD(rotary_embedding),
                         MXFA_METHOD(cache_append),
                         MXFA_METHOD(prefill_batch), MXFA_METHOD(pages_free), MXFA_METHOD(pages_fork),
                         MXFA_METHOD(pages_compact), MXFA_METHOD(pages_copy), MXFA_METHOD(cache_append_mx),
                         MXFA_METHOD(cache_read_mx), MXFA_METHOD(prefill_batch_mx), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module); }
