// The package's calls of the token embedding, of LayerNorm's gradient and of attention for plain tensors, in native code (see
// torch_calls.cpp, which does the same for the others).
#define MSD_CALLS(X)                                                                                        \
    X(msd_layernorm_backward) X(msd_layernorm_backward_workspace) X(msd_token_embedding)                    \
    X(msd_token_embedding_backward) X(msd_token_embedding_backward_workspace) X(msd_attention)              \
    X(msd_attention_backward) X(msd_attention_workspace)
#include <cmath>

#include "torch_calls.h"

namespace {

PyObject *wrapped(at::Tensor t) {
    if (t.defined()) return THPVariable_Wrap(std::move(t));
    Py_RETURN_NONE;
}

// A tuple of the objects, which it takes over; nullptr where one of them is.
PyObject *tuple_of(std::initializer_list<PyObject *> objects) {
    PyObject *t = PyTuple_New((Py_ssize_t)objects.size());
    Py_ssize_t i = 0;
    bool whole = t != nullptr;
    for (PyObject *o : objects) {
        whole = whole && o != nullptr;
        if (t != nullptr) PyTuple_SET_ITEM(t, i++, o);
        else Py_XDECREF(o);
    }
    if (!whole) Py_CLEAR(t);
    return t;
}

bool here(const at::Tensor &t) { return t.get_device() == c10::hip::current_device(); }
void *pointer(const at::Tensor *t) { return t != nullptr ? t->data_ptr() : nullptr; }
void *pointer(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

PyObject *layernorm_backward(PyObject *, Args a, Py_ssize_t n) {  // dy, x, gamma, eps, dsum, affine, out
    return plainly([&]() -> PyObject * {
        Call c(n, 7);
        int code = 0;
        const at::Tensor *dy = c.ok ? c.data(a[0], &code) : nullptr;
        if (!c.ok || dy->dim() == 0 || !here(*dy)) return nullptr;
        const int64_t count = dy->numel(), dim = dy->size(-1), rows = dim != 0 ? count / dim : 0;
        const at::Tensor *x = c.same(a[1], *dy, count);
        const float *gamma = c.affine(a[2], dim, *dy);
        const double eps = c.number(a[3]);
        const at::Tensor *dsum = a[4] != Py_None ? c.same(a[4], *dy, count) : nullptr;
        const int affine = c.truth(a[5]);
        Out out;
        out.take(c, a[6], *dy);
        size_t bytes = 0;
        if (!c.ok || abi.msd_layernorm_backward_workspace(rows, dim, code, &bytes) != 0) return nullptr;
        const at::Tensor workspace = new_tensor({(int64_t)bytes}, at::kByte, *dy);
        at::Tensor dgamma, dbeta;
        if (affine) {
            dgamma = new_tensor({dim}, at::kFloat, *dy);
            dbeta = new_tensor({dim}, at::kFloat, *dy);
        }
        const int rc = on_stream([&](void *s) {
            return abi.msd_layernorm_backward(dy->data_ptr(), x->data_ptr(), pointer(dsum), gamma, out.data,
                                              static_cast<float *>(pointer(dgamma)), static_cast<float *>(pointer(dbeta)), rows, dim,
                                              (float)eps, code, workspace.data_ptr(), bytes, s);
        });
        if (failed(rc)) return nullptr;
        return tuple_of({out.result(), wrapped(std::move(dgamma)), wrapped(std::move(dbeta))});
    });
}

// int64 ids [..., length] on the current device
const at::Tensor *token_ids(Call &c, PyObject *o) {
    const at::Tensor *ids = c.tensor(o);
    return ids != nullptr && ids->scalar_type() == at::kLong && ids->dim() != 0 && here(*ids) ? ids : c.fail();
}

std::vector<int64_t> rows_of(const at::Tensor &ids, int64_t dim) {
    std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(dim);
    return shape;
}

PyObject *token_embedding(PyObject *, Args a, Py_ssize_t n) {  // ids, table, positions, scale, out
    return plainly([&]() -> PyObject * {
        Call c(n, 5);
        if (!c.ok) return nullptr;
        int code = 0;
        const at::Tensor *ids = token_ids(c, a[0]), *table = c.data(a[1], &code), *positions = nullptr;
        if (!c.ok || table->dim() != 2 || !here(*table)) return nullptr;
        const int64_t vocab = table->size(0), dim = table->size(1), tokens = ids->numel(), length = ids->size(-1);
        if (a[2] != Py_None) {
            int other = 0;
            positions = c.data(a[2], &other);
            if (!c.ok || other != code || positions->dim() != 2 || positions->size(1) != dim || positions->size(0) < length || !here(*positions))
                return nullptr;
        }
        const double scale = c.number(a[3]);
        if (!c.ok) return nullptr;
        Out out;
        if (a[4] == Py_None) {
            out.make(new_tensor(rows_of(*ids, dim), table->scalar_type(), *table));
        } else if (const at::Tensor *t = c.same(a[4], *table, tokens * dim)) {
            out.object = a[4];
            out.data = t->data_ptr();
        }
        if (!c.ok) return nullptr;
        return finish(on_stream([&](void *s) {
            return abi.msd_token_embedding(static_cast<const int64_t *>(ids->data_ptr()), table->data_ptr(), pointer(positions), out.data,
                                           tokens, length, vocab, dim, (float)scale, code, s);
        }), out);
    });
}

PyObject *token_embedding_backward(PyObject *, Args a, Py_ssize_t n) {  // dy, ids, vocab, positions, scale
    return plainly([&]() -> PyObject * {
        Call c(n, 5);
        if (!c.ok) return nullptr;
        int code = 0;
        const at::Tensor *dy = c.data(a[0], &code), *ids = token_ids(c, a[1]);
        const int64_t vocab = c.integer(a[2]), positions = c.integer(a[3]);
        const double scale = c.number(a[4]);
        if (!c.ok || !here(*dy) || dy->dim() != ids->dim() + 1 || dy->sizes().slice(0, ids->dim()) != ids->sizes() || vocab < 0 || positions < 0)
            return nullptr;
        const int64_t dim = dy->size(-1), tokens = ids->numel(), length = ids->size(-1);
        if (positions != 0 && positions < length) return nullptr;
        size_t bytes = 0;
        if (abi.msd_token_embedding_backward_workspace(tokens, length, vocab, positions, dim, code, &bytes) != 0) return nullptr;
        const at::Tensor workspace = new_tensor({(int64_t)bytes}, at::kByte, *dy);
        at::Tensor dtable = new_tensor({vocab, dim}, dy->scalar_type(), *dy), dpositions;
        if (positions != 0) dpositions = new_tensor({positions, dim}, dy->scalar_type(), *dy);
        const int rc = on_stream([&](void *s) {
            return abi.msd_token_embedding_backward(static_cast<const int64_t *>(ids->data_ptr()), dy->data_ptr(), dtable.data_ptr(),
                                                    pointer(dpositions), tokens, length, vocab, positions, dim, (float)scale, code,
                                                    workspace.data_ptr(), bytes, s);
        });
        if (failed(rc)) return nullptr;
        return tuple_of({wrapped(std::move(dtable)), wrapped(std::move(dpositions))});
    });
}

// The sizes and strides of an attention call.
struct Heads {
    size_t batch = 0, q_rows = 0, k_rows = 0, heads = 0, kv_heads = 0, dim = 0;
    size_t strides[24];
    const int32_t *q_offsets = nullptr, *k_offsets = nullptr;
    const at::Tensor *q = nullptr, *k = nullptr, *v = nullptr;
    int code = 0;

    // a [batch, rows, heads, dim] or packed [rows, heads, dim] tensor of q's type, its strides as number `i`
    const at::Tensor *view(Call &c, PyObject *o, int i) {
        const at::Tensor *t = c.strided(o);
        if (t == nullptr || !here(*t) || (t->dim() != 3 && t->dim() != 4) || (t->size(-1) > 1 && t->stride(-1) != 1)) return c.fail();
        if (q != nullptr && (t->scalar_type() != q->scalar_type() || t->dim() != q->dim())) return c.fail();
        const int64_t d = t->dim();
        strides[3 * i] = d == 4 ? t->stride(0) : 0;
        strides[3 * i + 1] = t->stride(d - 3);
        strides[3 * i + 2] = t->stride(d - 2);
        return t;
    }
    // int32 [sequences + 1], of as many as `other` where that is not null
    const at::Tensor *offsets(Call &c, PyObject *o, const at::Tensor *other) {
        const at::Tensor *t = c.tensor(o);
        if (t == nullptr) return nullptr;
        if (t->scalar_type() != at::kInt || t->dim() != 1 || t->numel() == 0 || !here(*t)) return c.fail();
        return other == nullptr || t->numel() == other->numel() ? t : c.fail();
    }
    Heads(Call &c, PyObject *qo, PyObject *ko, PyObject *vo, PyObject *offsets_q, PyObject *offsets_k) {
        q = view(c, qo, 0);
        k = c.ok ? view(c, ko, 1) : nullptr;
        v = c.ok ? view(c, vo, 2) : nullptr;
        if (!c.ok) return;
        if (q->scalar_type() == at::kFloat) code = MSD_DTYPE_F32;
        else if (q->scalar_type() == at::kHalf) code = MSD_DTYPE_F16;
        else c.ok = false;
        const int64_t d = q->dim();
        if (k->sizes() != v->sizes() || k->size(-1) != q->size(-1)) c.ok = false;
        q_rows = q->size(d - 3);
        k_rows = k->size(d - 3);
        heads = q->size(d - 2);
        kv_heads = k->size(d - 2);
        dim = q->size(d - 1);
        if (d == 4) {
            if (offsets_q != Py_None || offsets_k != Py_None || q->size(0) != k->size(0)) c.ok = false;
            batch = q->size(0);
        } else if (c.ok) {
            if (offsets_k == Py_None && k_rows != q_rows) c.ok = false;
            const at::Tensor *of_q = c.ok ? offsets(c, offsets_q, nullptr) : nullptr;
            const at::Tensor *of_k = !c.ok || offsets_k == Py_None ? of_q : offsets(c, offsets_k, of_q);
            if (!c.ok) return;
            batch = (size_t)of_q->numel() - 1;
            q_offsets = static_cast<const int32_t *>(of_q->data_ptr());
            k_offsets = static_cast<const int32_t *>(of_k->data_ptr());
        }
        if (heads == 0 || kv_heads == 0 || heads % kv_heads != 0 || dim == 0) c.ok = false;
    }
    at::Tensor workspace(Call &c, int backward) const {
        size_t bytes = 0;
        if (!c.ok || abi.msd_attention_workspace(batch, q_rows, k_rows, heads, kv_heads, dim, q_offsets != nullptr, backward, code, &bytes) != 0) {
            c.ok = false;
            return at::Tensor();
        }
        return new_tensor({(int64_t)bytes}, at::kByte, *q);
    }
};

// q, k, v, causal, scale, offsets, offsets_k, out, keep -> out, or (out, lse, rest, scale) where `keep`
PyObject *attention(PyObject *, Args a, Py_ssize_t n) {
    return plainly([&]() -> PyObject * {
        Call c(n, 9);
        if (!c.ok) return nullptr;
        Heads h(c, a[0], a[1], a[2], a[5], a[6]);
        if (!c.ok) return nullptr;
        const int causal = c.truth(a[3]), keep = c.truth(a[8]);
        const double scale = a[4] == Py_None ? 1.0 / std::sqrt((double)h.dim) : c.number(a[4]);
        const at::Tensor workspace = h.workspace(c, 0);
        if (!c.ok) return nullptr;
        Out out;
        if (a[7] == Py_None) {
            out.make(new_tensor(h.q->sizes(), h.q->scalar_type(), *h.q));
            h.strides[9] = h.q_rows * h.heads * h.dim;
            h.strides[10] = h.heads * h.dim;
            h.strides[11] = h.dim;
        } else if (const at::Tensor *t = h.view(c, a[7], 3)) {
            if (t->sizes() != h.q->sizes()) return nullptr;
            out.object = a[7];
            out.data = t->data_ptr();
        }
        if (!c.ok) return nullptr;
        at::Tensor lse, rest;
        if (keep) {
            lse = new_tensor(h.q->sizes().slice(0, h.q->dim() - 1), at::kFloat, *h.q);
            if (h.code == MSD_DTYPE_F16) rest = new_tensor(h.q->sizes(), at::kHalf, *h.q);
        }
        const int rc = on_stream([&](void *s) {
            return abi.msd_attention(h.q->data_ptr(), h.k->data_ptr(), h.v->data_ptr(), out.data, static_cast<float *>(pointer(lse)),
                                     pointer(rest), h.q_offsets, h.k_offsets, h.batch, h.q_rows, h.k_rows, h.heads, h.kv_heads, h.dim,
                                     h.strides, (float)scale, causal, h.code, workspace.data_ptr(), workspace.numel(), s);
        });
        if (failed(rc)) return nullptr;
        if (!keep) return out.result();
        return tuple_of({out.result(), wrapped(std::move(lse)), wrapped(std::move(rest)), PyFloat_FromDouble(scale)});
    });
}

// dout, out (None), and the fields of a KeptAttention -> dq, dk, dv
PyObject *attention_backward(PyObject *, Args a, Py_ssize_t n) {
    return plainly([&]() -> PyObject * {
        Call c(n, 12);
        if (!c.ok || a[1] != Py_None) return nullptr;
        PyObject *const *kept = a + 2;  // q k v out lse rest causal scale offsets offsets_k
        Heads h(c, kept[0], kept[1], kept[2], kept[8], kept[9]);
        if (!c.ok) return nullptr;
        const at::Tensor *out = h.view(c, kept[3], 3), *dout = h.view(c, a[0], 4);
        const int causal = c.truth(kept[6]);
        const double scale = c.number(kept[7]);
        const at::Tensor workspace = h.workspace(c, causal ? 1 : 2);
        if (!c.ok || out->sizes() != h.q->sizes() || dout->sizes() != h.q->sizes()) return nullptr;
        const int64_t rows = h.q->numel() / (int64_t)h.dim;
        const float *lse = c.affine(kept[4], rows, *h.q);
        const at::Tensor *rest = kept[5] != Py_None ? c.same(kept[5], *h.q, h.q->numel()) : nullptr;
        if (!c.ok) return nullptr;
        at::Tensor to[3];
        const at::Tensor *const like[3] = {h.q, h.k, h.k};
        for (int i = 0; i < 3; i++) {
            to[i] = new_tensor(like[i]->sizes(), h.q->scalar_type(), *h.q);
            const size_t heads = i == 0 ? h.heads : h.kv_heads;
            h.strides[15 + 3 * i] = (i == 0 ? h.q_rows : h.k_rows) * heads * h.dim;
            h.strides[16 + 3 * i] = heads * h.dim;
            h.strides[17 + 3 * i] = h.dim;
        }
        const int rc = on_stream([&](void *s) {
            return abi.msd_attention_backward(dout->data_ptr(), h.q->data_ptr(), h.k->data_ptr(), h.v->data_ptr(), out->data_ptr(), lse,
                                              pointer(rest), to[0].data_ptr(), to[1].data_ptr(), to[2].data_ptr(), h.q_offsets, h.k_offsets,
                                              h.batch, h.q_rows, h.k_rows, h.heads, h.kv_heads, h.dim, h.strides, (float)scale, causal,
                                              h.code, workspace.data_ptr(), workspace.numel(), s);
        });
        if (failed(rc)) return nullptr;
        return tuple_of({wrapped(std::move(to[0])), wrapped(std::move(to[1])), wrapped(std::move(to[2]))});
    });
}

PyMethodDef methods[] = {
    FAST(layernorm_backward), FAST(token_embedding), FAST(token_embedding_backward), FAST(attention), FAST(attention_backward),
    {"bind", bind, METH_VARARGS, nullptr}, {"names", names, METH_NOARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "msd_torch_calls_text", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_msd_torch_calls_text(void) { return make_module(&module); }
