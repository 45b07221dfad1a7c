// The package's calls of the channels-last GroupNorm and of the Linear rows with 4-bit weights for plain tensors, in native
// code (see torch_calls.cpp, which does the same for the others): a call of the channels-last norm of 1280 channels at 8 x 8
// takes 9.9 us by Python's path and 5.1 so, its forward and gradient of 2560 at 9 x 7 28.4 and 14.8, 22 grouped projections 72 and 8.5.
#define MSD_CALLS(X)                                                                              \
    X(msd_groupnorm_channels_last) X(msd_groupnorm_channels_last_workspace)                       \
    X(msd_groupnorm_channels_last_backward) X(msd_linear_rows_q4) X(msd_linear_rows_q4_grouped)
#include "torch_calls.h"

namespace {

// A float32 or float16 tensor [batch, C, H, W] in channels-last order or contiguous [batch, positions, C], with the strides
// that a new one gets, on the current device.
struct Image {
    const at::Tensor *t = nullptr;
    int code = 0;
    int64_t batch = 0, positions = 0, channels = 0;

    Image(Call &c, PyObject *o) {
        const at::Tensor *x = c.strided(o);
        if (x == nullptr) return;
        if (x->scalar_type() == at::kFloat) code = MSD_DTYPE_F32;
        else if (x->scalar_type() == at::kHalf) code = MSD_DTYPE_F16;
        else c.ok = false;
        if (!c.ok || !plain(*x) || x->get_device() != c10::hip::current_device()) {
            c.ok = false;
            return;
        }
        t = x;
        batch = x->size(0);
        channels = x->size(x->dim() == 4 ? 1 : 2);
        positions = x->dim() == 4 ? x->size(2) * x->size(3) : x->size(1);
    }
    static bool plain(const at::Tensor &x) {
        if (x.dim() == 3) return plain_strides(x);
        if (x.dim() != 4) return false;
        int64_t stride = 1;
        for (const int i : {1, 3, 2, 0}) {
            if (x.stride(i) != stride) return false;
            stride *= std::max<int64_t>(x.size(i), 1);
        }
        return true;
    }
    at::Tensor like(at::ScalarType type) const {
        return at::Tensor(at::detail::empty_cuda(t->sizes(), type, t->device(),
                                                 t->dim() == 4 ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous));
    }
    // another such tensor of the same shape and of type `type`
    const at::Tensor *same(Call &c, PyObject *o, at::ScalarType type) const {
        const at::Tensor *x = c.strided(o);
        if (x == nullptr) return nullptr;
        if (x->scalar_type() != type || x->sizes() != t->sizes() || !plain(*x) || x->get_device() != t->get_device()) return c.fail();
        return x;
    }
    void take(Call &c, PyObject *o, Out &out) const {  // a new tensor like this one, or the caller's
        if (!c.ok) return;
        if (o == Py_None) out.make(like(t->scalar_type()));
        else if (const at::Tensor *x = same(c, o, t->scalar_type())) {
            out.object = o;
            out.data = x->data_ptr();
        }
    }
    at::Tensor workspace(Call &c, int64_t groups, int backward) const {
        size_t bytes = 0;
        if (!c.ok || groups <= 0 || channels % groups != 0 ||
            abi.msd_groupnorm_channels_last_workspace(batch, positions, channels, groups, code, backward, &bytes) != 0) {
            c.ok = false;
            return at::Tensor();
        }
        return new_tensor({(int64_t)bytes}, at::kByte, *t);
    }
};

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

// x, gamma, beta, groups, eps, fuse_silu, chunk, out: a[0 ... 7]
PyObject *forward(Call &c, Args a, bool kept, bool keep8) {
    const Image x(c, c.ok ? a[0] : nullptr);
    if (!c.ok) return nullptr;
    const float *g = c.affine(a[1], x.channels, *x.t), *b = c.affine(a[2], x.channels, *x.t);
    const int64_t groups = c.integer(a[3]);
    const double eps = c.number(a[4]);
    const int silu = c.truth(a[5]);
    const at::Tensor *chunk = a[6] != Py_None ? c.same(a[6], *x.t, x.batch * x.channels) : nullptr;
    Out out;
    x.take(c, a[7], out);
    const at::Tensor workspace = x.workspace(c, groups, 0);
    if (!c.ok || (kept && !keep8 && out.data == x.t->data_ptr() && x.t->numel() != 0)) return nullptr;
    at::Tensor stats, codes, scales;
    if (kept) stats = new_tensor({x.batch, groups, 2}, at::kFloat, *x.t);
    if (keep8) {
        codes = x.like(at::kChar);
        scales = new_tensor({x.batch, x.positions, (x.channels + MSD_CODE_BLOCK - 1) / MSD_CODE_BLOCK}, at::kFloat, *x.t);
    }
    auto at_or_null = [](const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
    const void *xp = x.t->data_ptr(), *cp = chunk != nullptr ? chunk->data_ptr() : nullptr;
    const int rc = on_stream([&](void *s) {
        return abi.msd_groupnorm_channels_last(xp, cp, out.data, g, b, x.batch, x.positions, x.channels, groups, (float)eps, silu,
                                               x.code, static_cast<float *>(at_or_null(stats)), static_cast<int8_t *>(at_or_null(codes)),
                                               static_cast<float *>(at_or_null(scales)), workspace.data_ptr(), workspace.numel(), s);
    });
    if (failed(rc)) return nullptr;
    if (!kept) return out.result();
    return tuple_of({out.result(), wrapped(std::move(codes)), wrapped(std::move(scales)), wrapped(std::move(stats))});
}

PyObject *groupnorm_channels_last(PyObject *, Args a, Py_ssize_t n) {  // x, gamma, beta, groups, eps, fuse_silu, chunk, out
    return plainly([&]() -> PyObject * {
        Call c(n, 8);
        return c.ok ? forward(c, a, false, false) : nullptr;
    });
}

PyObject *groupnorm_channels_last_kept(PyObject *, Args a, Py_ssize_t n) {  // the same and keep8 -> y, codes, scales, stats
    return plainly([&]() -> PyObject * {
        Call c(n, 9);
        if (!c.ok) return nullptr;
        const int keep8 = c.truth(a[8]);
        return c.ok ? forward(c, a, true, keep8 != 0) : nullptr;
    });
}

// dy, affine, out, and the fields of a KeptNorm -> dx, dgamma, dbeta, dchunk
PyObject *groupnorm_channels_last_backward(PyObject *, Args a, Py_ssize_t n) {
    return plainly([&]() -> PyObject * {
        Call c(n, 13);
        if (!c.ok) return nullptr;
        const Image dy(c, a[0]);
        const int affine = c.truth(a[1]);
        if (!c.ok) return nullptr;
        PyObject *const *kept = a + 3;  // x chunk codes scales stats gamma beta groups fuse_silu with_chunk
        const int64_t groups = c.integer(kept[7]);
        const int silu = c.truth(kept[8]), with_chunk = c.truth(kept[9]);
        if (!c.ok || groups <= 0) return nullptr;
        const at::Tensor *x = nullptr, *chunk = nullptr, *codes = nullptr;
        const float *scales = nullptr;
        if (kept[2] != Py_None) {
            codes = dy.same(c, kept[2], at::kChar);
            scales = c.affine(kept[3], dy.batch * dy.positions * ((dy.channels + MSD_CODE_BLOCK - 1) / MSD_CODE_BLOCK), *dy.t);
        } else {
            x = dy.same(c, kept[0], dy.t->scalar_type());
            if (kept[1] != Py_None) chunk = c.same(kept[1], *dy.t, dy.batch * dy.channels);
        }
        const float *stats = c.affine(kept[4], 2 * dy.batch * groups, *dy.t);
        const float *g = c.affine(kept[5], dy.channels, *dy.t), *b = c.affine(kept[6], dy.channels, *dy.t);
        Out out;
        dy.take(c, a[2], out);
        const at::Tensor workspace = dy.workspace(c, groups, 1);
        if (!c.ok) return nullptr;
        at::Tensor dgamma, dbeta, dchunk;
        if (affine) {
            dgamma = new_tensor({dy.channels}, at::kFloat, *dy.t);
            dbeta = new_tensor({dy.channels}, at::kFloat, *dy.t);
        }
        if (with_chunk) dchunk = new_tensor({dy.batch, dy.channels}, dy.t->scalar_type(), *dy.t);
        auto pointer = [](const at::Tensor *t) { return t != nullptr ? t->data_ptr() : nullptr; };
        float *dg = affine ? static_cast<float *>(dgamma.data_ptr()) : nullptr, *db = affine ? static_cast<float *>(dbeta.data_ptr()) : nullptr;
        void *dc = with_chunk ? dchunk.data_ptr() : nullptr;
        const int rc = on_stream([&](void *s) {
            return abi.msd_groupnorm_channels_last_backward(dy.t->data_ptr(), pointer(x), pointer(chunk), static_cast<const int8_t *>(pointer(codes)),
                                                            scales, stats, g, b, out.data, dg, db, dc, dy.batch, dy.positions, dy.channels,
                                                            groups, silu, dy.code, workspace.data_ptr(), workspace.numel(), s);
        });
        if (failed(rc)) return nullptr;
        return tuple_of({out.result(), wrapped(std::move(dgamma)), wrapped(std::move(dbeta)), wrapped(std::move(dchunk))});
    });
}

// x [m, k] on the current device and what its layers share
struct Q4Rows {
    const at::Tensor *x = nullptr;
    int code = 0;
    int64_t m = 0, k = 0, group = 0;

    Q4Rows(Call &c, PyObject *o) {
        x = c.data(o, &code);
        if (!c.ok || x->dim() != 2 || x->get_device() != c10::hip::current_device()) {
            c.ok = false;
            return;
        }
        m = x->size(0);
        k = x->size(1);
    }
    // codes and scales of a layer; the first one's say how many weights share a scale
    bool layer(Call &c, PyObject *packed, PyObject *scales, const uint8_t **q, const void **s, int64_t *n) {
        const at::Tensor *p = c.tensor(packed), *t = c.tensor(scales);
        if (!c.ok || p->dim() != 2 || t->dim() != 2 || p->scalar_type() != at::kByte || t->scalar_type() != x->scalar_type() ||
            p->get_device() != x->get_device() || t->get_device() != x->get_device() || 2 * p->size(1) != k || t->size(1) == 0)
            return c.ok = false;
        if (group == 0) group = k / t->size(1);
        if (group * t->size(1) != k || t->size(0) != p->size(0) || (group != 32 && group != 64 && group != 128)) return c.ok = false;
        *q = static_cast<const uint8_t *>(p->data_ptr());
        *s = t->data_ptr();
        *n = p->size(0);
        return true;
    }
};

PyObject *linear_rows_q4(PyObject *, Args a, Py_ssize_t n) {  // x, packed, scales, bias, act_in, act_out, out
    return plainly([&]() -> PyObject * {
        Call c(n, 7);
        if (!c.ok) return nullptr;
        Q4Rows r(c, a[0]);
        const uint8_t *packed = nullptr;
        const void *scales = nullptr;
        int64_t cols = 0;
        if (!c.ok || !r.layer(c, a[1], a[2], &packed, &scales, &cols)) return nullptr;
        const float *bias = a[3] == Py_None ? nullptr : c.affine(a[3], cols, *r.x);
        const int act_in = c.code(a[4]), act_out = c.code(a[5]);
        if (!c.ok) return nullptr;
        Out out;
        if (a[6] == Py_None) {
            out.make(new_tensor({r.m, cols}, r.x->scalar_type(), *r.x));
        } else if (const at::Tensor *t = c.same(a[6], *r.x, r.m * cols)) {
            out.object = a[6];
            out.data = t->data_ptr();
        }
        if (!c.ok) return nullptr;
        const void *xp = r.x->data_ptr();
        return finish(on_stream([&](void *s) {
            return abi.msd_linear_rows_q4(xp, packed, scales, bias, out.data, r.m, cols, r.k, r.group, act_in, act_out, r.code, s);
        }), out);
    });
}

// Tensors [m, n] for every n, side by side in one allocation at multiples of 256 bytes (22 allocations of their own: 5 us more).
std::vector<at::Tensor> parts_of_one(const std::vector<size_t> &ns, int64_t m, const at::Tensor &like) {
    const int64_t unit = 256 / (int64_t)like.element_size();
    int64_t total = 0;
    for (const size_t n : ns) total += (m * (int64_t)n + unit - 1) / unit * unit;
    const at::Tensor whole = new_tensor({total}, like.scalar_type(), like);
    std::vector<at::Tensor> parts;
    parts.reserve(ns.size());
    int64_t at = 0;
    for (const size_t n : ns) {
        auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
        impl->set_sizes_contiguous({m, (int64_t)n});
        impl->set_storage_offset(at);
        parts.emplace_back(std::move(impl));
        at += (m * (int64_t)n + unit - 1) / unit * unit;
    }
    return parts;
}

PyObject *linear_rows_q4_grouped(PyObject *, Args a, Py_ssize_t n) {  // x, packed, scales, biases, act_in, act_out
    return plainly([&]() -> PyObject * {
        Call c(n, 6);
        if (!c.ok || !PyList_CheckExact(a[1]) || !PyList_CheckExact(a[2]) || !(a[3] == Py_None || PyList_CheckExact(a[3]))) return nullptr;
        Q4Rows r(c, a[0]);
        const Py_ssize_t count = PyList_GET_SIZE(a[1]);
        if (!c.ok || count == 0 || PyList_GET_SIZE(a[2]) != count || (a[3] != Py_None && PyList_GET_SIZE(a[3]) != count)) return nullptr;
        const int act_in = c.code(a[4]), act_out = c.code(a[5]);
        std::vector<const uint8_t *> qs(count);
        std::vector<const void *> ss(count);
        std::vector<const float *> bs(count);
        std::vector<size_t> ns(count);
        for (Py_ssize_t i = 0; i < count; i++) {
            int64_t cols = 0;
            if (!r.layer(c, PyList_GET_ITEM(a[1], i), PyList_GET_ITEM(a[2], i), &qs[i], &ss[i], &cols)) return nullptr;
            PyObject *b = a[3] == Py_None ? Py_None : PyList_GET_ITEM(a[3], i);
            bs[i] = b == Py_None ? nullptr : c.affine(b, cols, *r.x);
            ns[i] = (size_t)cols;
        }
        if (!c.ok) return nullptr;
        std::vector<at::Tensor> outs = parts_of_one(ns, r.m, *r.x);
        std::vector<void *> ys(count);
        for (Py_ssize_t i = 0; i < count; i++) ys[i] = outs[i].data_ptr();
        const void *xp = r.x->data_ptr();
        const int rc = on_stream([&](void *s) {
            return abi.msd_linear_rows_q4_grouped(xp, qs.data(), ss.data(), bs.data(), ys.data(), ns.data(), count, r.m, r.k, r.group,
                                                  act_in, act_out, r.code, s);
        });
        if (failed(rc)) return nullptr;
        PyObject *list = PyList_New(count);
        if (list == nullptr) return nullptr;
        for (Py_ssize_t i = 0; i < count; i++) PyList_SET_ITEM(list, i, THPVariable_Wrap(std::move(outs[i])));
        return list;
    });
}

PyMethodDef methods[] = {
    FAST(groupnorm_channels_last), FAST(groupnorm_channels_last_kept), FAST(groupnorm_channels_last_backward), FAST(linear_rows_q4),
    FAST(linear_rows_q4_grouped), {"bind", bind, METH_VARARGS, nullptr}, {"names", names, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "msd_torch_calls_cl_q4", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_msd_torch_calls_cl_q4(void) { return make_module(&module); }
