"""Token embedding, LayerNorm's gradient, attention: sizes of workspaces and refusals, without a GPU (addresses are made up: a refused
call reads none); the 64-bit plain forms against differentiation."""
import ctypes

import pytest
import torch

import plain_text as plain

F32, F16 = 0, 1


def _bytes(msd, name, *args):
    size = ctypes.c_size_t(0)
    rc = getattr(msd.load_library(), name)(*args, ctypes.byref(size))
    return size.value if rc == 0 else None


def test_attention_gradient_workspace_holds_the_parts_of_a_causal_call(msd):
    """Under a mask the rows are cut into two parts where they are not without it: the bytes are those of the larger."""
    batch, rows, heads, kv_heads, dim = 4, 4000, 16, 4, 128
    got = _bytes(msd, "msd_attention_workspace", batch, rows, rows, heads, kv_heads, dim, 0, 1, F16)
    vectors = 4 * (2 * batch * rows * heads + batch * rows * kv_heads)
    part = 4 * 2 * dim * batch * rows * kv_heads
    assert got >= vectors + 2 * part


# ---- refusals --------------------------------------------------------------------------------
p, f = ctypes.c_void_p, ctypes.c_float
A, B, C, D, E, G, H, I, J, K, L, M = (p((i + 1) << 24) for i in range(12))
NEED = 1 << 23


def _shift(a, n):
    return p(a.value + n)


def test_layernorm_gradient_refusals(msd):
    lib = msd.load_library()

    def call(dy=A, x=B, dsum=None, gamma=C, dx=D, dgamma=E, dbeta=G, rows=64, dim=40, eps=1e-5, dtype=F16, workspace=H, size=NEED):
        return lib.msd_layernorm_backward(dy, x, dsum, gamma, dx, dgamma, dbeta, rows, dim, f(eps), dtype, workspace, size, None)

    for change in (dict(dy=None), dict(x=None), dict(gamma=None), dict(dx=None), dict(dgamma=None), dict(dbeta=None), dict(dtype=2), dict(dtype=-1),
                   dict(workspace=None), dict(size=16), dict(workspace=_shift(H, 8)), dict(dx=_shift(A, 2)), dict(dx=B), dict(dx=C),
                   dict(dsum=I, dx=_shift(I, 2)), dict(dgamma=A), dict(dgamma=G), dict(dbeta=B), dict(dgamma=D), dict(dbeta=C), dict(dsum=E),
                   dict(workspace=A), dict(workspace=D), dict(workspace=E), dict(workspace=C), dict(rows=1 << 60, dim=1 << 10), dict(dim=1 << 40)):
        assert call(**change) == 1, change
    # nothing to do: no dx, and no sums wanted
    assert call(rows=0, dy=None, x=None, dx=None, dgamma=None, dbeta=None, workspace=None, size=0) == 0
    assert call(dim=0, dy=None, x=None, dx=None, gamma=None, workspace=None, size=0) == 0
    assert _bytes(msd, "msd_layernorm_backward_workspace", 64, 40, 5) is None and _bytes(msd, "msd_layernorm_backward_workspace", 64, 40, F16) > 0
    assert lib.msd_layernorm_backward_workspace(64, 40, F16, None) == 1


def test_token_embedding_refusals(msd):
    lib = msd.load_library()

    def call(ids=A, table=B, positions=C, y=D, tokens=154, length=77, vocab=100, dim=8, dtype=F16):
        return lib.msd_token_embedding(ids, table, positions, y, tokens, length, vocab, dim, f(1.0), dtype, None)

    for change in (dict(ids=None), dict(table=None), dict(y=None), dict(vocab=0), dict(dtype=3), dict(length=0), dict(length=76), dict(y=A), dict(y=B),
                   dict(y=C), dict(y=_shift(B, 100 * 8 * 2 - 2)), dict(ids=_shift(D, 154 * 8 * 2 - 2)), dict(tokens=1 << 26, length=1),
                   dict(vocab=(1 << 28) + 1), dict(dim=(1 << 20) + 1), dict(tokens=1 << 25, length=1 << 25, dim=64)):
        assert call(**change) == 1, change
    assert call(tokens=0, ids=None, table=None, y=None) == 0 and call(dim=0, ids=None, table=None, y=None) == 0

    def back(ids=A, dy=B, dtable=C, dpositions=D, tokens=154, length=77, vocab=100, positions=77, dim=8, dtype=F16, workspace=E, size=NEED):
        return lib.msd_token_embedding_backward(ids, dy, dtable, dpositions, tokens, length, vocab, positions, dim, f(1.0), dtype, workspace,
                                                size, None)

    for change in (dict(ids=None), dict(dy=None), dict(dtable=None), dict(dpositions=None), dict(positions=0), dict(positions=76), dict(length=5),
                   dict(dtype=9), dict(workspace=None), dict(size=64), dict(workspace=_shift(E, 4)), dict(dtable=A), dict(dtable=B), dict(dpositions=B),
                   dict(dtable=D), dict(dtable=E), dict(workspace=A), dict(workspace=B), dict(dpositions=_shift(C, 100 * 8 * 2 - 2)),
                   dict(vocab=1 << 29), dict(positions=1 << 31)):
        assert back(**change) == 1, change
    assert back(dim=0, ids=None, dy=None) == 0 and back(vocab=0, positions=0, dtable=None, dpositions=None, tokens=0) == 0
    assert lib.msd_token_embedding_backward_workspace(4, 4, 4, 4, 4, F16, None) == 1


def _attention(lib, q=A, k=B, v=C, out=D, lse=E, rest=G, qo=None, ko=None, batch=2, rows=50, keys=60, heads=4, kv_heads=2, dim=64, strides=None,
               scale=0.125, causal=0, dtype=F16, workspace=H, size=NEED):
    s = (ctypes.c_size_t * 12)(*strides) if strides else None
    return lib.msd_attention(q, k, v, out, lse, rest, qo, ko, batch, rows, keys, heads, kv_heads, dim, s, f(scale), causal, dtype, workspace, size, None)


FEW = dict(batch=1, rows=1, keys=9000)  # (in parts, so that there is a workspace)


def test_attention_refusals(msd):
    lib = msd.load_library()
    inf, nan = float("inf"), float("nan")
    assert _bytes(msd, "msd_attention_workspace", 1, 1, 9000, 4, 2, 64, 0, 0, F16) > 0
    dense = [50 * 256, 256, 64, 60 * 128, 128, 64, 60 * 128, 128, 64, 50 * 256, 256, 64]

    def strided(**at):
        return dict(strides=[at.get("s%d" % i, n) for i, n in enumerate(dense)])

    for change in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(dim=0), dict(dim=129),
                   dict(dtype=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=inf), dict(scale=nan), dict(qo=I), dict(ko=I),
                   dict(out=A), dict(out=B), dict(out=C), dict(out=_shift(A, 2)), dict(out=E), dict(out=G), dict(lse=A), dict(lse=B), dict(lse=G), dict(rest=A),
                   dict(rest=C), dict(FEW, workspace=None), dict(FEW, size=100), dict(FEW, workspace=_shift(H, 8)), dict(FEW, workspace=A),
                   dict(FEW, workspace=D), dict(FEW, workspace=E), dict(FEW, workspace=G), dict(qo=D, ko=I), dict(qo=I, ko=E),
                   strided(s9=0), strided(s10=255), strided(s10=0), strided(s11=63), strided(s9=50 * 256 - 1), strided(s0=1 << 62), strided(s10=1 << 62),
                   dict(batch=1 << 28), dict(rows=1 << 28), dict(keys=1 << 28), dict(heads=1 << 21, kv_heads=1), dict(rows=1 << 26, batch=1),
                   dict(batch=1 << 22, rows=1, keys=1, kv_heads=4), dict(scale=1e30), dict(qo=I, ko=J, batch=(1 << 16) + 1, rows=1 << 17, keys=1 << 17),
                   dict(rows=1 << 24, keys=1, heads=8, kv_heads=1)):
        assert _attention(lib, **change) == 1, change
    assert _attention(lib, batch=0, q=None, k=None, v=None, out=None, lse=None, rest=None, workspace=None) == 0
    assert _attention(lib, rows=0, q=None, out=None, lse=None, rest=None, workspace=None) == 0
    assert lib.msd_attention_workspace(1, 1, 1, 1, 1, 64, 0, 0, F16, None) == 1 and _bytes(msd, "msd_attention_workspace", 1, 1, 1, 3, 2, 64, 0, 0, F16) is None


def _attention_backward(lib, at=(A, B, C, D, E, G, H, I), lse=J, rest=None, qo=None, ko=None, batch=2, rows=50, keys=60, heads=4, kv_heads=2, dim=64,
                        strides=None, scale=0.125, dtype=F16, workspace=K, size=NEED):
    q, k, v, out, dout, dq, dk, dv = at
    s = (ctypes.c_size_t * 24)(*strides) if strides else None
    return lib.msd_attention_backward(dout, q, k, v, out, lse, rest, dq, dk, dv, qo, ko, batch, rows, keys, heads, kv_heads, dim, s, f(scale), 0, dtype,
                                      workspace, size, None)


def test_attention_gradient_refusals(msd):
    lib = msd.load_library()
    base = (A, B, C, D, E, G, H, I)

    def swapped(i, to):
        return dict(at=base[:i] + (to,) + base[i + 1:])

    bad = [swapped(i, None) for i in range(8)] + [swapped(i, base[j]) for i in range(5, 8) for j in range(i)] + [swapped(5, J), swapped(6, K), swapped(7, _shift(A, 2))]
    for change in bad + [dict(lse=None), dict(rest=H), dict(rest=K), dict(qo=L), dict(ko=L), dict(qo=G, ko=L), dict(workspace=None), dict(size=64),
                         dict(workspace=_shift(K, 4)), dict(workspace=A), dict(workspace=J), dict(scale=-0.5), dict(dim=200), dict(heads=3), dict(dtype=4)]:
        assert _attention_backward(lib, **change) == 1, change
    assert _attention_backward(lib, batch=0, at=(None,) * 8, lse=None, workspace=None) == 0


@pytest.mark.parametrize("layout", ["rows", "sequences"])
def test_gradients_into_each_other(msd, layout):
    """dk one element too far in front, among the rows (sequences) of dq.  (In their places they are let through: that runs on a GPU.)"""
    lib = msd.load_library()
    rows, heads, dim = 50, 4, 64
    if layout == "rows":
        strides, step = [rows * 3 * heads * dim, 3 * heads * dim, dim], heads * dim * 2
    else:
        strides, step = [3 * heads * rows * dim, dim, rows * dim], heads * rows * dim * 2
    dense = [rows * heads * dim, heads * dim, dim]
    at = (A, B, C, D, E, G, _shift(G, step - 2), _shift(G, 2 * step))
    assert _attention_backward(lib, at=at, keys=rows, kv_heads=heads, strides=dense * 5 + strides * 3) == 1


# ---- the plain forms -------------------------------------------------------------------------
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[(5, 9)], [(9, 5), (0, 3), (2, 0), (4, 4)]], ids=["one", "four"])
def test_plain_attention_has_the_gradients_that_differentiation_gives(causal, lengths):
    nq, nk, heads, kv_heads, dim, scale = sum(a for a, _ in lengths), sum(b for _, b in lengths), 4, 2, 6, 0.4
    gen = torch.Generator().manual_seed(3)
    q, k, v, dout = (torch.randn(n, h, dim, generator=gen).double() for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads), (nq, heads)))
    plain.HALF[torch.float64] = plain.TINY[torch.float64] = 0.0
    try:
        got = plain.attention(q, k, v, causal, scale, dout, lengths)
    finally:
        del plain.HALF[torch.float64], plain.TINY[torch.float64]
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    total, outs, q0, k0 = 0.0, [], 0, 0
    for lq, lk in lengths:
        kk, vv = (t[k0:k0 + lk].repeat_interleave(heads // kv_heads, 1) for t in leaves[1:])
        for i in range(q0, q0 + lq):  # a row at a time, over the keys that it sees
            n = min(lk, max(0, i - q0 + 1 + lk - lq)) if causal else lk
            if n == 0:
                outs.append(torch.zeros(heads, dim, dtype=torch.float64))
                continue
            weights = torch.softmax(scale * torch.einsum("hd,nhd->hn", leaves[0][i], kk[:n]), 1)
            outs.append(torch.einsum("hn,nhd->hd", weights, vv[:n]))
        q0, k0 = q0 + lq, k0 + lk
    out = torch.stack(outs)
    (out * dout).sum().backward()
    for (value, _), want in zip(got, (out.detach(), leaves[0].grad, leaves[1].grad, leaves[2].grad)):
        assert torch.allclose(value, torch.zeros_like(value) if want is None else want, atol=1e-12, rtol=1e-12)


def test_plain_embedding_and_layernorm_have_the_gradients_that_differentiation_gives():
    gen = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 7, (3, 5), generator=gen)
    dy = torch.randn(3, 5, 6, generator=gen)
    table, places = torch.randn(7, 6, generator=gen).double().requires_grad_(), torch.randn(8, 6, generator=gen).double().requires_grad_()
    ((1.5 * table[ids] + places[:5]) * dy.double()).sum().backward()
    (dtable, _), (dplaces, _) = plain.embedding_backward(dy, ids, 7, 8, 1.5)
    assert torch.allclose(dtable, table.grad, atol=1e-12) and torch.allclose(dplaces, places.grad, atol=1e-12)

    x, gamma, dy, dsum = torch.randn(4, 9, generator=gen), torch.randn(9, generator=gen), torch.randn(4, 9, generator=gen), torch.randn(4, 9, generator=gen)
    leaves = [x.double().requires_grad_(), gamma.double().requires_grad_(), torch.zeros(9, dtype=torch.float64, requires_grad=True)]
    y = torch.nn.functional.layer_norm(leaves[0], (9,), leaves[1], leaves[2], 1e-5)
    ((y * dy.double()).sum() + (leaves[0] * dsum.double()).sum()).backward()
    for (value, _), leaf in zip(plain.layernorm_backward(dy, x, gamma, 1e-5, dsum), leaves):
        assert torch.allclose(value, leaf.grad, atol=1e-12)
