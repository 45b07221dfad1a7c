"""LayerNorm's gradient, attention and its gradient at the ends of what their calls allow."""
import ctypes
import math

import pytest
import torch

import plain_text as plain
from test_gpu_text_training import DTYPES, _normal, _offsets, _pack
from test_gpu_torch_calls import _General

pytestmark = pytest.mark.gpu


# ---- LayerNorm's gradient ----------------------------------------------------------------------
# (rows that are no multiple of what a workgroup has at a time: 16, 8 or 4 of them by vectors, 4 by single values)
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,dim", [(1, 64), (17, 64), (1, 320), (19, 400), (33, 640), (5, 1000), (1, 77), (6, 777), (154, 768), (3, 2048), (2, 1100)])
@pytest.mark.parametrize("add", [False, True])
def test_layernorm_gradient_without_eps(msd, cuda, dtype, rows, dim, add):
    t = DTYPES[dtype]
    x, dy, gamma = (2 * _normal(1, rows, dim) + 1).to(t), _normal(2, rows, dim).to(t), 1 + 0.2 * _normal(3, dim)
    dsum = _normal(4, rows, dim).to(t) if add else None
    got = msd.layernorm_backward(dy.to(cuda), x.to(cuda), gamma.to(cuda), 0.0, None if dsum is None else dsum.to(cuda))
    for g, w, what in zip(got, plain.layernorm_backward(dy, x, gamma, 0.0, dsum), ("dx", "dgamma", "dbeta")):
        plain.check(g, w, what)


# ---- packed sequences ----------------------------------------------------------------------------
@pytest.mark.parametrize("counts,counts_k", [([], [6]), ([], [2, 3, 1]), ([6], []), ([3, 3], [6]), ([6], [3, 3])])
def test_offsets_of_different_lengths_are_refused(msd, cuda, monkeypatch, counts, counts_k):
    """Also where one of them has no sequence at all."""
    q, k = torch.ones(6, 4, 16, device=cuda), torch.ones(6, 2, 16, device=cuda)
    o, ok = _offsets(counts, cuda), _offsets(counts_k, cuda)
    kept = msd.attention_kept(q, k, k, offsets=_offsets([6], cuda))[1]._replace(offsets=o, offsets_k=ok)
    for native in (msd._bind_native_text(), _General()):
        monkeypatch.setattr(msd, "_native_text", native)
        for call in (lambda: msd.attention(q, k, k, offsets=o, offsets_k=ok), lambda: msd.attention_kept(q, k, k, offsets=o, offsets_k=ok),
                     lambda: msd.attention_backward(q, kept)):
            with pytest.raises(msd.MsdError):
                call()


def test_offsets_of_one_element(msd, cuda):
    """No sequence: every row stays as it was."""
    q, k = torch.ones(6, 4, 16, device=cuda), torch.ones(5, 2, 16, device=cuda)
    none = _offsets([], cuda)
    out, kept = msd.attention_kept(q, k, k, offsets=none, offsets_k=none, out=torch.full_like(q, 3.0))
    grads = msd.attention_backward(q, kept, tuple(torch.full_like(t, 3.0) for t in (q, k, k)))
    assert all(bool((t == 3).all()) for t in (out,) + grads)


# ---- workspaces ------------------------------------------------------------------------------------
def _backward(msd, dout, kept, more, causal):
    """msd_attention_backward of dense tensors with `more` bytes of workspace than it asks for."""
    lib, (q, k, v) = msd.load_library(), (kept.q, kept.k, kept.v)
    code = {torch.float32: msd.DTYPE_F32, torch.float16: msd.DTYPE_F16}[q.dtype]
    sizes = (q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3])
    need = ctypes.c_size_t(0)
    assert lib.msd_attention_workspace(*sizes, 0, 1, code, ctypes.byref(need)) == 0
    workspace = torch.empty(need.value + more, dtype=torch.uint8, device=q.device)
    grads = [torch.full_like(t, 9.0) for t in (q, k, v)]
    rc = lib.msd_attention_backward(*[t.data_ptr() if t is not None else None for t in (dout, q, k, v, kept.out, kept.lse, kept.rest, *grads)], None, None,
                                    *sizes, None, kept.scale, int(causal), code, workspace.data_ptr(), workspace.numel(),
                                    torch.cuda.current_stream().cuda_stream)
    return rc, grads


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows,keys", [(1024, 0), (0, 1024), (600, 600), (2000, 40), (3, 2500)])
@pytest.mark.parametrize("more", [8, 1 << 24])
def test_more_workspace_than_needed(msd, cuda, dtype, causal, rows, keys, more):
    """Also where one side has no rows: the other's gradients are zeros."""
    t = DTYPES[dtype]
    q, k, v, dout = (_normal(i, 1, n, h, 40).to(t).to(cuda) for i, (n, h) in enumerate([(rows, 4), (keys, 2), (keys, 2), (rows, 4)]))
    kept = msd.attention_kept(q, k, v, causal)[1]
    rc, grads = _backward(msd, dout, kept, more, causal)
    assert rc == 0
    want = msd.attention_backward(dout, kept)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    if rows == 0 or keys == 0:
        assert not any(bool(g.any()) for g in grads)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("native", [False, True])
def test_a_gradient_without_the_mask_takes_its_own_bytes(msd, cuda, monkeypatch, dtype, native):
    t = DTYPES[dtype]
    q, k, v, dout = (_normal(i, 8, 1500, h, 64).to(t).to(cuda) for i, h in enumerate((8, 4, 4, 8)))
    monkeypatch.setattr(msd, "_native_text", msd._bind_native_text() if native else _General())
    peak = {}
    for causal in (True, False):
        kept = msd.attention_kept(q, k, v, causal)[1]
        rc, want = _backward(msd, dout, kept, 0, causal)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        grads = msd.attention_backward(dout, kept)
        peak[causal] = torch.cuda.max_memory_allocated() - before - sum(g.numel() * g.element_size() for g in grads)
        assert rc == 0 and all(torch.equal(a, b) for a, b in zip(grads, want))
        del kept, grads, want
    parts = 2 * 2 * 4 * k.numel()  # two parts of dk and dv in float32, under the mask alone
    assert peak[True] >= parts and peak[False] <= parts / 2


# ---- gradients that are zero in whole tiles ----------------------------------------------------------
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows,keys", [(264, 1000), (700, 1000)])
def test_rows_without_a_gradient_take_no_digits_from_the_others(msd, cuda, causal, dim, rows, keys):
    """The last 64 rows are left out of the loss.  Score gradients are near 10^-11 (float16's least step is 6 10^-8), large queries bring
    those of the keys back to 10^-3."""
    q, k, v, dout = _pack([(rows, keys)], 2, 1, dim, torch.float16)
    q, k, v = (q * 600).half(), (k * 2.0 ** -24).half(), (v * 0.01).half()
    dout = (dout * 1e-7).half()
    dout[-64:] = 0
    want = plain.attention(q, k, v, causal, 2000.0, dout, [(rows, keys)])
    d = [x[None].to(cuda) for x in (q, k, v, dout)]
    kept = msd.attention_kept(d[0], d[1], d[2], causal, 2000.0)[1]
    for g, w, what in zip(msd.attention_backward(d[3], kept), want[1:], ("dq", "dk", "dv")):
        plain.check(g[0], w, what)


# ---- keys that no row sees -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_of_sequences_without_rows(msd, cuda, dtype, causal, dim):
    """Their gradients are zeros, and the sequences between them (whose workgroups run where theirs have been) have theirs."""
    lengths = [(0, 500), (130, 130)] * 8 + [(0, 1000)]
    q, k, v, dout = _pack(lengths, 4, 2, dim, DTYPES[dtype])
    want = plain.attention(q, k, v, causal, 0.1, dout, lengths)
    o, ok = _offsets([a for a, _ in lengths], cuda), _offsets([b for _, b in lengths], cuda)
    out, kept = msd.attention_kept(q.to(cuda), k.to(cuda), v.to(cuda), causal, 0.1, o, ok)
    grads = msd.attention_backward(dout.to(cuda), kept)
    for g, w, what in zip((out,) + grads, want, ("out", "dq", "dk", "dv")):
        plain.check(g, w, what)
    for g in grads[1:]:
        assert not g[:500].any() and not g[-1000:].any()


@pytest.mark.parametrize("count", [0, 1, 2, 4, 5])
def test_gradients_into_another_number_of_tensors_are_refused(msd, cuda, count):
    q, k = torch.ones(1, 6, 4, 16, device=cuda), torch.ones(1, 6, 4, 16, device=cuda)
    kept = msd.attention_kept(q, k, k)[1]
    packed = msd.attention_kept(q[0], k[0], k[0], offsets=_offsets([6], cuda))[1]
    for case, like in ((kept, q), (packed, q[0])):
        with pytest.raises(msd.MsdError):
            msd.attention_backward(like, case, tuple(torch.empty_like(like) for _ in range(count)))


# ---- parts of rows that are no whole vectors ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [33, 127])
@pytest.mark.parametrize("lengths", [[(3, 2500)], [(2, 1500), (0, 4), (9, 700), (5, 0)], [(1500, 20)]], ids=lambda l: "-".join("%dx%d" % p for p in l))
def test_parts_of_an_odd_number_of_columns(msd, cuda, dtype, causal, dim, lengths):
    """Keys in parts for dq (and out), rows in parts for dk and dv."""
    q, k, v, dout = _pack(lengths, 4, 2, dim, DTYPES[dtype])
    want = plain.attention(q, k, v, causal, 0.2, dout, lengths)
    o, ok = _offsets([a for a, _ in lengths], cuda), _offsets([b for _, b in lengths], cuda)
    out, kept = msd.attention_kept(q.to(cuda), k.to(cuda), v.to(cuda), causal, 0.2, o, ok)
    for g, w, what in zip((out,) + msd.attention_backward(dout.to(cuda), kept), want, ("out", "dq", "dk", "dv")):
        plain.check(g, w, what)


# ---- the largest scores ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows,keys", [(70, 200), (2, 2000), (600, 600)])
def test_scores_of_the_largest_size(msd, cuda, dtype, dim, rows, keys):
    """Scores up to 2^21, 1024 apart: each row has one key.  Out is its values, off by the weight's rounding (float16) and the result's; the
    gradient's weights are off by 2^-23 times the score, 1/4 of themselves."""
    t, gen = DTYPES[dtype], torch.Generator().manual_seed(rows)
    q, k, v, dout = _pack([(rows, keys)], 1, 1, dim, t, 5)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q[:, 0, 1] = torch.where(torch.rand(rows, generator=gen) < 0.5, -1024.0, 1024.0).to(t)
    k[:, 0, 1] = (torch.randperm(2 * keys, generator=gen)[:keys] - keys).clamp(-2047, 2047).to(t)
    k[3, 0, 1], k[keys - 2, 0, 1] = 2048.0, -2048.0
    d = [x[None].to(cuda) for x in (q, k, v, dout)]
    out, kept = msd.attention_kept(d[0], d[1], d[2], False, 1.0)
    best = torch.where(q[:, 0, 1] > 0, 3, keys - 2)
    off = 2 * plain.HALF[t] + 2.0 ** -20
    assert bool(((out[0, :, 0].cpu().double() - v[best, 0].double()).abs() <= off * v[best, 0].double().abs() + plain.TINY[t]).all())
    dq, dk, dv = msd.attention_backward(d[3], kept)
    want = torch.zeros(keys, dim, dtype=torch.float64).index_add_(0, best, dout[:, 0].double())
    size = torch.zeros(keys, dim, dtype=torch.float64).index_add_(0, best, dout[:, 0].double().abs())
    assert bool(((dv[0, :, 0].cpu().double() - want).abs() <= 0.26 * size + plain.TINY[t]).all())
    assert bool(torch.isfinite(dq).all()) and bool(torch.isfinite(dk).all())


# ---- infinities that rows see -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("at", [5, 70, 149])
def test_infinities_without_weight_leave_nothing_finite(msd, cuda, dtype, causal, at):
    """A key far below the others: its infinite value times a weight of zero is an infinity or NaN in that column, and nowhere else."""
    t, n = DTYPES[dtype], 150
    q, k, v, _ = _pack([(n, n)], 1, 1, 64, t, 11)
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[at, 0, 0] = -1000.0
    v[at, 0, 9] = math.inf
    out = msd.attention(*(x[None].to(cuda) for x in (q, k, v)), causal)[0, :, 0].cpu()
    sees = torch.arange(n) >= at if causal else torch.ones(n, dtype=torch.bool)
    assert not torch.isfinite(out[sees, 9]).any() and torch.isfinite(out[~sees, 9]).all()
    assert torch.isfinite(out[:, [c for c in range(64) if c != 9]]).all()
