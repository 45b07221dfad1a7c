"""Token embedding, LayerNorm's gradient, attention and its gradient against 64-bit plain forms (plain_text.py), within bounds
derived there."""
import itertools
import math

import pytest
import torch

import plain_text as plain

DTYPES = {"f16": torch.float16, "f32": torch.float32}


def _normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


# ---- token embedding ---------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("batch,length,vocab,dim,places,scale", [
    (2, 77, 1000, 768, 77, 1.0), (1, 1, 1, 1, 0, 3.0), (3, 5, 7, 33, 9, 0.5), (40, 61, 513, 40, 61, 25.5), (70, 77, 300, 24, 80, 1.0),
    (1, 64, 2, 8, 0, 1.0), (1, 65, 2, 8, 64 + 1, -2.0), (16, 64, 5000, 650, 64, 1.0), (25, 41, 5000, 650, 41, 1.0), (64, 16, 300, 12, 20, 1.0), (65, 15, 300, 12, 20, 1.0),
    (1, 1024, 100, 1025, 0, 1.0), (1, 1024, 5, 1024, 0, 1.0), (3, 100, 2049, 4, 100, 1.0), (1, 700, 1, 20000, 0, 1.0), (100, 90, 70000, 8, 90, 1.0), (5, 0, 10, 16, 3, 1.0), (0, 4, 10, 16, 5, 1.0),
])
def test_token_embedding_and_its_gradient(msd, cuda, dtype, batch, length, vocab, dim, places, scale):
    t = DTYPES[dtype]
    gen = torch.Generator().manual_seed(batch * 1000 + length)
    ids = (torch.rand((batch, length), generator=gen) ** 3 * vocab).long().clamp_(0, vocab - 1)
    if ids.numel() > 10:  # a token that is most of the text, and some that are in no table
        ids[:, length // 3:] = vocab - 1
        ids.view(-1)[3], ids.view(-1)[5] = -1, vocab
    table, dy = _normal(1, vocab, dim).to(t), _normal(3, batch, length, dim).to(t)
    positions = _normal(2, places, dim).to(t) if places else None
    y = msd.token_embedding(ids.to(cuda), table.to(cuda), None if positions is None else positions.to(cuda), scale)
    plain.check(y, plain.embedding(ids, table, positions, scale), "y")
    got = msd.token_embedding_backward(dy.to(cuda), ids.to(cuda), vocab, places, scale)
    again = msd.token_embedding_backward(dy.to(cuda), ids.to(cuda), vocab, places, scale)
    want = plain.embedding_backward(dy, ids, vocab, places, scale)
    plain.check(got[0], want[0], "dtable")
    assert torch.equal(got[0], again[0])
    if places:
        plain.check(got[1], want[1], "dpositions")
        assert torch.equal(got[1], again[1])
    else:
        assert got[1] is None


@pytest.mark.gpu
def test_token_embedding_takes_unaligned_tables(msd, cuda):
    table = _normal(1, 101 * 24 + 1).half().to(cuda)[1:].view(101, 24)
    ids = torch.arange(101, device=cuda)
    assert torch.equal(msd.token_embedding(ids, table), table)


# ---- LayerNorm's gradient ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,dim", [
    (154, 768), (1, 1), (3, 5), (7, 64), (33, 320), (1000, 40), (17, 1280), (9, 2048), (5, 4096), (300, 777), (2, 4099), (3, 9000), (2, 8192), (5000, 8), (129, 256),
    (70, 384), (70, 392), (70, 512), (70, 776), (40, 1024), (40, 1536), (40, 1544), (9, 6152), (40, 1100), (9, 2049),
])
@pytest.mark.parametrize("add", [False, True])
def test_layernorm_gradient(msd, cuda, dtype, rows, dim, add):
    t = DTYPES[dtype]
    x = (_normal(1, rows, dim) * (0.5 + torch.rand(dim)) + 2).to(t)
    dy, gamma = _normal(2, rows, dim).to(t), 1 + 0.2 * _normal(3, dim)
    dsum = _normal(4, rows, dim).to(t) if add else None
    want = plain.layernorm_backward(dy, x, gamma, 1e-5, dsum)
    args = [a.to(cuda) if a is not None else None for a in (dy, x, gamma, dsum)]
    got = msd.layernorm_backward(args[0], args[1], args[2], 1e-5, args[3])
    for g, w, what in zip(got, want, ("dx", "dgamma", "dbeta")):
        plain.check(g, w, what)
    again = msd.layernorm_backward(args[0], args[1], args[2], 1e-5, args[3])
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # in place of dy, or of what comes back past the norm; without the sums over rows
    for place in (0, 3) if add else (0,):
        other = [a.clone() if a is not None else None for a in args]
        dx, dgamma, dbeta = msd.layernorm_backward(other[0], other[1], other[2], 1e-5, other[3], affine=False, out=other[place])
        assert dx is other[place] and dgamma is None and dbeta is None and torch.equal(dx, got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_layernorm_gradient_of_unaligned_rows_and_of_none(msd, cuda, dtype):
    t = DTYPES[dtype]
    dy, x, gamma = _normal(1, 50 * 64 + 1).to(t)[1:].view(50, 64), _normal(2, 50, 64).to(t), _normal(3, 64)
    want = plain.layernorm_backward(dy, x, gamma, 1e-5, None)
    shifted = _normal(1, 50 * 64 + 1).to(t).to(cuda)[1:].view(50, 64)
    for g, w in zip(msd.layernorm_backward(shifted, x.to(cuda), gamma.to(cuda)), want):
        plain.check(g, w)
    dx, dgamma, dbeta = msd.layernorm_backward(x[:0].to(cuda), x[:0].to(cuda), gamma.to(cuda))
    assert dx.shape == (0, 64) and not dgamma.any() and not dbeta.any() and dgamma.shape == (64,)


# ---- attention -------------------------------------------------------------------------------
def _pack(lengths, heads, kv_heads, dim, t, seed=0):
    nq, nk = sum(q for q, _ in lengths), sum(k for _, k in lengths)
    return ((1.5 * _normal(seed, nq, heads, dim)).to(t), _normal(seed + 1, nk, kv_heads, dim).to(t), _normal(seed + 2, nk, kv_heads, dim).to(t),
            _normal(seed + 3, nq, heads, dim).to(t))


def _offsets(counts, device):
    return torch.tensor([0] + list(itertools.accumulate(counts)), dtype=torch.int32, device=device)


LENGTHS = [
    [(77, 77), (77, 77)],
    [(1, 1)], [(1, 300)], [(5, 3)], [(3, 5)],
    [(1, 700), (2, 64), (0, 5), (4, 0), (130, 65), (33, 33), (64, 64), (65, 129)],
    [(300, 20), (20, 300)],
    [(257, 257), (1, 1), (31, 31)],
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (6, 2, 128), (4, 1, 40), (3, 3, 33), (2, 1, 1), (8, 1, 80)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda l: "-".join("%dx%d" % p for p in l))
def test_attention_and_its_gradient(msd, cuda, dtype, causal, heads, kv_heads, dim, lengths):
    t, scale = DTYPES[dtype], 1 / math.sqrt(dim)
    q, k, v, dout = _pack(lengths, heads, kv_heads, dim, t)
    want = plain.attention(q, k, v, causal, scale, dout, lengths)
    offsets, offsets_k = _offsets([a for a, _ in lengths], cuda), _offsets([b for _, b in lengths], cuda)
    d = [x.to(cuda) for x in (q, k, v, dout)]
    out, kept = msd.attention_kept(d[0], d[1], d[2], causal, None, offsets, offsets_k)
    plain.check(out, want[0], "out")
    assert torch.equal(out, msd.attention(d[0], d[1], d[2], causal, scale, offsets, offsets_k))
    grads = msd.attention_backward(d[3], kept)
    for g, w, what in zip(grads, want[1:], ("dq", "dk", "dv")):
        plain.check(g, w, what)
    assert all(torch.equal(a, b) for a, b in zip(grads, msd.attention_backward(d[3], kept)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("layout", ["fused", "heads first", "unaligned"])
def test_attention_of_views(msd, cuda, dtype, layout):
    """Views of one projection, [batch, heads, rows, dim] memory, rows that begin at odd elements: the same bits as dense tensors."""
    t, b, n, heads, dim = DTYPES[dtype], 2, 70, 4, 64
    dense = [_normal(i, b, n, heads, dim).to(t).to(cuda) for i in range(4)]
    if layout == "fused":
        q, k, v = torch.cat(dense[:3], dim=2).split(heads, dim=2)
        dout = dense[3]
        grads_out = torch.empty(b, n, 3 * heads, dim, dtype=t, device=cuda).split(heads, dim=2)
    elif layout == "heads first":
        q, k, v, dout = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in dense)
        grads_out = [torch.empty(b, heads, n, dim, dtype=t, device=cuda).transpose(1, 2) for _ in range(3)]
    else:
        def odd(x):
            whole = torch.empty(x.numel() + 1, dtype=t, device=cuda)
            whole[1:] = x.flatten()
            return whole[1:].view(x.shape)
        q, k, v, dout = (odd(x) for x in dense)
        grads_out = None
    out, kept = msd.attention_kept(q, k, v, True)
    dense_out, dense_kept = msd.attention_kept(*dense[:3], True)
    assert torch.equal(out, dense_out) and torch.equal(kept.lse, dense_kept.lse)
    got, want = msd.attention_backward(dout, kept, grads_out), msd.attention_backward(dense[3], dense_kept)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_long_sequences_of_few_rows_are_cut_and_joined(msd, cuda, dtype):
    lengths = [(1, 5001), (3, 900), (1, 0), (2, 7000)]
    q, k, v, _ = _pack(lengths, 8, 2, 128, DTYPES[dtype])
    want = plain.attention(q, k, v, True, 0.1, None, lengths)
    offsets, offsets_k = _offsets([a for a, _ in lengths], cuda), _offsets([b for _, b in lengths], cuda)
    out = msd.attention(q.to(cuda), k.to(cuda), v.to(cuda), True, 0.1, offsets, offsets_k)
    plain.check(out, want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_what_a_row_does_not_see_has_no_part_in_it(msd, cuda, dtype, value):
    """Odd values at one position: rows in front of it (and the other sequence) keep their bits, in the gradient too."""
    t, n, at = DTYPES[dtype], 100, 45
    q, k, v, dout = (x.to(cuda) for x in _pack([(n, n), (40, 40)], 2, 1, 64, t))
    offsets = _offsets([n, 40], cuda)

    def run(q, k, v, dout):
        out, kept = msd.attention_kept(q, k, v, True, None, offsets)
        return (out,) + msd.attention_backward(dout, kept)

    clean = run(q, k, v, dout)
    for which in range(3):
        bad = [q.clone(), k.clone(), v.clone(), dout.clone()]
        bad[which][at] = value
        if which == 0:
            bad[3][at] = value
        got = run(*bad)
        rows = list(range(at)) + list(range(n, n + 40))
        if which == 0:  # a row's own values reach the keys that it sees, and itself
            assert torch.equal(got[0][rows + list(range(at + 1, n))], clean[0][rows + list(range(at + 1, n))])
            assert torch.equal(got[1][rows], clean[1][rows])
            later = list(range(at + 1, n + 40))
            assert torch.equal(got[2][later], clean[2][later]) and torch.equal(got[3][later], clean[3][later])
        else:  # a key's reach the rows from it on
            assert torch.equal(got[0][rows], clean[0][rows]) and torch.equal(got[1][rows], clean[1][rows])
            assert not torch.isfinite(got[0][at:n].float()).all(dim=-1).any()


@pytest.mark.gpu
def test_visible_infinities_reach_the_rows_that_see_them(msd, cuda):
    q, k, v, _ = (x.to(cuda) for x in _pack([(40, 40)], 1, 1, 64, torch.float16))
    v[7, 0, 3], v[9, 0, 4] = math.inf, -math.inf
    out = msd.attention(q, k, v, True, None, _offsets([40], cuda))
    assert (out[7:, 0, 3] == math.inf).all() and (out[9:, 0, 4] == -math.inf).all()
    assert torch.isfinite(out[:7]).all() and torch.isfinite(out[:, :, 5:]).all()


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_stay_as_they_were(msd, cuda):
    q, k, v, dout = (x.to(cuda) for x in _pack([(90, 90)], 2, 2, 64, torch.float16))
    offsets = torch.tensor([3, 20, 20, 61], dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 7.0)
    kept = msd.attention_kept(q, k, v, True, None, offsets, out=out)[1]
    grads = msd.attention_backward(dout, kept, tuple(torch.full_like(x, 7.0) for x in (q, k, v)))
    for x in (out,) + grads:
        assert (x[:3] == 7).all() and (x[61:] == 7).all() and not (x[3:61] == 7).all(dim=-1).any()
    few = torch.tensor([1, 2], dtype=torch.int32, device=cuda)  # (cut into parts and joined)
    many_k, many_v = (_normal(i, 6000, 2, 64).half().to(cuda) for i in (5, 6))
    out = msd.attention(q[:4], many_k, many_v, True, None, few, torch.tensor([0, 6000], dtype=torch.int32, device=cuda),
                        out=torch.full_like(q[:4], 7.0))
    assert (out[0] == 7).all() and (out[2:] == 7).all() and not (out[1] == 7).any()


@pytest.mark.gpu
def test_offsets_beyond_the_tensors_are_cut_off(msd, cuda):
    q, k, v, dout = (x.to(cuda) for x in _pack([(50, 50)], 2, 2, 64, torch.float16))
    bad = torch.tensor([-5, 30, 900], dtype=torch.int32, device=cuda)
    good = torch.tensor([0, 30, 50], dtype=torch.int32, device=cuda)
    got, kept = msd.attention_kept(q, k, v, True, None, bad)
    want, kept_good = msd.attention_kept(q, k, v, True, None, good)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(msd.attention_backward(dout, kept), msd.attention_backward(dout, kept_good)))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-4, 1.0, 3e3])
def test_float16_gradients_keep_their_digits_at_any_size(msd, cuda, size):
    lengths = [(200, 200)]
    q, k, v, dout = _pack(lengths, 2, 1, 64, torch.float16)
    dout = (dout * size).half()
    want = plain.attention(q, k, v, False, 0.125, dout, lengths)
    d = [x.to(cuda) for x in (q, k, v, dout)]
    kept = msd.attention_kept(d[0], d[1], d[2], False, 0.125, _offsets([200], cuda))[1]
    for g, w in zip(msd.attention_backward(d[3], kept), want[1:]):
        plain.check(g, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal,lengths", [(False, [(2100, 77)]), (True, [(900, 900)]), (False, [(1500, 20), (0, 5), (3, 0), (700, 130)]),
                                            (False, [(3, 2500)]), (True, [(2, 1500), (0, 4), (9, 700), (5, 0)])])
def test_gradients_of_few_keys_and_of_few_rows(msd, cuda, dtype, causal, lengths):
    """Few keys and many rows, few rows and many keys: the many are cut into parts that are added afterwards."""
    q, k, v, dout = _pack(lengths, 4, 2, 48, DTYPES[dtype])
    want = plain.attention(q, k, v, causal, 0.2, dout, lengths)
    offsets, offsets_k = _offsets([a for a, _ in lengths], cuda), _offsets([b for _, b in lengths], cuda)
    d = [x.to(cuda) for x in (q, k, v, dout)]
    kept = msd.attention_kept(d[0], d[1], d[2], causal, 0.2, offsets, offsets_k)[1]
    grads = msd.attention_backward(d[3], kept)
    for g, w, what in zip(grads, want[1:], ("dq", "dk", "dv")):
        plain.check(g, w, what)
    if len(lengths) == 1:  # the same as a dense batch of one
        dense = [x[None] for x in d]
        kept = msd.attention_kept(dense[0], dense[1], dense[2], causal, 0.2)[1]
        for g, w in zip(msd.attention_backward(dense[3], kept), grads):
            plain.check(g[0], (w.cpu().double(), 2 * want[1:][[x is w for x in grads].index(True)][1]))
