"""Token embedding, LayerNorm's gradient and attention as they are used: together, captured, on other streams, with memory beyond 2^31
values, with random sizes; gradients against differences; native calls against the general path; refusals of the package."""
import itertools
import math

import pytest
import torch

import plain_text as plain
from test_gpu_text_training import DTYPES, _normal, _offsets, _pack
from test_gpu_torch_calls import _General, _Recorder

pytestmark = pytest.mark.gpu


# ---- together ----------------------------------------------------------------------------------
HEADS, DIM = 2, 64
WIDTH = 3 * HEADS * DIM


def _text(t, batch, length, vocab, device):
    gen = torch.Generator().manual_seed(batch * 100 + length)
    host = {"ids": torch.randint(0, vocab, (batch, length), generator=gen), "table": _normal(1, vocab, WIDTH).to(t),
            "places": (0.1 * _normal(2, length + 3, WIDTH)).to(t), "g1": 1 + 0.2 * _normal(3, WIDTH), "b1": 0.1 * _normal(4, WIDTH),
            "g2": 1 + 0.2 * _normal(5, HEADS * DIM), "b2": 0.1 * _normal(6, HEADS * DIM), "dn": _normal(7, batch, length, HEADS * DIM).to(t)}
    return host, {k: v.to(device) for k, v in host.items()}


def _step(msd, d):
    """Embedding, norm, causal attention over views of it, a residual and a norm; and all gradients."""
    batch, length = d["ids"].shape
    r = {"x": msd.token_embedding(d["ids"], d["table"], d["places"])}
    r["y"] = msd.layernorm(r["x"], d["g1"], d["b1"])
    q, k, v = r["y"].view(batch, length, 3 * HEADS, DIM).split(HEADS, dim=2)
    r["out"], kept = msd.attention_kept(q, k, v, causal=True)
    r["sum"], r["n"] = msd.add_layernorm(r["out"].view(batch, length, -1), r["x"][..., :HEADS * DIM].contiguous(), d["g2"], d["b2"])
    r["dsum"], r["dg2"], r["db2"] = msd.layernorm_backward(d["dn"], r["sum"], d["g2"])
    r["dy"] = torch.empty_like(r["y"])
    msd.attention_backward(r["dsum"].view(batch, length, HEADS, DIM), kept, r["dy"].view(batch, length, 3 * HEADS, DIM).split(HEADS, dim=2))
    past = torch.zeros_like(r["x"])
    past[..., :HEADS * DIM] = r["dsum"]
    r["dx"], r["dg1"], r["db1"] = msd.layernorm_backward(r["dy"], r["x"], d["g1"], 1e-5, past)
    r["dtable"], r["dplaces"] = msd.token_embedding_backward(r["dx"], d["ids"], d["table"].shape[0], d["places"].shape[0])
    return r


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("batch,length", [(2, 77), (1, 1), (5, 33)])
def test_a_text_block_and_its_gradients(msd, cuda, dtype, batch, length):
    """Each plain form starts from what the operator before it gave."""
    t = DTYPES[dtype]
    host, d = _text(t, batch, length, 100, cuda)
    dev = _step(msd, d)
    r = {k: v.cpu() for k, v in dev.items()}
    plain.check(dev["x"], plain.embedding(host["ids"], host["table"], host["places"], 1.0), "x")
    q, k, v = (x.reshape(-1, HEADS, DIM) for x in r["y"].view(batch, length, 3 * HEADS, DIM).split(HEADS, dim=2))
    want = plain.attention(q, k, v, True, DIM ** -0.5, r["dsum"].view(-1, HEADS, DIM), [(length, length)] * batch)
    plain.check(dev["out"].view(-1, HEADS, DIM), want[0], "out")
    grads = dev["dy"].view(batch, length, 3 * HEADS, DIM).split(HEADS, dim=2)
    for got, w, what in zip(grads, want[1:], ("dq", "dk", "dv")):
        plain.check(got.reshape(-1, HEADS, DIM), w, what)
    rows = batch * length
    for got, w, what in zip((dev["dsum"], dev["dg2"], dev["db2"]),
                            plain.layernorm_backward(host["dn"].view(rows, -1), r["sum"].view(rows, -1), host["g2"], 1e-5, None), ("dsum", "dg2", "db2")):
        plain.check(got.view(w[0].shape), w, what)
    past = torch.zeros(rows, WIDTH, dtype=t)
    past[:, :HEADS * DIM] = r["dsum"].view(rows, -1)
    for got, w, what in zip((dev["dx"], dev["dg1"], dev["db1"]),
                            plain.layernorm_backward(r["dy"].view(rows, -1), r["x"].view(rows, -1), host["g1"], 1e-5, past), ("dx", "dg1", "db1")):
        plain.check(got.view(w[0].shape), w, what)
    want = plain.embedding_backward(r["dx"], host["ids"], 100, length + 3, 1.0)
    plain.check(dev["dtable"], want[0], "dtable")
    plain.check(dev["dplaces"], want[1], "dplaces")


def test_captured_and_replayed_beside_eager_calls(msd, cuda):
    """Two graphs of the same operands on two streams, replayed at once, with eager work between: none shares a workspace."""
    _, d = _text(torch.float16, 3, 50, 100, cuda)
    _step(msd, d)
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            captured = _step(msd, d)
        graphs.append((graph, captured))
    for turn in range(4):
        d["ids"].copy_((d["ids"] * 7 + turn) % 100)
        d["table"].mul_(0.875)
        want = {k: v.clone() for k, v in _step(msd, d).items()}
        for _, captured in graphs:
            for x in captured.values():
                x.fill_(5.0)
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, captured in graphs:
            assert all(torch.equal(captured[k], want[k]) for k in want), turn


def test_cut_sequences_captured_and_replayed(msd, cuda):
    """The calls with parts (few rows and many keys; few keys and many rows) have workspaces, also in a graph."""
    q, k, v, dout = (x.to(cuda) for x in _pack([(2, 3000), (1500, 20)], 4, 2, 64, torch.float16))
    o, ok = _offsets([2, 1500], cuda), _offsets([3000, 20], cuda)
    one = [q[None, :2], k[None, :3000], v[None, :3000]]

    def run():
        out, kept = msd.attention_kept(q, k, v, False, None, o, ok)
        return (out, msd.attention(*one)) + msd.attention_backward(dout, kept)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for turn in range(4):
        q.mul_(0.9)
        want = [x.clone() for x in run()]
        for x in captured:
            x.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), turn


def test_calls_use_the_current_stream(msd, cuda):
    """Operands are written behind work that takes far longer than the host needs to reach the calls' launches."""
    stream = torch.cuda.Stream()
    ids, g = torch.zeros(2, 5, dtype=torch.int64, device=cuda), torch.ones(64, device=cuda)
    with torch.cuda.stream(stream):
        big, x = torch.empty(1 << 28, device=cuda), torch.full((10, 64), -1.0, device=cuda)
        for k in range(1, 4):
            x.fill_(-1.0)
            heads = x.view(2, 5, 1, 64)
            stream.synchronize()
            for _ in range(16):
                big.fill_(float(k))
            x.fill_(float(k))
            waits = not stream.query()
            y = msd.token_embedding(ids, x)
            dtable, _ = msd.token_embedding_backward(x.view(2, 5, 64), ids, 3)
            out, kept = msd.attention_kept(heads, heads, heads)
            dv = msd.attention_backward(heads, kept)[2]
            dbeta = msd.layernorm_backward(x, x, g)[2]
            assert waits and bool((y == k).all()) and bool((dtable[0] == 10.0 * k).all()) and not dtable[1:].any()
            assert bool((out - k).abs().max() <= 1e-5) and bool((dv - k).abs().max() <= 1e-5) and bool((dbeta == 10.0 * k).all())


def test_two_threads_at_once(msd, cuda):
    """Each with operands and a stream of its own: the results of the calls one after another."""
    import threading
    texts = [_text(torch.float16, 2 + i, 40 + 30 * i, 100, cuda)[1] for i in range(2)]
    want = [{k: v.clone() for k, v in _step(msd, d).items()} for d in texts]
    torch.cuda.synchronize()
    wrong, begin = [], threading.Barrier(2, timeout=60)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            begin.wait()
            with torch.cuda.stream(stream):
                got = [_step(msd, texts[i]) for _ in range(20)]
            stream.synchronize()
            wrong.extend((i, k) for r in got for k in r if not torch.equal(r[k], want[i][k]))
        except Exception as e:  # (to the test's own thread)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not wrong and not any(t.is_alive() for t in threads)


# ---- memory beyond 2^31 values ---------------------------------------------------------------------
@pytest.mark.parametrize("shift", [0, 1], ids=["aligned", "unaligned"])
def test_attention_over_a_cache_beyond_32_bits(msd, cuda, shift):
    """Keys and values are heads of a cache of 2.3 * 10^9 values: the bits of a call with dense tensors."""
    rows, wide = 70001, 256
    cache = torch.empty(rows * wide * 128 + 1, dtype=torch.float16, device=cuda)[shift:shift + rows * wide * 128].view(rows, wide, 128)
    k, v = cache[:, 1:3], cache[:, 254:256]
    k.copy_(torch.randn(rows, 2, 128, device=cuda))
    v.copy_(torch.randn(rows, 2, 128, device=cuda))
    q, dout = torch.randn(2, 5, 4, 128, device=cuda).half().unbind(0)
    o, ok = _offsets([2, 3], cuda), _offsets([1000, 69001], cuda)
    out, kept = msd.attention_kept(q, k, v, True, None, o, ok)
    dense, dense_kept = msd.attention_kept(q, k.contiguous(), v.contiguous(), True, None, o, ok)
    assert torch.equal(out, dense) and torch.equal(kept.lse, dense_kept.lse)
    dcache = torch.empty_like(cache)
    grads = msd.attention_backward(dout, kept, (torch.empty_like(q), dcache[:, 1:3], dcache[:, 254:256]))
    assert all(torch.equal(a, b) for a, b in zip(grads, msd.attention_backward(dout, dense_kept)))
    tail = slice(69990, 70001)
    want = plain.attention(q[2:].cpu(), k[1000:].cpu(), v[1000:].cpu(), True, 128 ** -0.5, dout[2:].cpu(), [(3, 69001)])
    plain.check(out[2:], want[0])
    plain.check(grads[1][tail], tuple(x[-11:] for x in want[2]))


def test_queries_beyond_32_bits(msd, cuda):
    """140000 rows of 128 heads of 128: only the last 40 have an incoming gradient."""
    rows, heads, dim, keys = 140000, 128, 128, 16
    q = torch.randn(1, 1, heads, dim, device=cuda).half().expand(1, rows, heads, dim).contiguous()
    k, v = (torch.randn(1, keys, 4, dim, device=cuda).half() for _ in range(2))
    q[0, -40:] = torch.randn(40, heads, dim, device=cuda).half()
    out, kept = msd.attention_kept(q, k, v)
    dout = torch.zeros_like(q)
    dout[0, -40:] = torch.randn(40, heads, dim, device=cuda).half()
    last = [x[0, -40:].cpu() for x in (q, dout)]
    want = plain.attention(last[0], k[0].cpu(), v[0].cpu(), False, dim ** -0.5, last[1], [(40, keys)])
    plain.check(out[0, -40:], want[0])
    assert bool((out[0, :-40] == out[0, :1]).all())
    dq, dk, dv = msd.attention_backward(dout, kept)
    plain.check(dq[0, -40:], want[1])
    assert not dq[0, :-40].any()
    plain.check(dk[0], want[2])
    plain.check(dv[0], want[3])


def test_embedding_and_layernorm_beyond_32_bits(msd, cuda):
    vocab, dim = 2200000, 1000
    table = torch.empty(vocab, dim, dtype=torch.float16, device=cuda)
    ids = torch.tensor([[vocab - 1, 0, vocab - 2], [vocab - 1, vocab // 2, 5]], device=cuda)
    table[ids.flatten()] = torch.randn(6, dim, device=cuda).half()
    assert torch.equal(msd.token_embedding(ids, table), table[ids])
    dy = torch.randn(2, 3, dim, device=cuda).half()
    dtable, _ = msd.token_embedding_backward(dy, ids, vocab)
    assert torch.equal(dtable[vocab - 2], dy[0, 2]) and torch.equal(dtable[5], dy[1, 2]) and torch.equal(dtable[vocab // 2], dy[1, 1])
    assert torch.equal(dtable[vocab - 1], (dy[0, 0].float() + dy[1, 0].float()).half())
    assert int(torch.count_nonzero(dtable.any(dim=1))) == 5
    del dtable

    x, g = table, torch.rand(dim, device=cuda) + 0.5  # (as rows of a norm)
    x.normal_()
    d = torch.zeros_like(x)
    d[-20:] = torch.randn(20, dim, device=cuda).half()
    dx, dgamma, dbeta = msd.layernorm_backward(d, x, g)
    want = plain.layernorm_backward(d[-20:].cpu(), x[-20:].cpu(), g.cpu(), 1e-5, None)
    plain.check(dx[-20:], want[0])
    plain.check(dgamma, want[1])
    plain.check(dbeta, want[2])
    assert not dx[:-20].any()


# ---- random sizes ------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(40))
def test_attention_of_random_sizes(msd, cuda, seed):
    gen = torch.Generator().manual_seed(seed)

    def pick(*of):
        return of[int(torch.randint(0, len(of), (1,), generator=gen))]

    t, causal, kv_heads, group = pick(torch.float16, torch.float32), pick(False, True), pick(1, 2, 3), pick(1, 2, 3, 5, 8)
    dim = pick(64, 128, 32, 96, int(torch.randint(1, 129, (1,), generator=gen)))
    longest = pick(8, 100, 400)
    lengths = [tuple(int(x) for x in torch.randint(0, longest + 1, (2,), generator=gen)) for _ in range(pick(1, 2, 5))]
    if pick(False, True):
        lengths = [(a, a) for a, _ in lengths]
    scale = pick(1 / math.sqrt(dim), 0.02, 2.0)
    q, k, v, dout = _pack(lengths, group * kv_heads, kv_heads, dim, t, seed)
    want = plain.attention(q, k, v, causal, scale, dout, lengths)
    o, ok = _offsets([a for a, _ in lengths], cuda), _offsets([b for _, b in lengths], cuda)
    out, kept = msd.attention_kept(q.to(cuda), k.to(cuda), v.to(cuda), causal, scale, o, ok)
    plain.check(out, want[0], "out")
    for g, w, what in zip(msd.attention_backward(dout.to(cuda), kept), want[1:], ("dq", "dk", "dv")):
        plain.check(g, w, what)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
def test_log_sums(msd, cuda, dtype, causal):
    """lse is log2 of the weights' sum, within what its scores' float32 sums may be off (see plain_text)."""
    t, lq, lk, dim, scale = DTYPES[dtype], 70, 50, 40, 0.3
    q, k, v, _ = _pack([(lq, lk)], 2, 1, dim, t)
    _, kept = msd.attention_kept(*(x[None].to(cuda) for x in (q, k, v)), causal, scale)
    for h in range(2):
        score = torch.where(plain.visible(lq, lk, causal), scale * q[:, h].double() @ k[:, 0].double().t(), -math.inf)
        size = scale * (q[:, h].double().abs() @ k[:, 0].double().abs().t()).amax(1)
        want, got = torch.logsumexp(score, 1) / math.log(2), kept.lse[0, :, h].cpu().double()
        none = want == -math.inf
        assert torch.equal(got == -math.inf, none) and (not causal or int(none.sum()) == lq - lk)
        off = ((dim + 12) * size + (lk / 32 + 40) + 4 * want.abs().nan_to_num(0, 0, 0) + 4 * size) * plain.EPS / math.log(2)
        assert bool(((got - want).abs() <= off)[~none].all())


# ---- gradients against differences ---------------------------------------------------------------------
@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradients_against_differences(msd, cuda, causal):
    """Along a direction u, with 64-bit values on both sides: (L(x + hu) - L(x - hu)) / 2h is off by h^2 / 6 of the third derivative
    (1e-3 of the slope's scale at h = 1e-3 would be 1e-6) and 2^-52 L / h."""
    lengths, scale, h = [(30, 45), (3, 3)], 0.2, 1e-3
    q, k, v, dout = _pack(lengths, 4, 2, 32, torch.float32)
    o, ok = _offsets([30, 3], cuda), _offsets([45, 3], cuda)
    _, kept = msd.attention_kept(q.to(cuda), k.to(cuda), v.to(cuda), causal, scale, o, ok)
    grads = [g.cpu().double() for g in msd.attention_backward(dout.to(cuda), kept)]
    plain.HALF[torch.float64] = plain.TINY[torch.float64] = 0.0
    try:
        for n in range(3):
            u = _normal(50 + n, *(q, k, v)[n].shape).double()
            u /= u.norm()

            def loss(step):
                at = [x.double() for x in (q, k, v)]
                at[n] = at[n] + step * u
                return float((plain.attention(*at, causal, scale, None, lengths)[0][0] * dout.double()).sum())

            slope, wide = (loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)
            bound = plain.attention(q, k, v, causal, scale, dout, lengths)[1 + n][1]
            # (wide - slope is three times slope's own error)
            assert abs(float((grads[n] * u).sum()) - slope) <= float((bound * u.abs()).sum()) + abs(wide - slope) + 1e-11
    finally:
        del plain.HALF[torch.float64], plain.TINY[torch.float64]


def test_layernorm_gradient_against_differences(msd, cuda):
    rows, dim, h = 20, 70, 1e-3
    x, dy, gamma = _normal(1, rows, dim), _normal(2, rows, dim), 1 + 0.3 * _normal(3, dim)
    got = [g.cpu().double() for g in msd.layernorm_backward(dy.to(cuda), x.to(cuda), gamma.to(cuda))]
    bounds = [b for _, b in plain.layernorm_backward(dy, x, gamma, 1e-5, None)]
    at = [x.double(), gamma.double(), torch.zeros(dim, dtype=torch.float64)]
    for n in range(3):
        u = _normal(60 + n, *at[n].shape).double()
        u /= u.norm()

        def loss(step):
            a = [t + step * u if i == n else t for i, t in enumerate(at)]
            return float((torch.nn.functional.layer_norm(a[0], (dim,), a[1], a[2], 1e-5) * dy.double()).sum())

        slope, wide = (loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)
        assert abs(float((got[n] * u).sum()) - slope) <= float((bounds[n] * u.abs()).sum()) + abs(wide - slope) + 1e-11


# ---- views that lie between each other ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_gradients_as_views_of_one_projection_by_sequence(msd, cuda, dtype):
    """[batch, 3, heads, rows, dim] memory for the operands and for their gradients."""
    t, b, heads, n, dim = DTYPES[dtype], 3, 2, 37, 64
    whole = _normal(1, b, 3, heads, n, dim).to(t).to(cuda)
    q, k, v = (x.transpose(1, 2) for x in whole.unbind(1))
    dout = _normal(2, b, n, heads, dim).to(t).to(cuda)
    grads = torch.full_like(whole, 9.0)
    got = msd.attention_backward(dout, msd.attention_kept(q, k, v)[1], [x.transpose(1, 2) for x in grads.unbind(1)])
    want = msd.attention_backward(dout, msd.attention_kept(q.contiguous(), k.contiguous(), v.contiguous())[1])
    assert all(torch.equal(a, c) for a, c in zip(got, want)) and got[1].data_ptr() == grads[:, 1].data_ptr()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_broadcast_operands(msd, cuda, dtype):
    """One key sequence for a batch, one head for all: views with strides of zero.  Their gradients come back for every copy."""
    t = DTYPES[dtype]
    q, k = _normal(1, 1, 40, 1, 64).to(t).to(cuda), _normal(2, 1, 90, 2, 64).to(t).to(cuda)
    wide = [q.expand(3, 40, 4, 64), k.expand(3, 90, 2, 64), k.expand(3, 90, 2, 64)]
    out, kept = msd.attention_kept(*wide, True)
    dense, dense_kept = msd.attention_kept(*(x.contiguous() for x in wide), True)
    dout = _normal(3, 3, 40, 4, 64).to(t).to(cuda)
    assert torch.equal(out, dense)
    grads = msd.attention_backward(dout, kept)
    assert all(torch.equal(a, b) and a.is_contiguous() for a, b in zip(grads, msd.attention_backward(dout, dense_kept)))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rows_whose_scores_are_all_minus_infinity_give_zeros(msd, cuda, dtype):
    t = DTYPES[dtype]
    q, k, v = (_normal(i, 1, 70, 2, 64).to(t).to(cuda) for i in range(3))
    q[..., 0] = q[..., 0].abs() + 0.5
    k[:, :30, :, 0] = -math.inf  # (causal: rows 0 to 29 see no other keys)
    out, kept = msd.attention_kept(q, k, v, True)
    assert not out[:, :30].any() and bool((kept.lse[:, :30] == -math.inf).all())
    want = plain.attention(q[0, 30:].cpu(), k[0, 30:].cpu(), v[0, 30:].cpu(), True, 64 ** -0.5, None, [(40, 40)])
    plain.check(out[0, 30:], want[0])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("causal,dim", [(False, 64), (True, 64), (False, 128), (True, 128), (False, 40)])
def test_visible_infinities_are_those_of_the_formula(msd, cuda, dtype, causal, dim):
    """Keys of minus infinity have no weight, values of infinity reach all rows that see them; operands of few digits, whose products
    with infinities must not become NaN."""
    t, n = DTYPES[dtype], 150
    q, k, v, dout = _pack([(n, n)], 2, 2, dim, t, 3)
    q[..., 0], q[..., 1] = 1.0, 0.5
    k[20, 0, 0] = k[100, 0, 1] = -math.inf
    v[140, 1, 7], v[9, 1, 5] = math.inf, -math.inf
    d = [x[None].to(cuda) for x in (q, k, v)]
    out, kept = msd.attention_kept(*d, causal, 0.1)
    gone = k.clone()
    gone[[20, 100], 0] = 0
    rest = torch.arange(n) != 20
    rest &= torch.arange(n) != 100
    sees = plain.visible(n, n, causal) & rest
    score = torch.where(sees, 0.1 * q[:, 0].double() @ gone[:, 0].double().t(), -math.inf)
    want = torch.softmax(score, 1) @ v[:, 0].double()
    size = torch.softmax(score, 1) @ v[:, 0].double().abs()
    assert bool(((out[0, :, 0].cpu().double() - want).abs() <= 4 * plain.HALF[t] * size + 2000 * plain.EPS * size + 2.0 ** -24).all())
    row = torch.arange(n)
    up, down = out[0, :, 1, 7].cpu(), out[0, :, 1, 5].cpu()
    assert bool((up == math.inf)[(row >= 140) | torch.tensor(not causal)].all()) and bool((down == -math.inf)[(row >= 9) | torch.tensor(not causal)].all())
    if causal:
        assert torch.isfinite(up[:140]).all() and torch.isfinite(down[:9]).all()
    others = [c for c in range(dim) if c not in (5, 7)]
    assert torch.isfinite(out[0, :, 1][:, others]).all()
    # what the keys without weight give back is nothing, and the others' gradients are finite
    clean = d[2].clone()
    clean[0, 140, 1, 7] = clean[0, 9, 1, 5] = 0
    out, kept = msd.attention_kept(d[0], d[1], clean, causal, 0.1)
    dq, dk, dv = msd.attention_backward(dout[None].to(cuda), kept)
    assert not dv[0, [20, 100], 0].any() and not dk[0, [20, 100], 0].any()
    assert torch.isfinite(dk).all() and torch.isfinite(dv).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", [30.0, 1e-3])
def test_scores_of_any_size(msd, cuda, dtype, size):
    """Weights of one key alone, and all alike."""
    t, lengths = DTYPES[dtype], [(150, 150)]
    q, k, v, dout = _pack(lengths, 2, 1, 64, t, 9)
    q = (q * size).to(t)
    want = plain.attention(q, k, v, True, 0.5, dout, lengths)
    out, kept = msd.attention_kept(*(x[None].to(cuda) for x in (q, k, v)), True, 0.5)
    plain.check(out[0], want[0], "out")
    for g, w, what in zip(msd.attention_backward(dout[None].to(cuda), kept), want[1:], ("dq", "dk", "dv")):
        plain.check(g[0], w, what)


@pytest.mark.parametrize("count", [63, 64, 65, 1000])
def test_many_packed_sequences(msd, cuda, count):
    gen = torch.Generator().manual_seed(count)
    lengths = [(int(a), int(b)) for a, b in torch.randint(0, 9, (count, 2), generator=gen)]
    q, k, v, dout = _pack(lengths, 2, 1, 16, torch.float32, count)
    want = plain.attention(q, k, v, True, 0.25, dout, lengths)
    o, ok = _offsets([a for a, _ in lengths], cuda), _offsets([b for _, b in lengths], cuda)
    out, kept = msd.attention_kept(q.to(cuda), k.to(cuda), v.to(cuda), True, 0.25, o, ok)
    plain.check(out, want[0], "out")
    for g, w, what in zip(msd.attention_backward(dout.to(cuda), kept), want[1:], ("dq", "dk", "dv")):
        plain.check(g, w, what)


@pytest.mark.parametrize("dim", [20000, 100001])
def test_layernorm_gradient_of_long_rows(msd, cuda, dim):
    dy, x, gamma, dsum = _normal(1, 3, dim), _normal(2, 3, dim) + 1, 1 + 0.1 * _normal(3, dim), _normal(4, 3, dim)
    want = plain.layernorm_backward(dy, x, gamma, 1e-5, dsum)
    for g, w in zip(msd.layernorm_backward(dy.to(cuda), x.to(cuda), gamma.to(cuda), 1e-5, dsum.to(cuda)), want):
        plain.check(g, w)


# ---- native calls ---------------------------------------------------------------------------------------
def _cases(msd, cuda, half):
    gen = torch.Generator(device=cuda).manual_seed(6)
    t = torch.float16 if half else torch.float32

    def rnd(*shape):
        return torch.randn(shape, device=cuda, generator=gen).to(t)

    def floats(n):
        return torch.randn(n, device=cuda, generator=gen)

    ids = torch.randint(0, 30, (2, 9), device=cuda, generator=gen)
    table, places, g = rnd(30, 64), rnd(12, 64), floats(64)
    embeds = [(ids, table), (ids, table, places, 2.0), (ids, table, places, 1.0, rnd(2, 9, 64)), (ids[0], table, None), (ids, table, rnd(8, 64)),
              (ids.int(), table), (ids, table.double()), (ids, table, places.double()), (ids.cpu(), table), (ids, table.cpu()), (ids.t(), table),
              (ids[:0], table), (ids, table, places[:, :63]), (ids, table, None, 1), (ids, table, None, 1.0, rnd(2, 9, 63)), (ids, table[0]),
              (ids, torch.nn.Parameter(table), places), (ids, table[:0])]
    dy = rnd(2, 9, 64)
    backs = [(dy, ids, 30), (dy, ids, 30, 12, 0.5), (dy[0], ids[0], 40, 9), (dy, ids, 30, 8), (dy, ids[:1], 30), (dy, ids, -1), (dy.double(), ids, 30),
             (dy[:0], ids[:0], 30, 3), (dy, ids, 0), (dy, ids.int(), 30), (dy.cpu(), ids, 30), (dy.transpose(0, 1), ids.t(), 30), (dy, ids, 30, -3)]
    x = rnd(2, 9, 64)
    norms = [(dy, x, g), (dy, x, g, 1e-3, rnd(2, 9, 64)), (dy, x, g, 1e-5, None, False), (dy, x, g, 1e-5, None, True, rnd(2, 9, 64)), (dy, x[:1], g),
             (dy, x, g[:63]), (dy, x, g.to(torch.float64)), (dy, x.double(), g), (dy.double(), x.double(), g), (dy, x.cpu(), g), (dy[:0], x[:0], g),
             (dy, x, torch.nn.Parameter(g)), (dy, x, None), (dy, x, g, 1e-5, None, True, x)]
    q, k, v = rnd(2, 9, 4, 64), rnd(2, 7, 2, 64), rnd(2, 7, 2, 64)
    o = torch.tensor([0, 4, 9], dtype=torch.int32, device=cuda)
    ok = torch.tensor([0, 7, 7], dtype=torch.int32, device=cuda)
    fused = rnd(2, 9, 8, 64)
    attends = [(q, k, v), (q, k, v, True, 0.5), (q, k, v, True, None, None, None, rnd(2, 9, 4, 64)), (q[0], k[0], v[0], False, None, o, ok),
               (q[0], q[1], q[0], True, None, o), (q[0], k[0], v[0], False, None, o), (q[0], k[0], v[0]), (q, k, v, False, None, o), (q, k, v[:, :6]),
               (q, k[:1], v[:1]), (q, rnd(2, 7, 3, 64), rnd(2, 7, 3, 64)), (q, k.double(), v), (q.double(), k.double(), v.double()), (q.cpu(), k, v),
               (q[..., ::2], k[..., ::2], v[..., ::2]), (q, k, v, False, -1.0), (q, k, v, False, 0.5, None, None, q), (q, k, v, False, 0.5, None, None, q[:1]),
               (q[0], k[0], v[0], False, None, o.long(), ok), (q[0], k[0], v[0], False, None, o, ok[:2]), (q[:0], k[:0], v[:0]), (q[:, :0], k, v),
               (q, k[:, :0], v[:, :0]), tuple(fused.split((4, 2, 2), dim=2)), (q, k, v, 1), (q[0, 0], k[0, 0], v[0, 0]), (torch.nn.Parameter(q), k, v),
               (rnd(1, 3, 1, 129), rnd(1, 3, 1, 129), rnd(1, 3, 1, 129)), (q, k, v, True, None, None, None, None)]
    kept = msd.attention_kept(q, k, v, True)[1]
    packed = msd.attention_kept(q[0], k[0], v[0], False, 0.3, o, ok)[1]
    plain_set = {0, 1, 2, 3, 4, 15, 16, 20, 21, 22, 23, 26, 28}  # (15, 16: refused by the library itself)
    dout = rnd(2, 9, 4, 64)
    grads = [(dout, kept), (dout[0], packed), (dout.transpose(1, 2).contiguous().transpose(1, 2), kept), (dout, kept, (rnd(2, 9, 4, 64), rnd(2, 7, 2, 64), rnd(2, 7, 2, 64))),
             (dout[:1], kept), (dout.double(), kept), (dout.cpu(), kept), (dout, kept._replace(lse=kept.lse[:1])), (dout, kept._replace(rest=None)),
             (dout, kept._replace(scale=0.0)), (dout, kept._replace(out=kept.out[:1])), (dout, kept._replace(lse=kept.lse.double())),
             (dout, kept._replace(k=k[:, :6])), (dout, kept, (kept.q, rnd(2, 7, 2, 64), rnd(2, 7, 2, 64)))]
    return {"token_embedding": (embeds, {0, 1, 2, 3, 11, 13, 16, 17}), "token_embedding_backward": (backs, {0, 1, 2, 8}),
            "layernorm_backward": (norms, {0, 1, 2, 3, 10, 11, 13}),
            "attention": (attends, plain_set), "attention_kept": (attends, plain_set), "attention_backward": (grads, {0, 1, 2, 8, 9})}


def _outcome(call, args):
    try:
        got = call(*args)
    except Exception as e:  # (TypeError, MsdError, ctypes.ArgumentError, ...)
        return type(e).__name__
    flat = [got] if torch.is_tensor(got) else [t for x in got for t in (x if isinstance(x, tuple) else (x,))]
    return [type(got).__name__] + [t.clone(memory_format=torch.preserve_format) if torch.is_tensor(t) else t for t in flat]


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_native_calls_are_the_general_ones(msd, cuda, half, monkeypatch):
    native, general = _cases(msd, cuda, half), _cases(msd, cuda, half)  # (some calls write into what later ones read)
    made = msd._bind_native_text()
    names = {n for n in dir(made) if not n.startswith("__")} - {"bind", "names", "built_for"}
    assert names | {"attention_kept"} == set(native)
    for name, (calls, plainly) in native.items():
        for i, args in enumerate(calls):
            recorder = _Recorder(made)
            with monkeypatch.context() as m:
                m.setattr(msd, "_native_text", recorder)
                a = _outcome(getattr(msd, name), args)
            with monkeypatch.context() as m:
                m.setattr(msd, "_native_text", _General())
                b = _outcome(getattr(msd, name), general[name][0][i])
            assert ((name.replace("_kept", ""), True) in recorder.made) == (i in plainly), (name, i, a if isinstance(a, str) else a[0])
            assert type(a) is type(b) and len(a) == len(b) and (a == b if isinstance(a, str) else a[0] == b[0]), (name, i, a, b)
            for s, t in zip(a[1:], b[1:]) if not isinstance(a, str) else ():
                if torch.is_tensor(s):
                    assert s.dtype == t.dtype and s.shape == t.shape and s.stride() == t.stride(), (name, i)
                    assert torch.equal(s, t), (name, i)
                else:
                    assert s == t, (name, i, s, t)


# ---- refusals of the package ------------------------------------------------------------------------------
def test_operands_that_do_not_fit(msd, cuda):
    ids, table, x, g = torch.zeros(2, 5, dtype=torch.int64, device=cuda), torch.zeros(9, 16, device=cuda), torch.zeros(2, 5, 16, device=cuda), torch.ones(16, device=cuda)
    q, k = torch.zeros(2, 5, 4, 16, device=cuda), torch.zeros(2, 6, 2, 16, device=cuda)
    o, ok = _offsets([5], cuda), _offsets([6], cuda)
    kept = msd.attention_kept(q, k, k)[1]
    n = torch.empty_like
    refused = [
        lambda: msd.token_embedding(ids.int(), table), lambda: msd.token_embedding(ids, table.bfloat16()), lambda: msd.token_embedding(ids, table[0]),
        lambda: msd.token_embedding(ids, table, table[:4]), lambda: msd.token_embedding(ids, table, table[:, :8]), lambda: msd.token_embedding(ids, table, table.half()),
        lambda: msd.token_embedding(ids, table, out=x[:1]), lambda: msd.token_embedding(ids, table, out=x.half()), lambda: msd.token_embedding(ids[0, 0], table),
        lambda: msd.token_embedding(ids.cpu(), table), lambda: msd.token_embedding(ids, table.cpu()), lambda: msd.token_embedding(ids, table[:0]),
        lambda: msd.token_embedding(ids.t(), table), lambda: msd.token_embedding(ids, table.t()),
        lambda: msd.token_embedding_backward(x, ids[:1], 9), lambda: msd.token_embedding_backward(x, ids, 9, 4), lambda: msd.token_embedding_backward(x.bfloat16(), ids, 9),
        lambda: msd.token_embedding_backward(x.cpu(), ids, 9), lambda: msd.token_embedding_backward(x, ids.int(), 9),
        lambda: msd.layernorm_backward(x, x[:1], g), lambda: msd.layernorm_backward(x, x, g.half()), lambda: msd.layernorm_backward(x, x, g[:8]),
        lambda: msd.layernorm_backward(x, x.half(), g), lambda: msd.layernorm_backward(x, x, g, out=x), lambda: msd.layernorm_backward(x.cpu(), x, g),
        lambda: msd.layernorm_backward(x, x, g, 1e-5, x[:1]), lambda: msd.layernorm_backward(x.bfloat16(), x.bfloat16(), g),
        lambda: msd.attention(q, k, k[:, :5]), lambda: msd.attention(q, k[:1], k[:1]), lambda: msd.attention(q, k.half(), k), lambda: msd.attention(q.bfloat16(), k.bfloat16(), k.bfloat16()),
        lambda: msd.attention(q, k[..., :8], k[..., :8]), lambda: msd.attention(q[:, :, :3], k, k), lambda: msd.attention(q, k, k, offsets=o), lambda: msd.attention(q[0], k[0], k[0]),
        lambda: msd.attention(q[0], k[0], k[0], offsets=o), lambda: msd.attention(q[0], k[0], k[0], offsets=o.long(), offsets_k=ok.long()),
        lambda: msd.attention(q[0], k[0], k[0], offsets=o, offsets_k=torch.cat([ok, ok[1:]])), lambda: msd.attention(q[0], k[0], k[0], offsets=o.cpu(), offsets_k=ok),
        lambda: msd.attention(q, k, k, scale=0.0), lambda: msd.attention(q, k, k, scale=math.inf), lambda: msd.attention(q, k, k, scale=math.nan), lambda: msd.attention(q, k, k, out=q),
        lambda: msd.attention(q, k, k, out=n(q)[:1]), lambda: msd.attention(q, k, k, out=n(q).half()), lambda: msd.attention(q, k, k, out=q[:1, :1, :1].expand(2, 5, 4, 16)),
        lambda: msd.attention(q.cpu(), k, k), lambda: msd.attention(q, k.cpu(), k.cpu()), lambda: msd.attention(q.transpose(2, 3), k.transpose(2, 3), k.transpose(2, 3)),
        lambda: msd.attention(*(torch.zeros(1, 2, 1, 136, device=cuda) for _ in range(3))), lambda: msd.attention(q[0, 0], k[0, 0], k[0, 0]),
        lambda: msd.attention_backward(q[:1], kept), lambda: msd.attention_backward(q.half(), kept), lambda: msd.attention_backward(q.cpu(), kept),
        lambda: msd.attention_backward(q, kept, (n(q), n(k), k)), lambda: msd.attention_backward(q, kept, (n(k), n(k), n(q))),
        lambda: msd.attention_backward(q, kept._replace(lse=kept.lse[:1])), lambda: msd.attention_backward(q, kept._replace(lse=kept.lse.half())),
        lambda: msd.attention_backward(q, kept._replace(offsets=o)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(msd.MsdError):
            call()
            pytest.fail("call %d was not refused" % i)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_calls_with_nothing_to_do(msd, cuda, dtype):
    t = DTYPES[dtype]
    q, k = torch.ones(2, 5, 4, 16, dtype=t, device=cuda), torch.ones(2, 6, 2, 16, dtype=t, device=cuda)
    out, kept = msd.attention_kept(q, k[:, :0], k[:, :0])
    assert not out.any() and bool((kept.lse == -math.inf).all())
    dq, dk, dv = msd.attention_backward(q, kept)
    assert not dq.any() and dk.shape == (2, 0, 2, 16)
    out, kept = msd.attention_kept(q[:, :0], k, k)
    dq, dk, dv = msd.attention_backward(q[:, :0], kept)
    assert out.shape == dq.shape == (2, 0, 4, 16) and not dk.any() and not dv.any()
    for cut in (q[:0], k[:0]), :
        out, kept = msd.attention_kept(cut[0], cut[1], cut[1])
        assert out.shape == (0, 5, 4, 16) and [x.shape[0] for x in msd.attention_backward(cut[0], kept)] == [0, 0, 0]
    none = torch.zeros(1, dtype=torch.int32, device=cuda)  # no sequence: every row stays
    out = msd.attention(q[0], q[1], q[1], offsets=none, out=torch.full_like(q[0], 3.0))
    assert bool((out == 3).all())
    assert not msd.token_embedding_backward(q.view(-1)[:0].view(0, 4, 16), torch.zeros(0, 4, dtype=torch.int64, device=cuda), 7, 4)[0].any()
