"""Linear rows with 4-bit weights against their plain form in 64 bits.

Tolerance: with e = 2^-24 and S the sum of the magnitudes of a sum's terms, every term is off by a dozen roundings (SiLU's
exponential by |x| log2 e more, |x| < 6 here unless said; the products; the split of x), and the additions of k terms in chains of
float32 by about sqrt(k) e S: (32 + 4 sqrt(k)) e S, and half a step of float16 where that is the type."""
import numpy as np
import pytest

import plain_q4 as plain
from tolerances import ulp16

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24


def _layer(torch, n, k, group, half, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = ((torch.rand((n, k // group), generator=g) + 0.5) * 0.2 / k ** 0.5).to(torch.float16 if half else torch.float32)
    return codes, scales, 0.1 * torch.randn(n, generator=g) if bias else None


def _rows(torch, m, k, half, seed):
    return torch.randn((m, k), generator=torch.Generator().manual_seed(seed)).to(torch.float16 if half else torch.float32)


def _check(got, x, layer, act_in, act_out, what):
    ref, size = (t.numpy() for t in plain.linear(x, *layer, act_in, act_out))
    half = got.dtype.itemsize == 2
    tol = (32 + 4 * np.sqrt(x.shape[1])) * E32 * size + (0.5 * ulp16(ref) * (1 + 1e-6) if half else 0)
    err = np.abs(got.double().cpu().numpy() - ref)
    bad = ~(err <= tol)
    assert got.shape == ref.shape and not bad.any(), "%s: %d of %d off, worst %.3e at %.3e (allowed %.3e)" % (
        what, bad.sum(), bad.size, err[bad].max(), ref[bad][np.argmax(err[bad])], tol[bad][np.argmax(err[bad])])


def _call(msd, cuda, x, layer, act_in=0, act_out=0, out=None):
    codes, scales, bias = layer
    return msd.linear_rows_q4(x.to(cuda), plain.bytes_of(codes).to(cuda), scales.to(cuda), bias.to(cuda) if bias is not None else None,
                              act_in, act_out, out)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("m,n,k,group", [(1, 1280, 1280, 64), (2, 320, 1280, 32), (8, 640, 1280, 128), (3, 1237, 2048, 32),
                                         (1, 1, 32, 32), (8, 1, 64, 64), (5, 17, 96, 32), (4, 16, 128, 128), (7, 33, 1184, 32),
                                         (6, 50, 1088, 64), (2, 15, 8192, 128), (8, 4097, 1152, 128), (1, 70, 10240, 64), (8, 8200, 256, 64)])
def test_shapes(msd, cuda, m, n, k, group, half):
    import torch
    for i, (act_in, act_out, bias) in enumerate(((0, 0, False), (1, 0, True), (0, 1, True))):
        layer, x = _layer(torch, n, k, group, half, 100 * i + n + k, bias), _rows(torch, m, k, half, 7 + i + k)
        _check(_call(msd, cuda, x, layer, act_in, act_out), x, layer, act_in, act_out, "%s acts %d %d" % ((m, n, k, group), act_in, act_out))


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_a_row_has_the_same_bits_in_any_company(msd, cuda, half):
    """Other rows, and other layers, more of them than one launch takes."""
    import torch
    for k, group in ((1280, 64), (352, 32)):
        ns = [320, 1, 640, 17, 0, 1280] * 7
        layers = [_layer(torch, n, k, group, half, 300 + i, i % 3 != 0) for i, n in enumerate(ns)]
        for act_in in (0, 1):
            x = _rows(torch, 8, k, half, 31)
            packed = [plain.bytes_of(c).to(cuda) for c, _, _ in layers]
            scales = [s.to(cuda) for _, s, _ in layers]
            biases = [b.to(cuda) if b is not None else None for _, _, b in layers]
            grouped = msd.linear_rows_q4_grouped(x.to(cuda), packed, scales, biases, act_in)
            assert [tuple(y.shape) for y in grouped] == [(8, n) for n in ns]
            for i in (0, 1, 2, 3, 4, 5, 31, 41):
                if ns[i]:
                    _check(grouped[i], x, layers[i], act_in, 0, "grouped %d" % i)
                for rows in (slice(0, 8), slice(0, 1), slice(2, 5), slice(7, 8)):
                    assert torch.equal(_call(msd, cuda, x[rows], layers[i], act_in), grouped[i][rows]), (k, i, rows)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_any_alignment_and_a_given_output(msd, cuda, half):
    import torch
    layer, x = _layer(torch, 40, 320, 32, half, 5), _rows(torch, 3, 320, half, 6)

    def shifted(t):
        big = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape)
        return big.copy_(t)

    packed, scales, bias = plain.bytes_of(layer[0]), layer[1], layer[2]
    for args in ((shifted(x), packed.to(cuda), scales.to(cuda), bias.to(cuda)), (x.to(cuda), shifted(packed), scales.to(cuda), bias.to(cuda)),
                 (x.to(cuda), packed.to(cuda), shifted(scales), shifted(bias))):
        for act_in in (0, 1):
            _check(msd.linear_rows_q4(*args, act_in), x, layer, act_in, 0, "shifted")
    out = shifted(torch.zeros((3, 40), dtype=x.dtype))
    assert _call(msd, cuda, x, layer, out=out) is out
    assert torch.equal(out, _call(msd, cuda, x, layer))
    assert _call(msd, cuda, x[:0], layer).shape == (0, 40)
    assert msd.linear_rows_q4_grouped(x.to(cuda), [], []) == []


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_values_of_every_size(msd, cuda, half):
    """Rows from the smallest values of the type to the largest, and rows of ordinary values with a few 2^12 times as large."""
    import torch
    k = 640
    layer, x = _layer(torch, 24, k, 32, half, 15, False), _rows(torch, 8, k, False, 16)
    if half:
        factors = torch.tensor([2.0 ** -22, 2.0 ** -14, 1.0, 2.0 ** 5, 1.0, 2.0 ** -18, 2.0 ** 8, 2.0 ** 10])
    else:
        factors = torch.tensor([2.0 ** -120, 2.0 ** -60, 1.0, 2.0 ** 60, 1.0, 2.0 ** -100, 2.0 ** 110, 2.0 ** 17])
    x = (x * factors[:, None]).to(torch.float16 if half else torch.float32)
    x[4, ::97] *= 4096 if not half else 2.0 ** 10
    _check(_call(msd, cuda, x, layer), x, layer, 0, 0, "sizes")  # (relative to each output's own summands)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_infinities_and_nan_reach_the_outputs_they_reach_in_a_sum(msd, cuda, half):
    import torch
    k = 256
    codes, scales, _ = _layer(torch, 20, k, 32, half, 25, False)
    codes[:, 70] = torch.arange(20) % 16
    x = _rows(torch, 5, k, half, 26)
    x[1, 70], x[2, 70], x[3, 70] = float("inf"), float("-inf"), float("nan")
    x[4, 200] = torch.finfo(x.dtype).max / 2
    y = _call(msd, cuda, x, (codes, scales, None)).cpu()
    want = plain.linear(x, codes, scales, None, 0, 0)[0].to(x.dtype)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.equal(y[torch.isinf(y)], want[torch.isinf(y)])
    _check(y[0:1], x[0:1], (codes, scales, None), 0, 0, "clean row")


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_packing(msd, cuda, half, group):
    import torch
    g = torch.Generator().manual_seed(group)
    w = (torch.randn((37, 384), generator=g) * 0.05).to(torch.float16 if half else torch.float32)
    w[3, :group], w[4, 5], w[5, 9], w[6, 130], w[7] = 0.0, float("inf"), float("nan"), 30.0, w[7] * 1e-6
    if not half:
        w[8], w[9] = w[8] * 1e-32, w[9] * 1e30
    packed, scales = msd.q4_pack(w.to(cuda), group)
    codes, want = plain.pack(w, group)
    assert torch.equal(scales.cpu(), want) and torch.equal(packed.cpu(), plain.bytes_of(codes))
    shifted = torch.empty(w.numel() + 1, dtype=w.dtype, device=cuda)[1:].view(w.shape).copy_(w)
    again = msd.q4_pack(shifted, group)
    assert torch.equal(again[0], packed) and torch.equal(again[1], scales)
    clean = torch.isfinite(w).all(1) & (w.abs().amax(1) >= 1e-4)
    off = ((codes.float() - 8) * want.float().repeat_interleave(group, 1) - w.float()).abs()[clean]
    # half a step; a float16 scale is off by 2^-11 of itself, seven steps of which a code can be away from zero
    step = want.float().repeat_interleave(group, 1)[clean]
    assert bool((off <= step * (0.5 + 8 * 2.0 ** -11) * (1 + 1e-6)).all())
    assert msd.q4_pack(w[:0].to(cuda), group)[0].shape == (0, 192)


def test_streams_and_graphs(msd, cuda):
    import torch
    layers = [_layer(torch, n, 1280, 64, True, 50 + n) for n in (320, 1280, 77)]
    packed = [plain.bytes_of(c).to(cuda) for c, _, _ in layers]
    scales, biases = [s.to(cuda) for _, s, _ in layers], [b.to(cuda) for _, _, b in layers]
    x = _rows(torch, 2, 1280, True, 51).to(cuda)
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    runs = [lambda: msd.linear_rows_q4_grouped(x, packed, scales, biases, msd.ACT_SILU),
            lambda: [msd.linear_rows_q4(x, packed[1], scales[1], biases[1])]]
    for run, stream in zip(runs, streams):
        want = run()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = run()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run()
        graphs.append((graph, out))
    for turn in range(4):
        x.mul_(0.75)
        want = [run() for run in runs]
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for (_, out), w in zip(graphs, want) for a, b in zip(out, w)), turn
