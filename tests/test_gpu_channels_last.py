"""The channels-last GroupNorm, its gradient and its 8-bit checkpoint against plain forms in 64 bits.

Tolerances.  The kernels work in float32 (unit rounding e = 2^-24).  A normalised value is off by a few e of itself, of
|mean| rstd and of the statistics; y is held to 1e-5 max(1, |y|) as every norm of the framework (tolerances.py), float16 to
half a step of its own beyond that.  A gradient is a sum of terms whose magnitudes plain.gradients adds up (S): each term is off
by at most a dozen roundings, SiLU's slope by the roundings of its exponential's argument (|z| log2 e e, |z| < 16 here: 24 e) and 2
e each for the exponential and the reciprocal, and the additions of N terms in chains of float32 by about sqrt(N) e S: together
(64 + 4 sqrt(N)) e S, and half a step of float16 where that is the type."""
import numpy as np
import pytest

import plain_channels_last as plain
from tolerances import assert_close_f16, assert_close_f32, ulp16

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24


def _inputs(torch, b, p, c, half, chunk, seed=0, level=0.5):
    g = torch.Generator().manual_seed(1000 * seed + 7 * b + 11 * p + 13 * c)
    dtype = torch.float16 if half else torch.float32
    x = (torch.randn((b, p, c), generator=g) * (0.5 + torch.rand(c, generator=g)) + level * torch.randn(c, generator=g)).to(dtype)
    add = torch.randn((b, c), generator=g).mul(0.5).to(dtype) if chunk else None
    gamma, beta = 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)
    dy = torch.randn((b, p, c), generator=g).to(dtype)
    return x, add, gamma, beta, dy


def _close(got, ref, half, what):
    got, ref = got.double().cpu().numpy(), ref.numpy()
    if half:
        assert_close_f16(got, ref, what)
    else:
        assert_close_f32(got, ref, what=what)


def _check_gradients(got, want, half, n, what):
    for name, value in got.items():
        if value is None:
            continue
        ref, size = (t.numpy() for t in want[name])
        # (dchunk: the kernel multiplies sums instead of summing products: the same terms)
        tol = (64 + 4 * np.sqrt(n)) * E32 * size
        if half and name in ("dx", "dchunk"):
            tol = tol + 0.5 * ulp16(ref) * (1 + 1e-6)
        err = np.abs(value.double().cpu().numpy().reshape(ref.shape) - ref)
        bad = ~(err <= tol)
        assert not bad.any(), "%s %s: %d of %d off, worst %.3e at %.3e (allowed %.3e)" % (
            what, name, bad.sum(), bad.size, err[bad].max(), ref[bad][np.argmax(err[bad])], tol[bad][np.argmax(err[bad])])


def _train(msd, cuda, x, add, gamma, beta, dy, groups, act, keep8, eps=1e-5):
    to = lambda t: t.to(cuda) if t is not None else None  # noqa: E731
    y, kept = msd.groupnorm_channels_last_kept(to(x), to(gamma), to(beta), groups, eps, act, to(add), keep8)
    dx, dgamma, dbeta, dchunk = msd.groupnorm_channels_last_backward(to(dy), kept)
    return y, kept, {"dx": dx, "dgamma": dgamma, "dbeta": dbeta, "dchunk": dchunk}


# batch, positions, channels, groups
SHAPES = [
    (2, 64, 320, 32), (1, 63, 1280, 32), (2, 4096, 320, 32), (3, 35, 2560, 32),   # of the UNet
    (2, 1, 32, 8), (1, 1, 1, 1), (4, 1, 96, 96), (1, 7, 5, 1), (2, 3, 8, 8),      # one position, one channel, one of each
    (2, 33, 99, 9), (1, 50, 482, 2), (2, 17, 258, 1), (1, 9, 1001, 7),            # no whole vectors
    (2, 20, 2561, 1), (1, 6, 2560, 1), (1, 5, 7680, 3), (1, 40, 1288, 7),         # groups longer than a workgroup is wide
    (1, 70000, 32, 32), (2, 9000, 8, 2), (1, 150000, 3, 1),                       # many positions of few channels
    (5, 300, 72, 3), (2, 100, 40, 4), (1, 260, 136, 8),                           # whole vectors, no whole blocks of codes
]


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("b,p,c,groups", SHAPES)
def test_forward_and_gradients(msd, cuda, b, p, c, groups, half):
    import torch
    for i, (act, chunk, keep8) in enumerate([(True, False, False), (True, True, True), (False, True, False), (False, False, True)]):
        x, add, gamma, beta, dy = _inputs(torch, b, p, c, half, chunk, seed=i)
        what = "%s act %d chunk %d keep8 %d" % ((b, p, c, groups), act, chunk, keep8)
        y, kept, got = _train(msd, cuda, x, add, gamma, beta, dy, groups, act, keep8)
        h = plain.added(x.double(), add, x.dtype)
        mean, rstd = plain.stats(h, groups, 1e-5)
        g64, b64 = gamma.double(), beta.double()
        _close(y, plain.forward(h, g64, b64, groups, 1e-5, act), half, "channels-last norm")
        only = msd.groupnorm_channels_last(x.to(cuda), gamma.to(cuda), beta.to(cuda), groups, 1e-5, act,
                                           add.to(cuda) if chunk else None)
        assert torch.equal(only, y), what
        err = (kept.stats.cpu().double() - torch.stack((mean, rstd), -1)).abs()
        assert bool((err[..., 0] <= 1e-6 * (1 + mean.abs()) / rstd.clamp(max=1)).all()) and bool((err[..., 1] <= 1e-5 * rstd).all()), what
        if keep8:
            codes, scales = plain.checkpoint(h)
            assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales), what
            h = plain.restored(codes, scales)
        # the statistics are those that the forward call kept, rounded to float32
        mean, rstd = kept.stats.cpu().double().unbind(-1)
        _check_gradients(got, plain.gradients(dy.double(), h, mean, rstd, g64, b64, groups, act), half, b * p * (c // groups), what)
        assert (got["dchunk"] is not None) == chunk


def test_gradients_against_differences_of_the_forward_call(msd, cuda):
    """Through the calls alone: the change of sum(y w) along random directions, from float32 outputs summed in 64 bits."""
    import torch
    b, p, c, groups = 2, 12, 24, 3
    for act in (False, True):
        x, add, gamma, beta, dy = _inputs(torch, b, p, c, False, True, seed=40 + act)
        _, _, got = _train(msd, cuda, x, add, gamma, beta, dy, groups, act, False)
        g = torch.Generator().manual_seed(5)
        for name, i in (("dx", 0), ("dchunk", 1), ("dgamma", 2), ("dbeta", 3)):
            values = [x, add, gamma, beta]
            way = torch.randn(values[i].shape, generator=g)
            ends = []
            step = 1.0 / 64  # (a power of two: the moved inputs carry one rounding of 2^-24 each, measured below as it is)
            for sign in (1, -1):
                moved = list(values)
                moved[i] = values[i] + sign * step * way
                y = msd.groupnorm_channels_last(moved[0].to(cuda), moved[2].to(cuda), moved[3].to(cuda), groups, 1e-5, act,
                                                moved[1].to(cuda))
                ends.append((y.cpu().double() * dy.double()).sum())
            along = ((ends[0] - ends[1]) / (2 * step)).item()
            said = (got[name].cpu().double() * way.double()).sum().item()
            # y is off by some 1e-6 a value, divided by 2 step and summed over 576 of them at random: 2e-3 at most; the curvature
            # step^2 / 6 x third derivative, with |way| of about sqrt(576) along normalised values: below 0.5 % of the scale
            scale = float(torch.linalg.vector_norm(got[name].cpu().double()) * torch.linalg.vector_norm(way.double()))
            assert abs(along - said) <= 2e-3 + 5e-3 * scale, (name, act, along, said)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_images_in_channels_last_order(msd, cuda, half):
    import torch
    x, add, gamma, beta, dy = _inputs(torch, 2, 35, 64, half, True)
    image = lambda t: t.to(cuda).view(2, 7, 5, 64).permute(0, 3, 1, 2)  # noqa: E731
    y, kept, got = _train(msd, cuda, x, add, gamma, beta, dy, 8, True, True)
    y4, kept4 = msd.groupnorm_channels_last_kept(image(x), gamma.to(cuda), beta.to(cuda), 8, 1e-5, True, add.to(cuda), True)
    grads4 = msd.groupnorm_channels_last_backward(image(dy), kept4)
    assert y4.shape == (2, 64, 7, 5) and y4.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(y4, image(y.cpu())) and torch.equal(grads4[0], image(got["dx"].cpu()))
    assert grads4[0].is_contiguous(memory_format=torch.channels_last)
    assert all(torch.equal(a, got[n]) for a, n in zip(grads4[1:], ("dgamma", "dbeta", "dchunk")))
    one = image(x)[:, :, :1, :1].contiguous(memory_format=torch.channels_last)  # both orders at once
    assert torch.equal(msd.groupnorm_channels_last(one, gamma.to(cuda), beta.to(cuda), 8).flatten(1),
                       msd.groupnorm_channels_last(one.flatten(2).permute(0, 2, 1).contiguous(), gamma.to(cuda), beta.to(cuda), 8).flatten(1))


@pytest.mark.parametrize("c", [320, 99])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_in_place_and_at_any_alignment(msd, cuda, half, c):
    import torch
    groups = 32 if c == 320 else 11
    x, add, gamma, beta, dy = (t.to(cuda) for t in _inputs(torch, 2, 90, c, half, True))
    y, kept = msd.groupnorm_channels_last_kept(x, gamma, beta, groups, 1e-5, True, add, True)
    want = msd.groupnorm_channels_last_backward(dy, kept)
    x2, dy2 = x.clone(), dy.clone()
    y2, kept2 = msd.groupnorm_channels_last_kept(x2, gamma, beta, groups, 1e-5, True, add, True, out=x2)
    assert y2 is x2 and torch.equal(y2, y) and torch.equal(kept2.codes, kept.codes) and torch.equal(kept2.scales, kept.scales)
    got = msd.groupnorm_channels_last_backward(dy2, kept2, out=dy2)
    assert got[0] is dy2 and all(torch.equal(a, b) for a, b in zip(got, want))

    def shifted(t):  # one element past a 16-byte boundary
        big = t.new_empty(t.numel() + 1)[1:].view(t.shape)
        return big.copy_(t)

    z, kept3 = msd.groupnorm_channels_last_kept(shifted(x), shifted(gamma), shifted(beta), groups, 1e-5, True, shifted(add), True)
    got = msd.groupnorm_channels_last_backward(shifted(dy), kept3)
    assert torch.equal(kept3.codes, kept.codes)
    for a, b in zip((z,) + got, (y,) + want):  # (other slices of positions: float32 sums in another order, of some 1e-6)
        tol = 1e-5 * (1 + b.abs().float().max().item()) + (2.0 ** -10 * b.abs().float() if b.dtype == torch.float16 else 0)
        assert bool(((a.float() - b.float()).abs() <= tol).all())
    none = msd.groupnorm_channels_last_backward(dy, kept, affine=False)
    assert none[1] is None and none[2] is None and torch.equal(none[0], want[0]) and torch.equal(none[3], want[3])


def test_a_mean_far_from_zero_costs_no_digits(msd, cuda):
    """Level 2000, spread 1: x itself has steps of 1.2e-4; means off by 2^-24 of 2000 move a normalised value by 1.2e-4."""
    import torch
    x, _, gamma, beta, _ = _inputs(torch, 2, 777, 64, False, False)
    x = x + 2000
    y = msd.groupnorm_channels_last(x.to(cuda), gamma.to(cuda), beta.to(cuda), 8).cpu().double()
    ref = plain.forward(x.double(), gamma.double(), beta.double(), 8, 1e-5, False)
    assert float((y - ref).abs().max()) <= 4 * 1.2e-4 * 2  # (mean, its products with gamma of up to 2: four roundings of it)


def test_infinities_and_nan_stay_in_their_group(msd, cuda):
    import torch
    x, add, gamma, beta, dy = _inputs(torch, 2, 40, 64, False, True)
    clean = _train(msd, cuda, x, add, gamma, beta, dy, 8, True, False)
    for bad in (float("inf"), float("-inf"), float("nan")):
        z = x.clone()
        z[1, 7, 21] = bad  # group 2 of sample 1
        for keep8 in (False, True):
            y, kept, got = _train(msd, cuda, z, add, gamma, beta, dy, 8, True, keep8)
            hit = torch.zeros((2, 1, 64), dtype=torch.bool)
            hit[1, 0, 16:24] = True
            for t in (y, got["dx"]):
                assert bool(torch.isnan(t.cpu()).logical_or(~hit).all()) and bool(torch.isfinite(t.cpu()).logical_or(hit).all())
            keep = ~hit.expand_as(y.cpu())
            assert torch.equal(y.cpu()[keep], clean[0].cpu()[keep])
            if not keep8:
                assert torch.equal(got["dx"].cpu()[keep], clean[2]["dx"].cpu()[keep])
            assert bool(torch.isnan(got["dchunk"].cpu()[1, 16:24]).all()) and bool(torch.isfinite(got["dchunk"].cpu()[0]).all())


def test_nothing_to_do(msd, cuda):
    import torch
    gamma, beta = torch.ones(16, device=cuda), torch.zeros(16, device=cuda)
    for shape in ((0, 5, 16), (2, 0, 16), (0, 16, 3, 3)):
        x = torch.empty(shape, device=cuda)
        x = x.to(memory_format=torch.channels_last) if len(shape) == 4 else x
        chunk = torch.ones((shape[0], 16), device=cuda)
        for keep8 in (False, True):
            y, kept = msd.groupnorm_channels_last_kept(x, gamma, beta, 4, 1e-5, True, chunk, keep8)
            dx, dgamma, dbeta, dchunk = msd.groupnorm_channels_last_backward(x, kept)
            assert y.shape == dx.shape == x.shape and dchunk.shape == (shape[0], 16)
            assert not bool(dgamma.any()) and not bool(dbeta.any()) and not bool(dchunk.any())


def test_the_same_bits_every_time_on_any_stream_and_in_graphs(msd, cuda):
    import torch
    cases = []
    for (b, p, c, groups), half, keep8 in (((2, 1024, 320, 32), True, True), ((1, 60000, 32, 4), False, False)):
        x, add, gamma, beta, dy = (t.to(cuda) for t in _inputs(torch, b, p, c, half, True))
        run = lambda x=x, add=add, gamma=gamma, beta=beta, dy=dy, groups=groups, keep8=keep8: (  # noqa: E731
            lambda pair: (pair[0],) + tuple(msd.groupnorm_channels_last_backward(dy, pair[1])))(
                msd.groupnorm_channels_last_kept(x, gamma, beta, groups, 1e-5, True, add, keep8))
        cases.append((run, [t.clone() for t in run()], x))
    streams = [torch.cuda.Stream() for _ in cases]
    graphs = []
    for (run, want, x), stream in zip(cases, streams):
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
        for (run, _, x), (graph, out) in zip(cases, graphs):
            x.mul_(0.5 + 0.25 * turn)
            [t.fill_(7.0) for t in out]
        want = [[t.clone() for t in run()] for run, _, _ in cases]
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):  # both at once: neither shares memory with the other
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w)), turn


def test_tensors_of_more_than_four_gigabytes(msd, cuda):
    """2^31 + some elements: offsets pass 32 bits in elements and bytes.  Every position holds one of seven rows, so that the
    statistics are those of the rows, weighted."""
    import torch
    p, c, groups = (1 << 22) + 1021, 512, 32
    g = torch.Generator().manual_seed(9)
    rows = torch.randn((7, c), generator=g).half()
    gamma, beta = 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)
    x = rows.to(cuda).repeat(-(-p // 7), 1)[:p].unsqueeze(0)
    counts = torch.tensor([len(range(i, p, 7)) for i in range(7)], dtype=torch.float64)[:, None]
    r = rows.double()
    wide = lambda v: v.view(groups, -1).mean(1).repeat_interleave(c // groups)  # noqa: E731
    mean = wide((r * counts).sum(0) / p)
    rstd = (wide(((r - mean) ** 2 * counts).sum(0) / p) + 1e-5) ** -0.5
    want = plain.silu((r - mean) * rstd * gamma.double() + beta.double())
    y = msd.groupnorm_channels_last(x, gamma.to(cuda), beta.to(cuda), groups, 1e-5, True, out=x)
    for i in range(7):
        mine = y[0, i::7]
        assert bool((mine == mine[0]).all())
        _close(mine[0], want[i], True, "channels-last norm of 4 GiB")
