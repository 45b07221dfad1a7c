"""The kernels of the channels-last GroupNorm and of the Linear rows with 4-bit weights that the UNet's levels, its 22 projections and
large layers are given, one by one, and seeded random shapes of both.  Tolerances as in test_gpu_channels_last.py and
test_gpu_linear_q4.py."""
import numpy as np
import pytest

import plain_channels_last as plain
import plain_q4
from test_gpu_channels_last import E32, _inputs
from test_gpu_channels_last_limits import _check as check_norm
from test_gpu_linear_q4 import _call, _check, _layer, _rows

pytestmark = pytest.mark.gpu


# 16 x 16: four rows a lane in the kernels that have all positions of a sample; 8 x 8: one
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("b,p,c", [(2, 256, 1280), (1, 256, 1920), (2, 256, 2560), (2, 256, 640), (2, 64, 1280), (1, 64, 2560), (1, 253, 1920),
                                   (2, 1024, 640), (1, 1024, 960)])
def test_levels_of_the_unet(msd, cuda, b, p, c, half):
    for i, (act, chunk, keep8) in enumerate(((True, True, False), (True, False, True), (False, True, True))):
        check_norm(msd, cuda, b, p, c, 32, half, act, chunk, keep8, seed=i)


# by the rule on tiles of 16 columns: one, two and four of them a workgroup, for one or two rows and for more
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 4000, 384), (2, 5200, 1280), (2, 16400, 512), (1, 16397, 384), (3, 4999, 640), (8, 5200, 1280), (5, 10300, 512),
                                   (8, 10243, 1280)])
def test_tiles_and_rows(msd, cuda, m, n, k, group, half):
    import torch
    for i, (act_in, act_out, bias) in enumerate(((0, 0, False), (1, 1, True))):
        layer, x = _layer(torch, n, k, group, half, 7 * i + n, bias), _rows(torch, m, k, half, i + k)
        _check(_call(msd, cuda, x, layer, act_in, act_out), x, layer, act_in, act_out, "acts %d %d" % (act_in, act_out))


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("m,group", [(1, 64), (2, 64), (2, 32), (8, 32), (8, 128), (3, 64)])
def test_22_projections(msd, cuda, m, group, half):
    import torch
    ns = [320, 320, 640, 640] + [1280] * 12 + [640] * 3 + [320] * 3
    layers, x = [_layer(torch, n, 1280, group, half, 400 + i) for i, n in enumerate(ns)], _rows(torch, m, 1280, half, 9)
    got = msd.linear_rows_q4_grouped(x.to(cuda), [plain_q4.bytes_of(c).to(cuda) for c, _, _ in layers], [s.to(cuda) for _, s, _ in layers],
                                     [b.to(cuda) for _, _, b in layers], msd.ACT_SILU)
    for i, layer in enumerate(layers):
        _check(got[i], x, layer, 1, 0, "projection %d" % i)


@pytest.mark.parametrize("seed", [21, 22, 23, 24])
def test_random_norms(msd, cuda, seed):
    rng = np.random.default_rng(seed)
    for i in range(40):
        groups = int(rng.choice([1, 2, 3, 8, 16, 32]))
        c = groups * int(rng.choice([rng.integers(1, 13), rng.integers(1, 200), 10, 20, 40, 80]))
        b = int(rng.choice([1, 2, 3, 5, 8, 17]))
        p = int(rng.choice([rng.integers(1, 40), rng.integers(1, 5000), 64, 256, 1024]))
        p = max(1, min(p, 600000 // (b * c)))
        check_norm(msd, cuda, b, p, c, groups, bool(rng.integers(2)), bool(rng.integers(2)), bool(rng.integers(2)), bool(rng.integers(2)), seed=100 * seed + i)


@pytest.mark.parametrize("seed", [31, 32, 33, 34])
def test_random_layers(msd, cuda, seed):
    import torch
    rng = np.random.default_rng(seed)
    for i in range(40):
        group, half = int(rng.choice([32, 64, 128])), bool(rng.integers(2))
        k = group * int(rng.choice([rng.integers(1, 5), rng.integers(1, 2560 // group + 1)]))
        m, act_in, act_out = int(rng.integers(1, 9)), int(rng.integers(2)), int(rng.integers(2))
        x, count = _rows(torch, m, k, half, 1000 * seed + i), int(rng.choice([1, 1, 3, 36]))
        ns = [int(rng.choice([rng.integers(1, 60), rng.integers(1, 1500)])) if count > 1 else int(rng.integers(1, 6000)) for _ in range(count)]
        layers = [_layer(torch, n, k, group, half, 5000 * seed + 50 * i + j, bool(rng.integers(2))) for j, n in enumerate(ns)]
        got = msd.linear_rows_q4_grouped(x.to(cuda), [plain_q4.bytes_of(c).to(cuda) for c, _, _ in layers], [s.to(cuda) for _, s, _ in layers],
                                         [v.to(cuda) if v is not None else None for _, _, v in layers], act_in, act_out)
        for n, y, layer in zip(ns, got, layers):
            _check(y, x, layer, act_in, act_out, "%s" % ((m, n, k, group, half, act_in, act_out),))
        if count == 1:
            assert torch.equal(got[0], _call(msd, cuda, x, layers[0], act_in, act_out))
        weight = torch.randn((int(rng.integers(1, 200)), k), generator=torch.Generator().manual_seed(i)).to(x.dtype)
        packed, scales = msd.q4_pack(weight.to(cuda), group)
        codes, want = plain_q4.pack(weight, group)
        assert torch.equal(packed.cpu(), plain_q4.bytes_of(codes)) and torch.equal(scales.cpu(), want)


@pytest.mark.parametrize("keep8", [False, True], ids=["x", "codes"])
def test_gradients_of_more_than_four_gigabytes(msd, cuda, keep8):
    """2^31 + some elements: offsets pass 32 bits in elements and bytes.  Every position holds one of seven pairs of rows of x and dy, so
    that all sums are those of the pairs, weighted."""
    import torch
    p, c, groups = (1 << 22) + 1021, 512, 32
    per = c // groups
    rows, _, gamma, beta, dys = _inputs(torch, 1, 7, c, True, False, seed=77)
    tiled = lambda t: t[0].to(cuda).repeat(-(-p // 7), 1)[:p].unsqueeze(0)  # noqa: E731
    x, dy = tiled(rows), tiled(dys)
    y, kept = msd.groupnorm_channels_last_kept(x, gamma.to(cuda), beta.to(cuda), groups, 1e-5, True, torch.zeros((1, c), device=cuda).half(), keep8)
    del y
    counts = torch.tensor([len(range(i, p, 7)) for i in range(7)], dtype=torch.float64)[:, None]
    h = rows[0].double()
    if keep8:
        codes, scales = plain.checkpoint(rows.double())
        for i in range(7):
            assert bool((kept.codes[0, i::7] == codes[0, i].to(cuda)).all()) and bool((kept.scales[0, i::7] == scales[0, i].to(cuda)).all())
        h = plain.restored(codes, scales)[0]
    dx, dgamma, dbeta, dchunk = msd.groupnorm_channels_last_backward(dy, kept, out=dy)
    mean, rstd = (v.repeat_interleave(per) for v in kept.stats.cpu().double()[0].unbind(-1))
    g64 = gamma.double()
    u = (h - mean) * rstd
    z = u * g64 + beta.double()
    s = 1 / (1 + torch.exp(-z))
    d = dys[0].double()
    dz, size = d * s * (1 + z * (1 - s)), d.abs() * s * (1 + z.abs() * (1 - s))
    wide = lambda v: ((v * counts).sum(0).view(groups, per).sum(1) / (p * per)).repeat_interleave(per)  # noqa: E731
    v, vs = dz * g64, (size * g64).abs()
    want = rstd * (v - wide(v) - u * wide(v * u))
    dx_size = rstd * (vs + wide(vs) + u.abs() * wide(vs * u.abs()))
    n = p * per
    slack = (64 + 4 * n ** 0.5) * E32
    for i in range(7):
        mine = dx[0, i::7]
        assert bool((mine == mine[0]).all())
        off = (mine[0].cpu().double() - want[i]).abs()
        assert bool((off <= slack * dx_size[i] + 2.0 ** -11 * (1 + 1e-6) * want[i].abs() + 2.0 ** -25).all()), i
    for got, ref, most in ((dgamma, dz * u, size * u.abs()), (dbeta, dz, size)):
        assert bool(((got.cpu().double() - (ref * counts).sum(0)).abs() <= slack * (most * counts).sum(0)).all())
    # sums of 2^22 positions: what is 65520 (half a step above the largest float16) and more is an infinity
    total, got = (want * counts).sum(0), dchunk[0].cpu().double()
    slack = slack * (dx_size * counts).sum(0)
    near = (got - total).abs() <= slack + 2.0 ** -11 * total.abs() + 2.0 ** -25
    beyond = (got == total.sign() * float("inf")) & (total.abs() + slack >= 65520)
    assert bool((near & (total.abs() - slack < 65520) | beyond).all())
