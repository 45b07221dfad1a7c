"""Linear rows with 4-bit weights where a row's values of 128 are of very different sizes, and the large ones meet weights of zero: what
is left is the sum of the small ones.  Tolerance as in test_gpu_linear_q4.py, relative to the summands that are not zero."""
import pytest

import plain_q4 as plain
from test_gpu_linear_q4 import E32, _call, _check, _layer, _rows

pytestmark = pytest.mark.gpu


def _wide(torch, m, n, k, group, half, seed):
    """A row of small values with a large one in every 128, whose weights are zero by the code or by the scale."""
    codes, scales, bias = _layer(torch, n, k, group, half, seed, False)
    x = _rows(torch, m, k, False, seed + 1)
    large = torch.arange(5, k, 128)
    codes[:, large[0::2]] = 8
    for at in large[1::2].tolist():
        scales[:, at // group] = 0.0
    return x, large, (codes, scales, bias)


@pytest.mark.parametrize("m,n,k,group", [(1, 40, 256, 32), (2, 330, 384, 64), (3, 17, 1184, 32), (8, 5200, 640, 128), (5, 10300, 512, 64),
                                         (2, 5200, 1280, 128), (1, 16400, 512, 32), (8, 33, 8192, 128)])
@pytest.mark.parametrize("factor", [1e9, 1e12, 1e14, 1e30])
def test_float32_rows(msd, cuda, m, n, k, group, factor):
    import torch
    x, large, layer = _wide(torch, m, n, k, group, False, 17 + n)
    x = x * 1e-3
    x[:, large] = torch.randn((m, len(large)), generator=torch.Generator().manual_seed(3)) * factor
    x[m - 1] *= 1e-6 if factor < 1e30 else 1.0
    y = _call(msd, cuda, x, layer)
    _check(y, x, layer, 0, 0, "%g" % factor)
    for rows in (slice(0, 1), slice(m - 1, m)):
        assert torch.equal(_call(msd, cuda, x[rows], layer), y[rows])


@pytest.mark.parametrize("m,n,k,group", [(1, 40, 256, 32), (2, 5200, 384, 64), (8, 5200, 640, 128), (7, 33, 1184, 32)])
def test_activated_rows(msd, cuda, m, n, k, group):
    """SiLU(-25) is -3.5e-10, SiLU(11) 11: 2^35 apart."""
    import torch
    for half in (False, True):
        x, large, layer = _wide(torch, m, n, k, group, half, 90 + n)
        layer = (layer[0], layer[1] * 2.0 ** 10, None)  # (float16 outputs hold 6e-8 and more)
        x = (x - 25)
        x[:, large] = 11
        x = x.half() if half else x
        _check(_call(msd, cuda, x, layer, 1), x, layer, 1, 0, "half %d" % half)


def test_every_size_in_one_row(msd, cuda):
    """Values from 2^-140 to 2^100 in steps of 2^2, each with a column of its own in which the others have the weight zero.  An output has
    one product, rounded once: to half of 2^-149, the step below 2^-126, or as in the tolerance above."""
    import torch
    k, group = 128, 32
    exponents = torch.arange(-140, 101, 2).float()
    x = torch.zeros((3, k))
    x[1, :len(exponents)] = torch.exp2(exponents) * 1.7
    x[0], x[2] = -x[1], torch.flip(x[1], (0,))
    codes = torch.full((k, k), 8, dtype=torch.uint8)
    codes.fill_diagonal_(13)
    layer = (codes, torch.full((k, k // group), 0.25), None)
    y, (ref, size) = _call(msd, cuda, x, layer).cpu().double(), plain.linear(x, *layer, 0, 0)
    assert bool(((y - ref).abs() <= 2.0 ** -150 + (32 + 4 * k ** 0.5) * E32 * size).all())


def test_rows_of_ordinary_and_of_infinite_values_beside_them(msd, cuda):
    import torch
    x, large, layer = _wide(torch, 4, 70, 512, 64, False, 5)
    x[1, large] = 1e13
    x[2, 77], x[3, 200] = float("inf"), float("nan")
    y = _call(msd, cuda, x, layer).cpu()
    want = plain.linear(x, *layer, 0, 0)[0]
    assert torch.equal(torch.isfinite(y), torch.isfinite(want)) and torch.equal(torch.isnan(y), torch.isnan(want))
    _check(y[:2], x[:2], layer, 0, 0, "finite rows")


@pytest.mark.parametrize("k", [1184, 8192, 131072])
def test_small_values_in_one_step_of_one_row(msd, cuda, k):
    """A row that is zero but for 128 values, in every tenth part of k in turn, beside rows of ordinary values."""
    import torch
    codes, scales, _ = _layer(torch, 37, k, 32, False, 8, False)
    for part in range(11):
        first = min(k * part // 10, k - 128) // 128 * 128 if part < 10 else k - 128
        at = first + 37
        x = _rows(torch, 3, k, False, part)
        x[1] = 0
        x[1, first:first + 128] = 1e-3 * _rows(torch, 1, 128, False, 50 + part)[0]
        x[1, at] = 1e13
        mine = codes.clone()
        mine[:, at] = 8
        layer = (mine, scales, None)
        _check(_call(msd, cuda, x, layer), x, layer, 0, 0, "part %d" % part)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_packing_groups_of_nothing_but_zeros_infinities_and_nan(msd, cuda, half):
    import torch
    w = _rows(torch, 5, 128, half, 70)
    w[1:4, 32:64] = 0.0
    w[1, 40], w[2, 33], w[3, 63] = float("inf"), float("nan"), float("-inf")
    packed, scales = msd.q4_pack(w.to(cuda), 32)
    assert bool((packed.cpu()[1:4, 16:32] == 0x88).all()) and not bool(scales.cpu()[1:4, 1].any())
    codes, want = plain.pack(w, 32)
    codes[1:4, 32:64] = 8
    assert torch.equal(packed.cpu(), plain.bytes_of(codes)) and torch.equal(scales.cpu(), want)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_a_layer_of_another_alignment_leaves_the_others_as_they_are(msd, cuda, half):
    import torch
    layers = [_layer(torch, n, 640, 64, half, 80 + n, False) for n in (320, 33, 640)]
    x = _rows(torch, 5, 640, half, 81).to(cuda)
    packed, scales = [plain.bytes_of(c).to(cuda) for c, _, _ in layers], [s.to(cuda) for _, s, _ in layers]
    alone = [msd.linear_rows_q4(x, p, s) for p, s in zip(packed, scales)]
    for i in range(3):
        moved = list(packed)
        moved[i] = torch.empty(packed[i].numel() + 1, dtype=torch.uint8, device=cuda)[1:].view(packed[i].shape).copy_(packed[i])
        got = msd.linear_rows_q4_grouped(x, moved, scales)
        assert all(torch.equal(a, b) for k, (a, b) in enumerate(zip(got, alone)) if k != i), i
        assert torch.equal(got[i], msd.linear_rows_q4(x, moved[i], scales[i]))
        _check(got[i], x.cpu(), layers[i], 0, 0, "moved %d" % i)
