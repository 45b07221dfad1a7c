"""Statistics of the channels-last GroupNorm where some rows are nothing like the others: a border of zeros, a zero corner, a channel
that is off, in front of values of 100 +- 0.01.

Tolerance: the squared deviations are sums of products that are never less than zero, in chains of a few hundred additions at
most, each off by 2^-24 of what it has: 1 / sqrt(variance) is held to 1e-5 of itself, as elsewhere.  The mean of values around 100 is held to
four roundings of 100 (2^-24 of it each), y to what that makes of it."""
import pytest

import plain_channels_last as plain

pytestmark = pytest.mark.gpu

SHAPES = [(1, 262144, 32, 8), (16, 65536, 32, 8), (2, 4096, 320, 32), (1, 30000, 5, 1), (1, 200, 2561, 1), (3, 4097, 72, 3),  # in slices
          (2, 64, 1280, 32), (1, 4096, 8, 2), (2, 63, 2560, 32), (1, 1000, 4, 4), (2, 16, 48, 1)]                             # in one launch


def _rows(torch, device, b, p, c, groups, what):
    g = torch.Generator(device=device).manual_seed(b + p + c)
    x = 100 + 0.01 * torch.randn((b, p, c), device=device, generator=g)
    if what == "first":
        x[:, 0] = 0
    elif what == "corner":
        x[:, :min(16, p - 1)] = 0
    elif what == "last":
        x[:, -1] = 0
    elif what == "half":
        x[:, :(p + 1) // 2] = 0
    elif what == "channel":
        x[:, :, ::c // groups] = 0
    return x


@pytest.mark.parametrize("what", ["first", "corner", "last", "half", "channel", "level"])
@pytest.mark.parametrize("b,p,c,groups", SHAPES)
def test_rows_unlike_the_others(msd, cuda, b, p, c, groups, what):
    import torch
    x = _rows(torch, cuda, b, p, c, groups, what)
    gamma, beta = torch.ones(c, device=cuda), torch.zeros(c, device=cuda)
    y, kept = msd.groupnorm_channels_last_kept(x, gamma, beta, groups, 1e-5)
    mean, rstd = plain.stats(x.double(), groups, 1e-5)
    got_mean, got_rstd = kept.stats.double().unbind(-1)
    ulp = 100 * 2.0 ** -24
    if what == "channel" and c // groups == 1:
        return  # (nothing but zeros)
    assert float((got_mean - mean).abs().max()) <= 4 * ulp, float((got_mean - mean).abs().max())
    if what == "level":  # the spread is 0.01: x has no more than that of it, and the mean's roundings add their square
        assert float((got_rstd / rstd - 1).abs().max()) <= 1e-5 + (4 * ulp / 0.01) ** 2
        return
    worst = float((got_rstd / rstd - 1).abs().max())
    assert worst <= 1e-5, worst
    ref = plain.forward(x.double(), gamma.double(), beta.double(), groups, 1e-5, False)
    off = (y.double() - ref).abs() - 1e-5 * ref.abs() - 8 * ulp * rstd.repeat_interleave(c // groups, dim=1)[:, None, :]
    assert float(off.max()) <= 0, float(off.max())
