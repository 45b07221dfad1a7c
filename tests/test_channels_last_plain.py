"""The plain 64-bit forms that the GPU tests of the channels-last GroupNorm compare with, against central differences."""
import pytest
import torch

import plain_channels_last as plain


@pytest.mark.parametrize("act", [False, True], ids=["plain", "silu"])
@pytest.mark.parametrize("b,p,c,groups", [(2, 5, 12, 3), (1, 1, 8, 2), (3, 4, 6, 6), (1, 7, 5, 1)])
def test_plain_gradients_against_differences(b, p, c, groups, act):
    g = torch.Generator().manual_seed(b * 100 + p * 10 + c)
    x, chunk, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((b, p, c), (b, c), (b, p, c)))
    gamma, beta = 1 + 0.3 * torch.randn(c, generator=g, dtype=torch.float64), torch.randn(c, generator=g, dtype=torch.float64)
    eps = 1e-2

    def loss(x, chunk, gamma, beta):
        return (dy * plain.forward(x + chunk[:, None, :], gamma, beta, groups, eps, act)).sum()

    h = x + chunk[:, None, :]
    got = plain.gradients(dy, h, *plain.stats(h, groups, eps), gamma, beta, groups, act)
    args = {"dx": 0, "dchunk": 1, "dgamma": 2, "dbeta": 3}
    values = [x, chunk, gamma, beta]
    step = 1e-5
    for name, i in args.items():
        flat = values[i].reshape(-1)
        for j in range(0, flat.numel(), max(1, flat.numel() // 17)):
            ends = []
            for sign in (1, -1):
                moved = [v.clone() for v in values]
                moved[i].reshape(-1)[j] += sign * step
                ends.append(loss(*moved))
            difference = (ends[0] - ends[1]) / (2 * step)
            # error of a central difference: step^2 / 6 times a third derivative of order (2 / sqrt(eps))^3, and 1e-16 / step
            assert abs(difference - got[name][0].reshape(-1)[j]) <= 1e-5 * (1 + abs(difference)), (name, j)


def test_plain_checkpoint_holds_a_value_within_half_a_step():
    g = torch.Generator().manual_seed(3)
    h = torch.randn((2, 9, 70), generator=g).double()
    h[0, 0, :32], h[1, 2, 5], h[1, 3, 66] = 0.0, 1e4, 1e-33
    codes, scales = plain.checkpoint(h)
    assert codes.shape == h.shape and scales.shape == (2, 9, 3)
    half_step = scales.double().repeat_interleave(32, dim=2)[:, :, :70] * 0.5
    assert bool(((plain.restored(codes, scales) - h).abs() <= half_step * (1 + 1e-6) + plain.TINY).all())
    assert int(codes[0, 0, :32].abs().max()) == 0 and float(scales[0, 0, 0]) == 0.0
