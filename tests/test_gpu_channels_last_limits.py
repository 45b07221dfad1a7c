"""The channels-last GroupNorm and its gradient where a workgroup's own limits decide how a call is made.  Tolerances as in
test_gpu_channels_last.py."""
import pytest

import plain_channels_last as plain
from test_gpu_channels_last import _check_gradients, _close, _inputs, _train

pytestmark = pytest.mark.gpu


def _check(msd, cuda, b, p, c, groups, half, act, chunk, keep8, seed=0):
    import torch
    x, add, gamma, beta, dy = _inputs(torch, b, p, c, half, chunk, seed=seed)
    what = "%s half %d act %d chunk %d keep8 %d" % ((b, p, c, groups), half, act, chunk, keep8)
    y, kept, got = _train(msd, cuda, x, add, gamma, beta, dy, groups, act, keep8)
    h = plain.added(x.double(), add, x.dtype)
    mean, rstd = plain.stats(h, groups, 1e-5)
    g64, b64 = gamma.double(), beta.double()
    _close(y, plain.forward(h, g64, b64, groups, 1e-5, act), half, what)
    err = (kept.stats.cpu().double() - torch.stack((mean, rstd), -1)).abs()
    assert bool((err[..., 0] <= 1e-6 * (1 + mean.abs()) / rstd.clamp(max=1)).all()) and bool((err[..., 1] <= 1e-5 * rstd).all()), what
    if keep8:
        codes, scales = plain.checkpoint(h)
        assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales), what
        h = plain.restored(codes, scales)
    mean, rstd = kept.stats.cpu().double().unbind(-1)
    _check_gradients(got, plain.gradients(dy.double(), h, mean, rstd, g64, b64, groups, act), half, b * p * (c // groups), what)


# a gradient's sums of 8192 channels (of 1023 in 32 groups: 8184 at a time) and what weights them are more than the 160 KB of LDS;
# 8160 channels are the most that fit
@pytest.mark.parametrize("b,p,c,groups", [(2, 1, 8192, 1), (1, 2, 16384, 2), (1, 1, 1023 * 32, 32), (2, 2, 8160, 1)])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_groups_that_fill_a_workgroups_lds(msd, cuda, b, p, c, groups, half):
    for act, chunk, keep8 in ((True, False, False), (False, True, False), (True, True, True)):
        _check(msd, cuda, b, p, c, groups, half, act, chunk, keep8)


# more than 256 chunks of 320 columns share a group, whose parts are then joined by a launch of their own
@pytest.mark.parametrize("b,p,c,groups,half", [(1, 3, 82001, 1, False), (2, 2, 2 * 82001, 2, True), (1, 2, 4 * 82080, 1, False), (2, 1, 8 * 82080, 1, True)])
def test_groups_over_more_chunks_than_a_workgroup_joins(msd, cuda, b, p, c, groups, half):
    for act, chunk, keep8 in ((True, True, False), (False, False, True)):
        _check(msd, cuda, b, p, c, groups, half, act, chunk, keep8)


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("c", [64, 72])
def test_blocks_of_nothing_but_zeros_infinities_and_nan_have_codes_of_zero(msd, cuda, c, half):
    import torch
    x, _, gamma, beta, _ = _inputs(torch, 2, 5, c, half, False)
    x[0, 1, 32:64], x[1, 2, 32:64], x[1, 3, 32:64] = 0.0, 0.0, 0.0
    x[0, 1, 40], x[1, 2, 33], x[1, 3, 63] = float("inf"), float("nan"), float("-inf")
    _, kept = msd.groupnorm_channels_last_kept(x.to(cuda), gamma.to(cuda), beta.to(cuda), c // 8, keep8=True)
    codes, scales = kept.codes.cpu(), kept.scales.cpu()
    for b, p in ((0, 1), (1, 2), (1, 3)):
        assert not bool(codes[b, p, 32:64].any()) and float(scales[b, p, 1]) == 0.0
    want = plain.checkpoint(x.double())
    others = torch.ones((2, 5, c), dtype=torch.bool)
    others[0, 1, 32:64] = others[1, 2:4, 32:64] = False
    assert torch.equal(codes[others], want[0][others]) and torch.equal(scales, want[1])
