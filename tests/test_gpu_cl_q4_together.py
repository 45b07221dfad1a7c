"""The channels-last GroupNorm with 4-bit projections as they are used together: the time embedding's projections of two residual
blocks in one launch, their outputs as the norms' addends, an 8-bit checkpoint in between, and the gradient back to the
projections' outputs; eagerly, and captured and replayed beside eager work.

Tolerances are those of the operators' own tests: each plain form starts from what the operator before it gave."""
import numpy as np
import pytest

import plain_channels_last as plain
import plain_q4
from test_gpu_channels_last import _check_gradients, _close
from tolerances import ulp16

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24
WIDTH, GROUP, EPS = 320, 64, 1e-5
BLOCKS = [(6, 7, 64, 32), (5, 3, 320, 32)]  # h, w, channels, groups


def _blocks(torch, half, batch, device):
    g = torch.Generator().manual_seed(77 + batch)
    dtype = torch.float16 if half else torch.float32
    emb = torch.randn((batch, WIDTH), generator=g).to(dtype)
    blocks = []
    for h, w, c, groups in BLOCKS:
        weight = (torch.randn((c, WIDTH), generator=g) / WIDTH ** 0.5).to(dtype)
        blocks.append({
            "weight": weight, "codes": plain_q4.pack(weight, GROUP), "groups": groups, "bias": 0.1 * torch.randn(c, generator=g),
            "gamma": 1 + 0.2 * torch.randn(c, generator=g), "beta": 0.2 * torch.randn(c, generator=g),
            "x": torch.randn((batch, c, h, w), generator=g).to(dtype).contiguous(memory_format=torch.channels_last),
            "dy": torch.randn((batch, c, h, w), generator=g).to(dtype).contiguous(memory_format=torch.channels_last)})
    dev = [{k: v.to(device) for k, v in b.items() if torch.is_tensor(v)} for b in blocks]
    return emb, emb.to(device), blocks, dev


def _step(msd, emb, blocks, dev, packed, keep8):
    chunks = msd.linear_rows_q4_grouped(emb, [p for p, _ in packed], [s for _, s in packed], [d["bias"] for d in dev],
                                        act_in=msd.ACT_SILU)
    out = []
    for b, d, chunk in zip(blocks, dev, chunks):
        y, kept = msd.groupnorm_channels_last_kept(d["x"], d["gamma"], d["beta"], b["groups"], EPS, True, chunk, keep8)
        out.append((chunk, y, kept) + tuple(msd.groupnorm_channels_last_backward(d["dy"], kept)))
    return out


def _rows(t):
    """[batch, C, H, W] in channels-last order -> [batch, positions, C] on the CPU"""
    return t.permute(0, 2, 3, 1).reshape(t.shape[0], -1, t.shape[1]).cpu()


@pytest.mark.parametrize("keep8", [False, True], ids=["kept", "kept8"])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
@pytest.mark.parametrize("batch", [1, 3, 8])
def test_projections_norms_and_gradients(msd, cuda, batch, half, keep8):
    import torch
    emb, emb_dev, blocks, dev = _blocks(torch, half, batch, cuda)
    packed = [msd.q4_pack(d["weight"], GROUP) for d in dev]
    for b, (p, s) in zip(blocks, packed):
        assert torch.equal(p.cpu(), plain_q4.bytes_of(b["codes"][0])) and torch.equal(s.cpu(), b["codes"][1])
    for b, d, (chunk, y, kept, dx, dgamma, dbeta, dchunk) in zip(blocks, dev, _step(msd, emb_dev, blocks, dev, packed, keep8)):
        ref, size = plain_q4.linear(emb, *b["codes"], b["bias"], True, False)
        tol = (32 + 4 * np.sqrt(WIDTH)) * E32 * size.numpy() + (0.5 * ulp16(ref.numpy()) * (1 + 1e-6) if half else 0)
        assert (np.abs(chunk.cpu().double().numpy() - ref.numpy()) <= tol).all()
        add, groups, g64, b64 = chunk.cpu(), b["groups"], b["gamma"].double(), b["beta"].double()
        h = plain.added(_rows(b["x"]), add, b["x"].dtype)
        _close(_rows(y), plain.forward(h, g64, b64, groups, EPS, True), half, "norm of the projections")
        if keep8:
            codes, scales = plain.checkpoint(h)
            assert torch.equal(_rows(kept.codes), codes) and torch.equal(kept.scales.cpu(), scales)
            h = plain.restored(codes, scales)
        mean, rstd = kept.stats.cpu().double().unbind(-1)
        want = plain.gradients(_rows(b["dy"]).double(), h, mean, rstd, g64, b64, groups, True)
        got = {"dx": _rows(dx), "dgamma": dgamma, "dbeta": dbeta, "dchunk": dchunk}
        _check_gradients(got, want, half, h.shape[0] * h.shape[1] * (h.shape[2] // groups), "batch %d" % batch)


def test_captured_and_replayed_beside_eager_calls(msd, cuda):
    import torch
    _, emb, blocks, dev = _blocks(torch, True, 2, cuda)
    packed = [msd.q4_pack(d["weight"], GROUP) for d in dev]
    flat = lambda out: [t for o in out for t in (o[0], o[1]) + o[3:]]  # noqa: E731
    _step(msd, emb, blocks, dev, packed, True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = flat(_step(msd, emb, blocks, dev, packed, True))
    for turn in range(4):
        emb.mul_(0.75)
        for d in dev:
            d["x"].add_(0.125 * turn)
        for t in captured:
            t.fill_(5.0)
        want = [t.clone() for t in flat(_step(msd, emb, blocks, dev, packed, True))]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), turn
