"""Plain forms, in 64 bits, of the channels-last GroupNorm, its 8-bit checkpoint and its gradient, for the tests.  Arrays are
float64 torch tensors [batch, positions, channels] on the CPU."""
import torch

BLOCK, TINY = 32, 1e-30


def silu(z):
    return z / (1 + torch.exp(-z))


def added(x, chunk, dtype):
    """x + chunk in the storage type, as float64."""
    x = x.to(dtype)
    return (x.float() + chunk.to(dtype).float()[:, None, :]).to(dtype).double() if chunk is not None else x.double()


def stats(h, groups, eps):
    b, p, c = h.shape
    g = h.reshape(b, p, groups, -1)
    mean = g.mean(dim=(1, 3))
    var = ((g - mean[:, None, :, None]) ** 2).mean(dim=(1, 3))
    return mean, (var + eps) ** -0.5


def _channels(v, c):
    """[batch, groups] -> [batch, 1, channels]"""
    return v.repeat_interleave(c // v.shape[1], dim=1)[:, None, :]


def forward(h, gamma, beta, groups, eps, act):
    mean, rstd = stats(h, groups, eps)
    c = h.shape[2]
    z = (h - _channels(mean, c)) * _channels(rstd, c) * gamma + beta
    return silu(z) if act else z


def checkpoint(h):
    """(codes, scales) of h, whose values are float32 or float16 ones; every step rounded to float32 as the definition has it."""
    b, p, c = h.shape
    blocks = torch.nn.functional.pad(h.float(), (0, -c % BLOCK)).reshape(b, p, -1, BLOCK)
    finite = torch.where(blocks.abs() <= torch.finfo(torch.float32).max, blocks.abs(), torch.zeros(()))
    most = finite.amax(dim=-1)
    empty = most < TINY
    inv = torch.where(empty, torch.zeros(()), torch.tensor(127.0) * (torch.tensor(1.0) / most))
    codes = torch.round(blocks * inv[..., None]).nan_to_num(-127.0).clamp(-127, 127).to(torch.int8)
    return codes.reshape(b, p, -1)[:, :, :c].contiguous(), torch.where(empty, torch.zeros(()), most * (torch.tensor(1.0) / torch.tensor(127.0)))


def restored(codes, scales):
    """What the codes stand for (the product is exact in 64 bits)."""
    c = codes.shape[2]
    return codes.double() * scales.double().repeat_interleave(BLOCK, dim=2)[:, :, :c]


def gradients(dy, h, mean, rstd, gamma, beta, groups, act):
    """dx, dgamma, dbeta, dchunk, and for each the sum of the magnitudes of its summands: what roundings are relative to."""
    b, p, c = dy.shape
    wide = lambda v: _channels(v, c)  # noqa: E731
    u = (h - wide(mean)) * wide(rstd)
    z = u * gamma + beta
    s = 1 / (1 + torch.exp(-z))
    dz = dy * s * (1 + z * (1 - s)) if act else dy
    # silu'(z) is computed from terms of size s and s |z| (1 - s), whose roundings do not cancel as they do
    size = dy.abs() * s * (1 + z.abs() * (1 - s)) if act else dy.abs()
    group_mean = lambda v: v.reshape(b, p, groups, -1).mean(dim=(1, 3))  # noqa: E731
    v = dz * gamma
    m1, m2 = wide(group_mean(v)), wide(group_mean(v * u))
    a1, a2 = wide(group_mean((size * gamma).abs())), wide(group_mean((size * gamma * u).abs()))
    r = wide(rstd)
    dx = r * (v - m1 - u * m2)
    dx_size = r * ((size * gamma).abs() + a1 + u.abs() * a2)
    return {"dx": (dx, dx_size), "dgamma": ((dz * u).sum((0, 1)), (size * u).abs().sum((0, 1))),
            "dbeta": (dz.sum((0, 1)), size.sum((0, 1))), "dchunk": (dx.sum(1), dx_size.sum(1))}
