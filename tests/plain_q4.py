"""Plain forms of the Linear rows with 4-bit weights, for the tests."""
import torch

TINY = 1e-30


def pack(w, group):
    """Codes [n, k] (0 ... 15) and scales of a float32 or float16 weight, every step rounded to float32 as the definition has it."""
    n, k = w.shape
    g = w.float().view(n, -1, group)
    finite = torch.where(torch.isfinite(g), g.abs(), torch.zeros(()))
    most = finite.amax(-1)
    scale = torch.where(most < TINY, torch.zeros(()), (most / torch.tensor(7.0)).to(w.dtype).float())
    inv = torch.where(scale > 0, torch.tensor(1.0) / scale, torch.zeros(()))
    codes = torch.round(g * inv[..., None]).nan_to_num(-7.0).clamp(-7, 7) + 8
    return codes.view(n, k).to(torch.uint8), scale.to(w.dtype)


def bytes_of(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def linear(x, codes, scales, bias, act_in, act_out):
    """y in 64 bits, and what roundings of its sum are relative to: the sum of the summands' magnitudes."""
    x = x.double()
    if act_in:
        x = x / (1 + torch.exp(-x))
    group = codes.shape[1] // scales.shape[1]
    w = (codes.double() - 8) * scales.double().repeat_interleave(group, dim=1)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    if act_out:
        z = y
        y = z / (1 + torch.exp(-z))
        size = 1.1 * size + (1 + z.abs()) * y.abs()  # (SiLU's slope is below 1.1; its own roundings)
    return y, size
