"""Timed cases of the channels-last GroupNorm, its gradient, its 8-bit checkpoint and the Linear rows with 4-bit weights.

Five kinds of pass:

  norm           GroupNorm over channels-last tensors, with or without the embedding add in front and SiLU behind
  train          the same as a training step has it: forward, then the gradients from dy and what the forward kept
  train8         ... where the forward keeps its input in 8 bits (blocks of 32 channels with one scale)
  rows4          a Linear layer on a few rows, its weight in 4 bits with one scale per 32, 64 or 128 of them
  rows4_grouped  several such layers on the same rows (the per-ResBlock projections of the time embedding)

Latents of a 512-pixel image are 64 x 64 with 320 channels; the UNet halves the sides three times (other aspect ratios
give odd ones) and goes up to 2560 channels; the decoder ends at 512 x 512 with 128.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "f32": torch.float32}
BLOCK = 32        # channels of one position that share a scale in the 8-bit checkpoint
TINY = 1e-30      # a block whose largest value is below this is kept as zeros
EPS = 1e-5

# output channels of the 22 ResBlocks of one UNet step, in execution order
RESBLOCK_COUT = [320, 320, 640, 640] + [1280] * 12 + [640] * 3 + [320] * 3


# ----------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------
def listed():
    return [
        # the deepest level, one sample: the smallest norm there is
        {"name": "norm_1280_8x8_b1_f16", "kind": "norm", "batch": 1, "channels": 1280, "h": 8, "w": 8, "groups": 32,
         "add": False, "silu": True, "dtype": "f16"},
        # a ResBlock's out-norm, one image with guidance: the embedding add, the norm, SiLU
        {"name": "norm_320_64x64_b2_f16", "kind": "norm", "batch": 2, "channels": 320, "h": 64, "w": 64, "groups": 32,
         "add": True, "silu": True, "dtype": "f16"},
        # the decoder's last level at full resolution, the largest tensors of the path
        {"name": "norm_128_512x512_b1_f32", "kind": "norm", "batch": 1, "channels": 128, "h": 512, "w": 512, "groups": 32,
         "add": False, "silu": True, "dtype": "f32"},
        # the deepest level of a 576 x 448 image, two samples, after a skip concatenation: 63 positions
        {"name": "train_2560_9x7_b2_f32", "kind": "train", "batch": 2, "channels": 2560, "h": 9, "w": 7, "groups": 32,
         "add": False, "silu": True, "dtype": "f32"},
        # fine-tuning the widest level, eight images, gradients of the embedding add among them
        {"name": "train_320_64x64_b8_f16", "kind": "train", "batch": 8, "channels": 320, "h": 64, "w": 64, "groups": 32,
         "add": True, "silu": True, "dtype": "f16"},
        # the second level in float32, four images, the norm's input kept in 8 bits
        {"name": "train8_640_32x32_b4_f32", "kind": "train8", "batch": 4, "channels": 640, "h": 32, "w": 32, "groups": 32,
         "add": True, "silu": True, "dtype": "f32"},
        # the widest level at a batch that needs the memory
        {"name": "train8_320_64x64_b16_f16", "kind": "train8", "batch": 16, "channels": 320, "h": 64, "w": 64, "groups": 32,
         "add": True, "silu": True, "dtype": "f16"},
        # the second layer of the time embedding, one row
        {"name": "rows4_1280x1280_m1_f16", "kind": "rows4", "m": 1, "n": 1280, "k": 1280, "group": 64, "act_in": False,
         "act_out": False, "bias": True, "dtype": "f16"},
        # float32 as the framework ships it, an odd number of columns, three rows, SiLU on both sides
        {"name": "rows4_1237x2048_m3_f32", "kind": "rows4", "m": 3, "n": 1237, "k": 2048, "group": 32, "act_in": True,
         "act_out": True, "bias": True, "dtype": "f32"},
        # a large generic layer at the most rows
        {"name": "rows4_16384x8192_m8_f16", "kind": "rows4", "m": 8, "n": 16384, "k": 8192, "group": 128, "act_in": False,
         "act_out": False, "bias": False, "dtype": "f16"},
        # SiLU(embedding) through the projections of all 22 ResBlocks of a step, one image with guidance
        {"name": "rows4_22_projections_m2_f16", "kind": "rows4_grouped", "m": 2, "layers": 22, "k": 1280, "group": 64,
         "act_in": True, "bias": True, "seed_n": 0, "dtype": "f16"},
        # the same for eight rows in float32
        {"name": "rows4_22_projections_m8_f32", "kind": "rows4_grouped", "m": 8, "layers": 22, "k": 1280, "group": 32,
         "act_in": True, "bias": True, "seed_n": 0, "dtype": "f32"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "train", "train8", "rows4", "rows4", "rows4_grouped"])
    dtype = rng.choice(["f16", "f32"])
    if kind in ("norm", "train", "train8"):
        groups = rng.choice([32, 32, 32, 16, 8, 1])
        per_group = rng.choice([1, 2, 3, 4, 5, 8, 10, 15, 20, 30, 40, 60, 80])
        if groups < 32:
            per_group = min(2560, per_group * 32) // groups + rng.randint(0, 3)
        channels = groups * max(1, per_group)
        batch = rng.choice([1, 2, 2, 3, 4, 8, 16])
        most = (33_000_000 if kind == "norm" else 12_000_000) // (batch * channels)
        positions = _log_int(rng, 1, max(1, min(512 * 512, most)))
        w = max(1, min(512, int(math.sqrt(positions)) + rng.randint(-1, 1)))
        return {"kind": kind, "batch": batch, "channels": channels, "h": max(1, positions // w), "w": w, "groups": groups,
                "add": rng.random() < 0.5, "silu": rng.random() < 0.75, "dtype": dtype}
    group = rng.choice([32, 64, 128])
    m = rng.randint(1, 8)
    if kind == "rows4":
        k = group * _log_int(rng, 1, 8192 // group)
        return {"kind": kind, "m": m, "n": _log_int(rng, 1, 16384), "k": k, "group": group, "act_in": rng.random() < 0.5,
                "act_out": rng.random() < 0.3, "bias": rng.random() < 0.6, "dtype": dtype}
    return {"kind": kind, "m": m, "layers": rng.randint(1, 40), "k": group * _log_int(rng, 1, 2560 // group), "group": group,
            "act_in": rng.random() < 0.7, "bias": rng.random() < 0.7, "seed_n": rng.randint(1, 1 << 20), "dtype": dtype}


def _columns(case):
    """Output columns of each layer of a grouped case."""
    if case["seed_n"] == 0:
        return RESBLOCK_COUT[:case["layers"]]
    return [1 + (case["seed_n"] * (i + 7) * 2654435761 >> 7) % 1500 for i in range(case["layers"])]


# ----------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------
def _weight4(gen, n, k, group, dtype):
    """Codes as a trained layer's have them (around the middle, few at the ends) and scales that give a unit output."""
    q = (torch.randn((n, k), device="cuda", generator=gen) * 2.5 + 8).round_().clamp_(0, 15).to(torch.uint8)
    packed = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
    scales = (torch.rand((n, k // group), device="cuda", generator=gen) + 0.5) * (0.4 / math.sqrt(k))
    return packed, scales.to(dtype)


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s = {"case": case}
    if own:
        s["msd"] = importlib.import_module("mobile-stable-diffusion_amd")
    if case["kind"] in ("norm", "train", "train8"):
        b, c, h, w = case["batch"], case["channels"], case["h"], case["w"]
        # channels of a trained network differ in level and spread
        x = normal(b, h, w, c) * (0.5 + torch.rand(c, device="cuda", generator=gen)) + 0.5 * normal(c)
        s["x"] = x.to(dtype).permute(0, 3, 1, 2)
        s["chunk"] = (0.5 * normal(b, c)).to(dtype) if case["add"] else None
        s["gamma"], s["beta"] = 1 + 0.2 * normal(c), 0.2 * normal(c)
        if case["kind"] != "norm":
            s["dy"] = normal(b, h, w, c).to(dtype).permute(0, 3, 1, 2)
        return s
    m, k, group = case["m"], case["k"], case["group"]
    s["x"] = normal(m, k).to(dtype)
    columns = [case["n"]] if case["kind"] == "rows4" else _columns(case)
    pairs = [_weight4(gen, n, k, group, dtype) for n in columns]
    s["packed"], s["scales"] = [p for p, _ in pairs], [t for _, t in pairs]
    s["biases"] = [0.1 * normal(n) for n in columns] if case["bias"] else None
    return s


# ----------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------
def _positions_last(t):
    """[batch, positions, channels] of a channels-last [batch, channels, h, w]."""
    return t.permute(0, 2, 3, 1).reshape(t.shape[0], -1, t.shape[1])


def _like_image(t, x):
    b, c, h, w = x.shape
    return t.view(b, h, w, c).permute(0, 3, 1, 2)


def _plain_norm(s):
    """y and what the gradient needs, all in float32 but for y."""
    case, x = s["case"], s["x"]
    h = _positions_last(x)
    b, p, c = h.shape
    if s["chunk"] is not None:
        h = (h.float() + s["chunk"].float()[:, None, :]).to(x.dtype)
    h = h.float()
    grouped = h.view(b, p, case["groups"], -1)
    mean = grouped.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((grouped - mean).square().mean(dim=(1, 3), keepdim=True) + EPS)
    normed = ((grouped - mean) * rstd).view(b, p, c)
    z = normed * s["gamma"] + s["beta"]
    y = z / (1 + torch.exp(-z)) if case["silu"] else z
    return _like_image(y.to(x.dtype), x), h, mean, rstd, normed


def _plain_checkpoint(h):
    """h through the 8-bit checkpoint and back."""
    c = h.shape[-1]
    padded = torch.nn.functional.pad(h, (0, -c % BLOCK)).unflatten(-1, (-1, BLOCK))
    most = padded.abs().amax(dim=-1, keepdim=True)
    empty = most < TINY
    inv = torch.where(empty, torch.zeros_like(most), 127.0 / most)
    codes = torch.round(padded * inv).clamp(-127, 127).to(torch.int8)
    scale = torch.where(empty, torch.zeros_like(most), most / 127.0)
    return (codes.float() * scale).flatten(-2)[..., :c]


def _plain_train(s):
    case, x = s["case"], s["x"]
    y, h, mean, rstd, normed = _plain_norm(s)
    b, p, c = h.shape
    groups = case["groups"]
    if case["kind"] == "train8":
        normed = ((_plain_checkpoint(h).view(b, p, groups, -1) - mean) * rstd).view(b, p, c)
    dz = _positions_last(s["dy"]).float()
    if case["silu"]:
        z = normed * s["gamma"] + s["beta"]
        sig = 1 / (1 + torch.exp(-z))
        dz = dz * sig * (1 + z * (1 - sig))
    d_gamma, d_beta = (dz * normed).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    dn = (dz * s["gamma"]).view(b, p, groups, -1)
    normed = normed.view(b, p, groups, -1)
    m1, m2 = dn.mean(dim=(1, 3), keepdim=True), (dn * normed).mean(dim=(1, 3), keepdim=True)
    dx = (rstd * (dn - m1 - normed * m2)).view(b, p, c)
    out = {"y": y, "dx": _like_image(dx.to(x.dtype), x), "dgamma": d_gamma, "dbeta": d_beta}
    if case["add"]:
        out["dchunk"] = dx.sum(dim=1).to(x.dtype)
    return out


def _plain_rows4(s, packed, scales, bias):
    case, x = s["case"], s["x"].float()
    n = packed.shape[0]
    if case["act_in"]:
        x = x / (1 + torch.exp(-x))
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).view(n, -1, case["group"])
    w = ((codes.float() - 8) * scales.float()[:, :, None]).view(n, -1)
    y = x @ w.t()
    if bias is not None:
        y = y + bias
    if case.get("act_out"):
        y = y / (1 + torch.exp(-y))
    return y.to(s["x"].dtype)


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "norm":
        return _plain_norm(s)[0]
    if kind in ("train", "train8"):
        return _plain_train(s)
    biases = s["biases"] or [None] * len(s["packed"])
    outs = [_plain_rows4(s, q, t, b) for q, t, b in zip(s["packed"], s["scales"], biases)]
    return outs[0] if kind == "rows4" else outs


def _own(s):
    msd, case, kind = s["msd"], s["case"], s["case"]["kind"]
    if kind == "norm":
        return msd.groupnorm_channels_last(s["x"], s["gamma"], s["beta"], case["groups"], EPS, case["silu"], s["chunk"])
    if kind in ("train", "train8"):
        y, kept = msd.groupnorm_channels_last_kept(s["x"], s["gamma"], s["beta"], case["groups"], EPS, case["silu"], s["chunk"],
                                                   keep8=kind == "train8")
        dx, d_gamma, d_beta, d_chunk = msd.groupnorm_channels_last_backward(s["dy"], kept)
        out = {"y": y, "dx": dx, "dgamma": d_gamma, "dbeta": d_beta}
        if case["add"]:
            out["dchunk"] = d_chunk
        return out
    act_in = msd.ACT_SILU if case["act_in"] else msd.ACT_NONE
    if kind == "rows4":
        act_out = msd.ACT_SILU if case["act_out"] else msd.ACT_NONE
        bias = s["biases"][0] if s["biases"] else None
        return msd.linear_rows_q4(s["x"], s["packed"][0], s["scales"][0], bias, act_in, act_out)
    return msd.linear_rows_q4_grouped(s["x"], s["packed"], s["scales"], s["biases"], act_in)


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "f16" else 4
    if case["kind"] in ("norm", "train", "train8"):
        rows = case["batch"] * case["h"] * case["w"]
        n = rows * case["channels"]
        vectors = 2 * 4 * case["channels"] + (size * case["batch"] * case["channels"] if case["add"] else 0)
        codes = n + 4 * rows * -(-case["channels"] // BLOCK)
        # elementwise operations per value, exponentials counted as one
        if case["kind"] == "norm":
            return {"bytes": 2 * size * n + vectors, "flops": 12 * n}
        if case["kind"] == "train":
            return {"bytes": 5 * size * n + 4 * vectors, "flops": 40 * n}
        return {"bytes": 4 * size * n + 2 * codes + 4 * vectors, "flops": 46 * n}
    columns = case["n"] if case["kind"] == "rows4" else sum(_columns(case))
    m, k = case["m"], case["k"]
    return {"bytes": columns * (k // 2 + size * (k // case["group"]) + size * m + (4 if case["bias"] else 0)) + size * m * k,
            "flops": 2 * m * k * columns}


# ----------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ----------------------------------------------------------------------------------------
def _exact_sigmoid(v):
    e = torch.exp(-v.abs())
    return torch.where(v >= 0, 1 / (1 + e), e / (1 + e))


def _exact_kept(h, dtype):
    """Values an 8-bit checkpoint of h [positions, channels] stands for: whole steps of the block's largest value / 127, the
    quotient, the product and the scale rounded to float32 as the definition has it."""
    got = torch.zeros_like(h)
    for first in range(0, h.shape[1], BLOCK):
        block = h[:, first:first + BLOCK].to(torch.float32)
        most = block.abs().max(dim=1).values
        live = most >= TINY
        if not bool(live.any()):
            continue
        steps = (127.0 / most[live])[:, None] * block[live]
        got[live, first:first + BLOCK] = steps.round().double() * (most[live] / 127.0).double()[:, None]
    return got


def _exact_norm_sample(case, s, b):
    """Outputs of one sample: y, and for a training step dx and the per-channel sums."""
    groups, dtype = case["groups"], s["x"].dtype
    c = case["channels"]
    h = s["x"][b].double().reshape(c, -1).t()
    if s["chunk"] is not None:
        h = (h + s["chunk"][b].double()).to(dtype).double()
    per, n = c // groups, h.shape[0] * (c // groups)
    of_group = torch.arange(c, device=h.device) // per

    def over_group(v):  # channel sums -> sums of the channel's group, one per channel
        return torch.zeros(groups, dtype=torch.float64, device=v.device).index_add_(0, of_group, v)[of_group]

    mean = over_group(h.sum(0)) / n
    rstd = (over_group(((h - mean) ** 2).sum(0)) / n + EPS) ** -0.5
    gamma, beta = s["gamma"].double(), s["beta"].double()
    z = (h - mean) * (rstd * gamma) + beta
    y = z * _exact_sigmoid(z) if case["silu"] else z
    if case["kind"] == "norm":
        return (y,)
    if case["kind"] == "train8":
        h = _exact_kept(h, dtype)
        z = (h - mean) * (rstd * gamma) + beta
    u = (h - mean) * rstd
    g = s["dy"][b].double().reshape(c, -1).t()
    if case["silu"]:
        sig = _exact_sigmoid(z)
        g = g * (sig + z * sig * _exact_sigmoid(-z))
    to_beta, to_gamma = g.sum(0), (g * u).sum(0)
    v = g * gamma
    dx = (v - over_group(v.sum(0)) / n - u * (over_group((v * u).sum(0)) / n)) * rstd
    return y, dx, to_gamma, to_beta, dx.sum(0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "train", "train8"):
        shape = s["x"].shape[1:]
        samples = [_exact_norm_sample(case, s, b) for b in range(case["batch"])]

        def image(i):
            return torch.stack([t[i].t().reshape(shape) for t in samples])

        if case["kind"] == "norm":
            return image(0)
        out = {"y": image(0), "dx": image(1), "dgamma": sum(t[2] for t in samples), "dbeta": sum(t[3] for t in samples)}
        if case["add"]:
            out["dchunk"] = torch.stack([t[4] for t in samples])
        return out
    x = s["x"].double()
    if case["act_in"]:
        x = x * _exact_sigmoid(x)
    outs = []
    for i, (packed, scales) in enumerate(zip(s["packed"], s["scales"])):
        y = torch.zeros((x.shape[0], packed.shape[0]), dtype=torch.float64, device=x.device)
        half = case["group"] // 2
        for j in range(scales.shape[1]):  # one group of weights after the other
            part = packed[:, j * half:(j + 1) * half].long()
            w = torch.empty((packed.shape[0], case["group"]), dtype=torch.float64, device=x.device)
            w[:, 0::2], w[:, 1::2] = (part % 16 - 8).double(), (part // 16 - 8).double()
            y += (x[:, j * case["group"]:(j + 1) * case["group"]] @ w.t()) * scales[:, j].double()
        if s["biases"] is not None:
            y = y + s["biases"][i].double()
        outs.append(y * _exact_sigmoid(y) if case.get("act_out") else y)
    return outs[0] if case["kind"] == "rows4" else outs
