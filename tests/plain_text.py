"""Token embedding, LayerNorm's gradient and attention with its gradient in 64 bits, from the formulas, and how far results in a
storage type may be from them.

Bounds: EPS = 2^-24 is half a step of float32, HALF[t] that of the storage type.  A float32 sum of n terms, whatever its order, is
within (n EPS) times the sum of the terms' sizes; the kernels add at most `steps` terms one after another."""
import math

import torch

EPS = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25}  # half the smallest step


# ---- token embedding -------------------------------------------------------------------
def embedding(ids, table, positions, scale):
    """(y, bound)"""
    dtype, vocab = table.dtype, table.shape[0]
    table = table.double()
    known = (ids >= 0) & (ids < vocab)
    y = torch.where(known[..., None], table[ids.clamp(0, vocab - 1)], 0.0) * scale
    size = y.abs()
    if positions is not None:
        p = positions[:ids.shape[-1]].double()
        y, size = y + p, size + p.abs()
    return y, HALF[dtype] * y.abs() + 2 * EPS * size + TINY[dtype]


def embedding_backward(dy, ids, vocab, positions, scale):
    """((dtable, bound), (dpositions, bound) or None)"""
    dtype, dim = dy.dtype, dy.shape[-1]
    flat, g = ids.reshape(-1), dy.double().reshape(-1, dim)
    known = (flat >= 0) & (flat < vocab)
    table, size = (torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, flat[known], t[known]) for t in (g * scale, (g * scale).abs()))
    steps = 64 + flat.numel() / 256 + 8
    out = table, HALF[dtype] * table.abs() + steps * EPS * size + TINY[dtype]
    if not positions:
        return out, None
    length = ids.shape[-1]
    whole, sizes = torch.zeros(2, positions, dim, dtype=torch.float64)
    if flat.numel():
        whole[:length], sizes[:length] = g.view(-1, length, dim).sum(0), g.abs().view(-1, length, dim).sum(0)
    steps = flat.numel() / max(1, length) + 4
    return out, (whole, HALF[dtype] * whole.abs() + steps * EPS * sizes + TINY[dtype])


# ---- LayerNorm's gradient ----------------------------------------------------------------
def layernorm_backward(dy, x, gamma, eps, dsum):
    """[(dx, bound), (dgamma, bound), (dbeta, bound)]"""
    dtype, (rows, dim) = dy.dtype, dy.shape
    d, x, g = dy.double(), x.double(), gamma.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    u, w = (x - mean) * rstd, d * g
    m1, m2 = w.mean(1, keepdim=True), (w * u).mean(1, keepdim=True)
    dx = rstd * (w - m1 - u * m2)
    # terms that a lane adds in a row, and the tree over the lanes
    n = (32 + dim / 256 + 10) * EPS
    du = 2 * n * u.abs() + n * rstd * x.abs().mean(1, keepdim=True) + 4 * EPS * rstd * x.abs()
    a1, a2 = w.abs().mean(1, keepdim=True), (w * u).abs().mean(1, keepdim=True)
    bound = rstd * (n * (w.abs() + a1 + u.abs() * a2) + du * a2 + u.abs() * (w.abs() * du).mean(1, keepdim=True)) + 3 * n * dx.abs()
    if dsum is not None:
        dx = dx + dsum.double()
        bound = bound + EPS * dsum.double().abs()
    steps = (rows / 64 + 16 + 140) * EPS  # rows of a lane, the teams, the partial sums
    dgamma, dbeta = (d * u).sum(0), d.sum(0)
    return [(dx, bound + HALF[dtype] * dx.abs() + TINY[dtype]),
            (dgamma, steps * (d * u).abs().sum(0) + (d.abs() * du).sum(0) + TINY[torch.float32]),
            (dbeta, steps * d.abs().sum(0) + TINY[torch.float32])]


# ---- attention ---------------------------------------------------------------------------
def visible(lq, lk, causal):
    seen = torch.ones(lq, lk, dtype=torch.bool)
    return seen.tril(lk - lq) if causal else seen


def attention_head(q, k, v, causal, scale, dout=None):
    """One query head of one sequence, q [lq, d], k and v [lk, d]: (out, bound) and, with dout, dq, dk, dv with theirs (before the
    storage type's rounding: see `rounded`)."""
    dtype = q.dtype
    weight_half = HALF[dtype] if dtype == torch.float16 else 0.0
    q, k, v = q.double(), k.double(), v.double()
    (lq, dim), lk = q.shape, k.shape[0]
    seen = visible(lq, lk, causal)
    score = torch.where(seen, scale * (q @ k.t()), -math.inf)
    size = torch.where(seen, scale * (q.abs() @ k.abs().t()), 0.0)
    top = score.amax(1, keepdim=True) if lk else torch.full((lq, 1), -math.inf, dtype=torch.float64)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(1, keepdim=True)
    p = torch.where(seen, e / torch.where(total == 0, 1.0, total), 0.0)

    # a score is a float32 sum of dim products and goes through a product and a difference more; the weights' sum takes in at
    # most lk / 32 terms one after another; exp2 and log2 are good to 2 steps
    score_off = (dim + 12) * EPS * (size.amax(1, keepdim=True) if lk else 0.0)
    weight_off = 2 * score_off + (lk / 32 + 40) * EPS
    out, out_size = p @ v, p @ v.abs()
    off = (weight_half + weight_off + (lk / 16 + 16) * EPS) * out_size + 2.0 ** -31 * v.abs().sum(0)
    # float32: a value's three bfloat16 have float32's exponents, and those below 2^-126 count as zero in a product: of a weight or
    # score gradient each is lost with at most 2^-126 of it, a term's loss is up to three of those times the other operand, and
    # weights below 2^-126, zero, take as much of dS as (dp - D) is large
    lost = 2.0 ** -124
    if dout is None:
        return (out, off),
    g = dout.double()
    dp, dp_size = g @ v.t(), g.abs() @ v.abs().t()
    stored = off + HALF[dtype] * (out.abs() + off) + TINY[dtype]
    delta, delta_off = (g * out).sum(1, keepdim=True), (g.abs() * stored).sum(1, keepdim=True) + dim * EPS * (g * out).abs().sum(1, keepdim=True)
    ds = torch.where(seen, p * (dp - delta), 0.0)
    ds_off = torch.where(seen, (weight_half + 2 * EPS) * ds.abs() + p * ((dim + 8) * EPS * dp_size + delta_off)
                         + weight_off * p * (dp.abs() + delta.abs()), 0.0)
    # (float16: what is far below the largest it can be keeps no digits)
    if weight_half:
        ds_off = ds_off + torch.where(seen, 2.0 ** -37 * ((g.norm(dim=1, keepdim=True) * v.norm(dim=1).amax() if lk else 0.0) + delta.abs().amax()), 0.0)
    if not weight_half:
        ds_off = ds_off + torch.where(seen, lost * (1 + dp.abs() + delta.abs()), 0.0)
    n = (max(lq, lk) / 16 + 40) * EPS
    dq, dq_off = scale * (ds @ k), scale * (ds_off + n * ds.abs()) @ k.abs()
    dk, dk_off = scale * (ds.t() @ q), scale * (ds_off + n * ds.abs()).t() @ q.abs()
    p_off = (weight_half + n) * p + weight_off * p + (2.0 ** -40 if weight_half else lost)
    dv, dv_off = p.t() @ g, torch.where(seen, p_off, 0.0).t() @ g.abs()
    return (out, off), (dq, dq_off), (dk, dk_off), (dv, dv_off)


def rounded(value, off, dtype):
    return value, off + HALF[dtype] * (value.abs() + off) + TINY[dtype]


def attention(q, k, v, causal, scale, dout=None, lengths=None):
    """Packed [rows, heads, dim] tensors on the CPU, lengths = [(queries, keys), ...]: [(out, bound), (dq, ..), (dk, ..), (dv, ..)]."""
    group = q.shape[1] // k.shape[1]
    shapes = (q, q, k, v) if dout is not None else (q,)
    got = [(torch.zeros(t.shape, dtype=torch.float64), torch.zeros(t.shape, dtype=torch.float64)) for t in shapes]
    q0 = k0 = 0
    for lq, lk in lengths:
        rows, keys = slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk
        if lq == 0 or lk == 0:
            continue
        for h in range(q.shape[1]):
            kh = h // group
            parts = attention_head(q[rows, h], k[keys, kh], v[keys, kh], causal, scale, None if dout is None else dout[rows, h])
            for n, ((value, off), (to, to_off)) in enumerate(zip(parts, got)):
                at, head = (rows, h) if n < 2 else (keys, kh)
                to[at, head] += value
                to_off[at, head] += off
    return [rounded(value, off, q.dtype) for value, off in got]


def check(got, want, what=""):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got - value).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d beyond their bound, worst %.3g times it (got %g, want %g)" % (
        what, int(bad.sum()), bad.numel(), float((off / bound)[bad].max()), float(got[bad][0]), float(value[bad][0]))
