"""The native calls of csrc/torch_calls_cl_q4.cpp against their general path: the same bits, layouts and refusals; which calls the
extension makes; that it uses the current stream."""
import pytest

from test_gpu_torch_calls import _General, _Recorder

pytestmark = pytest.mark.gpu


def _cases(torch, msd, cuda, half):
    g = torch.Generator(device=cuda).manual_seed(5)
    dtype = torch.float16 if half else torch.float32

    def rnd(*shape):
        return torch.randn(shape, device=cuda, generator=g).to(dtype)

    def floats(n):
        return torch.randn(n, device=cuda, generator=g)

    image = rnd(2, 64, 8, 6).to(memory_format=torch.channels_last)
    x, emb, gamma, beta = rnd(2, 48, 64), rnd(2, 64), floats(64), floats(64)
    odd = image[:1, :, :1, :1]  # strides that a new tensor would not have
    keeps = [(x, gamma, beta, 8), (image, gamma, beta, 32, 1e-3, True, emb, True), (x, gamma, beta, 8, 1e-5, True, emb, False),
             (x, gamma, beta, 8, 1e-5, False, None, False, x), (x.clone(), gamma, beta, 8, 1e-5, False, None, True, torch.empty_like(x)),
             (x, gamma, beta, 0), (x, gamma, beta, 7), (x.double(), gamma, beta, 8), (x[:0], gamma, beta, 8)]
    norms = [(x, gamma, beta, 8), (image, gamma, beta, 8, 1e-3, True), (image, gamma, beta, 8, 1e-3, True, emb),
             (x, gamma, beta, 8, 1e-3, False, None, torch.empty_like(x)), (x, gamma, beta, 7), (x, gamma[:63], beta, 8), (x, gamma.half(), beta, 8),
             (x.cpu(), gamma, beta, 8), (image.contiguous(), gamma, beta, 8), (image, gamma, beta, 8, 1e-3, True, emb[:1]), (odd, gamma, beta, 8),
             (x, gamma, beta, -1), (x, gamma, beta, 2.0), (x, gamma, beta, 8, 1e-3, 1), (x[0], gamma, beta, 8), (image[:0], gamma, beta, 8),
             (image, gamma, beta, 8, 1e-3, False, None, torch.empty_like(image).contiguous()), (x, None, beta, 8),
             (x, torch.nn.Parameter(gamma), beta, 8), (x, gamma, beta, 8, 1e-3, False, rnd(128)), (x, gamma, beta, 8, 1e-3, False, x.view(-1)[:128].view(2, 64), x)]
    kept = msd.groupnorm_channels_last_kept(image, gamma, beta, 8, 1e-5, True, emb)[1]
    kept8 = msd.groupnorm_channels_last_kept(image, gamma, beta, 8, 1e-5, True, emb, True)[1]
    plain = msd.groupnorm_channels_last_kept(x, gamma, beta, 8)[1]
    backs = [(image, kept), (image, kept8), (x, plain), (x, plain, False), (image, kept, True, torch.empty_like(image)), (image, kept8, True, image.clone()),
             (x, kept), (image[:1], kept), (image.contiguous(), kept), (x, plain._replace(stats=plain.stats[:1])), (x.cpu(), plain),
             (x, plain._replace(groups=0)), (x, plain, 1)]
    rows = rnd(6, 64)
    q = [torch.randint(0, 256, (n, 32), device=cuda, generator=g, dtype=torch.uint8) for n in (3, 40, 1)]
    s, bs, e = [rnd(n, 2) for n in (3, 40, 1)], [floats(3), None, floats(1)], msd.ACT_SILU
    linears = [(rows, q[1], s[1]), (rows, q[1], s[1], None, e, e), (rows, q[0], s[0], bs[0], 0, 0, rnd(6, 3)), (rows, q[0], s[0], bs[0], 0, 0, rnd(6, 4)),
               (rows, q[0], s[0], bs[2]), (rows, q[0], s[1]), (rows, q[0], s[0].double()), (rnd(9, 64), q[0], s[0]), (rows, q[0], s[0], None, 3),
               (x, q[0], s[0]), (rows, q[0][:, :31], s[0]), (rows, q[0], rnd(3, 1)), (rows, q[0], rnd(3, 4)), (rows, q[0], rnd(3, 0)), (rows[:0], q[0], s[0])]
    groups = [(rows, q, s), (rows, q, s, bs, e), (rows, tuple(q), s, bs), (rows, q, s, bs[:1]), (rows, [], []), (rnd(9, 64), q, s),
              (rows, q, s, [None] * 3, 0, e), (rows, q, [s[0], s[1], rnd(1, 1)]), (rows, q, s[:2])]
    return {"groupnorm_channels_last": (norms, {0, 1, 2, 3, 15, 18, 19, 20}), "groupnorm_channels_last_kept": (keeps, {0, 1, 2, 4, 8}),
            "groupnorm_channels_last_backward": (backs, {0, 1, 2, 3, 4, 5}), "linear_rows_q4": (linears, {0, 1, 2, 7, 8, 11, 14}),
            "linear_rows_q4_grouped": (groups, {0, 1, 5, 6})}


def _flat(v):
    if isinstance(v, (list, tuple)):
        return [t for x in v for t in _flat(x)]
    return [v]


def _outcome(f, args):
    try:
        got = f(*args)
    except Exception as e:  # (TypeError, MsdError, ctypes.ArgumentError, ...)
        return type(e).__name__
    return [type(got).__name__] + [t.clone() if hasattr(t, "clone") else t for t in _flat(got)]


@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_native_calls_are_the_general_ones(msd, cuda, half, monkeypatch):
    import torch
    native, general = _cases(torch, msd, cuda, half), _cases(torch, msd, cuda, half)  # (some calls write into what later ones read)
    made = msd._bind_native_cl_q4()
    assert {n for n in dir(made) if not n.startswith("__")} - {"bind", "names", "built_for"} == set(native)
    for name, (calls, plain) in native.items():
        for i, args in enumerate(calls):
            recorder = _Recorder(made)
            with monkeypatch.context() as m:
                m.setattr(msd, "_native_cl_q4", recorder)
                a = _outcome(getattr(msd, name), args)
            with monkeypatch.context() as m:
                m.setattr(msd, "_native_cl_q4", _General())
                b = _outcome(getattr(msd, name), general[name][0][i])
            assert ((name, True) in recorder.made) == (i in plain), (name, i)
            assert type(a) is type(b) and len(a) == len(b) and (a == b if isinstance(a, str) else a[0] == b[0]), (name, i, a, b)
            for s, t in zip(a[1:], b[1:]) if not isinstance(a, str) else ():
                if isinstance(s, torch.Tensor):
                    assert s.dtype == t.dtype and s.shape == t.shape and s.stride() == t.stride(), (name, i)
                    assert torch.equal(s.nan_to_num(7.0) if s.is_floating_point() else s, t.nan_to_num(7.0) if t.is_floating_point() else t), (name, i)
                else:
                    assert s == t, (name, i)


def test_native_calls_use_the_current_stream(msd, cuda):
    """The operand is written behind work that takes far longer than the host needs to reach the call's launch."""
    import torch
    stream = torch.cuda.Stream()
    g, b = torch.ones(64, device=cuda), torch.zeros(64, device=cuda)
    q, s = torch.full((64, 32), 0x99, device=cuda, dtype=torch.uint8), torch.ones((64, 2), device=cuda)  # weights of one
    msd.groupnorm_channels_last(torch.ones(1, 4, 64, device=cuda), g, b, 8)
    with torch.cuda.stream(stream):
        big, x = torch.empty(1 << 28, device=cuda), torch.full((4, 64), -1.0, device=cuda)
        for k in range(1, 4):
            x.fill_(-1.0)
            stream.synchronize()
            for _ in range(16):
                big.fill_(float(k))
            x.fill_(float(k))
            waits = not stream.query()
            y, z = msd.linear_rows_q4(x, q, s), msd.groupnorm_channels_last(x[None], g, b + k, 8, 1e-5, False, None)
            assert waits and bool((y == 64.0 * k).all()) and bool((z == float(k)).all())


def test_native_calls_leave_subclasses_and_modes(msd, cuda):
    import torch
    native = msd._bind_native_cl_q4()
    x, g = torch.randn(1, 4, 64, device=cuda), torch.ones(64, device=cuda)

    class Sub(torch.Tensor):
        pass

    assert native.groupnorm_channels_last(x.as_subclass(Sub), g, g, 8, 1e-5, False, None, None) is None
    assert native.groupnorm_channels_last(x, g, g, 8) is None and native.linear_rows_q4() is None
    with torch.device(cuda):
        assert native.groupnorm_channels_last(x, g, g, 8, 1e-5, False, None, None) is None
        under_mode = msd.groupnorm_channels_last(x, g, g, 8)
    assert torch.equal(under_mode, msd.groupnorm_channels_last(x, g, g, 8))
