"""Refusals of the channels-last GroupNorm calls and of the Linear rows with 4-bit weights, before anything is launched: through
the C ABI with addresses that are never dereferenced, and through the package with tensors that are not on a device."""
import ctypes

import pytest

p, f = ctypes.c_void_p, ctypes.c_float
X, Y, W, G, B, S, C, Q, T, DY, DX, DG, DB, DC = (p((i + 1) << 24) for i in range(14))
NULL = None
NEED = 1 << 22


def _forward(lib, x=X, chunk=NULL, y=Y, gamma=G, beta=B, batch=2, positions=16, channels=64, groups=8, dtype=1, stats=NULL,
             codes=NULL, scales=NULL, workspace=W, size=NEED):
    return lib.msd_groupnorm_channels_last(x, chunk, y, gamma, beta, batch, positions, channels, groups, f(1e-5), 1, dtype, stats,
                                           codes, scales, workspace, size, None)


def _backward(lib, dy=DY, x=X, chunk=NULL, codes=NULL, scales=NULL, stats=T, gamma=G, beta=B, dx=DX, dgamma=DG, dbeta=DB, dchunk=NULL,
              batch=2, positions=16, channels=64, groups=8, dtype=1, workspace=W, size=NEED):
    return lib.msd_groupnorm_channels_last_backward(dy, x, chunk, codes, scales, stats, gamma, beta, dx, dgamma, dbeta, dchunk, batch,
                                                    positions, channels, groups, 1, dtype, workspace, size, None)


def test_channels_last_forward(msd):
    lib = msd.load_library()
    shift = lambda a, n: p(a.value + n)  # noqa: E731
    bad = [dict(x=NULL), dict(y=NULL), dict(gamma=NULL), dict(beta=NULL), dict(groups=0), dict(groups=7), dict(channels=0),
           dict(dtype=2), dict(dtype=-1), dict(workspace=NULL), dict(size=7), dict(workspace=shift(W, 4)), dict(stats=shift(T, 4)),
           dict(codes=C), dict(scales=S),
           dict(batch=1 << 40, positions=1 << 30), dict(positions=1 << 31, batch=1), dict(batch=1 << 32, positions=1),
           dict(y=shift(X, 2)), dict(y=shift(X, 4094)), dict(x=shift(Y, 2)),                    # shifted
           dict(chunk=Y), dict(chunk=shift(Y, 4094)), dict(gamma=Y), dict(stats=Y), dict(workspace=Y), dict(workspace=X),
           dict(stats=X), dict(stats=G), dict(stats=W), dict(workspace=G),
           dict(codes=X, scales=S), dict(codes=Y, scales=S), dict(codes=C, scales=X), dict(codes=C, scales=shift(C, 2044)),
           dict(codes=C, scales=S, workspace=C), dict(chunk=C, codes=C, scales=S), dict(stats=C, codes=C, scales=S)]
    for change in bad:
        assert _forward(lib, **change) == 1, change
    assert _forward(lib, batch=0) == 0 and _forward(lib, positions=0, x=NULL, workspace=NULL) == 0


def test_channels_last_backward(msd):
    lib = msd.load_library()
    shift = lambda a, n: p(a.value + n)  # noqa: E731
    kept = dict(x=NULL, codes=C, scales=S)
    bad = [dict(dy=NULL), dict(x=NULL), dict(stats=NULL), dict(gamma=NULL), dict(beta=NULL), dict(dx=NULL), dict(dgamma=NULL),
           dict(dbeta=NULL), dict(groups=0), dict(groups=7), dict(dtype=3), dict(workspace=NULL), dict(size=64),
           dict(workspace=shift(W, 4)), dict(stats=shift(T, 4)), dict(codes=C), dict(codes=C, scales=S),  # x and codes
           dict(kept, chunk=Q), dict(kept, scales=NULL), dict(x=NULL, scales=S),
           dict(dx=shift(DY, 2)), dict(dx=X), dict(dx=G), dict(dx=T), dict(dx=W), dict(dx=DG), dict(chunk=DX), dict(kept, dx=C), dict(kept, dx=S),
           dict(dgamma=DY), dict(dgamma=DB), dict(dgamma=G), dict(dbeta=X), dict(dbeta=B), dict(dbeta=T),
           dict(dchunk=DY), dict(dchunk=DX), dict(dchunk=DG), dict(chunk=Q, dchunk=Q), dict(dchunk=W),
           dict(workspace=DY), dict(workspace=X), dict(workspace=T), dict(kept, workspace=C),
           dict(positions=1 << 31, batch=1), dict(batch=1 << 40, positions=1 << 30)]
    for change in bad:
        assert _backward(lib, **change) == 1, change
    assert _backward(lib, batch=0, dgamma=NULL, dbeta=NULL) == 0


def test_workspace_bytes(msd):
    lib = msd.load_library()
    size = ctypes.c_size_t(7)
    ask = lambda *a: lib.msd_groupnorm_channels_last_workspace(*a, ctypes.byref(size))  # noqa: E731
    assert ask(2, 4096, 320, 32, 1, 0) == 0 and 0 < size.value < 1 << 22
    forward = size.value
    assert ask(2, 4096, 320, 32, 1, 1) == 0 and size.value > forward
    assert ask(0, 4096, 320, 32, 1, 1) == 0 and size.value == 0
    assert ask(2, 4096, 320, 33, 1, 0) == 1 and ask(2, 4096, 320, 32, 5, 0) == 1 and ask(2, 1 << 31, 320, 32, 1, 0) == 1
    assert lib.msd_groupnorm_channels_last_workspace(2, 4096, 320, 32, 1, 0, None) == 1


def test_q4_calls(msd):
    lib = msd.load_library()
    shift = lambda a, n: p(a.value + n)  # noqa: E731

    def one(x=X, packed=Q, scales=S, bias=B, y=Y, m=2, n=16, k=128, group=32, act_in=0, act_out=0, dtype=1):
        return lib.msd_linear_rows_q4(x, packed, scales, bias, y, m, n, k, group, act_in, act_out, dtype, None)

    for change in (dict(x=NULL), dict(packed=NULL), dict(scales=NULL), dict(y=NULL), dict(m=9), dict(group=16), dict(group=0), dict(group=256),
                   dict(k=80), dict(k=96, group=64), dict(act_in=2), dict(act_out=-1), dict(dtype=2), dict(y=X), dict(y=shift(X, 510)),
                   dict(y=Q), dict(y=S), dict(y=B), dict(y=shift(Q, 1023)), dict(n=(1 << 28) + 1), dict(k=(1 << 28) + 128)):
        assert one(**change) == 1, change
    assert one(m=0, x=NULL) == 0 and one(n=0, y=NULL) == 0

    def grouped(y0, y1, q1=Q, s1=S, b1=B, ys=True):
        table = lambda a, b: (p * 2)(a, b)  # noqa: E731
        ns = (ctypes.c_size_t * 2)(16, 16)
        return lib.msd_linear_rows_q4_grouped(X, table(Q, q1), table(S, s1), table(B, b1), table(y0, y1) if ys else None, ns, 2, 2, 128, 32,
                                              0, 0, 1, None)

    assert grouped(Y, Y) == 1 and grouped(Y, shift(Y, 62)) == 1 and grouped(Y, DX, ys=False) == 1  # [2, 16] fp16: 64 bytes
    assert grouped(Y, DX, q1=shift(Y, 32)) == 1 and grouped(Y, DX, s1=shift(Y, 32)) == 1 and grouped(Y, DX, b1=shift(DX, 60)) == 1
    assert grouped(Y, X) == 1 and grouped(Y, NULL) == 1
    assert lib.msd_linear_rows_q4_grouped(None, None, None, None, None, None, 0, 2, 128, 32, 0, 0, 1, None) == 0

    def pack(w=X, packed=Q, scales=S, n=16, k=128, group=32, dtype=1):
        return lib.msd_q4_pack(w, packed, scales, n, k, group, dtype, None)

    for change in (dict(w=NULL), dict(packed=NULL), dict(scales=NULL), dict(group=48), dict(k=100), dict(dtype=7), dict(packed=X),
                   dict(scales=shift(X, 4)), dict(scales=shift(Q, 8)), dict(n=1 << 29)):
        assert pack(**change) == 1, change
    assert pack(n=0, w=NULL) == 0


def test_tensors_off_the_device_are_refused(msd):
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():  # (the checks ask for the current device)
        pytest.skip("no GPU in this environment")
    x, g = torch.zeros(2, 5, 16), torch.ones(16)
    with pytest.raises(msd.MsdError):
        msd.groupnorm_channels_last(x, g, g, 4)
    with pytest.raises(msd.MsdError):
        msd.linear_rows_q4(torch.zeros(2, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1))


@pytest.mark.gpu
def test_operands_that_do_not_fit(msd, cuda):
    import torch
    x = torch.zeros(2, 5, 16, device=cuda)
    g = torch.ones(16, device=cuda)
    nchw = torch.zeros(2, 16, 3, 4, device=cuda)
    y, kept = msd.groupnorm_channels_last_kept(x, g, g, 4)
    refused = [
        lambda: msd.groupnorm_channels_last(nchw, g, g, 4), lambda: msd.groupnorm_channels_last(x.transpose(1, 2), g, g, 4),
        lambda: msd.groupnorm_channels_last(x[0], g, g, 4), lambda: msd.groupnorm_channels_last(x.double(), g, g, 4),
        lambda: msd.groupnorm_channels_last(x.bfloat16(), g, g, 4), lambda: msd.groupnorm_channels_last(x, g.half(), g, 4),
        lambda: msd.groupnorm_channels_last(x, g, g[:8], 4), lambda: msd.groupnorm_channels_last(x, g, g, 3),
        lambda: msd.groupnorm_channels_last(x, g, g, 0), lambda: msd.groupnorm_channels_last(x, g, g, -4),
        lambda: msd.groupnorm_channels_last(x, g, g, 4, chunk=x[:, 0].half()), lambda: msd.groupnorm_channels_last(x, g, g, 4, chunk=x[:1, 0]),
        lambda: msd.groupnorm_channels_last(x, g, g, 4, out=x.half()), lambda: msd.groupnorm_channels_last(x, g, g, 4, out=x.view(5, 2, 16)),
        lambda: msd.groupnorm_channels_last_kept(x, g, g, 4, out=x), lambda: msd.groupnorm_channels_last_kept(x, g, g, 0),
        lambda: msd.groupnorm_channels_last(nchw.to(memory_format=torch.channels_last), g, g, 4, out=nchw),
        lambda: msd.groupnorm_channels_last_backward(x[:1], kept), lambda: msd.groupnorm_channels_last_backward(x.half(), kept),
        lambda: msd.groupnorm_channels_last_backward(x.cpu(), kept), lambda: msd.groupnorm_channels_last_backward(x, kept, out=kept.x),
        lambda: msd.groupnorm_channels_last_backward(x, kept._replace(stats=kept.stats[:1])),
    ]
    r, q, s = torch.zeros(2, 64, device=cuda), torch.zeros(4, 32, dtype=torch.uint8, device=cuda), torch.zeros(4, 1, device=cuda)
    refused += [
        lambda: msd.linear_rows_q4(r.half(), q, s), lambda: msd.linear_rows_q4(r, q.to(torch.int8), s), lambda: msd.linear_rows_q4(r, q[:, :16], s),
        lambda: msd.linear_rows_q4(r, q, s[:3]), lambda: msd.linear_rows_q4(r, q, torch.zeros(4, 4, device=cuda)),
        lambda: msd.linear_rows_q4(r, q, torch.zeros(4, 0, device=cuda)), lambda: msd.linear_rows_q4(r[0], q, s),
        lambda: msd.linear_rows_q4(r, q, s, g), lambda: msd.linear_rows_q4(r.t(), q, s), lambda: msd.linear_rows_q4(torch.zeros(9, 64, device=cuda), q, s),
        lambda: msd.linear_rows_q4(r, q.cpu(), s), lambda: msd.linear_rows_q4(r, q, s, out=torch.zeros(3, 4, device=cuda)),
        lambda: msd.linear_rows_q4(r, q, s, None, 2), lambda: msd.linear_rows_q4_grouped(r, [q, q], [s]),
        lambda: msd.linear_rows_q4_grouped(r, [q], [s], []), lambda: msd.linear_rows_q4_grouped(r, [q, q[:, :16]], [s, s]),
        lambda: msd.q4_pack(r, 48), lambda: msd.q4_pack(r, 128), lambda: msd.q4_pack(r[0], 32), lambda: msd.q4_pack(r.cpu(), 32),
        lambda: msd.q4_pack(r.double(), 32),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(msd.MsdError):
            call()
            pytest.fail("call %d was not refused" % i)


def test_launches_of_more_lanes_than_a_grid_holds(msd):
    lib, size = msd.load_library(), ctypes.c_size_t(0)
    for batch, positions, channels, fits in ((1 << 22, 8, 320, True), (1 << 24, 8, 320, False), (1 << 23, 4096, 320, False),
                                             (1 << 20, 1, 2560, True), (1 << 23, 4096, 32, False)):
        for backward in (0, 1):
            rc = lib.msd_groupnorm_channels_last_workspace(batch, positions, channels, 32, 1, backward, ctypes.byref(size))
            assert (rc == 0) == fits, (batch, positions, channels, backward)
    at = [p((i + 1) << 42) for i in range(4)]  # 2^28 columns of 1024: apart from each other
    assert lib.msd_linear_rows_q4(at[0], at[1], at[2], None, at[3], 1, 1 << 28, 1024, 128, 0, 0, 1, None) == 1
