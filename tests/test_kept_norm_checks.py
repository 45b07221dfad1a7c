"""groupnorm_channels_last_backward checks everything that a KeptNorm hands to the kernels, before anything is launched: on the
CPU, with tensors that only say that they are on a device and a library that records what would be launched."""
import pytest

torch = pytest.importorskip("torch")


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on device 0."""
    is_cuda = True

    def get_device(self):
        return 0


def _on(t):
    return t.as_subclass(OnDevice)


class Library:
    """Stands for the loaded library: workspaces as it says, gradients recorded and not made."""

    def __init__(self, lib):
        self.lib, self.made = lib, []

    def msd_groupnorm_channels_last_backward(self, *args):
        self.made.append(args)
        return 0

    def __getattr__(self, name):
        return getattr(self.lib, name)


@pytest.fixture
def library(msd, monkeypatch):
    lib = Library(msd.load_library())
    monkeypatch.setattr(msd, "_lib", lib)
    monkeypatch.setattr(msd, "_native_cl_q4", msd._NoNative())
    monkeypatch.setattr(msd, "_stream", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return lib


def _kept(msd, b, p, c, groups, keep8):
    g = _on(torch.ones(c))
    x = codes = scales = None
    if keep8:
        codes, scales = _on(torch.zeros((b, p, c), dtype=torch.int8)), _on(torch.zeros((b, p, -(-c // 32))))
    else:
        x = _on(torch.zeros((b, p, c)))
    return msd.KeptNorm(x, None, codes, scales, _on(torch.ones((b, groups, 2))), g, _on(torch.zeros(c)), groups, True, False)


def test_a_kept_norm_that_fits_is_taken(msd, library):
    for keep8 in (False, True):
        msd.groupnorm_channels_last_backward(_on(torch.zeros(2, 5, 48)), _kept(msd, 2, 5, 48, 8, keep8))
    assert len(library.made) == 2


@pytest.mark.parametrize("change", [
    dict(scales=torch.zeros((2, 5, 2), dtype=torch.float16)), dict(scales=torch.zeros((2, 5, 2), dtype=torch.float64)),
    dict(scales=torch.zeros(2, 5, 1)), dict(scales=torch.zeros(2, 4, 2)), dict(scales=torch.zeros(2, 5, 3)), dict(scales=torch.zeros(0)),
    dict(scales=torch.zeros(2, 2, 5).transpose(1, 2)),
    dict(codes=torch.zeros((2, 5, 48), dtype=torch.uint8)), dict(codes=torch.zeros((2, 5, 48), dtype=torch.float16)),
    dict(codes=torch.zeros((2, 5, 47), dtype=torch.int8)), dict(codes=torch.zeros((1, 5, 48), dtype=torch.int8)),
    dict(codes=torch.zeros((2, 48, 5), dtype=torch.int8).transpose(1, 2)),
    dict(stats=torch.ones(2, 7, 2)), dict(stats=torch.ones((2, 8, 2), dtype=torch.float16)), dict(gamma=torch.ones(47)),
    dict(beta=torch.ones(48, dtype=torch.float16)), dict(groups=7), dict(groups=0),
], ids=lambda change: "-".join("%s %s %s" % (k, getattr(v, "dtype", v), tuple(getattr(v, "shape", ()))) for k, v in change.items()))
def test_kept_codes_and_scales_that_do_not_fit_are_refused(msd, library, change):
    kept = _kept(msd, 2, 5, 48, 8, True)._replace(**{k: _on(v) if torch.is_tensor(v) else v for k, v in change.items()})
    with pytest.raises(msd.MsdError):
        msd.groupnorm_channels_last_backward(_on(torch.zeros(2, 5, 48)), kept)
    assert not library.made


@pytest.mark.parametrize("name", ["codes", "scales"])
def test_codes_and_scales_elsewhere_are_refused(msd, library, name):
    kept = _kept(msd, 2, 5, 48, 8, True)
    with pytest.raises(msd.MsdError):
        msd.groupnorm_channels_last_backward(_on(torch.zeros(2, 5, 48)), kept._replace(**{name: getattr(kept, name).as_subclass(torch.Tensor)}))
    assert not library.made


@pytest.mark.gpu
def test_refused_on_the_device_too(msd, cuda):
    x, g = torch.randn(2, 5, 48, device=cuda), torch.ones(48, device=cuda)
    _, kept = msd.groupnorm_channels_last_kept(x, g, g, 8, keep8=True)
    for change in (dict(scales=kept.scales.half()), dict(scales=kept.scales[:1]), dict(scales=kept.scales.cpu()), dict(codes=kept.codes.view(torch.uint8)),
                   dict(codes=kept.codes.cpu())):
        with pytest.raises(msd.MsdError):
            msd.groupnorm_channels_last_backward(x, kept._replace(**change))


def test_gradients_of_gamma_and_beta_are_vectors_whatever_theirs_are(msd, library):
    kept = _kept(msd, 2, 5, 48, 8, False)
    kept = kept._replace(gamma=kept.gamma.view(1, 48, 1), beta=kept.beta.view(48, 1))
    _, dgamma, dbeta, _ = msd.groupnorm_channels_last_backward(_on(torch.zeros(2, 5, 48)), kept)
    assert dgamma.shape == dbeta.shape == (48,) and dgamma.dtype == dbeta.dtype == torch.float32


@pytest.mark.gpu
def test_gradients_of_gamma_and_beta_are_vectors_on_both_paths(msd, cuda, monkeypatch):
    x, g = torch.randn(2, 5, 48, device=cuda), torch.ones(1, 48, 1, device=cuda)
    _, kept = msd.groupnorm_channels_last_kept(x, g, g, 8)
    first = msd.groupnorm_channels_last_backward(x, kept)
    monkeypatch.setattr(msd, "_native_cl_q4", msd._NoNative())
    second = msd.groupnorm_channels_last_backward(x, kept)
    assert all(a.shape == b.shape and torch.equal(a, b) for a, b in zip(first[:3], second[:3])) and first[1].shape == (48,)


@pytest.mark.parametrize("groups", [0, -8, 7, 96, 10 ** 13])
def test_groups_that_do_not_divide_the_channels_are_refused_before_anything_is_allocated(msd, library, groups):
    x, g = _on(torch.zeros(2, 5, 48)), _on(torch.ones(48))
    for call in (lambda: msd.groupnorm_channels_last_kept(x, g, g, groups), lambda: msd.groupnorm_channels_last_kept(x, g, g, groups, keep8=True),
                 lambda: msd.groupnorm_channels_last(x, g, g, groups)):
        with pytest.raises(msd.MsdError):
            call()
