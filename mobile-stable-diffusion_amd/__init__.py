"""ctypes access to the MI355X norm / activation / embedding library.

The product is the native code under csrc/ (HIP kernels behind the C ABI of
include/msd_hip.h, and the C++ layer objects on top of it).  This module only
loads the built libraries and passes torch tensors' device pointers and the
current torch stream through the C ABI; torch is used for device memory and
streams, nothing else.  There is no fallback: if the library was not built
the loader raises.
"""
import collections
import ctypes
import functools
import importlib.util
import os
import sys
import warnings

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC_DIR = os.path.join(_PKG_DIR, "csrc")
LIB_HIP_PATH = os.path.join(CSRC_DIR, "libmsd_hip.so")
LIB_NN_PATH = os.path.join(CSRC_DIR, "libmsd_nn.so")
TORCH_CALLS_PATH = os.path.join(CSRC_DIR, "msd_torch_calls.so")
TORCH_CALLS_CL_Q4_PATH = os.path.join(CSRC_DIR, "msd_torch_calls_cl_q4.so")  # channels-last norms, 4-bit weights
TORCH_CALLS_TEXT_PATH = os.path.join(CSRC_DIR, "msd_torch_calls_text.so")  # token embedding, LayerNorm's gradient, attention

DTYPE_F32 = 0
DTYPE_F16 = 1
TUNE_GN_SPLIT, TUNE_GN_THREADS, TUNE_LN_CHUNK, TUNE_LN_THREADS, TUNE_GEGLU_VECTORS, TUNE_ACT_VECTORS, \
    TUNE_SOFTMAX_ROWS, TUNE_GN_SPIN_LIMIT, TUNE_GN_WRITERS, TUNE_DEVICE_CUS, TUNE_DEVICE_XCDS, \
    TUNE_GN_PLAN_RULE_ONLY = range(12)
ERR_SCRATCH_LIMIT = -2
CODE_BLOCK = 32  # channels that share a scale in an 8-bit checkpoint: MSD_CODE_BLOCK of include/msd_hip.h
TOKENS_WORKSPACE_BYTES = 128  # per (sample, group): MSD_TOKENS_WORKSPACE_BYTES of include/msd_hip.h

# every symbol include/msd_hip.h declares
C_ABI_SYMBOLS = (
    "msd_version", "msd_error_string", "msd_init", "msd_release", "msd_shutdown", "msd_status",
    "msd_gn_fallbacks", "msd_set_tuning", "msd_groupnorm", "msd_groupnorm_noalloc", "msd_groupnorm_plan", "msd_layernorm", "msd_geglu",
    "msd_silu", "msd_gelu", "msd_quick_gelu", "msd_timestep_embedding", "msd_ddim_timesteps",
    "msd_elemwise_add", "msd_chunkwise_add", "msd_chunk_add_groupnorm", "msd_add_layernorm", "msd_copy",
    "msd_groupnorm_tokens", "msd_groupnorm_tokens_workspace", "msd_permute_0_2_1",
    "msd_groupnorm_channels_last", "msd_groupnorm_channels_last_workspace", "msd_groupnorm_channels_last_backward",
    "msd_linear_rows", "msd_linear_rows_grouped", "msd_q4_pack", "msd_linear_rows_q4", "msd_linear_rows_q4_grouped",
    "msd_layernorm_backward", "msd_layernorm_backward_workspace", "msd_token_embedding", "msd_token_embedding_backward",
    "msd_token_embedding_backward_workspace", "msd_attention", "msd_attention_backward", "msd_attention_workspace",
    "msd_softmax", "msd_alphas_cumprod", "msd_ddim_schedule", "msd_ddim_update",
)
ACT_NONE, ACT_SILU = 0, 1

_lib = None


class MsdError(RuntimeError):
    pass


def load_library(path=None):
    """Loads libmsd_hip.so (built in-tree) and declares the C ABI signatures."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    path = path or LIB_HIP_PATH
    if not os.path.exists(path):
        raise MsdError(
            "native library %s is missing: build it with `python -c 'import __graft_entry__ as g;"
            " g.build()'` (there is no non-native fallback)" % path)
    lib = ctypes.CDLL(path, mode=ctypes.RTLD_GLOBAL)
    vp, sz, fl, it = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_float, ctypes.c_int
    lib.msd_version.restype = it
    lib.msd_error_string.restype = ctypes.c_char_p
    lib.msd_error_string.argtypes = [it]
    lib.msd_init.argtypes = [vp]
    lib.msd_shutdown.argtypes = []
    lib.msd_status.argtypes = [vp]
    lib.msd_release.argtypes = [vp]
    lib.msd_gn_fallbacks.argtypes = [vp, ctypes.POINTER(ctypes.c_uint), it]
    lib.msd_set_tuning.argtypes = [it, it]
    lib.msd_groupnorm.argtypes = [vp, vp, vp, vp, sz, sz, sz, sz, fl, it, it, vp]
    lib.msd_groupnorm_noalloc.argtypes = [vp, vp, vp, vp, sz, sz, sz, sz, fl, it, it, vp]
    lib.msd_groupnorm_plan.argtypes = [sz, sz, sz, sz, it, it, it] + [ctypes.POINTER(ctypes.c_int)] * 4
    lib.msd_layernorm.argtypes = [vp, vp, vp, vp, sz, sz, fl, it, vp]
    lib.msd_geglu.argtypes = [vp, vp, sz, sz, it, vp]
    lib.msd_copy.argtypes = [vp, vp, sz, vp]
    lib.msd_permute_0_2_1.argtypes = [vp, vp, sz, sz, sz, it, vp]
    lib.msd_groupnorm_tokens.argtypes = [vp, vp, vp, vp, sz, sz, sz, sz, fl, it, vp]
    lib.msd_groupnorm_tokens_workspace.argtypes = [vp, vp, vp, vp, sz, sz, sz, sz, fl, it, vp, sz, vp]
    lib.msd_groupnorm_channels_last.argtypes = [vp, vp, vp, vp, vp, sz, sz, sz, sz, fl, it, it, vp, vp, vp, vp, sz, vp]
    lib.msd_groupnorm_channels_last_workspace.argtypes = [sz, sz, sz, sz, it, it, ctypes.POINTER(sz)]
    lib.msd_groupnorm_channels_last_backward.argtypes = [vp] * 12 + [sz, sz, sz, sz, it, it, vp, sz, vp]
    lib.msd_elemwise_add.argtypes = [vp, vp, vp, sz, it, vp]
    lib.msd_chunkwise_add.argtypes = [vp, vp, vp, sz, sz, it, vp]
    lib.msd_chunk_add_groupnorm.argtypes = [vp, vp, vp, vp, vp, sz, sz, sz, sz, fl, it, it, vp]
    lib.msd_add_layernorm.argtypes = [vp, vp, vp, vp, vp, vp, sz, sz, fl, it, vp]
    for name in ("msd_silu", "msd_gelu", "msd_quick_gelu"):
        getattr(lib, name).argtypes = [vp, vp, sz, it, vp]
    lib.msd_timestep_embedding.argtypes = [vp, vp, sz, sz, fl, it, vp]
    lib.msd_ddim_timesteps.argtypes = [it, ctypes.POINTER(ctypes.c_int), it]
    lib.msd_linear_rows.argtypes = [vp, vp, vp, vp, sz, sz, sz, it, it, it, vp]
    lib.msd_softmax.argtypes = [vp, vp, sz, sz, it, it, vp]
    lib.msd_linear_rows_grouped.argtypes = [vp, ctypes.POINTER(vp), ctypes.POINTER(vp), ctypes.POINTER(vp),
                                            ctypes.POINTER(sz), sz, sz, sz, it, it, it, vp]
    lib.msd_q4_pack.argtypes = [vp, vp, vp, sz, sz, sz, it, vp]
    lib.msd_linear_rows_q4.argtypes = [vp, vp, vp, vp, vp, sz, sz, sz, sz, it, it, it, vp]
    lib.msd_linear_rows_q4_grouped.argtypes = [vp] + [ctypes.POINTER(vp)] * 4 + [ctypes.POINTER(sz), sz, sz, sz, sz, it, it, it, vp]
    lib.msd_layernorm_backward_workspace.argtypes = [sz, sz, it, ctypes.POINTER(sz)]
    lib.msd_layernorm_backward.argtypes = [vp] * 7 + [sz, sz, fl, it, vp, sz, vp]
    lib.msd_token_embedding.argtypes = [vp, vp, vp, vp, sz, sz, sz, sz, fl, it, vp]
    lib.msd_token_embedding_backward_workspace.argtypes = [sz] * 5 + [it, ctypes.POINTER(sz)]
    lib.msd_token_embedding_backward.argtypes = [vp] * 4 + [sz] * 5 + [fl, it, vp, sz, vp]
    lib.msd_attention_workspace.argtypes = [sz] * 6 + [it, it, it, ctypes.POINTER(sz)]
    lib.msd_attention.argtypes = [vp] * 8 + [sz] * 6 + [ctypes.POINTER(sz), fl, it, it, vp, sz, vp]
    lib.msd_attention_backward.argtypes = [vp] * 12 + [sz] * 6 + [ctypes.POINTER(sz), fl, it, it, vp, sz, vp]
    flp, inp = ctypes.POINTER(ctypes.c_float), ctypes.POINTER(ctypes.c_int)
    lib.msd_alphas_cumprod.argtypes = [flp]
    lib.msd_ddim_schedule.argtypes = [it, inp, flp, flp, flp, it]
    lib.msd_ddim_update.argtypes = [vp, vp, vp, sz, fl, fl, fl, it, vp]
    for name in C_ABI_SYMBOLS:
        if name != "msd_error_string":
            getattr(lib, name).restype = it
    _lib = lib
    for native in (_native, _native_cl_q4, _native_text):
        if not isinstance(native, _Unbound):
            _bind_addresses(native)
    return lib


def check(code):
    if code != 0:
        raise MsdError("msd call failed with code %d: %s"
                       % (code, load_library().msd_error_string(code).decode()))


# What a call does on the host is most of a small call's time (a LayerNorm of 154 rows: a kernel of 2.2 us behind 2.5 to
# 3.5 us of the runtime's launch), so plain calls (dense device tensors that fit each other, no mode or transform around
# them) go through csrc/torch_calls.cpp, which checks them, makes the outputs and calls the C ABI; it returns None for any
# other, which the general path below it then makes or refuses.  Eager passes, us, from Python and so: four calls of a
# sampler's tick 25.0 -> 14.4, the 49 of a text encoder 325 -> 198 (to 222), 22 grouped projections 53 -> 15.3, the 8 of a
# 640-channel transformer block 55.6 -> 35.8.
class _Unbound:
    """Stands for the native calls until the first one."""

    def __getattr__(self, name):
        return getattr(_bind_native(), name)


class _UnboundClQ4(_Unbound):
    def __getattr__(self, name):
        return getattr(_bind_native_cl_q4(), name)


class _UnboundText(_Unbound):
    def __getattr__(self, name):
        return getattr(_bind_native_text(), name)


class _NoNative:
    """Stands for the native calls where there are none: every call takes its general path."""

    def __getattr__(self, name):
        return lambda *args: None

    def names(self):
        return []

    def bind(self, addresses, check):
        pass


# (three extensions: csrc/torch_calls.cpp, csrc/torch_calls_cl_q4.cpp, csrc/torch_calls_text.cpp)
_native, _native_cl_q4, _native_text = _Unbound(), _UnboundClQ4(), _UnboundText()


def _bind_addresses(native):
    native.bind({name: ctypes.cast(getattr(_lib, name), ctypes.c_void_p).value for name in native.names()}, check)


def _running(torch):
    """The Python and the torch at hand, as build.py names those that the extension is compiled for."""
    return "Python %d.%d, torch %s (%s)" % (sys.version_info[:2] + (torch.version.__version__, torch.version.git_version))


def _load_native(torch, path=None):
    """The extension, or what stands for it where it is not built or was built for another torch: the C ABI takes tensors of
    any torch, but the extension reads them as its own torch lays them out."""
    path = path or TORCH_CALLS_PATH
    spec = importlib.util.spec_from_file_location(os.path.splitext(os.path.basename(path))[0], path)
    try:
        native = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(native)
        built_for = getattr(native, "built_for", "another torch")
        if built_for == _running(torch):
            return native
        why = "was built for %s, this is %s" % (built_for, _running(torch))
    except ImportError as e:  # (no such file, or symbols that this torch does not have)
        why = "does not load: %s" % e
    warnings.warn("%s %s; a call takes about 2.5 us longer without it (run __graft_entry__.build())" % (path, why),
                  RuntimeWarning, stacklevel=4)
    return _NoNative()


def _bind_native():
    global _native
    load_library()
    torch = _bind_torch()  # the extension's symbols are torch's
    if isinstance(_native, _Unbound):
        native = _load_native(torch)
        _bind_addresses(native)
        _native = native
    return _native


def _bind_native_cl_q4():
    global _native_cl_q4
    load_library()
    torch = _bind_torch()
    if isinstance(_native_cl_q4, _Unbound):
        native = _load_native(torch, TORCH_CALLS_CL_Q4_PATH)
        _bind_addresses(native)
        _native_cl_q4 = native
    return _native_cl_q4


def _bind_native_text():
    global _native_text
    load_library()
    torch = _bind_torch()
    if isinstance(_native_text, _Unbound):
        native = _load_native(torch, TORCH_CALLS_TEXT_PATH)
        _bind_addresses(native)
        _native_text = native
    return _native_text


_torch = None
_dtype_codes = {}
_raw_stream = _current_device = _capturing = None


def _bind_torch():
    """torch, imported by the first call that takes tensors (the host-only calls do without)."""
    global _torch, _capturing
    if _torch is None:
        import torch
        _capturing = torch.cuda.is_current_stream_capturing
        _dtype_codes.update({torch.float32: DTYPE_F32, torch.float16: DTYPE_F16})
        _torch = torch
    return _torch


def _dtype_code(t):
    code = _dtype_codes.get(t.dtype)
    if code is None:
        _bind_torch()
        code = _dtype_codes.get(t.dtype)
        if code is None:
            raise MsdError("unsupported storage dtype %s" % t.dtype)
    return code


def _stream():
    """The handle of torch's current stream on the current device.  Two private functions of torch's give it without
    a stream object (0.3 us against 1.6 a call); a torch that lacks them is asked through its public ones."""
    global _raw_stream, _current_device
    if _raw_stream is None:
        torch = _bind_torch()
        handle = torch.cuda.current_stream().cuda_stream  # initialises the device where nothing has yet
        _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda device: torch.cuda.current_stream(device).cuda_stream)
        return handle
    return _raw_stream(_current_device())


def _dev(t):
    if not t.is_cuda or not t.is_contiguous():
        raise MsdError("expected a contiguous device tensor")
    return t.data_ptr()


def _affine(t, n, like, what):
    """gamma / beta / bias: float32, n values, on the device of `like`."""
    if t.dtype != (_torch or _bind_torch()).float32 or t.numel() != n or t.get_device() != like.get_device():
        raise MsdError("%s must be float32 with %d values on %s (got %s, %d, %s)"
                       % (what, n, like.device, t.dtype, t.numel(), t.device))
    return _dev(t)


def _same(t, like, numel, what):
    """An output / second operand: dtype and device of `like`, `numel` elements."""
    if t.dtype != like.dtype or t.get_device() != like.get_device() or t.numel() != numel:
        raise MsdError("%s must be %s with %d elements on %s (got %s, %d, %s)"
                       % (what, like.dtype, numel, like.device, t.dtype, t.numel(), t.device))
    return _dev(t)


def _out_like(x, out, what="out"):
    """(output, its pointer): a new tensor like x, which _dev has checked, or the caller's."""
    if out is None:
        out = (_torch or _bind_torch()).empty_like(x)
        return out, out.data_ptr()
    return out, _same(out, x, x.numel(), what)


def init():
    check(load_library().msd_init(_stream()))


def status():
    return load_library().msd_status(_stream())


def gn_fallbacks(reset=False):
    """How often a GroupNorm workgroup computed a sibling's statistics itself (diagnostic)."""
    n = ctypes.c_uint(0)
    check(load_library().msd_gn_fallbacks(_stream(), ctypes.byref(n), int(reset)))
    return n.value


def _planes(x):
    """(batch, channels, positions per channel) of [batch, C, ...]."""
    shape = x.shape
    batch, channels = shape[0], shape[1]
    return batch, channels, x.numel() // (batch * channels) if batch * channels else 0


def groupnorm(x, gamma, beta, groups, eps=1e-5, fuse_silu=False, out=None, noalloc=False):
    """x: [batch, C, ...] device tensor; gamma/beta float32 [C]; out may be x (in place).
    noalloc: go through msd_groupnorm_noalloc (fixed scratch, batch * groups <= 1024)."""
    done = _native.groupnorm(x, gamma, beta, groups, eps, fuse_silu, out, noalloc)
    if done is not None:
        return done
    lib = _lib or load_library()
    batch, channels, hw = _planes(x)
    xp = _dev(x)
    out, yp = _out_like(x, out)
    check((lib.msd_groupnorm_noalloc if noalloc else lib.msd_groupnorm)(
        xp, yp, _affine(gamma, channels, x, "gamma"), _affine(beta, channels, x, "beta"), batch, channels, hw, groups,
        eps, int(fuse_silu), _dtype_code(x), _stream()))
    return out


def groupnorm_plan(batch, channels, hw, groups=32, dtype_code=DTYPE_F16, noalloc=False, in_place=False):
    """(split, threads, vectors per lane, writers) of the launch msd_groupnorm makes for this
    shape; (0, 0, 0, 1) = the general kernel; writers > 1 = that many workgroups share each whole
    (sample, group) and store a part of it each (never for a call in place).  Host arithmetic,
    no GPU needed."""
    out = [ctypes.c_int(0) for _ in range(4)]
    check(load_library().msd_groupnorm_plan(batch, channels, hw, groups, dtype_code, int(noalloc), int(in_place),
                                            *[ctypes.byref(o) for o in out]))
    return tuple(o.value for o in out)


def groupnorm_tokens(x, gamma, beta, groups, eps=1e-6):
    """x: [batch, C, ...] -> [batch, H*W, C] = GroupNorm(x) with channels last (no SiLU)."""
    done = _native.groupnorm_tokens(x, gamma, beta, groups, eps)
    if done is not None:
        return done
    lib = _lib or load_library()
    batch, channels, hw = _planes(x)
    xp = _dev(x)
    out = x.new_empty((batch, hw, channels))
    gp, bp = _affine(gamma, channels, x, "gamma"), _affine(beta, channels, x, "beta")
    if not _capturing():
        check(lib.msd_groupnorm_tokens(xp, out.data_ptr(), gp, bp, batch, channels, hw, groups, eps, _dtype_code(x),
                                       _stream()))
        return out
    size = TOKENS_WORKSPACE_BYTES * batch * groups
    workspace = x.new_empty(size, dtype=_torch.uint8)  # (the graph keeps it in its pool, apart from other graphs')
    check(lib.msd_groupnorm_tokens_workspace(xp, out.data_ptr(), gp, bp, batch, channels, hw, groups, eps, _dtype_code(x),
                                             workspace.data_ptr(), size, _stream()))
    return out


def _channels_last(x, what="x"):
    """(batch, positions, channels) of a [batch, C, H, W] tensor in torch.channels_last order or a contiguous
    [batch, positions, C] one, on the current device."""
    torch = _torch or _bind_torch()
    if not x.is_cuda or x.get_device() != torch.cuda.current_device():
        raise MsdError("%s must be on the current device (got %s)" % (what, x.device))
    if x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last):
        batch, channels, h, w = x.shape
        return batch, h * w, channels
    if x.dim() == 3 and x.is_contiguous():
        return tuple(x.shape)
    raise MsdError("%s must be [batch, C, H, W] in torch.channels_last order or a contiguous [batch, positions, C]" % what)


def _groups_fit(groups, channels):
    if groups <= 0 or channels % groups:
        raise MsdError("groups must divide the channels (got %d, %d)" % (groups, channels))


def _same_layout(t, like, what):
    """An operand laid out as `like`, which _channels_last has checked."""
    if t.shape != like.shape or t.dtype != like.dtype:
        raise MsdError("%s must be %s of shape %s (got %s, %s)" % (what, like.dtype, tuple(like.shape), t.dtype, tuple(t.shape)))
    _channels_last(t, what)
    return t.data_ptr()


@functools.lru_cache(maxsize=1024)
def _channels_last_workspace(batch, positions, channels, groups, dtype_code, backward):
    size = ctypes.c_size_t(0)
    check(load_library().msd_groupnorm_channels_last_workspace(batch, positions, channels, groups, dtype_code, backward,
                                                               ctypes.byref(size)))
    return size.value


KeptNorm = collections.namedtuple("KeptNorm", "x chunk codes scales stats gamma beta groups fuse_silu with_chunk")
KeptNorm.__doc__ = """What groupnorm_channels_last_kept keeps for the gradient: the mean and 1 / sqrt(variance + eps) of every group
(stats, float32 [batch, groups, 2]) and either x and chunk themselves or, in 8 bits, codes (int8, in the order of x) and scales
(float32 [batch, positions, ceil(C / 32)]; a code times its block's scale is the value it stands for)."""


def _pointer(t):
    return None if t is None else t.data_ptr()


def _channels_last_forward(x, gamma, beta, groups, eps, fuse_silu, chunk, out, stats, codes, scales):
    lib = _lib or load_library()
    batch, positions, channels = _channels_last(x)
    code = _dtype_code(x)
    if out is None:
        out = _torch.empty_like(x)
    yp = _same_layout(out, x, "out")
    cp = _same(chunk, x, batch * channels, "chunk") if chunk is not None else None
    gp, bp = _affine(gamma, channels, x, "gamma"), _affine(beta, channels, x, "beta")
    _groups_fit(groups, channels)
    size = _channels_last_workspace(batch, positions, channels, groups, code, 0)
    workspace = x.new_empty(size, dtype=_torch.uint8)
    check(lib.msd_groupnorm_channels_last(x.data_ptr(), cp, yp, gp, bp, batch, positions, channels, groups, eps, int(fuse_silu), code,
                                          _pointer(stats), _pointer(codes), _pointer(scales),
                                          workspace.data_ptr(), size, _stream()))
    return out


def groupnorm_channels_last(x, gamma, beta, groups, eps=1e-5, fuse_silu=False, chunk=None, out=None):
    """GroupNorm(x + chunk[:, :, None]) (+ SiLU) over channels-last tensors: x is [batch, C, H, W] in torch.channels_last order or a
    contiguous [batch, positions, C]; gamma / beta float32 [C]; chunk [batch, C] in x's dtype or None.  out may be x (in place)."""
    done = _native_cl_q4.groupnorm_channels_last(x, gamma, beta, groups, eps, fuse_silu, chunk, out)
    if done is not None:
        return done
    return _channels_last_forward(x, gamma, beta, groups, eps, fuse_silu, chunk, out, None, None, None)


def groupnorm_channels_last_kept(x, gamma, beta, groups, eps=1e-5, fuse_silu=False, chunk=None, keep8=False, out=None):
    """groupnorm_channels_last, and a KeptNorm for groupnorm_channels_last_backward.  It holds gamma and beta, and x and chunk (out
    must not be x) or, with keep8, the sum of these two in 8 bits, a quarter of float32 and a half of float16 (out may be x).
    What it holds must not change until then."""
    done = _native_cl_q4.groupnorm_channels_last_kept(x, gamma, beta, groups, eps, fuse_silu, chunk, out, keep8)
    if done is not None:
        y, codes, scales, stats = done
        return y, KeptNorm(None if keep8 else x, None if keep8 else chunk, codes, scales, stats, gamma, beta, groups, fuse_silu,
                           chunk is not None)
    batch, positions, channels = _channels_last(x)
    if out is not None and not keep8 and out.data_ptr() == x.data_ptr() and x.numel():
        raise MsdError("out must not be x unless keep8: the gradient needs x")
    torch = _torch
    _groups_fit(groups, channels)
    stats = x.new_empty((batch, groups, 2), dtype=torch.float32)
    codes = scales = None
    if keep8:
        codes = torch.empty_like(x, dtype=torch.int8)
        scales = x.new_empty((batch, positions, -(-channels // CODE_BLOCK)), dtype=torch.float32)
    y = _channels_last_forward(x, gamma, beta, groups, eps, fuse_silu, chunk, out, stats, codes, scales)
    return y, KeptNorm(None if keep8 else x, None if keep8 else chunk, codes, scales, stats, gamma, beta, groups, bool(fuse_silu),
                       chunk is not None)


def groupnorm_channels_last_backward(dy, kept, affine=True, out=None):
    """-> (dx, dgamma, dbeta, dchunk) from dy, laid out as the forward call's x, and what that call kept.  dgamma and dbeta are
    float32 [C] (None unless affine); dchunk is [batch, C] in dy's dtype (None where the forward call had no chunk).
    out: receives dx; may be dy."""
    done = _native_cl_q4.groupnorm_channels_last_backward(dy, affine, out, *kept)
    if done is not None:
        return done
    lib = _lib or load_library()
    batch, positions, channels = _channels_last(dy, "dy")
    code = _dtype_code(dy)
    if kept.codes is not None:
        if kept.codes.dtype != _torch.int8 or kept.codes.shape != dy.shape:
            raise MsdError("codes must be int8 of dy's shape %s (got %s, %s)" % (tuple(dy.shape), kept.codes.dtype, tuple(kept.codes.shape)))
        _channels_last(kept.codes, "codes")
        xp = cp = None
        qp, sp = kept.codes.data_ptr(), _affine(kept.scales, batch * positions * -(-channels // CODE_BLOCK), dy, "scales")
    else:
        xp = _same_layout(kept.x, dy, "the forward call's x")
        cp = _same(kept.chunk, dy, batch * channels, "chunk") if kept.chunk is not None else None
        qp = sp = None
    if out is None:
        out = _torch.empty_like(dy)
    dxp = _same_layout(out, dy, "out")
    gp, bp = _affine(kept.gamma, channels, dy, "gamma"), _affine(kept.beta, channels, dy, "beta")
    tp = _affine(kept.stats, 2 * batch * kept.groups, dy, "stats")
    dgamma = dbeta = dchunk = None
    if affine:
        dgamma, dbeta = (dy.new_empty(channels, dtype=_torch.float32) for _ in range(2))
    if kept.with_chunk:
        dchunk = dy.new_empty((batch, channels))
    size = _channels_last_workspace(batch, positions, channels, kept.groups, code, 1)
    workspace = dy.new_empty(size, dtype=_torch.uint8)
    check(lib.msd_groupnorm_channels_last_backward(
        dy.data_ptr(), xp, cp, qp, sp, tp, gp, bp, dxp, _pointer(dgamma), _pointer(dbeta), _pointer(dchunk), batch, positions, channels, kept.groups, int(kept.fuse_silu), code,
        workspace.data_ptr(), size, _stream()))
    return out, dgamma, dbeta, dchunk


def permute_0_2_1(x):
    """[i, j, k] -> [i, k, j] (new tensor)."""
    done = _native.permute_0_2_1(x)
    if done is not None:
        return done
    lib = _lib or load_library()
    i, j, k = x.shape
    xp = _dev(x)
    out = x.new_empty((i, k, j))
    check(lib.msd_permute_0_2_1(xp, out.data_ptr(), i, j, k, _dtype_code(x), _stream()))
    return out


def chunk_add_groupnorm(x, chunk, gamma, beta, groups, eps=1e-5, fuse_silu=False, out=None):
    """GroupNorm(x + chunk[:, :, None]) (+ SiLU); chunk: [batch, C] in x's dtype."""
    done = _native.chunk_add_groupnorm(x, chunk, gamma, beta, groups, eps, fuse_silu, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    batch, channels, hw = _planes(x)
    xp = _dev(x)
    cp = _same(chunk, x, batch * channels, "chunk")
    out, yp = _out_like(x, out)
    check(lib.msd_chunk_add_groupnorm(xp, cp, yp, _affine(gamma, channels, x, "gamma"), _affine(beta, channels, x, "beta"),
                                      batch, channels, hw, groups, eps, int(fuse_silu), _dtype_code(x), _stream()))
    return out


def add_layernorm(a, b, gamma, beta, eps=1e-5, sum_out=None, out=None):
    """Returns (a + b, LayerNorm(a + b)); sum_out may be a or b."""
    done = _native.add_layernorm(a, b, gamma, beta, eps, sum_out, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    n, dim = a.numel(), a.shape[-1]
    rows = n // dim if dim else 0
    ap, bp = _dev(a), _same(b, a, n, "b")
    sum_out, sp = _out_like(a, sum_out, "sum_out")
    out, yp = _out_like(a, out)
    check(lib.msd_add_layernorm(ap, bp, sp, yp, _affine(gamma, dim, a, "gamma"), _affine(beta, dim, a, "beta"), rows, dim,
                                eps, _dtype_code(a), _stream()))
    return sum_out, out


def elemwise_add(a, b, out=None):
    done = _native.elemwise_add(a, b, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    n = a.numel()
    ap, bp = _dev(a), _same(b, a, n, "b")
    out, yp = _out_like(a, out)
    check(lib.msd_elemwise_add(ap, bp, yp, n, _dtype_code(a), _stream()))
    return out


def chunkwise_add(a, chunk, chunk_size, out=None):
    done = _native.chunkwise_add(a, chunk, chunk_size, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    n = a.numel()
    if chunk_size <= 0 or n % chunk_size:
        raise MsdError("chunk_size must divide the element count")
    ap, cp = _dev(a), _same(chunk, a, n // chunk_size, "chunk")
    out, yp = _out_like(a, out)
    check(lib.msd_chunkwise_add(ap, cp, yp, n, chunk_size, _dtype_code(a), _stream()))
    return out


def layernorm(x, gamma, beta, eps=1e-5, out=None):
    done = _native.layernorm(x, gamma, beta, eps, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    dim = x.shape[-1]
    rows = x.numel() // dim if dim else 0
    xp = _dev(x)
    out, yp = _out_like(x, out)
    check(lib.msd_layernorm(xp, yp, _affine(gamma, dim, x, "gamma"), _affine(beta, dim, x, "beta"), rows, dim, eps,
                            _dtype_code(x), _stream()))
    return out


def _workspace(like, name, *args):
    """(tensor to keep until the call is made, its pointer, its bytes)."""
    size = ctypes.c_size_t(0)
    check(getattr(load_library(), name)(*args, ctypes.byref(size)))
    t = like.new_empty(size.value, dtype=_torch.uint8)
    return t, t.data_ptr(), size.value


def layernorm_backward(dy, x, gamma, eps=1e-5, dsum=None, affine=True, out=None):
    """Gradient of layernorm(x, gamma, beta, eps), or of add_layernorm's norm (x is then the sum it returned) -> (dx, dgamma, dbeta).
    dsum: what comes back to x past the norm (the gradient of add_layernorm's sum), added to dx.  dgamma and dbeta are float32 [dim]
    (None unless affine).  out: receives dx; may be dy or dsum."""
    done = _native_text.layernorm_backward(dy, x, gamma, eps, dsum, affine, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    dp = _on_current_device(dy, "dy")
    n, dim = dy.numel(), dy.shape[-1]
    rows = n // dim if dim else 0
    xp, sp = _same(x, dy, n, "x"), _same(dsum, dy, n, "dsum") if dsum is not None else None
    gp = _affine(gamma, dim, dy, "gamma")
    out, op = _out_like(dy, out)
    dgamma = dbeta = None
    if affine:
        dgamma, dbeta = (dy.new_empty(dim, dtype=_torch.float32) for _ in range(2))
    code = _dtype_code(dy)
    workspace, wp, size = _workspace(dy, "msd_layernorm_backward_workspace", rows, dim, code)
    check(lib.msd_layernorm_backward(dp, xp, sp, gp, op, _pointer(dgamma), _pointer(dbeta), rows, dim, eps, code, wp, size, _stream()))
    return out, dgamma, dbeta


def _token_ids(ids):
    """(pointer, tokens, tokens per row) of int64 ids [..., length] on the current device."""
    ip = _on_current_device(ids, "ids")
    if ids.dtype != _torch.int64 or ids.dim() == 0:
        raise MsdError("ids must be int64 [..., length] (got %s, %s)" % (ids.dtype, tuple(ids.shape)))
    return ip, ids.numel(), ids.shape[-1]


def token_embedding(ids, table, positions=None, scale=1.0, out=None):
    """scale * table[ids] + positions[:length]: ids int64 [..., length], table [vocab, dim], positions [length or more, dim] in its dtype
    or None -> [..., length, dim].  An id outside [0, vocab) stands for a row of zeros."""
    done = _native_text.token_embedding(ids, table, positions, scale, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    ip, tokens, length = _token_ids(ids)
    tp = _on_current_device(table, "table")
    if table.dim() != 2:
        raise MsdError("table must be [vocab, dim] (got %s)" % (tuple(table.shape),))
    vocab, dim = table.shape
    pp = None
    if positions is not None:
        if positions.dim() != 2 or positions.shape[1] != dim or positions.shape[0] < length:
            raise MsdError("positions must be [%d or more, %d] (got %s)" % (length, dim, tuple(positions.shape)))
        pp = _same(positions, table, positions.numel(), "positions")
    if out is None:
        out = table.new_empty(ids.shape + (dim,))
    check(lib.msd_token_embedding(ip, tp, pp, _same(out, table, tokens * dim, "out"), tokens, length, vocab, dim, scale,
                                  _dtype_code(table), _stream()))
    return out


def token_embedding_backward(dy, ids, vocab, positions=0, scale=1.0):
    """Gradients of token_embedding's table of `vocab` rows and of its `positions` rows (0: not wanted) from dy [..., length, dim]
    -> (dtable [vocab, dim], dpositions [positions, dim] or None) in dy's dtype, every row written."""
    done = _native_text.token_embedding_backward(dy, ids, vocab, positions, scale)
    if done is not None:
        return done
    lib = _lib or load_library()
    dp = _on_current_device(dy, "dy")
    ip, tokens, length = _token_ids(ids)
    if dy.shape[:-1] != ids.shape:
        raise MsdError("dy must be %s + (dim,) (got %s)" % (tuple(ids.shape), tuple(dy.shape)))
    dim, code = dy.shape[-1], _dtype_code(dy)
    if positions and positions < length:
        raise MsdError("positions must be 0 or at least %d (got %d)" % (length, positions))
    dtable = dy.new_empty((vocab, dim))
    dpositions = dy.new_empty((positions, dim)) if positions else None
    workspace, wp, size = _workspace(dy, "msd_token_embedding_backward_workspace", tokens, length, vocab, positions, dim, code)
    check(lib.msd_token_embedding_backward(ip, dp, dtable.data_ptr(), _pointer(dpositions), tokens, length, vocab, positions, dim, scale,
                                           code, wp, size, _stream()))
    return dtable, dpositions


def geglu(proj, out=None):
    """proj: [..., 2*inner] (value | gate) -> [..., inner]."""
    done = _native.geglu(proj, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    shape = proj.shape
    inner = shape[-1] // 2
    rows = proj.numel() // (2 * inner) if inner else 0
    pp = _dev(proj)
    if out is None:
        out = proj.new_empty(shape[:-1] + (inner,))
    check(lib.msd_geglu(pp, _same(out, proj, rows * inner, "out"), rows, inner, _dtype_code(proj), _stream()))
    return out


def _act(name, x, out):
    fn = getattr(_lib or load_library(), name)
    xp = _dev(x)
    out, yp = _out_like(x, out)
    check(fn(xp, yp, x.numel(), _dtype_code(x), _stream()))
    return out


def silu(x, out=None):
    done = _native.silu(x, out)
    return done if done is not None else _act("msd_silu", x, out)


def gelu(x, out=None):
    done = _native.gelu(x, out)
    return done if done is not None else _act("msd_gelu", x, out)


def quick_gelu(x, out=None):
    done = _native.quick_gelu(x, out)
    return done if done is not None else _act("msd_quick_gelu", x, out)


def timestep_embedding(timesteps, dim, max_period=10000.0, dtype=None):
    """timesteps: int64 device tensor [batch] -> [batch, dim] as [cos | sin]."""
    torch = _torch or _bind_torch()
    if dtype is None or dtype is torch.float32 or dtype is torch.float16:
        done = _native.timestep_embedding(timesteps, dim, max_period, dtype is torch.float16)
        if done is not None:
            return done
    lib = _lib or load_library()
    n = timesteps.numel()
    out = timesteps.new_empty((n, dim), dtype=dtype or torch.float32)
    check(lib.msd_timestep_embedding(_dev(timesteps), _dev(out), n, dim, max_period, _dtype_code(out), _stream()))
    return out


def ddim_timesteps(steps):
    """Ascending integer DDIM timestep list (host only)."""
    lib = load_library()
    n = lib.msd_ddim_timesteps(steps, None, 0)
    if n < 0:
        raise MsdError("ddim steps must be in [1, 1000]")
    buf = (ctypes.c_int * n)()
    lib.msd_ddim_timesteps(steps, buf, n)
    return list(buf)


def linear_rows(x, weight, bias=None, act_in=ACT_NONE, act_out=ACT_NONE, out=None):
    """x [m <= 8, k], weight [n, k] (x's dtype), bias float32 [n] or None -> [m, n]."""
    done = _native.linear_rows(x, weight, bias, act_in, act_out, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    m, k = x.shape
    n = weight.shape[0]
    if weight.shape[1] != k or weight.dtype != x.dtype:
        raise MsdError("weight must be [n, k] in the dtype of x")
    if weight.get_device() != x.get_device():
        raise MsdError("weight and x must share a device")
    xp, wp = _dev(x), _dev(weight)
    bp = _affine(bias, n, x, "bias") if bias is not None else None
    out = x.new_empty((m, n)) if out is None else out
    check(lib.msd_linear_rows(xp, wp, bp, _same(out, x, m * n, "out"), m, n, k, act_in, act_out, _dtype_code(x), _stream()))
    return out


def linear_rows_grouped(x, weights, biases=None, act_in=ACT_NONE, act_out=ACT_NONE):
    """One launch for several Linear layers on the same x [m <= 8, k]: weights[i] is [n_i, k] in
    x's dtype, biases[i] float32 [n_i] or None -> list of [m, n_i] tensors."""
    done = _native.linear_rows_grouped(x, weights, biases, act_in, act_out)
    if done is not None:
        return done
    lib = _lib or load_library()
    m, k = x.shape
    xp, dtype, device, new = _dev(x), x.dtype, x.get_device(), x.new_empty
    outs, wp, bp, yp, ns = [], [], [], [], []
    for i, w in enumerate(weights):
        shape = w.shape
        if len(shape) != 2 or shape[1] != k or w.dtype != dtype or w.get_device() != device:
            raise MsdError("weights[%d] must be [n, %d] in the dtype and on the device of x" % (i, k))
        n = shape[0]
        b = biases[i] if biases is not None else None
        bp.append(_affine(b, n, x, "biases[%d]" % i) if b is not None else None)
        if not w.is_contiguous():
            raise MsdError("expected contiguous weights")
        out = new((m, n))
        outs.append(out)
        wp.append(w.data_ptr())  # (0 for an empty tensor, as for the others)
        yp.append(out.data_ptr())
        ns.append(n)
    count = len(outs)
    pointers = ctypes.c_void_p * count
    check(lib.msd_linear_rows_grouped(xp, pointers(*wp), pointers(*bp), pointers(*yp), (ctypes.c_size_t * count)(*ns), count,
                                      m, k, act_in, act_out, _dtype_code(x), _stream()))
    return outs


def q4_pack(weight, group=64):
    """(packed, scales) of a weight [n, k] for linear_rows_q4: uint8 [n, k / 2], two 4-bit codes to a byte, and [n, k / group] in
    the weight's dtype; group is 32, 64 or 128 and divides k."""
    lib = _lib or load_library()
    wp = _on_current_device(weight, "weight")
    if weight.dim() != 2 or group not in (32, 64, 128) or weight.shape[1] % group:
        raise MsdError("weight must be [n, k] with k a multiple of group, which is 32, 64 or 128")
    n, k = weight.shape
    packed, scales = weight.new_empty((n, k // 2), dtype=_torch.uint8), weight.new_empty((n, k // group))
    check(lib.msd_q4_pack(wp, packed.data_ptr(), scales.data_ptr(), n, k, group, _dtype_code(weight), _stream()))
    return packed, scales


def _on_current_device(t, what):
    """A contiguous tensor on the device whose stream the call goes to."""
    torch = _torch or _bind_torch()
    if not t.is_cuda or t.get_device() != torch.cuda.current_device() or not t.is_contiguous():
        raise MsdError("%s must be a contiguous tensor on the current device (got %s)" % (what, t.device))
    return t.data_ptr()


def _q4_weight(packed, scales, x, k, group, what):
    """Columns of a packed weight that fits x [m, k] and the group."""
    if packed.dim() != 2 or packed.dtype != _torch.uint8 or 2 * packed.shape[1] != k or packed.get_device() != x.get_device() \
            or not packed.is_contiguous():
        raise MsdError("%spacked must be contiguous uint8 [n, %d] on %s" % (what, k // 2, x.device))
    if scales.shape != (packed.shape[0], k // group) or scales.dtype != x.dtype or scales.get_device() != x.get_device() \
            or not scales.is_contiguous():
        raise MsdError("%sscales must be contiguous %s [%d, %d] on %s" % (what, x.dtype, packed.shape[0], k // group, x.device))
    return packed.shape[0]


def _q4_group(x, scales):
    """Weights per scale, from x [m, k] and scales [n, k / group]."""
    if x.dim() != 2 or scales.dim() != 2:
        raise MsdError("x must be [m, k] and scales [n, k / group]")
    k, count = x.shape[1], scales.shape[1]
    group = k // count if count else 0
    if group not in (32, 64, 128) or group * count != k:
        raise MsdError("scales must hold one value per 32, 64 or 128 of k = %d (got %d)" % (k, count))
    return group


def linear_rows_q4(x, packed, scales, bias=None, act_in=ACT_NONE, act_out=ACT_NONE, out=None):
    """linear_rows with the weight in 4 bits: x [m <= 8, k], packed uint8 [n, k / 2] and scales [n, k / group] (x's dtype) as
    q4_pack makes them, bias float32 [n] or None -> [m, n]."""
    done = _native_cl_q4.linear_rows_q4(x, packed, scales, bias, act_in, act_out, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    xp = _on_current_device(x, "x")
    group = _q4_group(x, scales)
    m, k = x.shape
    n = _q4_weight(packed, scales, x, k, group, "")
    bp = _affine(bias, n, x, "bias") if bias is not None else None
    out = x.new_empty((m, n)) if out is None else out
    check(lib.msd_linear_rows_q4(xp, packed.data_ptr(), scales.data_ptr(), bp, _same(out, x, m * n, "out"), m, n, k, group, act_in,
                                 act_out, _dtype_code(x), _stream()))
    return out


def linear_rows_q4_grouped(x, packed, scales, biases=None, act_in=ACT_NONE, act_out=ACT_NONE):
    """One launch for several such layers on the same x [m <= 8, k], all with the same group: lists of packed weights, scales and
    biases (or None) -> list of [m, n_i] tensors, which share one allocation."""
    done = _native_cl_q4.linear_rows_q4_grouped(x, packed, scales, biases, act_in, act_out)
    if done is not None:
        return done
    lib = _lib or load_library()
    xp = _on_current_device(x, "x")
    if len(packed) != len(scales) or (biases is not None and len(biases) != len(packed)):
        raise MsdError("packed, scales and biases must be lists of one length")
    if not packed:
        return []
    group = _q4_group(x, scales[0])
    m, k = x.shape
    ns = [_q4_weight(p, s, x, k, group, "layer %d: " % i) for i, (p, s) in enumerate(zip(packed, scales))]
    bp = [_affine(b, n, x, "biases[%d]" % i) if b is not None else None for i, (b, n) in enumerate(zip(biases or [None] * len(ns), ns))]
    unit = 256 // x.element_size()
    whole = x.new_empty(sum(-(-m * n // unit) * unit for n in ns))
    outs, at = [], 0
    for n in ns:
        outs.append(whole[at:at + m * n].view(m, n))
        at += -(-m * n // unit) * unit
    count = len(ns)
    pointers = ctypes.c_void_p * count
    check(lib.msd_linear_rows_q4_grouped(xp, pointers(*[p.data_ptr() for p in packed]), pointers(*[s.data_ptr() for s in scales]),
                                         pointers(*bp), pointers(*[o.data_ptr() for o in outs]), (ctypes.c_size_t * count)(*ns), count,
                                         m, k, group, act_in, act_out, _dtype_code(x), _stream()))
    return outs


def softmax(x, stable=False, out=None):
    """Softmax over the last axis; out may be x (in place)."""
    done = _native.softmax(x, stable, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    xp = _dev(x)
    out, yp = _out_like(x, out)
    check(lib.msd_softmax(xp, yp, rows, cols, int(stable), _dtype_code(x), _stream()))
    return out


KeptAttention = collections.namedtuple("KeptAttention", "q k v out lse rest causal scale offsets offsets_k")
KeptAttention.__doc__ = """What attention_kept keeps for the gradient: the call's tensors, lse, float32 [rows of q, heads], the log2 of the weights'
sums, and for float16 rest, what the rounding of out took away."""


def _heads(t, what, like=None):
    """The strides of a [batch, rows, heads, dim] or packed [rows, heads, dim] tensor on the current device."""
    torch = _torch or _bind_torch()
    if not t.is_cuda or t.get_device() != torch.cuda.current_device() or t.dim() not in (3, 4) or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise MsdError("%s must be [batch, rows, heads, dim] or [rows, heads, dim] on the current device, the values of a head together "
                       "(got %s, strides %s, %s)" % (what, tuple(t.shape), t.stride(), t.device))
    if like is not None and (t.dtype != like.dtype or t.dim() != like.dim()):
        raise MsdError("%s must be %s with %d dimensions (got %s, %d)" % (what, like.dtype, like.dim(), t.dtype, t.dim()))
    strides = t.stride()[:-1]
    return strides if t.dim() == 4 else (0,) + strides


def _attention_sizes(q, k, v, offsets, offsets_k):
    """(batch, q_rows, k_rows, heads, kv_heads, dim), pointers of the offsets, checked."""
    if k.shape != v.shape or q.dim() != k.dim() or q.shape[-1] != k.shape[-1] or (q.dim() == 4 and q.shape[0] != k.shape[0]):
        raise MsdError("k and v must have one shape that fits q (got %s, %s, %s)" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    heads, kv_heads = q.shape[-2], k.shape[-2]
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise MsdError("heads must be a multiple of the key heads (got %d, %d)" % (heads, kv_heads))
    if q.dim() == 4:
        if offsets is not None or offsets_k is not None:
            raise MsdError("offsets go with packed [rows, heads, dim] tensors")
        return (q.shape[0], q.shape[1], k.shape[1], heads, kv_heads, q.shape[-1]), None, None
    if offsets is None:
        raise MsdError("packed [rows, heads, dim] tensors need offsets")
    if offsets_k is None:
        if k.shape[0] != q.shape[0]:
            raise MsdError("k has %d rows, q %d: pass offsets_k" % (k.shape[0], q.shape[0]))
        offsets_k = offsets
    pointers = []
    for o, what in ((offsets, "offsets"), (offsets_k, "offsets_k")):
        pointers.append(_on_current_device(o, what))
        if o.dtype != _torch.int32 or o.dim() != 1 or o.numel() != offsets.numel() or o.numel() == 0:
            raise MsdError("%s must be int32 [sequences + 1] (got %s, %s)" % (what, o.dtype, tuple(o.shape)))
    return (offsets.numel() - 1, q.shape[0], k.shape[0], heads, kv_heads, q.shape[-1]), pointers[0], pointers[1]


def _attention_forward(q, k, v, causal, scale, offsets, offsets_k, out, keep):
    lib = _lib or load_library()
    strides = _heads(q, "q") + _heads(k, "k", q) + _heads(v, "v", q)
    sizes, qo, ko = _attention_sizes(q, k, v, offsets, offsets_k)
    code = _dtype_code(q)
    if scale is None:
        scale = sizes[5] ** -0.5 if sizes[5] else 1.0
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape:
        raise MsdError("out must be %s (got %s)" % (tuple(q.shape), tuple(out.shape)))
    strides += _heads(out, "out", q)
    lse = q.new_empty(q.shape[:-1], dtype=_torch.float32) if keep else None
    rest = q.new_empty(q.shape) if keep and code == DTYPE_F16 else None
    workspace, wp, size = _workspace(q, "msd_attention_workspace", *sizes, int(qo is not None), 0, code)
    check(lib.msd_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _pointer(lse), _pointer(rest), qo, ko, *sizes,
                            (ctypes.c_size_t * 12)(*strides), scale, int(causal), code, wp, size, _stream()))
    return out, lse, rest, scale


def attention(q, k, v, causal=False, scale=None, offsets=None, offsets_k=None, out=None):
    """softmax(scale q k^T) v: q [batch, rows, heads, dim], k and v [batch, keys, kv_heads, dim], heads a multiple of kv_heads, dim up
    to 128; views are fine as long as a head's values lie together.  scale: 1 / sqrt(dim) unless given.  causal: the last query sees
    every key, the one before all but the last, ...  Packed sequences: [rows, heads, dim] tensors with offsets (and offsets_k for the
    keys, if they differ), int32 [sequences + 1] on the device; rows of no sequence stay as they were (in a new `out`: undefined).
    A row that sees no key gives zeros."""
    done = _native_text.attention(q, k, v, causal, scale, offsets, offsets_k, out, False)
    if done is not None:
        return done
    return _attention_forward(q, k, v, causal, scale, offsets, offsets_k, out, False)[0]


def attention_kept(q, k, v, causal=False, scale=None, offsets=None, offsets_k=None, out=None):
    """attention, and a KeptAttention for attention_backward.  What it holds must not change until then."""
    done = _native_text.attention(q, k, v, causal, scale, offsets, offsets_k, out, True)
    if done is None:
        done = _attention_forward(q, k, v, causal, scale, offsets, offsets_k, out, True)
    out, lse, rest, scale = done
    return out, KeptAttention(q, k, v, out, lse, rest, bool(causal), scale, offsets, offsets_k)


def attention_backward(dout, kept, out=None):
    """-> (dq, dk, dv) from dout (as the forward call's out) and what that call kept.  out: three tensors (views of one are fine) that
    receive them."""
    done = _native_text.attention_backward(dout, out, *kept)
    if done is not None:
        return done
    lib = _lib or load_library()
    q, k, v = kept.q, kept.k, kept.v
    sizes, qo, ko = _attention_sizes(q, k, v, kept.offsets, kept.offsets_k)
    out = (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)) if out is None else tuple(out)
    if len(out) != 3:
        raise MsdError("out must be three tensors (got %d)" % len(out))
    tensors = (q, k, v, kept.out, dout) + out
    strides = ()
    for t, like, what in zip(tensors, (q, k, k, q, q, q, k, k), ("q", "k", "v", "out", "dout", "dq", "dk", "dv")):
        if t.shape != like.shape:
            raise MsdError("%s must be %s (got %s)" % (what, tuple(like.shape), tuple(t.shape)))
        strides += _heads(t, what, q)
    code = _dtype_code(q)
    lp = _affine(kept.lse, q.numel() // sizes[5] if sizes[5] else 0, q, "lse")
    rp = _same(kept.rest, q, q.numel(), "rest") if kept.rest is not None else None
    workspace, wp, size = _workspace(q, "msd_attention_workspace", *sizes, int(qo is not None), 1 if kept.causal else 2, code)
    check(lib.msd_attention_backward(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), kept.out.data_ptr(), lp, rp,
                                     *[t.data_ptr() for t in out], qo, ko, *sizes, (ctypes.c_size_t * 24)(*strides), kept.scale,
                                     int(kept.causal), code, wp, size, _stream()))
    return out


def alphas_cumprod():
    """The sampler's 1000 cumulative alpha products as a list of floats (host only)."""
    buf = (ctypes.c_float * 1000)()
    check(load_library().msd_alphas_cumprod(buf))
    return list(buf)


def ddim_schedule(steps):
    """-> (timesteps, alphas, alphas_prev, sqrt_one_minus_alphas) as lists (host only)."""
    lib = load_library()
    n = lib.msd_ddim_schedule(steps, None, None, None, None, 0)
    if n < 0:
        raise MsdError("ddim steps must be in [1, 500] (code %d)" % n)
    ts = (ctypes.c_int * n)()
    a, ap, s1m = (ctypes.c_float * n)(), (ctypes.c_float * n)(), (ctypes.c_float * n)()
    lib.msd_ddim_schedule(steps, ts, a, ap, s1m, n)
    return list(ts), list(a), list(ap), list(s1m)


def ddim_update(x, e_t, a_t, a_prev, sqrt_one_minus_at, out=None):
    """One DDIM step (eta 0) on device tensors; out may be x."""
    done = _native.ddim_update(x, e_t, a_t, a_prev, sqrt_one_minus_at, out)
    if done is not None:
        return done
    lib = _lib or load_library()
    n = x.numel()
    xp, ep = _dev(x), _same(e_t, x, n, "e_t")
    out, yp = _out_like(x, out)
    check(lib.msd_ddim_update(xp, ep, yp, n, a_t, a_prev, sqrt_one_minus_at, _dtype_code(x), _stream()))
    return out


# ---------------------------------------------------------------------------------------
# C++ layer objects (libmsd_nn.so) through their plain-C handles
# ---------------------------------------------------------------------------------------
_nn = None
# int model(void *x, int t, void *e_t, size_t bytes, void *user): the sampler's noise-model callback
MODEL_FN = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t,
                            ctypes.c_void_p)


def load_nn_library(path=None):
    """Loads libmsd_nn.so (GroupNorm / LayerNorm / GEGLU objects, NPY loader, step runner)."""
    global _nn
    if _nn is not None and path is None:
        return _nn
    load_library()
    path = path or LIB_NN_PATH
    if not os.path.exists(path):
        raise MsdError("native library %s is missing: run __graft_entry__.build()" % path)
    nn = ctypes.CDLL(path)
    vp, sz, fl, it, cp = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_float, ctypes.c_int, ctypes.c_char_p
    szp = ctypes.POINTER(ctypes.c_size_t)
    flp = ctypes.POINTER(ctypes.c_float)
    lgp = ctypes.POINTER(ctypes.c_long)
    sig = {
        "msdnn_last_error": (cp, []),
        "msdnn_set_media_path": (None, [cp]),
        "msdnn_set_debug_timing": (None, [it]),
        "msdnn_npy_load": (it, [cp, flp, sz, szp, szp]),
        "msdnn_npy_save": (it, [cp, flp, sz]),
        "msdnn_groupnorm_create": (vp, [vp, sz, sz, fl, cp, cp, sz, it]),
        "msdnn_groupnorm_init": (it, [vp]),
        "msdnn_groupnorm_check": (it, [vp, sz, it]),
        "msdnn_groupnorm_forward": (it, [vp, vp, vp, sz, it]),
        "msdnn_groupnorm_forward_chunk": (it, [vp, vp, vp, sz, vp, sz, it]),
        "msdnn_groupnorm_forward_tokens": (it, [vp, vp, vp, sz, it]),
        "msdnn_groupnorm_destroy": (None, [vp]),
        "msdnn_layernorm_create": (vp, [vp, sz, cp, cp, fl]),
        "msdnn_layernorm_init": (it, [vp]),
        "msdnn_layernorm_check": (it, [vp, sz, it]),
        "msdnn_layernorm_forward": (it, [vp, vp, vp, sz, it]),
        "msdnn_layernorm_forward_add": (it, [vp, vp, vp, vp, vp, sz, it]),
        "msdnn_layernorm_destroy": (None, [vp]),
        "msdnn_geglu_create": (vp, [vp, sz, sz]),
        "msdnn_geglu_weight_shape": (it, [vp, szp, szp]),
        "msdnn_geglu_check": (it, [vp, sz, sz, it]),
        "msdnn_geglu_forward": (it, [vp, vp, sz, vp, sz, it]),
        "msdnn_geglu_destroy": (None, [vp]),
        "msdnn_activation": (it, [vp, it, vp, vp, sz, it]),
        "msdnn_timestep_embedding": (it, [vp, lgp, sz, flp]),
        "msdnn_ddim_timesteps": (it, [it, ctypes.POINTER(ctypes.c_int), it]),
        "msdnn_linear_create": (vp, [vp, sz, sz, cp, cp, it]),
        "msdnn_linear_init": (it, [vp]),
        "msdnn_linear_init_from": (it, [vp, flp, sz, flp, sz]),
        "msdnn_linear_forward": (it, [vp, vp, sz, vp, sz, it, it, it]),
        "msdnn_linear_forward_grouped": (it, [ctypes.POINTER(vp), sz, vp, sz, ctypes.POINTER(vp), szp, it, it, it]),
        "msdnn_linear_destroy": (None, [vp]),
        "msdnn_softmax": (it, [vp, vp, vp, sz, it, sz, it]),
        "msdnn_ddim_sample": (it, [vp, vp, sz, it, it, MODEL_FN, vp, vp]),
        "msdnn_ddim_make_schedule": (it, [ctypes.POINTER(ctypes.c_int), it, flp, flp]),
        "msdnn_test_buffer": (it, [vp, vp, sz, it, cp, flp, szp]),
        "msdnn_step_create": (vp, [vp, sz, it, it]),
        "msdnn_step_num_ops": (sz, [vp]),
        "msdnn_step_op_info": (it, [vp, sz, ctypes.POINTER(ctypes.c_int), szp, ctypes.POINTER(ctypes.c_int)]),
        "msdnn_step_download": (it, [vp, sz, it, flp, sz, szp]),
        "msdnn_step_affine": (it, [vp, sz, flp, flp, sz]),
        "msdnn_step_restore": (it, [vp]),
        "msdnn_step_bytes": (sz, [vp]),
        "msdnn_step_launches": (sz, [vp]),
        "msdnn_step_run": (it, [vp, it, it, lgp, sz]),
        "msdnn_step_destroy": (None, [vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(nn, name)
        fn.restype = res
        fn.argtypes = args
    _nn = nn
    return nn


def nn_last_error():
    return load_nn_library().msdnn_last_error().decode()
