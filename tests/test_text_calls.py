"""Token embedding, LayerNorm's gradient, attention: sizes of workspaces and refusals, without a GPU (pointers are made up: a refused
call reads none)."""
import ctypes

import pytest

F32, F16 = 0, 1


def _bytes(msd, name, *args):
    size = ctypes.c_size_t(0)
    rc = getattr(msd.load_library(), name)(*args, ctypes.byref(size))
    return size.value if rc == 0 else None


def test_attention_gradient_workspace_holds_the_parts_of_a_causal_call(msd):
    """Under a mask the rows are cut into two parts where they are not without it: the bytes are those of the larger."""
    batch, rows, heads, kv_heads, dim = 4, 4000, 16, 4, 128
    got = _bytes(msd, "msd_attention_workspace", batch, rows, rows, heads, kv_heads, dim, 0, 1, F16)
    vectors = 4 * (2 * batch * rows * heads + batch * rows * kv_heads)
    part = 4 * 2 * dim * batch * rows * kv_heads
    assert got >= vectors + 2 * part
