"""What msd_attention_workspace asks for, without a GPU (addresses are made up: a refused call reads none)."""
import ctypes

import pytest

F32, F16 = 0, 1


def _bytes(msd, batch, rows, keys, heads, kv_heads, dim, packed, backward, dtype):
    size = ctypes.c_size_t(0)
    assert msd.load_library().msd_attention_workspace(batch, rows, keys, heads, kv_heads, dim, packed, backward, dtype, ctypes.byref(size)) == 0
    return size.value


@pytest.mark.parametrize("dtype", [F32, F16])
def test_a_gradient_without_the_mask_needs_no_parts_of_a_causal_one(msd, dtype):
    """4 x 4000: rows are in two parts under the mask alone, each with dk and dv in float32."""
    sizes = 4, 4000, 4000, 16, 4, 128
    causal, open_ = (_bytes(msd, *sizes, 0, backward, dtype) for backward in (1, 2))
    assert causal - open_ == 2 * 2 * 4 * (4 * 4000 * 4 * 128)
    assert open_ <= 4 * (3 * 4 * 4000 * 16 + 4 * 4000 * 4 + 3)


@pytest.mark.parametrize("packed", [0, 1])
@pytest.mark.parametrize("sizes", [(2, 77, 77, 12, 12, 64), (1, 3, 2500, 4, 2, 48), (1, 2100, 77, 4, 2, 48), (1, 900, 900, 4, 2, 33), (8, 4096, 4096, 16, 16, 64)])
def test_bytes_for_either_mask_hold_both(msd, packed, sizes):
    for dtype in (F32, F16):
        assert _bytes(msd, *sizes, packed, 1, dtype) >= _bytes(msd, *sizes, packed, 2, dtype) > 0


def test_a_causal_gradient_is_refused_the_bytes_of_one_without_the_mask(msd):
    lib, p = msd.load_library(), ctypes.c_void_p
    at = [p((i + 1) << 32) for i in range(11)]
    sizes = 4, 4000, 4000, 16, 4, 128
    few = _bytes(msd, *sizes, 0, 2, F16)
    assert lib.msd_attention_backward(*at[:6], None, *at[6:9], None, None, *sizes, None, ctypes.c_float(0.1), 1, F16, at[9], few, None) == 1
