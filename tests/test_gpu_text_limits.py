"""LayerNorm's gradient, attention and its gradient at the ends of what their calls allow."""
import pytest

import plain_text as plain
from test_gpu_text_training import DTYPES, _normal

pytestmark = pytest.mark.gpu


# ---- LayerNorm's gradient ----------------------------------------------------------------------
# (rows that are no multiple of what a workgroup has at a time: 16, 8 or 4 of them by vectors, 4 by single values)
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,dim", [(1, 64), (17, 64), (1, 320), (19, 400), (33, 640), (5, 1000), (1, 77), (6, 777), (154, 768), (3, 2048), (2, 1100)])
@pytest.mark.parametrize("add", [False, True])
def test_layernorm_gradient_without_eps(msd, cuda, dtype, rows, dim, add):
    t = DTYPES[dtype]
    x, dy, gamma = (2 * _normal(1, rows, dim) + 1).to(t), _normal(2, rows, dim).to(t), 1 + 0.2 * _normal(3, dim)
    dsum = _normal(4, rows, dim).to(t) if add else None
    got = msd.layernorm_backward(dy.to(cuda), x.to(cuda), gamma.to(cuda), 0.0, None if dsum is None else dsum.to(cuda))
    for g, w, what in zip(got, plain.layernorm_backward(dy, x, gamma, 0.0, dsum), ("dx", "dgamma", "dbeta")):
        plain.check(g, w, what)
