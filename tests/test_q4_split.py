"""The split of a float32 value into two float16 that the Linear rows with 4-bit weights hand to the matrix cores (csrc/linear_q4.hip),
in numpy: what a row's values of a step are off by, from the largest of them down to 2^26 times less."""
import numpy as np
import pytest


def split(f, most):
    """The values that the two float16 stand for, in float64; most: the largest magnitude of the row's values of the step."""
    exponent = max(int(np.float32(most).view(np.uint32)) >> 23, 20)
    up = np.uint32((268 - exponent) << 23).view(np.float32)
    s = (f * up).astype(np.float32)
    hi = s.astype(np.float16)
    lo = ((s - hi.astype(np.float32)) * np.float32(2048)).astype(np.float16)
    return (hi.astype(np.float64) + lo.astype(np.float64) / 2048) / np.float64(up)


def smallest(most):
    exponent = int(np.float32(most).view(np.uint32)) >> 23
    return np.uint32((max(exponent, 26) - 26) << 23).view(np.float32)


@pytest.mark.parametrize("exponent", [-149, -140, -126, -110, -103, -101, -100, -99, -60, 0, 11, 100, 127])
def test_values_of_a_step_are_off_by_a_float32_rounding_or_two(exponent):
    rng = np.random.default_rng(exponent + 200)
    most = np.float32(np.ldexp(1.9, exponent)) if exponent > -149 else np.float32(np.ldexp(1.0, -149))
    for down in range(0, 60):
        f = np.ldexp(rng.uniform(0.5, 1.0, 4000), exponent + 1 - down).astype(np.float32)
        f = f[f <= most]
        f = np.concatenate([f, -f])
        taken = np.abs(f) >= smallest(most)
        off = np.abs(split(f, most) - f.astype(np.float64))
        assert (off[taken] <= 2.0 ** -23 * np.abs(f[taken].astype(np.float64))).all(), down
        if smallest(most) == 0:
            assert taken.all()
        elif down > 28:
            assert not taken.any()
    if smallest(most) == 0:  # as small as that, nothing is left out
        assert (off == 0).all()


def test_what_is_far_below_the_largest_would_be_lost():
    f = np.full(1, 1.2e-3, np.float32)
    assert [float(abs(split(f, m)[0] / f[0] - 1)) > t for m, t in ((1e9, 1e-4), (1e12, 0.1), (1e14, 0.99))] == [True] * 3
    assert all(f[0] < smallest(m) for m in (1e9, 1e12, 1e14))
