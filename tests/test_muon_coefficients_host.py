"""Which coefficients of an orthogonalised update are taken: against a fine sampling of the polynomial (no GPU needed)."""
import ctypes

import numpy as np
import pytest

pytest.importorskip("torch")

from f2cgt_amd import capi  # noqa: E402

UNSUPPORTED = -2


def _answer(coefficients, steps):
    return capi.lib().f2cgt_orthogonalize(None, capi.DT_F32, None, 0, 40, 40, steps, (ctypes.c_float * 3)(*coefficients), None, 0, None)


def _reach(coefficients, steps):
    """(largest singular value, largest multiplier) over all steps."""
    a, b, c = (float(np.float32(v)) for v in coefficients)
    reach, most, factor = 1.0, 0.0, 0.0
    for _ in range(steps):
        x = np.linspace(0.0, reach * 1.001, 20001)
        p = a + b * x ** 2 + c * x ** 4
        reach = float(np.abs(x * p).max())
        most, factor = max(most, reach), max(factor, float(np.abs(p).max()))
        if most > 100:
            break
    return most, factor


@pytest.mark.parametrize("steps", [1, 2, 5])
def test_what_leaves_the_range_is_refused(steps):
    rng = np.random.default_rng(steps)
    taken = refused = 0
    for i in range(1200):
        a = rng.uniform(-7.4, 7.4) if i % 2 else rng.uniform(1.0, 4.5)
        b = rng.uniform(-12.0, 12.0) if i % 2 else rng.uniform(-7.0, 0.0)
        c = (rng.choice([0.0, 1e-38, -1e-38, 1e-20, -1e-20, 1e-12, 1e-6, -1e-4]) if i % 3 == 0 else
             rng.uniform(-30.0, 30.0) if i % 3 == 1 else rng.uniform(0.0, 3.0))
        most, factor = _reach((a, b, c), steps)
        if abs(most - 2.5) < 0.05 or abs(factor - 7.5) < 0.05:      # (the check's own reserve)
            continue
        want = UNSUPPORTED if most > 2.5 or factor > 7.5 else 0
        assert _answer((a, b, c), steps) == want, (a, b, c, steps, most, factor)
        taken, refused = taken + (want == 0), refused + (want != 0)
    assert taken > 30 and refused > 30


@pytest.mark.parametrize("c", [0.0, 1e-38, 1e-20, -1e-20, 1e-15, 1e-8])
def test_a_vanishing_last_coefficient(c):
    # singular values near 0.577 become 2.85, whose squares times 8192 no fp16 number holds
    assert _answer((7.4, -7.4, c), 1) == UNSUPPORTED
    assert _answer((7.4, -7.4, c), 2) == UNSUPPORTED
