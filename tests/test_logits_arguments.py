"""Penalties as numbers, without a device."""
import math

import numpy as np
import pytest

from bgtq import _lib
from bgtq.serving import _per_row


@pytest.mark.parametrize("x", [1e39, -1e39, 1e300, math.inf, math.nan, np.float64(1e40)])
@pytest.mark.parametrize("name", ["repetition", "presence", "frequency"])
def test_penalties_that_fp32_does_not_hold_are_refused(x, name):
    with pytest.raises(_lib.RangeError, match="finite"):
        _per_row(x, 2, "cpu", name)


@pytest.mark.parametrize("x", [0.0, -1.0, 1e-50, 5e-46])
def test_a_repetition_that_fp32_rounds_to_zero_is_refused(x):
    with pytest.raises(_lib.RangeError, match="positive"):
        _per_row(x, 2, "cpu", "repetition")


@pytest.mark.parametrize("x", [1, 1.3, True, 3e38, 1e-45, np.float32(1.1), np.float64(1.1), np.int64(2)])
def test_other_numbers_are_filled_in(x):
    for name in ("repetition", "presence", "frequency"):
        got = _per_row(x, 3, "cpu", name)
        assert got.shape == (3,) and (got.numpy() == np.float32(x)).all()
    assert (_per_row(-0.0, 1, "cpu", "presence").numpy() == 0).all() and (_per_row(1e-50, 1, "cpu", "presence").numpy() == 0).all()
