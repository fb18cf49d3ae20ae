"""silu of gates of any size in stride_amd.mx.mlp13."""
import numpy as np
import pytest

import mx_plain
import test_gpu_mx as plain
from stride_amd import mx

pytestmark = pytest.mark.gpu

GATES = [0.0, 1.0, -1.0, 2.0 ** -20, -2.0 ** -20, 5.0, -5.0, 20.0, -20.0, 52.0, -52.0, 80.0, -80.0, 88.0, -88.0, 96.0, -96.0, 208.0, -208.0,
         1.25 * 2.0 ** 60, -1.25 * 2.0 ** 60, 1.25 * 2.0 ** 120, -1.25 * 2.0 ** 120]


@pytest.mark.parametrize("n", [32, 1040])
def test_gates_of_any_size(n):
    """A row's gates are all one number and its up values 1, so that z is silu of that number alone, in a
    block of its own: within half a step of e4m3 (2^-4) and the roundings of the two instructions (2^-20).
    Below -88.7 fp32 has no e^-x, and -88 lies where its inverse is no normal number: 0 there."""
    w = np.zeros((2, n, 512))
    w[0, :, 0], w[1, :, 32] = 1, 1
    x = np.zeros((len(GATES), 512))
    x[:, 0], x[:, 32] = GATES, 1
    w1, w3, xt = plain.held(w[0], 4), plain.held(w[1], 4), plain.held(x, 8)
    assert np.array_equal(mx_plain.values(xt, len(GATES), 512)[:, 0], GATES)
    z = mx_plain.values(mx.mlp13(w1, w3, xt, len(GATES)), len(GATES), n)
    for g, row in zip(GATES, z):
        want = g / (1 + np.exp(-g)) if g > -700 else 0.0
        if g <= -96:
            assert (row == 0).all(), g
        elif g == -88:
            assert (row == 0).all() or (np.abs(row - want) <= 2.0 ** -4 * abs(want)).all(), (g, row[0])
        else:
            assert (np.abs(row - want) <= (2.0 ** -4 + 2.0 ** -20) * abs(want)).all(), (g, row[0], want)
