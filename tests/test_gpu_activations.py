"""The activations of yx_linear_bf16_dev against 64 bits: as a share of the argument, as
include/yaxus_hip.h states it, and as a share of the result, into the tails.

Bounds on the result's relative error, in u = 2^-24. Constants and products before the
exponential: log2(e) in f32 is 0.23 u off and its product rounds by u, so e^-z is off by 1.23 u
|z| and its own 2 u (the hardware's e^x and 1/x are within 1 ulp, 2 u). silu, z = y: the sum 1 + e^-z
adds u, 1/x 2 u, the product u: 1.23 |y| + 6. gelu_tanh, z = y (a y^2 + b), with a 2.4 u, b 0.8 u
and a y u off and u each for the fused sum and the product: z itself is off by 5.4 u of it, so
6.63 |z| + 6. gelu, y erfc(-y / sqrt 2) / 2: the argument is off by 1.29 u, which erfc takes
y^2 + 0.8 |y| times for negative y; erfc is within 16 ulp (32 u), the product within u:
1.29 (y^2 + 0.8 |y|) + 33. All that while e^-z, 1 / (1 + e^-z) and the result are normal numbers."""

import math

import numpy as np
import pytest
from scipy.special import erfcx

from tests.test_gpu_linear import bf16_bits, run

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def exact(y, act):
    """(result, bound on its relative error, whether all steps are normal numbers)"""
    if act == "gelu":
        z = np.abs(y) / math.sqrt(2)
        tail = 0.5 * erfcx(z) * np.exp(-z * z)  # (erfcx: no loss in the tail)
        v = y * np.where(y < 0, tail, 1 - tail)
        return v, (1.29 * (y * y + 0.8 * np.abs(y)) + 33) * U, np.abs(v) >= 2.0 ** -125
    z = y if act == "silu" else 2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
    with np.errstate(over="ignore"):
        v = y / (1 + np.exp(-z))
    rel = 1.23 * np.abs(y) + 6 if act == "silu" else 6.63 * np.abs(z) + 6
    return v, rel * U, (z > -125 * math.log(2)) & (np.abs(v) >= 2.0 ** -125)


@pytest.mark.parametrize("act,share", [("silu", 2.0 ** -21), ("gelu_tanh", 2.0 ** -21), ("gelu", 2.0 ** -19)])
def test_activations_into_their_tails(hip, act, share):
    rng = np.random.default_rng(3)
    y = np.concatenate([np.linspace(-90, 90, 9001), np.linspace(-16, 4, 9001), rng.normal(size=20000) * 3,
                        np.geomspace(1e-30, 1e30, 2001), -np.geomspace(1e-30, 1e30, 2001)]).astype(np.float32)
    x = np.zeros((len(y), 8), np.float32)
    x[:, 3] = y
    w = np.zeros((16, 8), np.uint16)
    w[:, 3] = bf16_bits(np.ones(1, np.float32))[0]
    got = run(hip, x, w, act=act)
    assert (got == got[:, :1]).all()
    got, y = got[:, 0].astype(np.float64), y.astype(np.float64)
    want, rel, normal = exact(y, act)
    off = np.abs(got - want)
    assert np.all(off <= share * np.abs(y) + 2.0 ** -126)
    bad = normal & (off > rel * np.abs(want))
    assert not bad.any(), [(y[i], got[i], want[i]) for i in np.flatnonzero(bad)[:5]]
    # The tails are part of that: these results are at 2^-100 and below.
    assert (normal & (y < 0) & (np.abs(want) < 2.0 ** -100)).sum() > 50
