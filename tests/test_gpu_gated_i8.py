"""The activations of the gated products in 8-bit integers, in float32: each side's values come in as a bias (codes of 0 add nothing), so that a result is the activation itself.

Bounds in u = 2^-24 of the value, half a step of float32. silu and sigmoid: the hardware's 2^x is off by a step (2 u), what goes back in for its argument, the sum 1 + e and the quotient by half a
step each (3 u), ln 2 as a float32 by 2^-28 of the argument, second-order terms by less than 1 u. gelu, with v = log2(2 Phi(-a)) and a = |g|: v is off by 4 u of itself (the polynomial's last step and the
product with a by 1 u each, what its earlier steps are off by and the roundings of its coefficients by 1 u each of parts of it) and by what the polynomial leaves, `fit`; Phi(-a) by ln 2 times that and
2 u, 1 - Phi(-a) and the products by 1 u each."""
from math import erf, erfc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from excalibur_amd import hip
    c = hip.Ctx(0)
    yield c
    c.close()


def activation(ctx, gate, g, m=1, u=None):
    """act(g) * u in float32 as the product has it in each of m rows."""
    n = len(g)
    ones = np.ones(n, np.float32)
    w = ctx.array(np.ones((n, 16), np.int8))
    y = ctx.empty((m, n), np.float32)
    ctx.innerproduct_gated_i8(ctx.i8_desc(m, n, 16), ctx.array(np.zeros((m, 16), np.int8)), ctx.array(np.ones(m, np.float32)), ctx.pack_i8_weights(n, 16, w, w), ctx.array(ones), ctx.array(ones),
                              gate=gate, bias_gate=ctx.array(g), bias_up=ctx.array(ones if u is None else u), y_f32=y)
    y = y.download()
    assert np.array_equal(y.view(np.uint32), np.broadcast_to(y[0], y.shape).view(np.uint32))
    return y[0]


def gates(rng):
    g = np.concatenate([rng.standard_normal(20000) * 2, rng.uniform(-87, 87, 20000), np.ldexp(rng.uniform(-2, 2, 4000), rng.integers(-126, 0, 4000)), np.arange(-87, 88), [0.0, -0.0]])
    return g.astype(np.float32)


@pytest.mark.parametrize("m", [1, 200])
@pytest.mark.parametrize("gate", ["silu", "sigmoid"])
def test_silu_and_sigmoid_within_their_roundings(ctx, gate, m):
    g = gates(np.random.default_rng(1))
    got = activation(ctx, gate, g, m).astype(np.float64)
    v = g.astype(np.float64)
    want = (v if gate == "silu" else 1) / (1 + np.exp(-v))
    assert np.all(np.abs(got - want) <= np.abs(want) * (6 + np.abs(v) / 16) * U + 2.0 ** -149)


def phi_below(a):
    """Phi(-a), and log2(2 Phi(-a)), of a >= 0."""
    below = 0.5 * np.vectorize(erfc)(a * np.sqrt(0.5))
    with np.errstate(divide="ignore"):
        return below, np.log2(2 * below)


@pytest.mark.parametrize("m", [1, 200])
def test_gelu_within_its_roundings(ctx, m):
    g = gates(np.random.default_rng(2))
    got = activation(ctx, "gelu", g, m).astype(np.float64)
    a = np.abs(g.astype(np.float64))
    below, v = phi_below(a)
    # what the polynomial leaves of v: a tenth of u of Phi(-a), no more than u of v up to 4 and than 2^8 u at 6.5
    with np.errstate(all="ignore"):
        fit = np.minimum(0.11 / below, 0.74 * np.exp2(8 * np.clip((a - 4) / 2.5, 0, 1)) * np.maximum(-v, 0.2))
        own = 2.8 * -v + 2 + fit  # of Phi(-a), in u
        bound = a * np.where(g < 0, below * (own + 2), (1 - below) * 2 + below * own + 1) * U + 2.0 ** -149
    want = g * np.where(g < 0, below, 1 - below)
    here = a <= 6.5
    assert np.all(np.abs(got - want)[here] <= bound[here])
    # behind the polynomial's range: Phi(-a) falls from 4e-11, and is taken for no more
    far = ~here
    assert np.all(np.abs(got - want)[far] <= (a * (1.01 * phi_below(np.float64(6.5))[0] + 2 * U * (g > 0)))[far])


@pytest.mark.parametrize("gate", ["silu", "gelu", "sigmoid"])
def test_activations_are_as_exact_as_their_formulas_in_float32(ctx, gate):
    """Error in norm over gates of a normal distribution, and from -3 to -1, against the formulas with every step rounded to float32 and expf and erff without an error. The formulas' own is 0.6 u and more of
    the values' norm; the hardware's 2^x and 1 / x, a step each where those are off by nothing, may add half as much."""
    rng = np.random.default_rng(3)
    for g in (rng.standard_normal(60000).astype(np.float32), rng.uniform(-3, -1, 30000).astype(np.float32)):
        v, one = g.astype(np.float64), np.float32(1)
        if gate == "gelu":
            part = np.vectorize(erf)((g * np.float32(np.sqrt(0.5))).astype(np.float64)).astype(np.float32)
            formula, want = np.float32(0.5) * g * (one + part), v * np.where(v < 0, phi_below(np.abs(v))[0], 1 - phi_below(np.abs(v))[0])
        else:
            e = np.exp(-v).astype(np.float32)
            formula, want = (g if gate == "silu" else one) / (one + e), (v if gate == "silu" else 1) / (1 + np.exp(-v))
        error = lambda y: np.linalg.norm(y.astype(np.float64) - want) / np.linalg.norm(want)  # noqa: E731
        assert error(activation(ctx, gate, g)) <= 1.5 * error(formula)


@pytest.mark.parametrize("m", [1, 200])
@pytest.mark.parametrize("gate", ["silu", "gelu", "sigmoid", "relu"])
def test_activations_at_the_ends_of_float32(ctx, gate, m):
    largest = np.finfo(np.float32).max
    g = np.array([np.nan, np.inf, largest, 1e30, 200, 88.8, -88.8, -200, -1e30, -largest, -np.inf, 2, 2, 2], np.float32)
    u = np.array([1] * 11 + [np.inf, -np.inf, np.nan], np.float32)
    y = activation(ctx, gate, g, m, u)
    assert np.isnan(y[0]) and np.isnan(y[13])
    assert np.array_equal(y[1:6], np.ones(5, np.float32) if gate == "sigmoid" else g[1:6])
    assert np.all(np.abs(y[6:10]) <= 1.1e-36)  # zero, or the value where e^-g ends
    assert y[11] == np.inf and y[12] == -np.inf
