"""Sums of answers and orders by expert where something is missing or at an end, against their definitions (tests/i8ref.py)."""
import numpy as np
import pytest

from tests import i8ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from excalibur_amd import hip
    c = hip.Ctx(0)
    yield c
    c.close()


@pytest.mark.parametrize("each,n", [(1, 40), (6, 1029), (64, 520)])
def test_a_row_whose_weights_are_all_of_nothing_is_zero_whatever_its_answers(ctx, each, n):
    rng = np.random.default_rng(each)
    m, answers = 5, 5 * each
    z = rng.standard_normal((answers, n)).astype(np.float16)
    places = rng.permutation(answers).reshape(m, each).astype(np.int32)
    weights = rng.standard_normal((m, each)).astype(np.float32)
    empty = [1, 3]
    weights[empty] = -np.inf
    z[places[1]] = np.nan  # rows that nothing computed
    z[places[3]] = np.inf
    places[3, 0] = answers  # no such row
    y32, y16 = ctx.empty((m, n), np.float32), ctx.empty((m, n), np.uint16)
    dz, dp, dw = ctx.array(z.view(np.uint16)), ctx.array(places), ctx.array(weights)
    ctx.combine_rows(dz, dp, dw, kind="log_normalized", y_f32=y32)
    ctx.combine_rows(dz, dp, dw, kind="log_normalized", y_f16=y16)
    got, halves = y32.download(), y16.download()
    assert not got[empty].view(np.uint32).any() and not halves[empty].any()
    others = [0, 2, 4]
    want, bound = i8ref.combine(z, places[others], weights[others], "log_normalized")
    assert np.all(np.abs(got[others] - want) <= bound)
