"""Log probabilities, entropy and the largest classes against 64 bits.

With d = x - max x: a difference is off by 2^-24 |d|, an exponential of it by less than 2^-22 |d| + 2^-22 relative (its argument's product with log2 e, the
function), a sum of c of them over 256 lanes or more by (c / 256 + 64) 2^-24 relative. The logarithm of the sum is off by that and by its own 2^-23 relative,
a log probability by two more roundings; the entropy by the logarithm's error and, relative to the mean of |d|, by that of the two sums."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from excalibur_amd import hip
    c = hip.Ctx(0)
    yield c
    c.close()


def _reference(x):
    """(log probabilities, entropy, bound of one, bound of the other) of rows in 64 bits."""
    x = x.astype(np.float64)
    c = x.shape[1]
    with np.errstate(all="ignore"):
        most = x.max(1, keepdims=True)
        empty = most[:, 0] == -np.inf
        d = np.where(empty[:, None], -np.inf, x - np.where(np.isfinite(most), most, 0.0))
        d = np.where(most == np.inf, np.nan, d)
        e = np.exp(d)
        s = e.sum(1, keepdims=True)
        log_s = np.where(empty[:, None], 0.0, np.log(s))
        p = e / np.where(s == 0, 1, s)
        entropy = np.where(empty, 0.0, (log_s[:, 0] - np.where(p > 0, p * d, 0.0).sum(1)))
        mean = np.where(p > 0, p * -d, 0.0).sum(1)
        mean2 = np.where(p > 0, p * d * d, 0.0).sum(1)
        rel = mean * 2.0 ** -22 + 2.0 ** -22 + (c / 256 + 64) * 2.0 ** -24
        b = rel + np.abs(log_s[:, 0]) * 2.0 ** -23
        return d - log_s, entropy, b, b + mean * (rel + 2.0 ** -22) + mean2 * 2.0 ** -22


def _order(x, top):
    x = x.astype(np.float64)
    key = np.where(np.isnan(x), np.inf, x)
    rank = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -key, ~np.isnan(x)), axis=1)
    return rank[:, :top]


def _run(ctx, x, ids=None, top=0, stride=None, entropy=True):
    m, c = x.shape
    wide = np.full((m, stride or c), np.nan, x.dtype)
    wide[:, :c] = x
    dx = ctx.array(wide.view(np.uint16) if x.dtype == np.float16 else wide)
    out = dict(entropy=ctx.empty((m,), np.float32)) if entropy else {}
    if ids is not None:
        out["log_p"] = ctx.empty(ids.shape, np.float32)
    if top:
        out.update(top_ids=ctx.empty((m, top), np.int32), top_log_p=ctx.empty((m, top), np.float32))
    d_ids = None if ids is None else ctx.array(ids.astype(np.int32))
    ctx.log_probabilities(dx, c, ids=d_ids, top=top, **out)
    got = {name: a.download() for name, a in out.items()}
    for a in [dx, d_ids, *out.values()]:
        if a is not None:
            a.free()
    return got


def _same(got, want, bound):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    same = (got == want) | np.isnan(want)
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, np.abs(got - want) / bound)
    assert np.all(off <= 1), float(np.nanmax(off))


def _check(ctx, x, ids=None, top=0, stride=None):
    got = _run(ctx, x, ids, top, stride)
    log_p, entropy, b, be = _reference(x)
    _same(got["entropy"], entropy, be)
    if ids is not None:
        c = x.shape[1]
        want = np.take_along_axis(log_p, np.clip(ids, 0, c - 1), 1)
        want = np.where(ids < 0, 0.0, np.where(ids >= c, np.nan, want))
        with np.errstate(invalid="ignore"):
            _same(got["log_p"], want, b[:, None] + np.where(np.isfinite(want), np.abs(want), 0) * 2.0 ** -22)
    if top:
        order = _order(x, top)
        assert np.array_equal(got["top_ids"], order)
        want = np.take_along_axis(log_p, order, 1)
        _same(got["top_log_p"], want, b[:, None] + np.where(np.isfinite(want), np.abs(want), 0) * 2.0 ** -22)


def _logits(rng, m, c, dtype):
    x = rng.standard_normal((m, c)) * 2.5
    x[np.arange(m), rng.integers(0, c, m)] += rng.uniform(0, 20, m)
    return x.astype(dtype)


SIZES = [(1, 1), (1, 2), (3, 63), (2, 64), (5, 65), (1, 1000), (300, 257), (17, 4096), (4, 4097), (2, 16384), (3, 16385), (1, 32000), (2, 50001), (1, 131072), (1, 262144), (40, 8191)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("m,c", SIZES)
def test_sizes(ctx, m, c, dtype):
    rng = np.random.default_rng(m + c)
    x = _logits(rng, m, c, dtype)
    ids = rng.integers(0, c, (m, 3))
    _check(ctx, x, ids, min(c, 20), c + (m + c) % 4)
    _check(ctx, x, ids[:, :1])
    _check(ctx, x, None, min(c, 64))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("c", [40, 1000, 20001, 70000])
def test_masked_rows(ctx, c, dtype):
    rng = np.random.default_rng(c)
    low = np.finfo(dtype).min
    x = _logits(rng, 9, c, dtype)
    x[0, rng.random(c) < 0.7] = -np.inf
    x[1] = -np.inf                          # nothing is left
    x[2] = -np.inf
    x[2, c // 2] = -3.0                     # one class is left
    x[3, rng.random(c) < 0.9] = low         # masked with the type's lowest value
    x[4] = low
    x[5] = -np.inf
    x[5, [0, c - 1]] = low
    x[6, c // 3] = np.nan
    x[7, c // 3:c // 3 + 2] = np.inf
    x[8] = -np.inf
    x[8, 5] = np.nan
    ids = np.stack([rng.integers(0, c, 9), np.full(9, c // 2), np.full(9, -1), np.full(9, c)], 1)
    _check(ctx, x, ids, 20)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("c", [64, 999, 16384, 100003])
def test_equal_values_go_by_their_index(ctx, c, dtype):
    rng = np.random.default_rng(c + 1)
    x = np.zeros((6, c), dtype)
    x[1] = -0.0
    x[1, ::3] = 0.0                                   # the zeros are alike
    x[2] = rng.integers(0, 4, c)                      # a few values, each many times
    x[3] = np.sort(rng.standard_normal(c)).astype(dtype)  # rising: the largest are all at the end
    x[4] = x[3][::-1]
    x[5, 64 * np.arange(c // 64)] = 1.0               # one place of every 64
    _check(ctx, x, None, min(64, c))
    _check(ctx, x, None, 7)


def test_large_and_small_values(ctx):
    rng = np.random.default_rng(9)
    x = _logits(rng, 6, 5000, np.float32)
    x[0] += 1e4
    x[1] -= 1e4
    x[2] = np.float32(3e38)
    x[3] *= 1e-30
    x[4, 77] = 3e38
    x[5] *= 50
    _check(ctx, x, rng.integers(0, 5000, (6, 2)), 10)


@pytest.mark.parametrize("c", [777, 40000])
def test_rows_at_any_alignment(ctx, c):
    rng = np.random.default_rng(c)
    for dtype, first in ((np.float16, 1), (np.float16, 3), (np.float32, 1), (np.float32, 3)):
        x = _logits(rng, 3, c, dtype)
        buf = np.zeros(first + x.size, dtype)
        buf[first:] = x.ravel()
        raw = np.uint16 if dtype == np.float16 else np.float32
        d = ctx.array(buf.view(raw))
        ids, top = ctx.empty((3, 9), np.int32), ctx.empty((3, 9), np.float32)
        ctx.log_probabilities(ctx.view(d.ptr.value + first * buf.itemsize, (3, c), raw), top=9, top_ids=ids, top_log_p=top)
        assert np.array_equal(ids.download(), _order(x, 9))


def test_many_rows_and_only_what_is_asked(ctx):
    rng = np.random.default_rng(10)
    x = _logits(rng, 3000, 300, np.float16)
    _check(ctx, x, rng.integers(-1, 300, (3000, 1)), 3)
    alone = _run(ctx, x, entropy=False, top=3)
    assert np.array_equal(alone["top_ids"], _order(x, 3))


def test_many_candidates_of_a_row(ctx):
    rng = np.random.default_rng(13)
    x = _logits(rng, 2, 3001, np.float32)
    _check(ctx, x, rng.integers(0, 3001, (2, 1000)))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("c", [130, 513, 2049, 8200, 24999])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_more_candidates_than_are_ranked(ctx, c, top, dtype):
    rng = np.random.default_rng(c + top)
    x = np.zeros((11, c), dtype)
    low = np.finfo(dtype).min
    x[0, rng.permutation(c)[:130]] = np.nan              # more than are asked, few others
    x[1] = rng.standard_normal(c)
    x[1, rng.permutation(c)[:100]] = np.inf
    x[2] = np.sort(rng.standard_normal(c)).astype(dtype)
    x[3] = np.linspace(1, 2, c)                          # close to each other
    x[4] = rng.integers(0, 40, c)
    x[5] = low
    x[5, rng.permutation(c)[:top - 1]] = -1.0            # one of the masked ones is among the largest
    x[6] = -np.inf
    x[6, c // 2:] = low
    x[7] = -np.inf
    x[7, -1] = 0.0
    x[8] = np.nan
    x[9, ::-1] = np.repeat(np.arange(c // 70 + 1), 70)[:c] % 1500  # 70 alike of each
    x[10] = np.where(np.arange(c) < c - 50, 1.0, 0.5)
    got = _run(ctx, x, None, top)
    assert np.array_equal(got["top_ids"], _order(x, top))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("m,c", [(520, 8193), (520, 16384), (300, 16390), (270, 24999)])
def test_rows_enough_for_long_slices(ctx, m, c, dtype):
    rng = np.random.default_rng(m + c)
    x = _logits(rng, m, c, dtype)
    x[3] = 0.0
    x[4] = np.finfo(dtype).min
    x[4, ::c // 5] = 1.0
    x[5] = np.sort(rng.standard_normal(c)).astype(dtype)
    x[6, rng.permutation(c)[:200]] = np.nan
    x[7] = -np.inf
    x[8] = -np.inf
    x[8, -3:] = 2.0
    x[9] = rng.integers(0, 50, c)
    ids = rng.integers(0, c, (m, 2))
    _check(ctx, x, ids, 8, c + c % 3)
    _check(ctx, x, ids, 64)
    _check(ctx, x, ids)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("c", [8192, 16384, 32760, 32767, 32768, 65536])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_the_largest_of_a_whole_group_s_values(ctx, c, top, dtype):
    """As many values as a group holds and nearly so, every one of them above what the search begins with: rows of NaN, and of NaN but for a few."""
    rng = np.random.default_rng(c + top)
    x = np.full((6, c), np.nan, dtype)
    x[1, rng.permutation(c)[:5]] = 1.0
    x[2, -1] = -3.0
    x[3] = np.inf
    x[3, ::9] = np.nan
    x[4] = np.where(np.arange(c) % 2, rng.standard_normal(c), np.nan)
    x[5] = -np.inf
    x[5, c // 2:] = np.nan
    got = _run(ctx, x, None, top)
    assert np.array_equal(got["top_ids"], _order(x, top))
    assert np.all(np.isnan(got["top_log_p"])) and np.all(np.isnan(got["entropy"]))


@pytest.mark.parametrize("m,c,top", [(48, 131072, 20), (300, 65537, 5), (33, 140000, 64)])
def test_one_workspace_for_smaller_calls(ctx, m, c, top):
    """A workspace of the largest call takes smaller ones, and nothing behind it or behind any result changes."""
    rng = np.random.default_rng(m + c)
    x = (rng.standard_normal((m, c)) * 2.5).astype(np.float16)
    ids = rng.integers(0, c, (m, 2)).astype(np.int32)
    dx, d_ids = ctx.array(x.view(np.uint16)), ctx.array(ids)
    nbytes = ctx.log_probabilities_workspace(m, c, top)
    for rows, classes, largest in ((m, c, top), (32, c, top), (17, c, top), (m, c, 1), (m, c, 0), (20, c - 9000, top), (3, 999, top)):
        work = ctx.array(np.full(nbytes + 4096, 0xA5, np.uint8))
        out = dict(entropy=ctx.array(np.full(rows + 64, 7.25, np.float32)), log_p=ctx.array(np.full((rows + 8, 2), 7.25, np.float32)))
        if largest:
            out.update(top_ids=ctx.array(np.full((rows + 8, largest), 77, np.int32)), top_log_p=ctx.array(np.full((rows + 8, largest), 7.25, np.float32)))
        ctx.log_probabilities(ctx.view(dx.ptr.value, (rows, c), np.uint16), classes, ids=ctx.view(d_ids.ptr.value, (rows, 2), np.int32), top=largest, workspace=work, **out)
        got = {name: a.download() for name, a in out.items()}
        assert np.all(work.download()[nbytes:] == 0xA5), (rows, classes, largest)
        for name, a in got.items():
            assert np.all(a[rows:] == (77 if name == "top_ids" else 7.25)), (name, rows, classes, largest)
        log_p, entropy, b, be = _reference(x[:rows, :classes])
        _same(got["entropy"][:rows], entropy, be)
        if largest:
            assert np.array_equal(got["top_ids"][:rows], _order(x[:rows, :classes], largest))
        for a in [work, *out.values()]:
            a.free()
    dx.free()
    d_ids.free()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("c", [1, 40, 3000, 40000])
def test_no_probability_above_one(ctx, c, dtype):
    """Rows that are sure of one class, at values all over the type's range: log probabilities are not above 0 and entropies not below, whatever is rounded."""
    rng = np.random.default_rng(c)
    m = 3000 if c <= 40 else 60
    sure = rng.uniform(-6e4, 6e4, m)
    x = np.full((m, c), -np.inf, dtype)
    x[:, 1::2] = (sure[:, None] - rng.uniform(0, 40, (m, c // 2))).astype(dtype)
    at = rng.integers(0, c, m)
    x[np.arange(m), at] = sure
    out = _run(ctx, x, at[:, None], top=1)
    assert np.all(out["log_p"] <= 0) and np.all(out["top_log_p"] <= 0) and np.all(out["entropy"] >= 0)
