"""Kernels and branches of the 8-bit integer products and their quantizer that only some sizes, strides and divisions among experts reach (tests/i8ref.py has the definitions and bounds)."""
import numpy as np
import pytest

from tests import i8ref
from tests.test_gpu_inner_i8 import FORMS, GROUPED_FORMS, Operands, _check, _grouped, _split, _wide

pytestmark = pytest.mark.gpu
GATES = ("silu", "gelu", "sigmoid", "relu")


@pytest.fixture(scope="module")
def ctx():
    from excalibur_amd import hip
    c = hip.Ctx(0)
    yield c
    c.close()


@pytest.fixture
def pinned():
    from excalibur_amd import hip
    yield lambda form: hip.set_option("i8_form", form)
    hip.set_option("i8_form", 0)


# ---- the quantizer ----
# A wave's pieces are 256 floats or 512 halves: rows of up to three waves' with one wave each (from 512 rows of floats, 2048 and 3500 of halves on, none of these a multiple of a group's four) and with
# four; the longer forms of one row a group; more than 128 MB, the same rows again and again.
QUANTIZED = [(515, 300, 0), (515, 513, 3), (515, 700, 0), (515, 768, 1), (515, 1000, 0), (515, 1500, 5), (515, 1536, 0), (2051, 700, 1), (2051, 1024, 0), (3503, 1300, 3), (3503, 1536, 0), (5, 1500, 0), (5, 2048, 2), (5, 3500, 1), (5, 6000, 0), (5, 11264, 0), (6, 12289, 1),
             (4, 20000, 0)]
PAST_L2 = {"f32": [(8203, 4101, 0), (112003, 300, 1), (46001, 760, 0), (16387, 2050, 1), (3801, 9000, 0)], "f16": [(16391, 4101, 0), (96003, 700, 1), (46001, 1500, 0), (6001, 11264, 0), (4001, 17000, 0)]}


def _quantized(ctx, dtype, m, k, pad, distinct=None):
    rng = np.random.default_rng(m + k)
    distinct = m if distinct is None else distinct
    x = rng.standard_normal((distinct, k), np.float32)
    x *= np.exp(rng.standard_normal((distinct, 1))).astype(np.float32)
    x = x.astype(np.float16 if dtype == "f16" else np.float32)
    x[0] = 0
    x[1, -1] = np.nan
    x[distinct - 1, 0] = np.inf
    x[2] = np.where(rng.random(k) < 0.5, 1, -1)
    want, scale = i8ref.quantize_rows(x.astype(np.float32))
    dx = ctx.array(_wide(x, k + pad, np.nan)[np.arange(m) % distinct].view(np.uint16 if dtype == "f16" else np.float32))
    y = ctx.array(np.full((m + 1, (k + 15) // 16 * 16 + 16), 0x25, np.int8))
    scales = ctx.array(np.full(m + 1, 7.25, np.float32))
    ctx.quantize_rows_i8(dx, k, y=y, scale=scales)
    got, got_scale = y.download(), scales.download()
    for first in range(0, m, distinct):
        rows = slice(first, min(m, first + distinct))
        count = rows.stop - first
        assert np.array_equal(got_scale[rows], scale[:count], equal_nan=True)
        assert np.array_equal(got[rows, :k], want[:count])
    assert got_scale[m] == 7.25 and np.all(got[:m, k:] == 0x25) and np.all(got[m] == 0x25)
    for a in (dx, y, scales):
        a.free()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("m,k,pad", QUANTIZED)
def test_quantized_rows_of_every_kernel(ctx, dtype, m, k, pad):
    _quantized(ctx, dtype, m, k, pad)


@pytest.mark.parametrize("dtype,m,k,pad", [(t, *s) for t, sizes in PAST_L2.items() for s in sizes])
def test_quantized_rows_that_go_past_l2(ctx, dtype, m, k, pad):
    assert m * k * (4 if dtype == "f32" else 2) > 128 << 20
    _quantized(ctx, dtype, m, k, pad, distinct=1031)


# ---- results that begin on lines ----
def _on_lines(ctx, m, n, k, gate=None, experts=0, how="chance"):
    """A product whose result rows begin on 128 bytes in either type, with a guard behind the rows and behind each."""
    rng = np.random.default_rng(m + n + k)
    o = Operands(ctx, rng, m, n, k, sides=1 if gate is None else 2, bias=True, experts=max(1, experts))
    stride = (n + 64) // 64 * 64
    y32, y16 = ctx.array(np.full((m + 1, stride), 7.25, np.float32)), ctx.array(np.full((m + 1, stride), 0x4567, np.uint16))
    assert y32.ptr.value % 128 == 0 and y16.ptr.value % 128 == 0 and stride > n
    offsets = _split(rng, m, experts, how) if experts else np.array([0, m])
    more = dict(experts=experts, offsets=ctx.array(offsets)) if experts else {}
    o.run(ctx, o.desc(ctx, y_stride=stride), gate, y_f32=y32, y_f16=y16, **more)
    y32, y16 = y32.download(), y16.download()
    untouched = np.ones(m + 1, bool)
    for e in range(max(1, experts)):
        at = slice(offsets[e], offsets[e + 1])
        untouched[at] = False
        if at.stop > at.start:
            _check(np.ascontiguousarray(y32[at, :n]), np.ascontiguousarray(y16[at, :n]), *o.result(gate, rows=at, expert=e))
    for y, fill in ((y32, 7.25), (y16, 0x4567)):
        assert np.all(y[untouched] == fill) and np.all(y[:, n:] == fill)


@pytest.mark.parametrize("gate", [None, "gelu"])
@pytest.mark.parametrize("m,n,k", [(130, 257, 520), (300, 520, 200), (64, 127, 384)])
@pytest.mark.parametrize("form", range(1, FORMS + 1))
def test_results_that_begin_on_lines(ctx, pinned, form, m, n, k, gate):
    pinned(form)
    _on_lines(ctx, m, n, k, gate)


@pytest.mark.parametrize("gate", [None, "silu"])
@pytest.mark.parametrize("m,experts,n,k,how", [(300, 4, 530, 260, "inside"), (260, 70, 257, 130, "holes")])
@pytest.mark.parametrize("form", range(1, GROUPED_FORMS + 1))
def test_results_by_experts_that_begin_on_lines(ctx, pinned, form, m, experts, n, k, how, gate):
    pinned(form)
    _on_lines(ctx, m, n, k, gate, experts, how)


# ---- more experts than lanes, with several tiles each ----
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("gate", [None, "silu"])
@pytest.mark.parametrize("form", range(GROUPED_FORMS + 1))
def test_experts_that_share_a_lane_have_several_tiles(ctx, pinned, form, gate, gather):
    pinned(form)
    _grouped(ctx, 3000, 130, 300, 140, "chance", gate, gather, bias=True)
    _grouped(ctx, 700, 100, 530, 64, "one", gate, gather)
    _grouped(ctx, 900, 1000, 40, 32, "holes", gate, gather)


def test_all_rows_to_one_expert_of_many_weights(ctx, pinned):
    """More than 40 MB of weights for few rows each as far as the sizes say, and thirteen tiles of rows for the same weights in fact."""
    for form in (0, 1, 2, 3):
        pinned(form)
        _grouped(ctx, 200, 60, 700, 1100, "one", "gelu" if form % 2 else None, gather=True)


# ---- offsets that do not rise ----
@pytest.mark.parametrize("form", range(GROUPED_FORMS + 1))
@pytest.mark.parametrize("experts", [5, 150])
def test_offsets_that_do_not_rise_stay_within_the_rows(ctx, pinned, form, experts):
    """Which of the experts a row goes to is not said then; rows that lie between no two neighbouring offsets, and what lies around the result, stay as they are."""
    pinned(form)
    m, n, k = 200, 70, 96
    rng = np.random.default_rng(experts)
    o = Operands(ctx, rng, m, n, k, experts=experts)
    low, high = np.iinfo(np.int32).min, np.iinfo(np.int32).max
    for offsets in (rng.permutation(experts + 1) * m // experts, np.full(experts + 1, high), np.full(experts + 1, low), np.where(np.arange(experts + 1) % 2, high, low), np.linspace(m, 0, experts + 1),
                    rng.integers(-m, 2 * m, experts + 1), np.where(np.arange(experts + 1) % 2, 120, 37)):
        offsets = offsets.astype(np.int32)
        y = ctx.array(np.full((m + 2, n + 3), 7.25, np.float32))
        inside = ctx.view(y.ptr.value + 4 * (n + 3), (m, n + 3), np.float32)
        o.run(ctx, o.desc(ctx, m, n + 3), experts=experts, offsets=ctx.array(offsets), y_f32=inside)
        got = y.download()
        inside_some = np.zeros(m, bool)
        for a, b in zip(np.clip(offsets[:-1], 0, m), np.clip(offsets[1:], 0, m)):
            inside_some[a:b] = True
        assert np.all(got[[0, -1]] == 7.25) and np.all(got[:, n:] == 7.25) and np.all(got[1:-1][~inside_some] == 7.25)


# ---- the same bits from every kernel ----
@pytest.mark.parametrize("gate", [None, *GATES])
@pytest.mark.parametrize("form", range(1, GROUPED_FORMS + 1))
def test_every_form_by_experts_has_the_bits_of_the_product_without(ctx, pinned, form, gate):
    m, n, k, experts = 310, 290, 300, 6
    rng = np.random.default_rng(31)
    offsets = _split(rng, m, experts, "chance")
    o = Operands(ctx, rng, m, n, k, sides=1 if gate is None else 2, bias=True, experts=experts)
    y = ctx.empty((m, n), np.float32)
    pinned(form)
    o.run(ctx, o.desc(ctx), gate, experts=experts, offsets=ctx.array(offsets), y_f32=y)
    y = y.download()
    for other in (1, FORMS):
        pinned(other)
        for e in range(experts):
            first, count = int(offsets[e]), int(offsets[e + 1] - offsets[e])
            if count == 0:
                continue
            part = ctx.empty((count, n), np.float32)
            packed = ctx.pack_i8_weights(n, k, *[ctx.array(w[e]) for w in o.w])
            scales, biases = [s.at(4 * e * n) for s in o.dw_scale], [b.at(4 * e * n) for b in o.dbias]
            args = (o.desc(ctx, count), o.dx.at(first * o.stride), o.dx_scale.at(4 * first), packed)
            if gate is None:
                ctx.innerproduct_i8(*args, scales[0], biases[0], y_f32=part)
            else:
                ctx.innerproduct_gated_i8(*args, *scales, gate, *biases, y_f32=part)
            assert np.array_equal(part.download().view(np.uint32), y[first:first + count].view(np.uint32)), (other, e)


@pytest.mark.parametrize("gate", [None, *GATES])
def test_the_first_form_has_the_bits_of_the_others(ctx, pinned, gate):
    o = Operands(ctx, np.random.default_rng(22), 140, 210, 500, sides=1 if gate is None else 2, bias=True)
    results = []
    for form in range(FORMS + 1):
        pinned(form)
        y = ctx.empty((140, 210), np.float32)
        o.run(ctx, o.desc(ctx), gate, y_f32=y)
        results.append(y.download())
    for y in results[2:] + results[:1]:
        assert np.array_equal(y.view(np.uint32), results[1].view(np.uint32))


def test_operands_that_end_with_their_last_value(ctx):
    """The last row's last piece of 16 bytes is read whole: what lies behind the row's end counts for nothing, whatever it is."""
    m, n, k = 37, 50, 131
    rng = np.random.default_rng(5)
    codes, w = rng.integers(-128, 128, (m, k)).astype(np.int8), rng.integers(-128, 128, (n, k)).astype(np.int8)
    results = []
    for behind in (0, 127, -128):
        wide = _wide(codes, 144, behind)
        y = ctx.empty((m, n), np.float32)
        x = ctx.array(wide)
        ctx.innerproduct_i8(ctx.i8_desc(m, n, k, x_stride=144), ctx.view(x.ptr.value, ((m - 1) * 144 + k,), np.int8), ctx.array(np.ones(m, np.float32)), ctx.pack_i8_weights(n, k, ctx.array(w)),
                            ctx.array(np.ones(n, np.float32)), y_f32=y)
        results.append(y.download())
    want = (codes.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32)
    for y in results:
        assert np.array_equal(y, want)
