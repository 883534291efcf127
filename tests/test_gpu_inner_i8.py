"""The inner products in 8-bit integers and their quantizer, alone and by experts, against their definitions (tests/i8ref.py has the bounds)."""
import numpy as np
import pytest

from tests import f8ref, i8ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from excalibur_amd import hip
    c = hip.Ctx(0)
    yield c
    c.close()


def _wide(a, stride, fill):
    """Rows of `stride`, `fill` behind each."""
    out = np.full((a.shape[0], stride), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


# ---- the quantizer ----
QUANTIZED = [(1, 1, 0), (1, 128, 0), (3, 127, 1), (16, 129, 0), (17, 1000, 7), (130, 260, 3), (5, 4096, 0), (1, 5000, 0), (300, 64, 0), (7, 8192, 1), (3, 16384, 0), (2, 40001, 3), (9, 2050, 6)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("m,k,pad", QUANTIZED)
def test_quantized_rows_are_exactly_the_definition(ctx, dtype, m, k, pad):
    rng = np.random.default_rng(m * 1000 + k)
    x = (rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))).astype(np.float16 if dtype == "f16" else np.float32)
    if m > 1:
        x[0] = 0
        x[1, -1] = np.nan
    if m > 3:
        x[2, 0], x[3, k // 2] = np.inf, -np.inf
        x[4 % m] = np.where(rng.random(k) < 0.5, 1, -1)
    want, scale = i8ref.quantize_rows(x.astype(np.float32))
    dx = ctx.array(_wide(x, k + pad, np.nan).view(np.uint16 if dtype == "f16" else np.float32))
    y = ctx.array(np.full((m, (k + 15) // 16 * 16 + 16), 0x25, np.int8))
    got, got_scale = ctx.quantize_rows_i8(dx, k, y=y)
    got, got_scale = got.download(), got_scale.download()
    assert np.array_equal(got_scale, scale, equal_nan=True)
    assert np.array_equal(got[:, :k], want)
    assert np.all(got[:, k:] == 0x25)  # nothing behind the rows


def test_quantized_rows_take_ties_to_the_even_code(ctx):
    """Scales that are powers of two, and odd ones: values that stand exactly between two codes, and their neighbours on either side."""
    rng = np.random.default_rng(5)
    scale = np.concatenate([2.0 ** np.arange(-60, 60), rng.integers(1 << 15, 1 << 16, 200) * 2.0 ** -20]).astype(np.float32)
    x = np.empty((len(scale), 512), np.float32)
    tie = (rng.integers(-127, 127, x.shape) + 0.5) * scale[:, None].astype(np.float64)  # at most 8 + 16 bits: a float32
    x[:] = tie
    assert np.array_equal(x, tie)
    x[:, 1::3] = np.nextafter(x[:, 1::3], np.float32(np.inf))
    x[:, 2::3] = np.nextafter(x[:, 2::3], np.float32(-np.inf))
    x[:, 0] = 127 * scale
    x = np.where(np.abs(x) > x[:, :1], x[:, :1], x)
    got, got_scale = ctx.quantize_rows_i8(ctx.array(x))
    want, want_scale = i8ref.quantize_rows(x)
    assert np.array_equal(want_scale, scale)
    assert np.array_equal(got_scale.download(), want_scale) and np.array_equal(got.download(), want)


def test_quantized_rows_of_every_size_of_value(ctx):
    """From the smallest float to the largest: the scale's floor, rows of subnormal values."""
    rng = np.random.default_rng(4)
    x = np.ldexp(rng.uniform(-2, 2, (277, 96)), np.arange(-149, 128)[:, None] - rng.integers(0, 9, (277, 96))).astype(np.float32)
    assert np.isfinite(x).all()
    got, scale = ctx.quantize_rows_i8(ctx.array(x))
    want, want_scale = i8ref.quantize_rows(x)
    assert np.array_equal(scale.download(), want_scale) and np.array_equal(got.download(), want)


@pytest.mark.parametrize("k", [301, 5001])
def test_quantized_rows_at_any_alignment_of_their_type(ctx, k):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, k)).astype(np.float16)
    want, want_scale = i8ref.quantize_rows(x.astype(np.float32))
    for dtype, bits in ((np.float16, np.uint16), (np.float32, np.float32)):
        for first in (1, 2, 3):
            buf = np.zeros(first + x.size, dtype)
            buf[first:] = x.ravel()
            d = ctx.array(buf.view(bits))
            got, scale = ctx.quantize_rows_i8(ctx.view(d.ptr.value + buf.itemsize * first, (4, k), bits))
            assert np.array_equal(got.download()[:, :k], want) and np.array_equal(scale.download(), want_scale)


def test_quantized_rows_that_lie_behind_four_gigabytes(ctx):
    from excalibur_amd import hip
    stride = 1_100_000_000  # of halves: the third row's bytes begin behind 2^32
    x = ctx.empty((2 * stride + 128,), np.uint16)
    rows = np.random.default_rng(6).standard_normal((3, 100)).astype(np.float16)
    for r in range(3):
        hip._check(hip.lib().exhip_memcpy_h2d(ctx.h, x.at(2 * r * stride).ptr, rows[r].ctypes.data_as(hip.ctypes.c_void_p), hip.ctypes.c_size_t(200)))
    got, scale = ctx.quantize_rows_i8(ctx.view(x.ptr.value, (3, stride), np.uint16), 100, y=ctx.empty((3, 112), np.int8))
    want, want_scale = i8ref.quantize_rows(rows.astype(np.float32))
    assert np.array_equal(got.download()[:, :100], want) and np.array_equal(scale.download(), want_scale)
    x.free()


# ---- the products ----
class Operands:
    """Rows and weights as codes of every value, on the host and on the device; codes that are not zero stand behind every row's end."""

    def __init__(self, ctx, rng, m, n, k, sides=1, bias=False, pad=0, experts=1):
        self.m, self.n, self.k = m, n, k
        self.x = rng.integers(-128, 128, (m, k)).astype(np.int8)
        self.x_scale = np.exp(rng.standard_normal(m) - 4).astype(np.float32)
        self.stride = (k + 15) // 16 * 16 + pad
        self.w = [rng.integers(-128, 128, (experts, n, k)).astype(np.int8) for _ in range(sides)]
        self.w_scale = [(np.exp(rng.standard_normal((experts, n)) - 4) / np.sqrt(k)).astype(np.float32) for _ in range(sides)]
        self.bias = [rng.standard_normal((experts, n)).astype(np.float32) if bias else None for _ in range(sides)]
        self.dx, self.dx_scale = ctx.array(_wide(self.x, self.stride, 77)), ctx.array(self.x_scale)
        self.packed = ctx.pack_i8_weights(n, k, *[ctx.array(w) for w in self.w], experts=experts)
        self.dw_scale = [ctx.array(s) for s in self.w_scale]
        self.dbias = [ctx.array(b) if b is not None else None for b in self.bias]

    def desc(self, ctx, m=None, y_stride=None):
        return ctx.i8_desc(self.m if m is None else m, self.n, self.k, x_stride=self.stride, y_stride=y_stride)

    def want(self, side=0, rows=slice(None), expert=0):
        bias = self.bias[side]
        return i8ref.side(self.x[rows], self.x_scale[rows], self.w[side][expert], self.w_scale[side][expert], None if bias is None else bias[expert])

    def result(self, gate=None, **by):
        return self.want(**by) if gate is None else i8ref.gated(gate, self.want(0, **by), self.want(1, **by))

    def run(self, ctx, d, gate=None, **more):
        """The product, gated and by experts where there are such, with arguments named for both."""
        args = dict(x=self.dx, x_scale=self.dx_scale, w=self.packed, **more)
        if gate is None:
            args.update(w_scale=self.dw_scale[0], bias=self.dbias[0])
        else:
            args.update(gate=gate, w_scale_gate=self.dw_scale[0], w_scale_up=self.dw_scale[1], bias_gate=self.dbias[0], bias_up=self.dbias[1])
        name = "innerproduct" + ("_grouped" if "experts" in more else "") + ("" if gate is None else "_gated") + "_i8"
        getattr(ctx, name)(d, **args)


def _near(got, want, bound):
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= bound), (float((off - bound).max()), np.unravel_index(np.argmax(off - bound), off.shape))


def _check(y32, y16, want, bound):
    _near(y32, want, bound)
    with np.errstate(over="ignore"):
        assert np.array_equal(y16.view(np.float16), y32.astype(np.float16))  # one rounding of the same value


SIZES = [(1, 1, 1), (1, 16, 128), (1, 1000, 2200), (2, 17, 127), (7, 300, 1000), (15, 129, 129), (16, 128, 256), (17, 64, 16), (33, 1000, 300), (64, 200, 384), (65, 127, 1000),
         (130, 257, 520), (257, 100, 640), (300, 520, 1531), (512, 384, 512), (1, 4096, 4096)]


def _product(ctx, m, n, k, bias, gate=None):
    o = Operands(ctx, np.random.default_rng(m + 7 * n + 13 * k), m, n, k, sides=1 if gate is None else 2, bias=bias, pad=16 * (m % 3))
    extra = n % 5
    y32 = ctx.array(np.full((m + 1, n + extra), 7.25, np.float32))
    y16 = ctx.array(np.full((m + 1, n + extra), 0x4567, np.uint16))
    o.run(ctx, o.desc(ctx, y_stride=n + extra), gate, y_f32=y32, y_f16=y16)
    y32, y16 = y32.download(), y16.download()
    _check(np.ascontiguousarray(y32[:m, :n]), np.ascontiguousarray(y16[:m, :n]), *o.result(gate))
    for y, fill in ((y32, 7.25), (y16, 0x4567)):
        assert np.all(y[m] == fill) and np.all(y[:, n:] == fill)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_is_the_definition(ctx, m, n, k, bias):
    _product(ctx, m, n, k, bias)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated_product_within_its_roundings(ctx, m, n, k, bias):
    _product(ctx, m, n, k, bias, ("silu", "gelu", "sigmoid", "relu")[(m + n) % 4])


@pytest.mark.parametrize("gate", ["silu", "gelu", "sigmoid", "relu"])
def test_every_activation(ctx, gate):
    _product(ctx, 20, 70, 200, True, gate)


def test_the_longest_sums_fit(ctx):
    """-128 times -128 as often as a row may be long: 2^31 - 2^14, all of it in one sum."""
    k = 131071
    for m in (1, 70):
        x, w = np.full((m, k), -128, np.int8), np.full((33, k), -128, np.int8)
        w[1] = 127
        dx, y = ctx.array(_wide(x, 131072, -128)), ctx.empty((m, 33), np.float32)
        ctx.innerproduct_i8(ctx.i8_desc(m, 33, k), dx, ctx.array(np.ones(m, np.float32)), ctx.pack_i8_weights(33, k, ctx.array(w)), ctx.array(np.ones(33, np.float32)), y_f32=y)
        want = np.full((m, 33), np.float32(16384 * k))
        want[:, 1] = np.float32(-128 * 127 * k)
        assert np.array_equal(y.download(), want)


def test_rows_that_are_not_numbers_stay_among_themselves(ctx):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((40, 200)).astype(np.float32)
    x[3, 7], x[20, 0], x[39, 199] = np.nan, np.inf, -np.inf
    bad = [3, 20, 39]
    w = rng.standard_normal((50, 200)).astype(np.float32)
    (dx, dx_scale), (dw, dw_scale) = ctx.quantize_rows_i8(ctx.array(x)), ctx.quantize_rows_i8(ctx.array(w))
    codes = dw.download()[:, :200]
    y = ctx.empty((40, 50), np.float32)
    ctx.innerproduct_i8(ctx.i8_desc(40, 50, 200, x_stride=208), dx, dx_scale, ctx.pack_i8_weights(50, 200, ctx.array(np.ascontiguousarray(codes))), dw_scale, y_f32=y)
    y, fine = y.download(), np.setdiff1d(np.arange(40), bad)
    assert np.isnan(y[bad]).all()
    qx, sx = i8ref.quantize_rows(x)
    qw, sw = i8ref.quantize_rows(w)
    assert np.array_equal(y[fine], i8ref.side(qx[fine], sx[fine], qw, sw)[0])


def test_a_row_has_the_same_result_alone_as_among_others(ctx):
    o = Operands(ctx, np.random.default_rng(9), 600, 330, 700, sides=2, bias=True)
    y = ctx.empty((600, 330), np.float32)
    o.run(ctx, o.desc(ctx), "gelu", y_f32=y)
    y = y.download()
    for first, count in ((0, 1), (599, 1), (37, 20), (100, 130)):
        part = ctx.empty((count, 330), np.float32)
        args = dict(gate="gelu", w_scale_gate=o.dw_scale[0], w_scale_up=o.dw_scale[1], bias_gate=o.dbias[0], bias_up=o.dbias[1], y_f32=part)
        ctx.innerproduct_gated_i8(o.desc(ctx, count), o.dx.at(first * o.stride), o.dx_scale.at(4 * first), o.packed, **args)
        assert np.array_equal(part.download(), y[first:first + count])


def test_rows_that_lie_behind_two_gigabytes(ctx):
    """Offsets of the last rows do not fit 32 bits, of the input's bytes nor of the result's."""
    m, k, n, stride, y_stride = 70000, 40, 33, 32768, 8192
    x = ctx.empty((m * stride,), np.int8)
    y = ctx.empty((m * y_stride,), np.float32)
    rng = np.random.default_rng(10)
    codes, w = rng.integers(-128, 128, (130, k)).astype(np.int8), rng.integers(-128, 128, (n, k)).astype(np.int8)
    x.zero()
    from excalibur_amd import hip
    first = m - 130
    rows = _wide(codes, stride, 1)
    hip._check(hip.lib().exhip_memcpy_h2d(ctx.h, x.at(first * stride).ptr, rows.ctypes.data_as(hip.ctypes.c_void_p), hip.ctypes.c_size_t(rows.nbytes)))
    scale = np.linspace(1, 2, m).astype(np.float32)
    w_scale = np.linspace(0.5, 3, n).astype(np.float32)
    ctx.innerproduct_i8(ctx.i8_desc(m, n, k, x_stride=stride, y_stride=y_stride), x, ctx.array(scale), ctx.pack_i8_weights(n, k, ctx.array(w)), ctx.array(w_scale), y_f32=y)
    got = np.empty((130, y_stride), np.float32)
    hip._check(hip.lib().exhip_memcpy_d2h(ctx.h, got.ctypes.data_as(hip.ctypes.c_void_p), y.at(first * y_stride * 4).ptr, hip.ctypes.c_size_t(got.nbytes)))
    assert np.array_equal(got[:, :n], i8ref.side(codes, scale[first:], w, w_scale)[0])
    x.free()
    y.free()


# ---- by experts ----
def _split(rng, m, experts, how):
    """Offsets of m rows: spread evenly, by chance, all to one expert, every second one without rows, or some rows before the first and behind the last."""
    if how == "even":
        counts = np.full(experts, m // experts)
    elif how == "one":
        counts = np.zeros(experts, int)
        counts[experts // 2] = m
    elif how == "none":
        counts = np.zeros(experts, int)
    else:
        p = rng.random(experts) ** 3 * (np.arange(experts) % 2 if how == "holes" and experts > 1 else 1)
        counts = rng.multinomial(m if how != "inside" else m * 2 // 3, p / p.sum())
    first = m // 6 if how == "inside" else 0
    return (first + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)


def _grouped(ctx, m, experts, n, k, how, gate=None, gather=False, bias=False):
    rng = np.random.default_rng(m + 3 * experts + 7 * n + 13 * k)
    offsets = _split(rng, m, experts, how)
    tokens = max(1, m // 3) if gather else m
    o = Operands(ctx, rng, tokens, n, k, sides=1 if gate is None else 2, bias=bias, pad=16 * (m % 2), experts=experts)
    source = rng.integers(0, tokens, m).astype(np.int32) if gather else np.arange(m)
    y32 = ctx.array(np.full((m + 1, n + 3), 7.25, np.float32))
    y16 = ctx.array(np.full((m + 1, n + 3), 0x4567, np.uint16))
    more = dict(rows=ctx.array(source), x_rows=tokens) if gather else {}
    o.run(ctx, o.desc(ctx, m, n + 3), gate, experts=experts, offsets=ctx.array(offsets), y_f32=y32, y_f16=y16, **more)
    y32, y16 = y32.download(), y16.download()
    untouched = np.ones(m + 1, bool)
    for e in range(experts):
        at = slice(offsets[e], offsets[e + 1])
        untouched[at] = False
        if at.stop > at.start:
            _check(np.ascontiguousarray(y32[at, :n]), np.ascontiguousarray(y16[at, :n]), *o.result(gate, rows=source[at], expert=e))
    for y, fill in ((y32, 7.25), (y16, 0x4567)):
        assert np.all(y[untouched] == fill) and np.all(y[:, n:] == fill)


GROUPED = [(8, 8, 40, 200, "even"), (1, 1, 33, 64, "one"), (1, 5, 16, 16, "one"), (50, 3, 100, 300, "chance"), (130, 7, 129, 140, "holes"), (300, 4, 70, 520, "inside"), (700, 2, 260, 130, "chance"),
           (64, 100, 20, 128, "chance"), (200, 64, 48, 256, "chance"), (20, 6, 40, 100, "none"), (500, 9, 64, 128, "one"), (257, 130, 35, 40, "holes"), (600, 20, 300, 400, "inside")]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("m,experts,n,k,how", GROUPED)
def test_grouped_product_is_the_definition(ctx, m, experts, n, k, how, gather):
    _grouped(ctx, m, experts, n, k, how, gather=gather, bias=m % 2 == 0)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("m,experts,n,k,how", GROUPED)
def test_grouped_gated_product_within_its_roundings(ctx, m, experts, n, k, how, gather):
    _grouped(ctx, m, experts, n, k, how, gate=("silu", "gelu", "sigmoid", "relu")[m % 4], gather=gather, bias=m % 3 == 0)


def test_a_thousand_experts(ctx):
    _grouped(ctx, 1500, 1024, 20, 32, "chance", gather=True)
    _grouped(ctx, 40, 1024, 20, 32, "chance")


def test_one_expert_of_all_rows_is_the_product_without(ctx):
    o = Operands(ctx, np.random.default_rng(12), 333, 200, 300, bias=True)
    a, b = ctx.empty((333, 200), np.float32), ctx.empty((333, 200), np.float32)
    o.run(ctx, o.desc(ctx), y_f32=a)
    o.run(ctx, o.desc(ctx), experts=1, offsets=ctx.array(np.array([0, 333], np.int32)), y_f32=b)
    assert np.array_equal(a.download(), b.download())


@pytest.mark.parametrize("m", [40, 700])
def test_rows_that_the_input_does_not_have_are_not_numbers(ctx, m):
    rng = np.random.default_rng(13)
    o = Operands(ctx, rng, 9, 50, 100, experts=3)
    source = rng.integers(0, 9, m).astype(np.int32)
    source[[1, 17, 30]] = -1, 9, 2 ** 31 - 1
    source[m - 1] = -2 ** 31
    offsets = np.array([0, 15, 35, m], np.int32)
    y = ctx.empty((m, 50), np.float32)
    o.run(ctx, o.desc(ctx, m), experts=3, offsets=ctx.array(offsets), rows=ctx.array(source), x_rows=9, y_f32=y)
    y = y.download()
    for e in range(3):
        at = np.arange(offsets[e], offsets[e + 1])
        bad = (source[at] < 0) | (source[at] >= 9)
        assert np.isnan(y[at[bad]]).all()
        assert np.array_equal(y[at[~bad]], o.want(rows=source[at[~bad]], expert=e)[0])


# ---- every kernel at the sizes of the others ----
FORMS, GROUPED_FORMS = 11, 7


@pytest.fixture
def pinned():
    from excalibur_amd import hip
    yield lambda form: hip.set_option("i8_form", form)
    hip.set_option("i8_form", 0)


FORM_SIZES = [(1, 1, 1), (2, 17, 127), (33, 300, 129), (65, 513, 500), (130, 257, 520), (300, 520, 1531), (1, 96, 4200)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("form", range(1, FORMS + 1))
def test_every_form_at_the_sizes_of_the_others(ctx, pinned, form, gated):
    pinned(form)
    for m, n, k in FORM_SIZES:
        _product(ctx, m, n, k, m % 2 == 0, ("silu", "gelu", "sigmoid", "relu")[(form + m) % 4] if gated else None)


@pytest.mark.parametrize("gate", ["silu", "gelu", "sigmoid", "relu"])
def test_every_form_with_every_activation(ctx, pinned, gate):
    for form in range(1, FORMS + 1):
        pinned(form)
        _product(ctx, 70, 150, 200, form % 2 == 0, gate)


FORM_GROUPED = [(1, 1, 33, 64, "one"), (50, 3, 100, 300, "chance"), (130, 7, 129, 140, "holes"), (300, 4, 530, 520, "inside"), (64, 100, 20, 128, "chance"), (20, 6, 40, 100, "none"), (257, 130, 35, 40, "holes")]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("form", range(1, GROUPED_FORMS + 1))
def test_every_form_by_experts_at_the_sizes_of_the_others(ctx, pinned, form, gated):
    pinned(form)
    for m, experts, n, k, how in FORM_GROUPED:
        _grouped(ctx, m, experts, n, k, how, gate=("silu", "gelu", "sigmoid", "relu")[(form + m) % 4] if gated else None, gather=(form + m) % 2 == 0, bias=m % 3 == 0)


@pytest.mark.parametrize("form", range(1, FORMS + 1))
def test_every_form_has_the_same_bits(ctx, pinned, form):
    """Sums are exact and results are rounded in one order: which kernel takes a call changes nothing, an activation's value neither."""
    o = Operands(ctx, np.random.default_rng(21), 150, 290, 600, sides=2, bias=True, pad=16)
    want, got = ctx.empty((150, 290), np.float32), ctx.empty((150, 290), np.float32)
    for gate in (None, "gelu", "silu"):
        pinned(1)
        o.run(ctx, o.desc(ctx), gate, y_f32=want) if gate else ctx.innerproduct_i8(o.desc(ctx), o.dx, o.dx_scale, ctx.pack_i8_weights(290, 600, ctx.array(o.w[0])), o.dw_scale[0], o.dbias[0], y_f32=want)
        pinned(form)
        o.run(ctx, o.desc(ctx), gate, y_f32=got) if gate else ctx.innerproduct_i8(o.desc(ctx), o.dx, o.dx_scale, ctx.pack_i8_weights(290, 600, ctx.array(o.w[0])), o.dw_scale[0], o.dbias[0], y_f32=got)
        assert np.array_equal(want.download(), got.download()), gate


def test_weights_that_go_past_l2(ctx):
    """One tile of rows and more than 40 MB of weights: the form that reads them past L2, alone and by experts."""
    _product(ctx, 2, 11000, 4100, True)
    _grouped(ctx, 40, 30, 1000, 1500, "chance", gate="silu", gather=True)


# ---- recorded, and beside others ----
def test_products_recorded_and_replayed(ctx):
    """A quantizer and the products behind it in one graph, with other rows and other experts at every replay."""
    from tests.test_gpu_experts import recorded
    rng = np.random.default_rng(14)
    m, n, k, experts = 90, 130, 260, 5
    o = Operands(ctx, rng, m, n, k, sides=2, bias=True, experts=experts)
    x, codes, scale = ctx.empty((m, k), np.float32), ctx.empty((m, 272), np.int8), ctx.empty((m,), np.float32)
    offsets, h, hq, hs = ctx.empty((experts + 1,), np.int32), ctx.empty((m, n), np.uint16), ctx.empty((m, 144), np.int8), ctx.empty((m,), np.float32)
    y = ctx.empty((m, 70), np.float32)
    w2 = rng.integers(-128, 128, (70, n)).astype(np.int8)
    packed2, w2_scale = ctx.pack_i8_weights(70, n, ctx.array(w2)), rng.random(70).astype(np.float32)
    dw2_scale = ctx.array(w2_scale)
    o.dx, o.dx_scale = codes, scale

    def step():
        ctx.quantize_rows_i8(x, y=codes, scale=scale)
        o.run(ctx, ctx.i8_desc(m, n, k), "silu", experts=experts, offsets=offsets, y_f16=h)
        ctx.quantize_rows_i8(h, y=hq, scale=hs)
        ctx.innerproduct_i8(ctx.i8_desc(m, 70, n), hq, hs, packed2, dw2_scale, y_f32=y)

    def fill(i):
        x.upload(np.random.default_rng(i).standard_normal((m, k)).astype(np.float32))
        offsets.upload(_split(np.random.default_rng(i), m, experts, "chance"))

    recorded(ctx, step, fill, [codes, scale, h, hq, hs, y])


def test_two_contexts_at_once():
    from excalibur_amd import hip
    rng = np.random.default_rng(15)
    both = [hip.Ctx(0), hip.Ctx(0)]
    sets = [Operands(c, rng, 200 + 100 * i, 300, 500, bias=True) for i, c in enumerate(both)]
    results = [[c.empty((o.m, 300), np.float32) for _ in range(6)] for c, o in zip(both, sets)]
    for turn in range(6):
        for c, o, y in zip(both, sets, results):
            o.run(c, o.desc(c), y_f32=y[turn])
    for c, o, ys in zip(both, sets, results):
        for y in ys:
            _near(y.download(), *o.want())
    for c in both:
        c.close()
