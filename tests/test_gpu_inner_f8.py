"""The inner products in 8-bit floating point, their quantizers and what they refuse, against 64 bits (tests/f8ref.py has the bounds)."""
import ctypes

import numpy as np
import pytest

from tests import f8ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from excalibur_amd import hip
    c = hip.Ctx(0)
    yield c
    c.close()


def _rows(rng, m, k):
    x = rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))
    return x.astype(np.float32)


def _wide(a, stride, fill):
    """Rows of `stride`, `fill` behind each."""
    out = np.full((a.shape[0], stride), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


class Operands:
    """Rows and weights as codes, on the host and on the device; NaN codes stand behind every row's end."""

    def __init__(self, ctx, rng, m, n, k, sides=1, bias=False, pad=0):
        self.m, self.n, self.k = m, n, k
        self.x, self.x_scale = f8ref.quantize_rows(_rows(rng, m, k))
        self.stride = (k + 15) // 16 * 16 + pad
        self.w, self.w_scale, self.bias = [], [], []
        for _ in range(sides):
            w, s = f8ref.quantize_weights((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32))
            self.w.append(w)
            self.w_scale.append(s)
            self.bias.append(rng.standard_normal(n).astype(np.float32) if bias else None)
        self.dx, self.dx_scale = ctx.array(_wide(self.x, self.stride, 0x7F)), ctx.array(self.x_scale)
        self.packed = ctx.pack_f8_weights(n, k, *[ctx.array(w) for w in self.w])
        self.dw_scale = [ctx.array(s) for s in self.w_scale]
        self.dbias = [ctx.array(b) if b is not None else None for b in self.bias]

    def desc(self, ctx, y_stride=None):
        return ctx.f8_desc(self.m, self.n, self.k, x_stride=self.stride, y_stride=y_stride)

    def want(self, side=0):
        return f8ref.product(self.x, self.x_scale, self.w[side], self.w_scale[side], self.bias[side])


def _near(got, want, bound):
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= bound), (float((off / bound).max()), np.unravel_index(np.argmax(off / bound), off.shape))


# ---- quantizers ----
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("m,k,pad", [(1, 1, 0), (1, 128, 0), (3, 127, 1), (16, 129, 0), (17, 1000, 7), (130, 260, 3), (5, 4096, 0), (1, 5000, 0)])
def test_quantized_rows_are_exactly_the_definition(ctx, dtype, m, k, pad):
    rng = np.random.default_rng(m * 1000 + k)
    x = _rows(rng, m, k).astype(np.float16 if dtype == "f16" else np.float32)
    x[0, :min(k, 128)] = 0  # a block of zeros
    if m > 2:
        x[2, 0] = np.inf
        x[1, -1] = np.nan
        x[1, 0] = x.dtype.type(6e-8)
    want, scale = f8ref.quantize_rows(x.astype(np.float32))
    dx = ctx.array(_wide(x, k + pad, np.nan).view(np.uint16 if dtype == "f16" else np.float32))
    y = ctx.array(np.full((m, (k + 15) // 16 * 16 + 16), 0xA5, np.uint8))
    got, got_scale = ctx.quantize_rows_f8(dx, k, y=y)
    got, got_scale = got.download(), got_scale.download()
    assert np.array_equal(got_scale, scale)
    nan = np.isnan(f8ref.VALUES[want])
    assert np.array_equal(np.isnan(f8ref.VALUES[got[:, :k]]), nan)
    assert np.array_equal(got[:, :k][~nan], want[~nan])
    assert np.all(got[:, k:] == 0xA5)  # nothing behind the rows


def test_quantized_rows_at_any_alignment_of_their_type(ctx):
    rng = np.random.default_rng(3)
    x = _rows(rng, 4, 301).astype(np.float16)
    for first in (1, 2, 3):
        buf = np.zeros(first + x.size, np.float16)
        buf[first:] = x.ravel()
        d = ctx.array(buf.view(np.uint16))
        got, scale = ctx.quantize_rows_f8(ctx.view(d.ptr.value + 2 * first, (4, 301), np.uint16))
        want, want_scale = f8ref.quantize_rows(x.astype(np.float32))
        assert np.array_equal(got.download()[:, :301], want) and np.array_equal(scale.download(), want_scale)


def test_quantized_rows_of_every_size_of_value(ctx):
    """From the smallest float to the largest: the scale's floor, subnormal codes, values that round up to 448."""
    rng = np.random.default_rng(4)
    x = np.ldexp(rng.uniform(1, 2, (64, 256)), rng.integers(-149, 127, (64, 256))).astype(np.float32)
    x[:, 128:] = np.ldexp(rng.uniform(1, 2, (64, 128)), rng.integers(-12, 3, (64, 128))).astype(np.float32)
    got, scale = ctx.quantize_rows_f8(ctx.array(x))
    want, want_scale = f8ref.quantize_rows(x)
    assert np.array_equal(scale.download(), want_scale)
    assert np.array_equal(got.download(), want)


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 127), (300, 260), (5, 1000)])
def test_quantized_blocks_are_exactly_the_definition(ctx, n, k):
    w = np.random.default_rng(n + k).standard_normal((n, k)).astype(np.float32)
    got, scale = ctx.quantize_blocks_f8(ctx.array(w))
    want, want_scale = f8ref.quantize_weights(w)
    assert np.array_equal(got.download(), want) and np.array_equal(scale.download(), want_scale)


# ---- the product ----
SIZES = [(1, 1, 1), (1, 16, 128), (1, 1000, 2200), (2, 17, 127), (7, 300, 1000), (15, 129, 129), (16, 128, 256), (17, 64, 16), (33, 1000, 300), (64, 200, 384), (65, 127, 1000),
         (130, 257, 520), (257, 100, 640), (300, 520, 1531), (512, 384, 512), (1, 4096, 4096)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_within_its_roundings(ctx, m, n, k, bias):
    o = Operands(ctx, np.random.default_rng(m + 7 * n + 13 * k), m, n, k, bias=bias, pad=16 * (m % 3))
    want, bound = o.want()
    extra = n % 5
    y32 = ctx.array(np.full((m + 1, n + extra), 7.25, np.float32))
    y16 = ctx.array(np.full((m + 1, n + extra), 0x4567, np.uint16))
    ctx.innerproduct_f8(o.desc(ctx, n + extra), o.dx, o.dx_scale, o.packed, o.dw_scale[0], o.dbias[0], y_f32=y32, y_f16=y16)
    y32, y16 = y32.download(), y16.download()
    _near(y32[:m, :n], want, bound)
    _near(y16[:m, :n].view(np.float16), want, f8ref.half_bound(want, bound))
    assert np.array_equal(y16[:m, :n].view(np.float16), y32[:m, :n].astype(np.float16))  # one rounding of the same sum
    for y, fill in ((y32, 7.25), (y16, 0x4567)):
        assert np.all(y[m] == fill) and np.all(y[:, n:] == fill)


def test_product_of_whole_numbers_is_exact(ctx):
    """Codes of small whole numbers and scales of powers of two: every sum is a float32, so a wrong place or scale cannot hide in a bound."""
    rng = np.random.default_rng(11)
    for m, n, k in ((1, 48, 300), (40, 200, 384), (270, 300, 900)):
        o = Operands(ctx, rng, m, n, k)
        o.x = f8ref.encode(rng.integers(-8, 9, (m, k)))
        o.w[0] = f8ref.encode(rng.integers(-8, 9, (n, k)))
        o.x_scale = np.ldexp(1.0, rng.integers(-3, 4, o.x_scale.shape)).astype(np.float32)
        o.w_scale[0] = np.ldexp(1.0, rng.integers(-3, 4, o.w_scale[0].shape)).astype(np.float32)
        want, _ = o.want()
        y = ctx.empty((m, n), np.float32)
        ctx.innerproduct_f8(o.desc(ctx), ctx.array(_wide(o.x, o.stride, 0x7F)), ctx.array(o.x_scale), ctx.pack_f8_weights(n, k, ctx.array(o.w[0])), ctx.array(o.w_scale[0]), y_f32=y)
        assert np.array_equal(y.download().astype(np.float64), want)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_nan_stays_in_its_row_and_in_its_output(ctx, m):
    rng = np.random.default_rng(12)
    n, k = 150, 200
    o = Operands(ctx, rng, m, n, k)
    o.x[m - 1, 3] = 0x7F
    o.w[0][n - 1, k - 1] = 0xFF
    y = ctx.empty((m, n), np.float32)
    ctx.innerproduct_f8(o.desc(ctx), ctx.array(_wide(o.x, o.stride, 0x7F)), o.dx_scale, ctx.pack_f8_weights(n, k, ctx.array(o.w[0])), o.dw_scale[0], y_f32=y)
    want = np.zeros((m, n), bool)
    want[m - 1] = True
    want[:, n - 1] = True
    assert np.array_equal(np.isnan(y.download()), want)


def test_halves_beyond_their_range_are_infinite(ctx):
    x = np.full((2, 128), 1.0, np.float32)
    x[1] = -1
    codes, scale = f8ref.quantize_rows(x)
    scale[:] = 1e4
    w, ws = f8ref.quantize_weights(np.ones((3, 128), np.float32))
    y = ctx.empty((2, 3), np.uint16)
    ctx.innerproduct_f8(ctx.f8_desc(2, 3, 128), ctx.array(codes), ctx.array(scale), ctx.pack_f8_weights(3, 128, ctx.array(w)), ctx.array(ws), y_f16=y)
    y = y.download().view(np.float16)
    assert np.all(y[0] == np.inf) and np.all(y[1] == -np.inf)


# ---- the gated product ----
GATED = [(1, 1, 1), (1, 128, 128), (1, 1500, 1000), (3, 17, 127), (16, 130, 300), (17, 64, 16), (40, 300, 260), (64, 256, 384), (130, 257, 520), (300, 200, 640), (384, 512, 512)]


@pytest.mark.parametrize("gate", ["silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("m,n,k", GATED)
def test_gated_product_within_its_roundings(ctx, m, n, k, gate):
    o = Operands(ctx, np.random.default_rng(m + 5 * n + 11 * k), m, n, k, sides=2, bias=(m + n) % 2 == 1, pad=16 * (n % 2))
    h, bound = f8ref.gated(gate, *o.want(0), *o.want(1))
    args = (o.dx, o.dx_scale, o.packed, o.dw_scale[0], o.dw_scale[1], gate, o.dbias[0], o.dbias[1])
    extra = n % 3
    y = ctx.array(np.full((m + 1, n + extra), 0x4567, np.uint16))
    ctx.innerproduct_gated_f8(o.desc(ctx, n + extra), *args, y_f16=y)
    y = y.download()
    _near(y[:m, :n].view(np.float16), h, f8ref.half_bound(h, bound))
    assert np.all(y[m] == 0x4567) and np.all(y[:, n:] == 0x4567)
    stride, blocks = (n + 15) // 16 * 16 + 16, f8ref.blocks(n)
    codes, scale = ctx.array(np.full((m + 1, stride), 0xA5, np.uint8)), ctx.array(np.full((blocks + 1, m), 7.25, np.float32))
    ctx.innerproduct_gated_f8(o.desc(ctx, stride), *args, y_f8=codes, y_scale=scale)
    codes, scale = codes.download(), scale.download()
    assert np.all(codes[m] == 0xA5) and np.all(codes[:, n:] == 0xA5) and np.all(scale[blocks] == 7.25)
    scale = scale[:blocks]
    edge = np.zeros((m, blocks * 128))
    edge[:, :n] = np.abs(h)
    most = edge.reshape(m, blocks, 128).max(2).T
    edge[:, :n] = bound
    assert np.all(np.abs(scale - np.maximum(most / 448, 2.0 ** -100)) <= edge.reshape(m, blocks, 128).max(2).T / 448 + scale * 2.0 ** -22)
    _near(f8ref.rows_of(codes[:m, :n], scale), h, f8ref.code_bound(h, bound, scale))


def test_gated_codes_are_the_quantizer_s(ctx):
    """Whole-number operands through ReLU: h is exact, so codes and scales are those of the quantizer on it, bit for bit."""
    rng = np.random.default_rng(21)
    for m, n, k in ((1, 300, 128), (70, 200, 256), (300, 260, 128)):
        o = Operands(ctx, rng, m, n, k, sides=2)
        o.x = f8ref.encode(rng.integers(-4, 5, (m, k)))
        o.x_scale[:] = 1
        for s in range(2):
            o.w[s] = f8ref.encode(rng.integers(-4, 5, (n, k)))
            o.w_scale[s][:] = 2.0 ** -s
        h = f8ref.gate("relu", o.want(0)[0]) * o.want(1)[0]
        want, want_scale = f8ref.quantize_rows(h.astype(np.float32))
        stride = (n + 15) // 16 * 16
        codes, scale = ctx.empty((m, stride), np.uint8), ctx.empty(want_scale.shape, np.float32)
        ctx.innerproduct_gated_f8(o.desc(ctx, stride), ctx.array(_wide(o.x, o.stride, 0x7F)), ctx.array(o.x_scale), ctx.pack_f8_weights(n, k, ctx.array(o.w[0]), ctx.array(o.w[1])),
                                  ctx.array(o.w_scale[0]), ctx.array(o.w_scale[1]), "relu", y_f8=codes, y_scale=scale)
        assert np.array_equal(scale.download(), want_scale)
        assert np.array_equal(f8ref.VALUES[codes.download()[:, :n]], f8ref.VALUES[want])  # (a zero's sign is that of its product)


# ---- every kernel, at sizes that its rule would give to another ----
@pytest.fixture
def pin():
    from excalibur_amd import hip
    yield lambda form: hip.set_option("f8_form", form)
    hip.set_option("f8_form", 0)


FORM_SIZES = [(1, 1, 1), (16, 16, 128), (17, 130, 129), (130, 300, 1531), (257, 520, 384), (300, 257, 1000), (64, 128, 2049)]


@pytest.mark.parametrize("m,n,k", FORM_SIZES)
def test_every_form_of_the_product(ctx, pin, m, n, k):
    o = Operands(ctx, np.random.default_rng(m + 3 * n + 5 * k), m, n, k, bias=n % 2 == 0, pad=16 * (n % 2))
    want, bound = o.want()
    args = (o.dx, o.dx_scale, o.packed, o.dw_scale[0], o.dbias[0])
    cut = bound + f8ref.cut_bound(o.x, o.x_scale, o.w[0], o.w_scale[0])
    for form in range(1, 8):
        pin(form)
        for extra in (0, 3):
            y32, y16 = ctx.array(np.full((m + 1, n + extra), 7.25, np.float32)), ctx.array(np.full((m + 1, n + extra), 0x4567, np.uint16))
            d = o.desc(ctx, n + extra)
            ctx.innerproduct_f8(d, *args, y_f32=y32)
            ctx.innerproduct_f8(d, *args, y_f16=y16)
            y32, y16 = y32.download(), y16.download()
            _near(y32[:m, :n], want, bound)
            _near(y16[:m, :n].view(np.float16), want, f8ref.half_bound(want, cut))
            for y, fill in ((y32, 7.25), (y16, 0x4567)):
                assert np.all(y[m] == fill) and np.all(y[:, n:] == fill), form


@pytest.mark.parametrize("m,n,k", FORM_SIZES)
def test_every_form_of_the_gated_product(ctx, pin, m, n, k):
    o = Operands(ctx, np.random.default_rng(m + 3 * n + 7 * k), m, n, k, sides=2, bias=n % 2 == 0, pad=16 * (n % 2))
    (g, gb), (u, ub) = o.want(0), o.want(1)
    h, bound = f8ref.gated("silu", g, gb, u, ub)
    cut = f8ref.gated("silu", g, gb + f8ref.cut_bound(o.x, o.x_scale, o.w[0], o.w_scale[0]), u, ub + f8ref.cut_bound(o.x, o.x_scale, o.w[1], o.w_scale[1]))[1]
    args = (o.dx, o.dx_scale, o.packed, o.dw_scale[0], o.dw_scale[1], "silu", o.dbias[0], o.dbias[1])
    for form in range(1, 7):
        pin(form)
        y = ctx.array(np.full((m + 1, n + 3), 0x4567, np.uint16))
        ctx.innerproduct_gated_f8(o.desc(ctx, n + 3), *args, y_f16=y)
        y = y.download()
        _near(y[:m, :n].view(np.float16), h, f8ref.half_bound(h, cut))
        assert np.all(y[m] == 0x4567) and np.all(y[:, n:] == 0x4567), form
    stride, blocks = (n + 15) // 16 * 16 + 16, f8ref.blocks(n)
    for form in range(1, 4):
        pin(form)
        codes, scale = ctx.array(np.full((m + 1, stride), 0xA5, np.uint8)), ctx.array(np.full((blocks + 1, m), 7.25, np.float32))
        ctx.innerproduct_gated_f8(o.desc(ctx, stride), *args, y_f8=codes, y_scale=scale)
        codes, scale = codes.download(), scale.download()
        assert np.all(codes[m] == 0xA5) and np.all(codes[:, n:] == 0xA5) and np.all(scale[blocks] == 7.25), form
        _near(f8ref.rows_of(codes[:m, :n], scale[:blocks]), h, f8ref.code_bound(h, bound, scale[:blocks]))


def test_every_form_of_whole_numbers_is_exact(ctx, pin):
    """As test_product_of_whole_numbers_is_exact, of each kernel: values up to 8, so that nothing of eight products lies 13 bits beneath the largest."""
    rng = np.random.default_rng(61)
    for m, n, k in ((40, 200, 384), (270, 300, 905)):
        o = Operands(ctx, rng, m, n, k)
        o.x, o.w[0] = f8ref.encode(rng.integers(-8, 9, (m, k))), f8ref.encode(rng.integers(-8, 9, (n, k)))
        o.x_scale = np.ldexp(1.0, rng.integers(-2, 3, o.x_scale.shape)).astype(np.float32)
        o.w_scale[0] = np.ldexp(1.0, rng.integers(-2, 3, o.w_scale[0].shape)).astype(np.float32)
        want, _ = o.want()
        args = (ctx.array(_wide(o.x, o.stride, 0x7F)), ctx.array(o.x_scale), ctx.pack_f8_weights(n, k, ctx.array(o.w[0])), ctx.array(o.w_scale[0]))
        for form in range(1, 8):
            pin(form)
            y32, y16 = ctx.empty((m, n), np.float32), ctx.empty((m, n), np.uint16)
            ctx.innerproduct_f8(o.desc(ctx), *args, y_f32=y32)
            ctx.innerproduct_f8(o.desc(ctx), *args, y_f16=y16)
            assert np.array_equal(y32.download().astype(np.float64), want), form
            assert np.array_equal(y16.download().view(np.float16), want.astype(np.float16)), form


def test_every_form_keeps_a_nan_in_its_row(ctx, pin):
    rng = np.random.default_rng(62)
    m, n, k = 140, 150, 203
    o = Operands(ctx, rng, m, n, k)
    o.x[m - 1, 3] = 0x7F
    o.w[0][n - 1, k - 1] = 0xFF
    args = (ctx.array(_wide(o.x, o.stride, 0x7F)), o.dx_scale, ctx.pack_f8_weights(n, k, ctx.array(o.w[0])), o.dw_scale[0])
    want = np.zeros((m, n), bool)
    want[m - 1], want[:, n - 1] = True, True
    for form in range(1, 8):
        pin(form)
        y32, y16 = ctx.empty((m, n), np.float32), ctx.empty((m, n), np.uint16)
        ctx.innerproduct_f8(o.desc(ctx), *args, y_f32=y32)
        ctx.innerproduct_f8(o.desc(ctx), *args, y_f16=y16)
        assert np.array_equal(np.isnan(y32.download()), want) and np.array_equal(np.isnan(y16.download().view(np.float16)), want), form


def test_rows_far_into_a_large_tensor(ctx):
    """Offsets beyond 32 bits: rows of codes 2^22 bytes apart and results behind 4 GiB of others."""
    rng = np.random.default_rng(63)
    m, n, k = 1100, 96, 256
    o = Operands(ctx, rng, m, n, k)
    stride, y_stride = 1 << 22, 2_000_000
    x, y = ctx.empty((m, stride), np.uint8), ctx.empty((m, y_stride), np.float32)
    from excalibur_amd import hip
    for r in range(m):
        hip._check(hip.lib().exhip_memcpy_h2d(ctx.h, x.at(r * stride).ptr, ctypes.c_void_p(np.ascontiguousarray(o.x[r]).ctypes.data), ctypes.c_size_t(k)))
    ctx.innerproduct_f8(ctx.f8_desc(m, n, k, x_stride=stride, y_stride=y_stride), x, o.dx_scale, o.packed, o.dw_scale[0], y_f32=y)
    want, bound = o.want()
    got = np.empty((m, n), np.float32)
    for r in range(m):
        hip._check(hip.lib().exhip_memcpy_d2h(ctx.h, ctypes.c_void_p(got[r:].ctypes.data), y.at(r * y_stride * 4).ptr, ctypes.c_size_t(n * 4)))
    _near(got, want, bound)
    x.free()
    y.free()


# ---- as a program runs them ----
def _network(ctx, rng, m, hidden, k, classes):
    """rows -> codes -> gated product (codes) -> product (float32) -> log probabilities, all queued before anything is read."""
    gate, up = (f8ref.quantize_weights((rng.standard_normal((hidden, k)) / np.sqrt(k)).astype(np.float32)) for _ in range(2))
    head = f8ref.quantize_weights((rng.standard_normal((classes, hidden)) * 3 / np.sqrt(hidden)).astype(np.float32))
    dev = dict(gated=ctx.pack_f8_weights(hidden, k, ctx.array(gate[0]), ctx.array(up[0])), head=ctx.pack_f8_weights(classes, hidden, ctx.array(head[0])),
               scales=[ctx.array(s) for s in (gate[1], up[1], head[1])], ids=ctx.array(rng.integers(0, classes, (m, 2)).astype(np.int32)),
               x=ctx.empty((m, k), np.float32), codes=ctx.empty((m, (k + 15) // 16 * 16), np.uint8), scale=ctx.empty((f8ref.blocks(k), m), np.float32),
               h=ctx.empty((m, (hidden + 15) // 16 * 16), np.uint8), h_scale=ctx.empty((f8ref.blocks(hidden), m), np.float32), logits=ctx.empty((m, classes), np.float32),
               log_p=ctx.empty((m, 2), np.float32), entropy=ctx.empty((m,), np.float32), top_ids=ctx.empty((m, 5), np.int32), top_log_p=ctx.empty((m, 5), np.float32),
               work=ctx.empty((ctx.log_probabilities_workspace(m, classes, 5),), np.uint8))

    def forward():
        d = dev
        ctx.quantize_rows_f8(d["x"], k, y=d["codes"], scale=d["scale"])
        ctx.innerproduct_gated_f8(ctx.f8_desc(m, hidden, k, y_stride=d["h"].shape[1]), d["codes"], d["scale"], d["gated"], d["scales"][0], d["scales"][1], y_f8=d["h"], y_scale=d["h_scale"])
        ctx.innerproduct_f8(ctx.f8_desc(m, classes, hidden), d["h"], d["h_scale"], d["head"], d["scales"][2], y_f32=d["logits"])
        ctx.log_probabilities(d["logits"], ids=d["ids"], top=5, log_p=d["log_p"], entropy=d["entropy"], top_ids=d["top_ids"], top_log_p=d["top_log_p"], workspace=d["work"])

    def results():
        return {name: dev[name].download() for name in ("codes", "scale", "h", "h_scale", "logits", "log_p", "entropy", "top_ids", "top_log_p")}

    return dev, forward, results, (gate, up, head)


@pytest.mark.parametrize("m,hidden,k,classes", [(1, 700, 500, 1000), (19, 384, 256, 333), (200, 300, 260, 1000)])
def test_rows_to_log_probabilities(ctx, m, hidden, k, classes):
    rng = np.random.default_rng(31 + m)
    dev, forward, results, (gate, up, head) = _network(ctx, rng, m, hidden, k, classes)
    x = _rows(rng, m, k)
    dev["x"].upload(x)
    forward()
    got = results()
    codes, scale = f8ref.quantize_rows(x)
    assert np.array_equal(got["codes"][:, :k], codes) and np.array_equal(got["scale"], scale)
    h, bound = f8ref.gated("silu", *f8ref.product(codes, scale, *gate), *f8ref.product(codes, scale, *up))
    _near(f8ref.rows_of(got["h"][:, :hidden], got["h_scale"]), h, f8ref.code_bound(h, bound, got["h_scale"]))
    _near(got["logits"], *f8ref.product(got["h"][:, :hidden], got["h_scale"], *head))
    logits = got["logits"].astype(np.float64)
    log_p = logits - logits.max(1, keepdims=True)
    log_p -= np.log(np.exp(log_p).sum(1, keepdims=True))
    # (differences of a few tens, a sum of a few hundred terms: a hundred roundings at most of 64 at most)
    near = 100 * 64 * 2.0 ** -24
    order = np.argsort(-got["logits"], axis=1, kind="stable")[:, :5]
    assert np.array_equal(got["top_ids"], order)
    assert np.abs(got["top_log_p"] - np.take_along_axis(log_p, order, 1)).max() <= near
    assert np.abs(got["log_p"] - np.take_along_axis(log_p, dev["ids"].download().astype(np.int64), 1)).max() <= near
    assert np.abs(got["entropy"] + (np.exp(log_p) * log_p).sum(1)).max() <= near


def test_recorded_runs_are_the_direct_ones(ctx):
    from excalibur_amd import hip
    rng = np.random.default_rng(41)
    for m in (1, 70):
        dev, forward, results, _ = _network(ctx, rng, m, 300, 200, 1000)
        dev["x"].upload(_rows(rng, m, 200))
        forward()
        direct = results()
        graph = ctypes.c_void_p()
        hip._check(hip.lib().exhip_graph_begin(ctx.h))
        forward()
        hip._check(hip.lib().exhip_graph_end(ctx.h, ctypes.byref(graph)))
        for turn in range(4):
            x = _rows(rng, m, 200)
            dev["x"].upload(x)
            forward()
            direct = results()
            for name in direct:
                dev[name].zero()
            hip._check(hip.lib().exhip_graph_launch(ctx.h, graph))
            replayed = results()
            for name in direct:
                assert np.array_equal(replayed[name], direct[name]), (m, turn, name)
        hip._check(hip.lib().exhip_graph_destroy(graph))


def test_two_contexts_at_once(ctx):
    from excalibur_amd import hip
    other = hip.Ctx(0)
    rng = np.random.default_rng(51)
    both = [_network(c, rng, m, 384, 256, 1000) for c, m in ((ctx, 1), (other, 130))]
    alone = []
    for (dev, forward, results, _), m in zip(both, (1, 130)):
        dev["x"].upload(_rows(rng, m, 256))
        forward()
        alone.append(results())
    for _ in range(20):
        for _, forward, _, _ in both:
            forward()
    for (_, _, results, _), want in zip(both, alone):
        got = results()
        for name in want:
            assert np.array_equal(got[name], want[name]), name
    other.close()


@pytest.mark.parametrize("what,m,n,k", [("f32", 2060, 4087, 442), ("f16", 2895, 5799, 332), ("gated", 2076, 3892, 201)])
def test_last_rows_by_a_launch_of_their_own(ctx, what, m, n, k):
    o = Operands(ctx, np.random.default_rng(m + n + k), m, n, k, sides=2 if what == "gated" else 1, bias=True, pad=16)
    y = ctx.array(np.full((m + 1, n + 3), 7.25, np.float32) if what == "f32" else np.full((m + 1, n + 3), 0x4567, np.uint16))
    d, args = o.desc(ctx, n + 3), (o.dx, o.dx_scale, o.packed)
    some = np.r_[0:40, m // 2:m // 2 + 40, m - 300:m]  # the launches meet among the last rows
    x, x_scale = o.x[some], o.x_scale[:, some]
    want, bound = f8ref.product(x, x_scale, o.w[0], o.w_scale[0], o.bias[0])
    cut = bound + f8ref.cut_bound(x, x_scale, o.w[0], o.w_scale[0])
    if what == "gated":
        ctx.innerproduct_gated_f8(d, *args, *o.dw_scale, "silu", *o.dbias, y_f16=y)
        up, up_bound = f8ref.product(x, x_scale, o.w[1], o.w_scale[1], o.bias[1])
        want, bound = f8ref.gated("silu", want, cut, up, up_bound + f8ref.cut_bound(x, x_scale, o.w[1], o.w_scale[1]))
        bound = f8ref.half_bound(want, bound)
    else:
        ctx.innerproduct_f8(d, *args, o.dw_scale[0], o.dbias[0], **{"y_" + what: y})
        bound = bound if what == "f32" else f8ref.half_bound(want, cut)
    got, fill = y.download(), 7.25 if what == "f32" else 0x4567
    assert np.all(got[m] == fill) and np.all(got[:, n:] == fill) and not np.any(np.all(got[:m, :n] == fill, axis=1))
    _near((got if what == "f32" else got.view(np.float16))[some, :n], want, bound)


@pytest.fixture
def front(pin):
    from excalibur_amd import hip
    yield lambda rows: hip.set_option("f8_front", rows)
    hip.set_option("f8_front", 0)


@pytest.mark.parametrize("m,n,k,rows", [(5, 130, 129, 1), (97, 300, 260, 40), (300, 257, 1000, 129), (300, 140, 203, 299), (40, 64, 300, 40)])
def test_every_form_in_two_launches(ctx, pin, front, m, n, k, rows):
    """The first rows in a launch and the others in one: the results of one launch, whatever row the second begins with (a kernel's sums of a row do not depend on
    where it stands)."""
    o = Operands(ctx, np.random.default_rng(m + n + k), m, n, k, sides=2, bias=True, pad=16)
    args, single = (o.dx, o.dx_scale, o.packed), ctx.pack_f8_weights(n, k, ctx.array(o.w[0]))
    stride, blocks = (n + 15) // 16 * 16 + 16, f8ref.blocks(n)

    def calls():
        out = []
        for kw in (dict(y_f32=ctx.array(np.full((m + 1, n + 3), 7.25, np.float32))), dict(y_f16=ctx.array(np.full((m + 1, n + 3), 0x4567, np.uint16))),
                   dict(y_f16=ctx.array(np.full((m + 1, n + 3), 0x4567, np.uint16)), cut_sums=True)):
            ctx.innerproduct_f8(o.desc(ctx, n + 3), *args[:2], single, o.dw_scale[0], o.dbias[0], **kw)
            out += [a.download() for a in kw.values() if a is not True]
        for kw in (dict(y_f16=ctx.array(np.full((m + 1, n + 3), 0x4567, np.uint16))), dict(y_f16=ctx.array(np.full((m + 1, n + 3), 0x4567, np.uint16)), cut_sums=True)):
            ctx.innerproduct_gated_f8(o.desc(ctx, n + 3), *args, *o.dw_scale, "gelu", *o.dbias, **kw)
            out += [a.download() for a in kw.values() if a is not True]
        codes, scale = ctx.array(np.full((m + 1, stride), 0xA5, np.uint8)), ctx.array(np.full((blocks + 1, m), 7.25, np.float32))
        ctx.innerproduct_gated_f8(o.desc(ctx, stride), *args, *o.dw_scale, "gelu", *o.dbias, y_f8=codes, y_scale=scale)
        return out + [codes.download(), scale.download()]

    for form in range(1, 8):
        pin(form)
        front(0)
        one = calls()
        front(rows)
        for i, (a, b) in enumerate(zip(one, calls())):
            assert np.array_equal(a, b), (form, i)
    pin(0)
    calls()  # the rule's kernels for both


# ---- what sums keep ----
def _cancelling(rng, rows, k):
    """(values, the same with the large ones of every other group of eight negated): one of 448 in each of an even number of groups of eight of a block of
    128, and small whole numbers. The products of both cancel and leave those of the small ones."""
    at = np.array([8 * g + rng.integers(8) for g in range(k // 16 * 2)], int)
    out = []
    for m in rows:
        v = rng.integers(-2, 3, (m, k)).astype(np.float64)
        v[:, at] = 448
        out.append(v)
    out[1][:, at[1::2]] = -448
    return out


LOST = [(1, 48, 144), (17, 130, 144), (130, 300, 1536), (300, 257, 1000), (64, 128, 2064)]


def _exact_operands(ctx, rng, m, n, k, sides):
    o = Operands(ctx, rng, m, n, k, sides=sides)
    x, w = _cancelling(rng, (m, sides * n), k)
    o.x, o.w = f8ref.encode(x), list(f8ref.encode(w).reshape(sides, n, k))
    o.x_scale[:] = 1
    for s in o.w_scale:
        s[:] = 1
    return o, (ctx.array(_wide(o.x, o.stride, 0x7F)), ctx.array(o.x_scale), ctx.pack_f8_weights(n, k, *[ctx.array(np.ascontiguousarray(w)) for w in o.w]),
               *[ctx.array(s) for s in o.w_scale])


@pytest.mark.parametrize("m,n,k", LOST)
def test_sums_keep_what_large_products_leave(ctx, pin, m, n, k):
    """Every partial sum is a whole number below 2^24, so a float32 sum of the exact products is the result itself, in any order; of the matrix core's 8-bit
    products, which keep 13 bits beneath the largest of eight, nothing would be left of the small ones."""
    o, args = _exact_operands(ctx, np.random.default_rng(m + n + k), m, n, k, 1)
    want, _ = o.want()
    assert np.abs(want).max() <= 2048  # a half
    for form in range(0, 7):
        pin(form)
        y32, y16 = ctx.empty((m, n), np.float32), ctx.empty((m, n), np.uint16)
        ctx.innerproduct_f8(o.desc(ctx), *args, y_f32=y32)
        ctx.innerproduct_f8(o.desc(ctx), *args, y_f16=y16)
        assert np.array_equal(y32.download(), want), form
        assert np.array_equal(y16.download().view(np.float16), want), form


@pytest.mark.parametrize("m,n,k", LOST)
def test_gated_sums_keep_what_large_products_leave(ctx, pin, m, n, k):
    """As above, through ReLU: the codes are the quantizer's of the exact result, the halves its rounding."""
    o, args = _exact_operands(ctx, np.random.default_rng(m + n + k + 1), m, n, k, 2)
    h = f8ref.gate("relu", o.want(0)[0]) * o.want(1)[0]
    assert np.abs(h).max() < 2 ** 24
    want, want_scale = f8ref.quantize_rows(h.astype(np.float32))
    stride = (n + 15) // 16 * 16
    for form in range(0, 6):
        pin(form)
        y = ctx.empty((m, n), np.uint16)
        ctx.innerproduct_gated_f8(o.desc(ctx), *args, "relu", y_f16=y)
        assert np.array_equal(y.download().view(np.float16), h.astype(np.float16)), form
    for form in range(0, 4):
        pin(form)
        codes, scale = ctx.empty((m, stride), np.uint8), ctx.empty(want_scale.shape, np.float32)
        ctx.innerproduct_gated_f8(o.desc(ctx, stride), *args, "relu", y_f8=codes, y_scale=scale)
        assert np.array_equal(scale.download(), want_scale), form
        assert np.array_equal(f8ref.VALUES[codes.download()[:, :n]], f8ref.VALUES[want]), form


@pytest.mark.parametrize("m,n,k", [(1, 300, 1000), (17, 4096, 300), (64, 200, 2200), (256, 1030, 1100), (700, 520, 1531), (2100, 300, 260)])
def test_halves_are_the_float32_result_rounded_once(ctx, m, n, k):
    """Asked for alone, among few rows or many."""
    o = Operands(ctx, np.random.default_rng(m + n + k), m, n, k, bias=True)
    args = (o.dx, o.dx_scale, o.packed, o.dw_scale[0], o.dbias[0])
    y32, y16 = ctx.empty((m, n), np.float32), ctx.empty((m, n), np.uint16)
    ctx.innerproduct_f8(o.desc(ctx), *args, y_f32=y32)
    ctx.innerproduct_f8(o.desc(ctx), *args, y_f16=y16)
    assert np.array_equal(y16.download().view(np.float16), y32.download().astype(np.float16))


def _outliers(o, rng):
    """Channels of twenty times the size, as one in a hundred of a trained network's is: the largest of eight then stands far above the others."""
    x = _rows(rng, o.m, o.k) * np.where(rng.random(o.k) < 0.05, 20, 1).astype(np.float32)
    o.x, o.x_scale = f8ref.quantize_rows(x)


def _near_halves(got, want, bound):
    """As _near; what 65520, the border of the values that a half holds, is within reach of may be infinite."""
    beyond = np.isinf(got) & (np.signbit(got) == np.signbit(want)) & (np.abs(want) + bound >= 65520)
    _near(np.where(beyond, want, got), want, f8ref.half_bound(want, bound))


@pytest.mark.parametrize("outliers", [False, True])
@pytest.mark.parametrize("m,n,k", FORM_SIZES)
def test_every_form_of_cut_sums(ctx, pin, m, n, k, outliers):
    rng = np.random.default_rng(m + 3 * n + 9 * k)
    o = Operands(ctx, rng, m, n, k, sides=2, bias=n % 2 == 0, pad=16 * (n % 2))
    if outliers:
        _outliers(o, rng)
    dx, dx_scale = ctx.array(_wide(o.x, o.stride, 0x7F)), ctx.array(o.x_scale)
    packed = ctx.pack_f8_weights(n, k, ctx.array(o.w[0]))
    (g, gb), (u, ub) = o.want(0), o.want(1)
    gb, ub = gb + f8ref.cut_bound(o.x, o.x_scale, o.w[0], o.w_scale[0]), ub + f8ref.cut_bound(o.x, o.x_scale, o.w[1], o.w_scale[1])
    h, bound = f8ref.gated("silu", g, gb, u, ub)
    for form in range(0, 8):
        pin(form)
        for extra in (0, 3):
            y = ctx.array(np.full((m + 1, n + extra), 0x4567, np.uint16))
            ctx.innerproduct_f8(o.desc(ctx, n + extra), dx, dx_scale, packed, o.dw_scale[0], o.dbias[0], y_f16=y, cut_sums=True)
            got = y.download()
            _near_halves(got[:m, :n].view(np.float16), g, gb)
            assert np.all(got[m] == 0x4567) and np.all(got[:, n:] == 0x4567), form
            y = ctx.array(np.full((m + 1, n + extra), 0x4567, np.uint16))
            ctx.innerproduct_gated_f8(o.desc(ctx, n + extra), dx, dx_scale, o.packed, *o.dw_scale, "silu", *o.dbias, y_f16=y, cut_sums=True)
            got = y.download()
            _near_halves(got[:m, :n].view(np.float16), h, bound)
            assert np.all(got[m] == 0x4567) and np.all(got[:, n:] == 0x4567), form


def test_every_form_of_cut_sums_of_whole_numbers_and_nan(ctx, pin):
    """Values up to 8: nothing of eight products lies 13 bits beneath the largest, so places and scales cannot hide. A NaN stays in its row and its output."""
    rng = np.random.default_rng(71)
    m, n, k = 270, 300, 905
    o = Operands(ctx, rng, m, n, k)
    o.x, o.w[0] = f8ref.encode(rng.integers(-8, 9, (m, k))), f8ref.encode(rng.integers(-8, 9, (n, k)))
    o.x_scale = np.ldexp(1.0, rng.integers(-2, 3, o.x_scale.shape)).astype(np.float32)
    o.w_scale[0] = np.ldexp(1.0, rng.integers(-2, 3, o.w_scale[0].shape)).astype(np.float32)
    want, _ = o.want()
    o.x[m - 1, 3], o.w[0][n - 1, k - 1] = 0x7F, 0xFF
    want[m - 1], want[:, n - 1] = np.nan, np.nan
    args = (ctx.array(_wide(o.x, o.stride, 0x7F)), ctx.array(o.x_scale), ctx.pack_f8_weights(n, k, ctx.array(o.w[0])), ctx.array(o.w_scale[0]))
    for form in range(1, 8):
        pin(form)
        y = ctx.empty((m, n), np.uint16)
        ctx.innerproduct_f8(o.desc(ctx), *args, y_f16=y, cut_sums=True)
        assert np.array_equal(y.download().view(np.float16), want.astype(np.float16), equal_nan=True), form


def test_cut_sums_are_for_halves_alone(ctx):
    from excalibur_amd import hip
    o = Operands(ctx, np.random.default_rng(72), 3, 128, 128, sides=2)
    y32, y16, codes, scale = ctx.empty((3, 128), np.float32), ctx.empty((3, 128), np.uint16), ctx.empty((3, 128), np.uint8), ctx.empty((1, 3), np.float32)
    with pytest.raises(hip.ExhipError, match="halves alone"):
        ctx.innerproduct_f8(o.desc(ctx), o.dx, o.dx_scale, o.packed, o.dw_scale[0], y_f32=y32, y_f16=y16, cut_sums=True)
    with pytest.raises(hip.ExhipError, match="halves alone"):
        ctx.innerproduct_gated_f8(o.desc(ctx), o.dx, o.dx_scale, o.packed, *o.dw_scale, y_f8=codes, y_scale=scale, cut_sums=True)
    with pytest.raises(hip.ExhipError, match="no result"):
        ctx.innerproduct_f8(o.desc(ctx), o.dx, o.dx_scale, o.packed, o.dw_scale[0], cut_sums=True)
