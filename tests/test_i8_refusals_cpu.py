"""What the entry points of the 8-bit integer products and of rows by experts refuse: checked on the host, before a device is asked for anything."""
import ctypes

import numpy as np
import pytest

from tests import i8ref
from tests.test_f8_refusals_cpu import ERR_ARG, _lib, _status

X, Y, S, W, S2, B, B2, I, P, E = (0x10000 * (i + 1) for i in range(10))


@pytest.mark.parametrize("name", ["exhip_quantize_rows_f32_to_i8", "exhip_quantize_rows_f16_to_i8"])
def test_quantize_rows_refusals(name):
    entry = getattr(_lib(), name)
    good = [X, 100, 3, 100, Y, 112, S]
    assert _status(entry, *good) not in (0, ERR_ARG)
    for at, bad in ((0, None), (4, None), (6, None), (1, 99), (2, 0), (2, -1), (3, 0), (5, 96), (5, 120), (4, Y + 8), (0, X + 1), (6, S + 2), (5, 1 << 23), (2, 1 << 27)):
        args = list(good)
        args[at] = bad
        assert _status(entry, *args) == ERR_ARG, (at, bad)


def test_packed_bytes_and_pack_refusals():
    L = _lib()
    size = L.exhip_i8_packed_bytes
    assert size(1, 33, 129, 0) == 2 * 2 * 4096 and size(1, 33, 129, 1) == 3 * 2 * 4096 and size(5, 32, 128, 0) == 5 * 4096
    for bad in ((0, 5, 5, 0), (1025, 5, 5, 0), (-1, 5, 5, 0), (1, 0, 5, 0), (1, 5, -1, 0), (1, 5, 131072, 0), (1, (1 << 24) + 1, 5, 0)):
        assert size(*bad) == 0, bad
    assert size(1024, 1 << 24, 131071, 1) == 1024 * (1 << 20) * 1024 * 4096
    assert _status(L.exhip_i8_pack_weights, 2, 5, 7, X, W, Y) not in (0, ERR_ARG)
    for args in ((2, 5, 7, None, W, Y), (0, 5, 7, X, None, Y), (2, 5, 7, X, W, None), (2, 5, 7, X, W, Y + 8), (1, 5, 131072, X, None, Y), (1024, 1 << 24, 131071, X, None, Y)):
        assert _status(L.exhip_i8_pack_weights, *args) == ERR_ARG, args


def _desc(**change):
    from excalibur_amd import hip
    return ctypes.byref(hip.I8Desc(*[{**dict(m=3, n_out=40, k_in=100, x_stride=112, y_stride=48), **change}[f] for f, _ in hip.I8Desc._fields_]))


BAD_DESC = (dict(m=0), dict(n_out=0), dict(k_in=0), dict(m=-1), dict(x_stride=96), dict(x_stride=120), dict(y_stride=39), dict(x_stride=1 << 23), dict(k_in=131072, x_stride=131072),
            dict(m=1 << 30, n_out=1 << 24, y_stride=1 << 24))


def _refuses(entry, lead, good, bad, desc=_desc):
    assert _status(entry, desc(), *lead, *good) not in (0, ERR_ARG)
    for change in BAD_DESC:
        assert _status(entry, desc(**change), *lead, *good) == ERR_ARG, change
    assert _status(entry, None, *lead, *good) == ERR_ARG
    for at, value in bad:
        args = list(good)
        args[at] = value
        assert _status(entry, desc(), *lead, *args) == ERR_ARG, (at, value)


PLAIN = [X, S, W, S2, B, Y, None]
PLAIN_BAD = [(0, None), (1, None), (2, None), (3, None), (5, None), (0, X + 8), (1, S + 1), (2, W + 8), (3, S2 + 2), (4, B + 1), (5, Y + 2), (6, Y + 1)]
GATED = [X, S, W, S2, E, B, B2, None, Y]
GATED_BAD = [(0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (6, None), (8, None), (0, X + 8), (1, S + 1), (2, W + 8), (3, S2 + 2), (4, E + 1), (6, B2 + 2), (7, Y + 2), (8, Y + 1)]


def test_product_refusals():
    L = _lib()
    _refuses(L.exhip_innerproduct_i8, [], PLAIN, PLAIN_BAD)
    _refuses(L.exhip_innerproduct_gated_i8, [0], GATED, GATED_BAD)
    for gate in (-1, 4):
        assert _status(L.exhip_innerproduct_gated_i8, _desc(), gate, *GATED) == ERR_ARG


def test_grouped_product_refusals():
    L = _lib()
    for rows, x_rows in ((None, 0), (P, 5)):
        _refuses(L.exhip_innerproduct_grouped_i8, [4, I, rows, x_rows], PLAIN, PLAIN_BAD)
        _refuses(L.exhip_innerproduct_grouped_gated_i8, [2, 4, I, rows, x_rows], GATED, GATED_BAD)
    bad = ((0, I, None, 0), (-3, I, None, 0), (1025, I, None, 0), (4, None, None, 0), (4, I + 2, None, 0), (4, I, P + 1, 5), (4, I, P, 0), (4, I, P, -1), (4, I, P, (1 << 31) // 112 + 1))
    for lead in bad:
        assert _status(L.exhip_innerproduct_grouped_i8, _desc(), *lead, *PLAIN) == ERR_ARG, lead
        assert _status(L.exhip_innerproduct_grouped_gated_i8, _desc(), 0, *lead, *GATED) == ERR_ARG, lead
    assert _status(L.exhip_innerproduct_grouped_gated_i8, _desc(), 4, 4, I, None, 0, *GATED) == ERR_ARG


def test_group_rows_refusals():
    entry = _lib().exhip_group_rows
    good = [I, 5, 2, 8, X, Y, P]
    assert _status(entry, *good) not in (0, ERR_ARG)
    for at, bad in ((0, None), (4, None), (5, None), (6, None), (1, 0), (1, -1), (2, 0), (2, 65), (3, 0), (3, 1025), (1, 1 << 28), (0, I + 1), (4, X + 2), (5, Y + 3), (6, P + 1)):
        args = list(good)
        args[at] = bad
        assert _status(entry, *args) == ERR_ARG, (at, bad)


@pytest.mark.parametrize("name", ["exhip_combine_rows_f32", "exhip_combine_rows_f16"])
def test_combine_rows_refusals(name):
    entry = getattr(_lib(), name)
    #       z, z_stride, z_rows, places, weights, kind, m, each, n, y, y_stride
    good = [X, 104, 12, P, W, 2, 6, 2, 100, Y, 101]
    assert _status(entry, *good) not in (0, ERR_ARG)
    for at, bad in ((0, None), (3, None), (4, None), (9, None), (1, 99), (2, 0), (5, -1), (5, 3), (6, 0), (7, 0), (7, 65), (8, 0), (8, (1 << 24) + 1), (10, 99), (6, 1 << 28), (0, X + 1), (3, P + 2),
                    (4, W + 2), (9, Y + 1)):
        args = list(good)
        args[at] = bad
        assert _status(entry, *args) == ERR_ARG, (at, bad)


def test_a_null_context_is_refused():
    L = _lib()
    p = ctypes.c_void_p(0x10000)
    assert L.exhip_quantize_rows_f32_to_i8(None, p, 16, 1, 16, p, 16, p) == ERR_ARG
    assert L.exhip_i8_pack_weights(None, 1, 1, 1, p, None, p) == ERR_ARG
    assert L.exhip_innerproduct_i8(None, _desc(), p, p, p, p, None, p, None) == ERR_ARG
    assert L.exhip_innerproduct_grouped_i8(None, _desc(), 1, p, None, 0, p, p, p, p, None, p, None) == ERR_ARG
    assert L.exhip_group_rows(None, p, 1, 1, 1, p, p, p) == ERR_ARG
    assert L.exhip_combine_rows_f32(None, p, 4, 1, p, p, 0, 1, 1, 4, p, 4) == ERR_ARG


def test_the_python_face_refuses_operands_of_another_type_or_too_small():
    from excalibur_amd import hip
    ctx = hip.Ctx.__new__(hip.Ctx)
    ctx.h = None
    view = lambda shape, dtype: hip.View(0x10000, shape, dtype)  # noqa: E731
    f32, f16, i8, u8, i32 = np.float32, np.uint16, np.int8, np.uint8, np.int32

    def refused(call, text):
        with pytest.raises(hip.ExhipError, match=text):
            call()

    refused(lambda: ctx.quantize_rows_i8(view((3, 40), np.float64), y=view((3, 48), i8), scale=view((3,), f32)), "x is float64")
    refused(lambda: ctx.quantize_rows_i8(view((3, 40), f32), y=view((3, 32), i8), scale=view((3,), f32)), "y has 96 values, the call takes 104")
    refused(lambda: ctx.quantize_rows_i8(view((3, 40), f32), y=view((3, 48), i8), scale=view((2,), f32)), "scale has 2")
    d = ctx.i8_desc(3, 40, 100)
    args = dict(x=view((3, 112), i8), x_scale=view((3,), f32), w=view((2 * 4096,), u8), w_scale=view((40,), f32), bias=view((40,), f32), y_f32=view((3, 40), f32))
    for name, small, text in (("x", view((2, 112), i8), "x has"), ("x_scale", view((3,), f16), "x_scale is"), ("w", view((4096,), u8), "w has"), ("w_scale", view((39,), f32), "w_scale has"),
                              ("bias", view((39,), f32), "bias has"), ("y_f32", view((119,), f32), "y_f32 has")):
        refused(lambda: ctx.innerproduct_i8(d, **{**args, name: small}), text)
    by = dict(args, experts=2, offsets=view((3,), i32), w=view((4 * 4096,), u8), w_scale=view((80,), f32), bias=view((80,), f32))
    for name, small, text in (("w", view((2 * 4096,), u8), "w has"), ("w_scale", view((40,), f32), "w_scale has"), ("offsets", view((2,), i32), "offsets has"), ("offsets", view((3,), f32), "offsets is"),
                              ("rows", view((2,), i32), "rows has")):
        refused(lambda: ctx.innerproduct_grouped_i8(d, **{**by, "x_rows": 1, name: small}), text)
    refused(lambda: ctx.innerproduct_grouped_i8(d, **{**by, "rows": view((3,), i32), "x_rows": 4}), "x has")
    refused(lambda: ctx.group_rows(view((4, 2), i32), 3, offsets=view((3,), i32), rows=view((8,), i32), places=view((4, 2), i32)), "offsets has")
    refused(lambda: ctx.group_rows(view((4, 2), f32), 3, offsets=view((4,), i32), rows=view((8,), i32), places=view((4, 2), i32)), "ids is")
    combine = dict(z=view((8, 20), f16), places=view((4, 2), i32), weights=view((8,), f32))
    refused(lambda: ctx.combine_rows(**combine), "one result")
    refused(lambda: ctx.combine_rows(**combine, y_f32=view((4, 20), f32), y_f16=view((4, 20), f16)), "one result")
    refused(lambda: ctx.combine_rows(**combine, y_f32=view((3, 20), f32)), "y_f32 has")
    refused(lambda: ctx.combine_rows(**{**combine, "weights": view((7,), f32)}, y_f16=view((4, 20), f16)), "weights has")


def test_codes_of_the_oracle():
    """Scale 1, so that codes are the rounded values: ties go to the even one; rows of zeros, of one size, and with what is not a number."""
    x = np.array([[127, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5], [0] * 8, [-3] * 8, [np.nan] + [1] * 7, [1, -np.inf] + [2] * 6], np.float32)
    codes, scale = i8ref.quantize_rows(x)
    assert codes[0].tolist() == [127, 0, 2, 2, 0, -2, 126, -126] and scale[0] == 1
    assert not codes[1].any() and scale[1] == np.float32(2.0 ** -100)
    assert (codes[2] == -127).all() and scale[2] == np.float32(3) / np.float32(127)
    assert not codes[3:].any() and np.isnan(scale[3:]).all()


def test_order_of_the_oracle():
    offsets, rows, places = i8ref.group(np.array([[2, 0], [2, 2], [-1, 0], [7, 1]]), 3)
    assert offsets.tolist() == [0, 2, 3, 6] and rows.tolist() == [0, 2, 3, 0, 1, 1, -1, -1]
    assert places.tolist() == [[3, 0], [4, 5], [-1, 1], [-1, 2]]
