"""What the 8-bit floating point and log probability entry points refuse: checked on the host, before a device is asked for anything."""
import ctypes

import numpy as np
import pytest

from tests import f8ref

ERR_ARG = 10001


def _lib():
    from excalibur_amd import hip
    return hip.lib()


def _status(entry, *args):
    """For operands that are addresses only: what passes the checks ends in the runtime's own error where there is no GPU."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("operands are addresses only")
    ctx = ctypes.create_string_buffer(4096)
    return entry(ctx, *[ctypes.c_void_p(a) if isinstance(a, int) and a >= 0x10000 else a for a in args])


X, Y, S, W, S2, B, B2, I, P, E = (0x10000 * (i + 1) for i in range(10))


@pytest.mark.parametrize("name", ["exhip_quantize_rows_f32_to_f8", "exhip_quantize_rows_f16_to_f8"])
def test_quantize_rows_refusals(name):
    entry = getattr(_lib(), name)
    good = [X, 100, 3, 100, Y, 112, S]
    assert _status(entry, *good) not in (0, ERR_ARG)
    for at, bad in ((0, None), (4, None), (6, None), (1, 99), (2, 0), (2, -1), (3, 0), (5, 96), (5, 120), (4, Y + 8), (0, X + 1), (6, S + 2), (5, 1 << 23), (2, 1 << 27)):
        args = list(good)
        args[at] = bad
        assert _status(entry, *args) == ERR_ARG, (at, bad)


def test_quantize_blocks_and_pack_refusals():
    L = _lib()
    assert _status(L.exhip_quantize_blocks_f32_to_f8, X, 5, 7, Y, S) not in (0, ERR_ARG)
    for args in ((None, 5, 7, Y, S), (X, 0, 7, Y, S), (X, 5, -7, Y, S), (X, 5, 7, None, S), (X, 5, 7, Y, S + 1), (X + 2, 5, 7, Y, S), (X, 1 << 24, 1 << 22, Y, S)):
        assert _status(L.exhip_quantize_blocks_f32_to_f8, *args) == ERR_ARG, args
    assert _status(L.exhip_f8_pack_weights, 5, 7, X, W, Y) not in (0, ERR_ARG)
    for args in ((5, 7, None, W, Y), (0, 7, X, None, Y), (5, 7, X, W, None), (5, 7, X, W, Y + 8), (5, (1 << 22) + 1, X, None, Y), (1 << 24, 1 << 22, X, None, Y)):
        assert _status(L.exhip_f8_pack_weights, *args) == ERR_ARG, args
    assert L.exhip_f8_packed_bytes(17, 129, 0) == 2 * 2 * 2048 and L.exhip_f8_packed_bytes(17, 129, 1) == 2 * 2 * 2 * 2048
    assert L.exhip_f8_packed_bytes(0, 5, 0) == 0 and L.exhip_f8_packed_bytes(5, -1, 0) == 0
    assert L.exhip_f8_packed_bytes(1 << 24, 1 << 22, 0) == 1 << 46


def _desc(**change):
    from excalibur_amd import hip
    return ctypes.byref(hip.F8Desc(*[{**dict(m=3, n_out=40, k_in=100, x_stride=112, y_stride=48), **change}[f] for f, _ in hip.F8Desc._fields_]))


BAD_DESC = (dict(m=0), dict(n_out=0), dict(k_in=0), dict(m=-1), dict(x_stride=96), dict(x_stride=120), dict(y_stride=39), dict(x_stride=1 << 23), dict(k_in=1 << 23, x_stride=1 << 23),
            dict(m=1 << 30, n_out=1 << 24, y_stride=1 << 24))


def test_product_refusals():
    entry = _lib().exhip_innerproduct_f8
    good = [X, S, W, S2, B, Y, None]
    assert _status(entry, _desc(), *good) not in (0, ERR_ARG)
    assert _status(entry, _desc(), X, S, W, S2, None, None, Y) not in (0, ERR_ARG)
    for change in BAD_DESC:
        assert _status(entry, _desc(**change), *good) == ERR_ARG, change
    assert _status(entry, None, *good) == ERR_ARG
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (5, None), (0, X + 8), (1, S + 1), (2, W + 8), (3, S2 + 2), (4, B + 1), (5, Y + 2), (6, Y + 1)):
        args = list(good)
        args[at] = bad
        assert _status(entry, _desc(), *args) == ERR_ARG, (at, bad)


def test_gated_product_refusals():
    entry = _lib().exhip_innerproduct_gated_f8
    good = [0, X, S, W, S2, S2, B, B2, Y, None, None]
    codes = [0, X, S, W, S2, S2, B, B2, None, Y, P]
    assert _status(entry, _desc(), *good) not in (0, ERR_ARG)
    assert _status(entry, _desc(), *codes) not in (0, ERR_ARG)
    for change in BAD_DESC:
        assert _status(entry, _desc(**change), *good) == ERR_ARG, change
    assert _status(entry, _desc(y_stride=50), *codes) == ERR_ARG  # codes begin on 16 bytes
    for at, bad in ((0, -1), (0, 4), (1, None), (2, None), (3, None), (4, None), (5, None), (6, None), (7, None), (8, None), (8, Y + 1), (9, P), (10, P), (7, B2 + 2)):
        args = list(good)
        args[at] = bad
        assert _status(entry, _desc(), *args) == ERR_ARG, (at, bad)
    for at, bad in ((8, E), (9, None), (10, None), (9, Y + 8), (10, P + 2)):
        args = list(codes)
        args[at] = bad
        assert _status(entry, _desc(), *args) == ERR_ARG, (at, bad)


@pytest.mark.parametrize("name", ["exhip_log_probabilities_f32", "exhip_log_probabilities_f16"])
def test_log_probability_refusals(name):
    entry = getattr(_lib(), name)
    #       x, x_stride, m, c, ids, n_ids, log_p, entropy, top, top_ids, top_log_p, workspace
    good = [X, 100, 3, 100, I, 2, P, E, 5, Y, S, W]
    assert _status(entry, *good) not in (0, ERR_ARG)
    for at, bad in ((0, None), (0, X + 1), (1, 99), (2, 0), (3, 0), (3, -5), (4, None), (5, -1), (5, 0), (6, None), (8, -1), (8, 0), (8, 65), (9, None), (10, None), (11, None), (11, W + 8),
                    (4, I + 2), (6, P + 1), (7, E + 2), (9, Y + 1), (10, S + 3)):
        args = list(good)
        args[at] = bad
        assert _status(entry, *args) == ERR_ARG, (at, bad)
    assert _status(entry, X, 100, 3, 100, None, 0, None, None, 0, None, None, W) == ERR_ARG  # nothing is asked
    assert _status(entry, X, 100, 3, 4, None, 0, None, E, 5, Y, S, W) == ERR_ARG  # more classes than there are
    L = _lib()
    for args in ((0, 5, 0), (5, 0, 0), (5, 5, 6), (5, 100, 65), (5, 5, -1)):
        assert L.exhip_log_probabilities_workspace(*args) == 0, args
    assert L.exhip_log_probabilities_workspace(1, 1, 0) > 0


def test_a_null_context_is_refused():
    L = _lib()
    p = ctypes.c_void_p(0x10000)
    assert L.exhip_quantize_rows_f32_to_f8(None, p, 16, 1, 16, p, 16, p) == ERR_ARG
    assert L.exhip_f8_pack_weights(None, 1, 1, p, None, p) == ERR_ARG
    assert L.exhip_innerproduct_f8(None, _desc(), p, p, p, p, None, p, None) == ERR_ARG
    assert L.exhip_log_probabilities_f32(None, p, 16, 1, 16, None, 0, None, p, 0, None, None, p) == ERR_ARG


def test_codes_of_the_oracle():
    """The oracle's own codes: every value is its own code, ties go to the even one, the borders of the format."""
    finite = ~np.isnan(f8ref.VALUES)
    codes = np.arange(256, dtype=np.uint8)[finite]
    assert np.array_equal(f8ref.encode(f8ref.VALUES[finite]), codes)
    assert f8ref.VALUES.max(initial=0, where=finite) == 448 and f8ref.VALUES[1] == 2.0 ** -9 and f8ref.VALUES[8] == 2.0 ** -6
    assert f8ref.encode([2.0 ** -10, 3 * 2.0 ** -10, 17, 19, 460, -17, np.nan]).tolist() == [0, 2, 0x58, 0x5A, 0x7E, 0xD8, 0x7F]


def test_a_log_probability_workspace_is_enough_for_smaller_calls():
    """A server has one for its largest batch: the size never falls as rows, classes or the largest asked grow, and what is refused has none."""
    size = _lib().exhip_log_probabilities_workspace
    rows, classes, tops = (1, 2, 16, 17, 31, 32, 33, 48, 300, 4096), (64, 8192, 8193, 32767, 32768, 32769, 49153, 65536, 100003, 131071, 131072, 131073, 262144, 1000000), (0, 1, 2, 20, 64)
    sizes = np.array([[[size(m, c, top) for top in tops] for c in classes] for m in rows], np.int64)
    assert sizes.min() >= 16
    for axis in range(3):
        assert np.diff(sizes, axis=axis).min() >= 0, axis
    entry = _lib().exhip_log_probabilities_f32
    for m, c, top in ((1 << 22, 64, 0), (1 << 22, 64, 5), (1 << 19, 100000, 0), (1 << 20, 100000, 5)):
        assert size(m, c, top) == 0, (m, c, top)
        assert _status(entry, X, c, m, c, None, 0, None, E, top, Y if top else None, S if top else None, W) == ERR_ARG
        assert size(m // 16, c, top) > 0


def test_a_log_probability_workspace_holds_every_row_s_slices():
    """What the slices of a row need, counted from what a group holds: at least 8192 values of a row of more than 32768, sums of 16 bytes and 8 for each of the largest."""
    size = _lib().exhip_log_probabilities_workspace
    for m in (1, 32, 33, 700):
        for c in (32769, 40000, 65537, 131072, 131073, 500001):
            for top in (0, 1, 20, 64):
                assert size(m, c, top) >= m * -(-c // 8192) * (16 + 8 * top), (m, c, top)


def test_refusals_of_the_products_with_cut_sums():
    entry = _lib().exhip_innerproduct_cut_f8
    good = [X, S, W, S2, B, Y]
    assert _status(entry, _desc(), *good) not in (0, ERR_ARG)
    for change in BAD_DESC:
        assert _status(entry, _desc(**change), *good) == ERR_ARG, change
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (5, None), (0, X + 8), (1, S + 1), (2, W + 8), (3, S2 + 2), (4, B + 1), (5, Y + 1)):
        args = list(good)
        args[at] = bad
        assert _status(entry, _desc(), *args) == ERR_ARG, (at, bad)
    entry = _lib().exhip_innerproduct_gated_cut_f8
    good = [0, X, S, W, S2, S2, B, B2, Y]
    assert _status(entry, _desc(), *good) not in (0, ERR_ARG)
    for change in BAD_DESC:
        assert _status(entry, _desc(**change), *good) == ERR_ARG, change
    for at, bad in ((0, -1), (0, 4), (1, None), (2, None), (3, None), (4, None), (5, None), (6, None), (7, None), (8, None), (8, Y + 1), (7, B2 + 2)):
        args = list(good)
        args[at] = bad
        assert _status(entry, _desc(), *args) == ERR_ARG, (at, bad)


# ---- the Python face: operands of another type, or too small, never reach the library ----
def _face():
    from excalibur_amd import hip
    ctx = object.__new__(hip.Ctx)  # without a device: what passes the checks here is refused by the library for its missing context
    ctx.h = None
    return hip, ctx


def _refused(match, call, *args, **kw):
    hip, _ = _face()
    with pytest.raises(hip.ExhipError, match=match):
        call(*args, **kw)


PASSES = "NULL argument"  # the library's first check
OTHER_ROWS = (np.float64, np.int16, np.int32, np.uint8, np.dtype(">f4"), np.dtype(">f2"))


def test_face_refuses_other_rows_for_the_quantizers():
    hip, ctx = _face()
    view = lambda shape, dtype: hip.View(X, shape, dtype)
    y, scale = view((3, 112), np.uint8), view((1, 3), np.float32)
    for dtype in (np.float32, np.float16, np.uint16):
        _refused(PASSES, ctx.quantize_rows_f8, view((3, 100), dtype), y=y, scale=scale)
    for dtype in OTHER_ROWS:
        _refused("x is", ctx.quantize_rows_f8, view((3, 100), dtype), y=y, scale=scale)
    x = view((3, 100), np.float32)
    _refused("y is", ctx.quantize_rows_f8, x, y=view((3, 112), np.float32), scale=scale)
    _refused("y has", ctx.quantize_rows_f8, x, y=view((2, 112), np.uint8), scale=scale)
    _refused("scale is", ctx.quantize_rows_f8, x, y=y, scale=view((1, 3), np.float64))
    _refused("scale has", ctx.quantize_rows_f8, x, y=y, scale=view((1, 2), np.float32))
    _refused("x has", ctx.quantize_rows_f8, x, k=101, y=y, scale=scale)
    _refused("w is", ctx.quantize_blocks_f8, view((3, 100), np.float16))
    _refused("w is", ctx.pack_f8_weights, 3, 100, view((3, 100), np.float32))
    _refused("w has", ctx.pack_f8_weights, 4, 100, view((3, 100), np.uint8))
    _refused("w_up has", ctx.pack_f8_weights, 3, 100, view((3, 100), np.uint8), view((3, 99), np.uint8))
    _refused("packed has", ctx.pack_f8_weights, 3, 100, view((3, 100), np.uint8), packed=view((2047,), np.uint8))
    _refused(PASSES, ctx.pack_f8_weights, 3, 100, view((3, 100), np.uint8), packed=view((2048,), np.uint8))


def test_face_refuses_other_operands_of_the_products():
    hip, ctx = _face()
    view = lambda count, dtype: hip.View(X, (count,), dtype)
    d = ctx.f8_desc(3, 40, 100, y_stride=48)  # rows of 112 codes
    good = dict(x=view(2 * 112 + 100, np.uint8), x_scale=view(3, np.float32), w=view(3 * 2048, np.uint8), w_scale=view(1, np.float32), bias=view(40, np.float32),
                y_f32=view(2 * 48 + 40, np.float32), y_f16=view(2 * 48 + 40, np.float16))
    _refused(PASSES, ctx.innerproduct_f8, d, **good)
    _refused(PASSES, ctx.innerproduct_f8, d, **dict(good, y_f16=view(2 * 48 + 40, np.uint16)))
    for name, a in good.items():
        _refused(name + " has", ctx.innerproduct_f8, d, **dict(good, **{name: view(a.size - 1, a.dtype)}))
        _refused(name + " is", ctx.innerproduct_f8, d, **dict(good, **{name: view(a.size, np.int64)}))
    d.m = 4  # what a description says now counts
    _refused("x has", ctx.innerproduct_f8, d, **good)
    d.m = 3
    gated = dict(x=good["x"], x_scale=good["x_scale"], w=view(2 * 3 * 2048, np.uint8), w_scale_gate=good["w_scale"], w_scale_up=good["w_scale"], bias_gate=good["bias"], bias_up=good["bias"])
    for results in (dict(y_f16=view(2 * 48 + 40, np.uint16)), dict(y_f8=view(2 * 48 + 40, np.uint8), y_scale=view(3, np.float32))):
        call = dict(gated, **results)
        _refused(PASSES, ctx.innerproduct_gated_f8, d, **call)
        for name, a in call.items():
            _refused(" has", ctx.innerproduct_gated_f8, d, **dict(call, **{name: view(a.size - 1, a.dtype)}))
            _refused(" is", ctx.innerproduct_gated_f8, d, **dict(call, **{name: view(a.size, np.int64)}))
    _refused("more than a size of", ctx.f8_desc, 2 ** 32 + 3, 40, 100)
    _refused("more than a size of", ctx.f8_packed_bytes, 40, 2 ** 32 + 100)


def test_face_refuses_other_operands_of_the_log_probabilities():
    hip, ctx = _face()
    view = lambda shape, dtype: hip.View(X, shape, dtype)
    m, c, top = 3, 40000, 5
    good = dict(x=view((m, c), np.uint16), ids=view((m, 2), np.int32), log_p=view((m, 2), np.float32), entropy=view((m,), np.float32), top_ids=view((m, top), np.int32),
                top_log_p=view((m, top), np.float32), workspace=view((ctx.log_probabilities_workspace(m, c, top),), np.uint8))
    for dtype in (np.float32, np.float16, np.uint16):
        _refused(PASSES, ctx.log_probabilities, top=top, **dict(good, x=view((m, c), dtype)))
    for dtype in OTHER_ROWS:
        _refused("x is", ctx.log_probabilities, top=top, **dict(good, x=view((m, c), dtype)))
    _refused("ids is int64", ctx.log_probabilities, top=top, **dict(good, ids=view((m, 2), np.int64)))
    _refused("top_ids is", ctx.log_probabilities, top=top, **dict(good, top_ids=view((m, top), np.int64)))
    _refused("entropy is", ctx.log_probabilities, top=top, **dict(good, entropy=view((m,), np.float16)))
    for name in ("ids", "log_p", "top_ids", "top_log_p"):
        _refused(" has", ctx.log_probabilities, top=top, **dict(good, **{name: view((m - 1,) + good[name].shape[1:], good[name].dtype)}))
    _refused("entropy has", ctx.log_probabilities, top=top, **dict(good, entropy=view((m - 1,), np.float32)))
    _refused("workspace has", ctx.log_probabilities, top=top, **dict(good, workspace=view((good["workspace"].size - 1,), np.uint8)))
    _refused(PASSES, ctx.log_probabilities, top=top, **dict(good, workspace=view((-(-good["workspace"].size // 4),), np.float32)))
    _refused("x has", ctx.log_probabilities, c=c + 1, top=top, **good)
