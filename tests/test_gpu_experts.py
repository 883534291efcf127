"""Rows put in order by expert, the sum of their answers, and a layer of experts as a program runs it, against their definitions (tests/i8ref.py)."""
import ctypes

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


def recorded(ctx, step, fill, results, turns=4):
    """What a graph of step() leaves in `results` after each fill(i), against step() by itself."""
    from excalibur_amd import hip
    want = []
    for i in range(turns):
        fill(i)
        step()
        want.append([r.download() for r in results])
    graph = ctypes.c_void_p()
    hip._check(hip.lib().exhip_graph_begin(ctx.h))
    try:
        step()
    finally:
        hip._check(hip.lib().exhip_graph_end(ctx.h, ctypes.byref(graph)))
    for i in (*range(turns), 1):
        fill(i)
        for r in results:
            r.zero()
        hip._check(hip.lib().exhip_graph_launch(ctx.h, graph))
        for r, w in zip(results, want[i]):
            assert np.array_equal(r.download().view(np.uint8), w.view(np.uint8)), i
        step()  # the program's own work between the replays
        ctx.sync()
    hip._check(hip.lib().exhip_graph_destroy(graph))


# ---- in order by expert ----
GROUPS = [(1, 1, 1, "all"), (1, 8, 64, "all"), (3, 2, 5, "all"), (16, 8, 64, "all"), (63, 1, 2, "all"), (65, 1, 3, "some"), (100, 3, 20, "some"), (1024, 1, 7, "all"), (1025, 4, 256, "some"),
          (700, 64, 100, "all"), (5, 4, 1024, "some"), (3000, 6, 1, "some"), (4097, 8, 128, "one"), (200, 5, 33, "none"), (20000, 8, 300, "some"), (8191, 8, 64, "all"),
          (2048, 8, 256, "some"), (2049, 8, 7, "all"), (8191, 8, 256, "none"), (8191, 8, 1024, "all"), (3, 5, 600, "some"), (40000, 8, 2, "some"), (70000, 5, 1000, "some"), (300000, 1, 5, "all")]


@pytest.mark.parametrize("m,each,experts,which", GROUPS)
def test_order_is_that_of_the_experts_and_then_of_the_choices(ctx, m, each, experts, which):
    rng = np.random.default_rng(m + each)
    ids = rng.integers(0, experts, (m, each)).astype(np.int32)  # some experts more than once in a row
    if which == "some":
        ids[rng.random(ids.shape) < 0.3] = -1
        ids.ravel()[::97] = experts
        ids.ravel()[::89] = np.iinfo(np.int32).min
        ids.ravel()[::83] = np.iinfo(np.int32).max
    elif which == "one":
        ids[:] = experts - 1
    elif which == "none":
        ids[:] = -1
    want = i8ref.group(ids, experts)
    out = [ctx.array(np.full(w.size + 5, 99, np.int32)) for w in want]
    ctx.group_rows(ctx.array(ids), experts, *[ctx.view(o.ptr.value, w.shape, np.int32) for o, w in zip(out, want)])
    for o, w in zip(out, want):
        got = o.download()
        assert np.array_equal(got[:w.size], w.ravel()) and np.all(got[w.size:] == 99)


def test_orders_recorded_and_replayed(ctx):
    ids = ctx.empty((300, 4), np.int32)
    out = [ctx.empty((21,), np.int32), ctx.empty((1200,), np.int32), ctx.empty((300, 4), np.int32)]
    recorded(ctx, lambda: ctx.group_rows(ids, 20, *out), lambda i: ids.upload(np.random.default_rng(i).integers(-3, 22, (300, 4)).astype(np.int32)), out)


# ---- the sum of the answers ----
@pytest.mark.parametrize("kind", ["plain", "log", "log_normalized"])
@pytest.mark.parametrize("m,each,n,pad", [(1, 1, 1, 0), (1, 8, 4096, 0), (3, 2, 7, 1), (50, 6, 1023, 2), (17, 3, 1024, 0), (9, 64, 130, 6), (300, 4, 1029, 3), (2, 5, 5000, 0), (40, 1, 64, 8), (33, 7, 2056, 0)])
def test_combined_rows_within_their_roundings(ctx, m, each, n, pad, kind):
    rng = np.random.default_rng(m + each + n)
    z_rows = m * each + 3
    z = (rng.standard_normal((z_rows, n)) * 10).astype(np.float16)
    places = rng.permutation(z_rows)[:m * each].reshape(m, each).astype(np.int32)
    weights = rng.standard_normal((m, each)).astype(np.float32) * (1 if kind == "plain" else 4)
    if m > 2:
        places[rng.random(places.shape) < 0.2] = -1
        places[0] = -1
        z[np.setdiff1d(np.arange(z_rows), places)] = np.nan  # rows that nothing chose
        places[1, 0] = z_rows + 4  # no such row
        if kind != "plain":
            weights[2] = -np.inf
            weights[m - 1, 0] = -np.inf
    wide = np.full((z_rows, n + pad), np.nan, np.float16)
    wide[:, :n] = z
    dz, dp, dw = ctx.array(wide.view(np.uint16)), ctx.array(places), ctx.array(weights)
    y32, y16 = ctx.array(np.full((m + 1, n + pad), 7.25, np.float32)), ctx.array(np.full((m + 1, n + pad), 0x4567, np.uint16))
    ctx.combine_rows(dz, dp, dw, n, kind, y_f32=y32)
    ctx.combine_rows(dz, dp, dw, n, kind, y_f16=y16)
    y32, y16 = y32.download(), y16.download()
    want, bound = i8ref.combine(z, places, weights, kind)
    got = y32[:m, :n]
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad)
    assert np.all(np.abs(got.astype(np.float64) - want)[~bad] <= bound[~bad])
    with np.errstate(over="ignore"):
        assert np.array_equal(y16[:m, :n].copy().view(np.float16), got.astype(np.float16), equal_nan=True)
    for y, fill in ((y32, 7.25), (y16, 0x4567)):
        assert np.all(y[m] == fill) and np.all(y[:, n:] == fill)
    if m > 2:
        assert not got[0].any()


def test_combined_rows_at_any_alignment_of_their_types(ctx):
    rng = np.random.default_rng(2)
    z = rng.standard_normal((12, 1111)).astype(np.float16)
    places, weights = rng.permutation(12).reshape(4, 3).astype(np.int32), rng.random((4, 3)).astype(np.float32)
    want, bound = i8ref.combine(z, places, weights, "plain")
    for first in (0, 1, 2, 3, 5):
        buf = ctx.array(np.concatenate([np.zeros(first, np.float16), z.ravel()]).view(np.uint16))
        out = ctx.empty((first + 4 * 1111,), np.float32)
        ctx.combine_rows(ctx.view(buf.ptr.value + 2 * first, z.shape, np.uint16), ctx.array(places), ctx.array(weights), y_f32=ctx.view(out.ptr.value + 4 * first, (4, 1111), np.float32))
        assert np.all(np.abs(out.download()[first:].reshape(4, 1111) - want) <= bound)


def test_combined_rows_that_lie_behind_four_gigabytes(ctx):
    stride, rows = 1 << 20, 2100
    z = ctx.empty((rows * stride,), np.uint16)
    from excalibur_amd import hip
    values = np.arange(1, 9, dtype=np.float16)
    hip._check(hip.lib().exhip_memcpy_h2d(ctx.h, z.at((rows - 1) * stride * 2).ptr, values.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(16)))
    y = ctx.empty((1, 8), np.float32)
    ctx.combine_rows(ctx.view(z.ptr.value, (rows, stride), np.uint16), ctx.array(np.array([[rows - 1]], np.int32)), ctx.array(np.array([[2.0]], np.float32)), 8, y_f32=y)
    assert y.download().ravel().tolist() == [2, 4, 6, 8, 10, 12, 14, 16]
    z.free()


# ---- a layer of experts ----
def _layer(ctx, rng, tokens, each, experts, width, inner):
    """The router's largest classes, their rows in order, quantized rows through the experts' two products, the sum with the router's weights."""
    x = rng.standard_normal((tokens, width)).astype(np.float32)
    router = rng.standard_normal((experts, width)).astype(np.float32) / np.sqrt(width).astype(np.float32)
    w = [rng.standard_normal((experts, inner, width)).astype(np.float32) / np.sqrt(width).astype(np.float32) for _ in range(2)] + \
        [rng.standard_normal((experts, width, inner)).astype(np.float32) / np.sqrt(inner).astype(np.float32)]
    codes, scales, on_device = [], [], []
    for a in w:
        q, s = i8ref.quantize_rows(a.reshape(-1, a.shape[2]))
        codes.append(q.reshape(a.shape))
        scales.append(s.reshape(a.shape[:2]))
        on_device.append((ctx.array(codes[-1]), ctx.array(scales[-1])))
    gate_up = ctx.pack_i8_weights(inner, width, on_device[0][0], on_device[1][0], experts=experts)
    down = ctx.pack_i8_weights(width, inner, on_device[2][0], experts=experts)
    m = tokens * each
    dx = ctx.array(x)
    logits = ctx.innerproduct_f32(dx, ctx.array(router))
    log_p, ids = ctx.empty((tokens, each), np.float32), ctx.empty((tokens, each), np.int32)
    ctx.log_probabilities(ctx.view(logits.ptr.value, (tokens, experts), np.float32), top=each, top_ids=ids, top_log_p=log_p)
    offsets, rows, places = ctx.group_rows(ids, experts)
    xq, xs = ctx.quantize_rows_i8(dx)
    h = ctx.empty((m, inner), np.uint16)
    ctx.innerproduct_grouped_gated_i8(ctx.i8_desc(m, inner, width), experts, offsets, xq, xs, gate_up, on_device[0][1], on_device[1][1], rows=rows, x_rows=tokens, y_f16=h)
    hq, hs = ctx.quantize_rows_i8(h)
    z = ctx.empty((m, width), np.uint16)
    ctx.innerproduct_grouped_i8(ctx.i8_desc(m, width, inner), experts, offsets, hq, hs, down, on_device[2][1], y_f16=z)
    y = ctx.empty((tokens, width), np.float32)
    ctx.combine_rows(z, places, log_p, kind="log_normalized", y_f32=y)
    # in 64 bits, with the choices that the device made
    ids, log_p = ids.download(), log_p.download()
    order = np.sort(x.astype(np.float64) @ router.T.astype(np.float64), axis=1)[:, ::-1]
    chosen = np.take_along_axis(x.astype(np.float64) @ router.T.astype(np.float64), ids, 1)
    assert np.all(np.abs(chosen - order[:, :each]) <= width * 2.0 ** -23 * 10)
    q, s = i8ref.quantize_rows(x)
    want = np.zeros((tokens, width))
    p = np.exp(log_p.astype(np.float64))
    p /= p.sum(axis=1, keepdims=True)
    for e in range(experts):
        at, j = np.nonzero(ids == e)
        if not len(at):
            continue
        g, u = (i8ref.side(q[at], s[at], codes[i][e], scales[i][e]) for i in (0, 1))
        hq_e, hs_e = i8ref.quantize_rows(i8ref.gated("silu", g, u)[0].astype(np.float16).astype(np.float32))
        want[at] += p[at, j][:, None] * i8ref.side(hq_e, hs_e, codes[2][e], scales[2][e])[0]
    return y.download(), want


@pytest.mark.parametrize("tokens,each,experts,width,inner", [(1, 2, 8, 256, 96), (40, 4, 16, 300, 130), (600, 2, 6, 256, 200)])
def test_a_layer_of_experts(ctx, tokens, each, experts, width, inner):
    """Two roundings to halves (2^-11 each) and a code of h that the first of them moves by a step (a scale of 1/127 of the row's largest, on few of its `inner` values)
    are all that is between the two: 1 % of a row's size holds them."""
    got, want = _layer(ctx, np.random.default_rng(tokens), tokens, each, experts, width, inner)
    off = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
    assert np.all(off < 0.01), off.max()
