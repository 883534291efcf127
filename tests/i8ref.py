"""Operators on 8-bit integers with a scale for each row and each output, by their definitions: what the library's are tested against.

Sums of codes are whole numbers below 2^31 and exact. A float32 result without a bias is two products, each rounded to nearest, and is compared bit for bit (a product of two
float32 has 48 bits, float64 holds it, and rounding that to float32 is rounding the product). With a bias the last product and the sum are rounded once: off by
at most half a step, 2^-24 of the result or 2^-150 below the normal range, from the value that float64 gives, itself off by less than 2^-52 of its terms.
A gated result's sides have those bounds; the activation's are those of tests/f8ref.py."""
import numpy as np

from tests import f8ref


def quantize_rows(x):
    """(codes int8 [m][k], scales float32 [m]) of float32 rows."""
    x = np.asarray(x, np.float32)
    fine = np.isfinite(x).all(axis=1)
    most = np.abs(np.where(fine[:, None], x, 0)).max(axis=1)
    scale = np.maximum(most / np.float32(127), np.float32(2.0 ** -100)).astype(np.float32)
    codes = np.rint(np.where(fine[:, None], x, 0).astype(np.float64) / scale.astype(np.float64)[:, None]).astype(np.int8)
    return codes, np.where(fine, scale, np.float32(np.nan)).astype(np.float32)


def side(x, x_scale, w, w_scale, bias=None):
    """(y float64, bound) of one projection; the bound is 0 without a bias, where y is the float32 result itself."""
    sums = (x.astype(np.float64) @ w.astype(np.float64).T).astype(np.int64)  # below 2^53: exact
    with np.errstate(over="ignore", invalid="ignore"):
        scaled = sums.astype(np.float32) * x_scale.astype(np.float32)[:, None]
        if bias is None:
            return (scaled * w_scale.astype(np.float32)).astype(np.float64), np.zeros(sums.shape)
        product = scaled.astype(np.float64) * w_scale.astype(np.float64)
        y = product + bias.astype(np.float64)
    return y, np.abs(y) * 2.0 ** -24 + 2.0 ** -150 + (np.abs(product) + np.abs(bias)) * 2.0 ** -51


def gated(gate, g, u):
    return f8ref.gated(gate, *g, *u)


def group(ids, experts):
    flat = ids.ravel()
    chosen = [np.flatnonzero(flat == e) for e in range(experts)]
    offsets = np.concatenate([[0], np.cumsum([len(c) for c in chosen])]).astype(np.int32)
    order = np.concatenate(chosen)
    rows, places = np.full(flat.size, -1, np.int32), np.full(flat.size, -1, np.int32)
    rows[:len(order)] = order // ids.shape[1]
    places[order] = np.arange(len(order))
    return offsets, rows, places.reshape(ids.shape)


def combine(z, places, weights, kind):
    """(y, bound on a float32 result's error): `each` multiply-adds, each off by half a step of what stands so far, and weights that are logarithms off by 2^-16 of
    theirs: an argument of at most 128 rounded by 2^-24 of it (2^-17), exp within two units, the sum of up to 64 and the division (2^-18 together)."""
    each = places.shape[1]
    w = weights.astype(np.float64)
    if kind != "plain":
        with np.errstate(invalid="ignore"):
            top = w.max(axis=1, keepdims=True) if kind == "log_normalized" else np.zeros((len(w), 1))
            w = np.exp(w - np.where(np.isneginf(top), 0, top))
            if kind == "log_normalized":
                total = w.sum(axis=1, keepdims=True)
                w = np.where(total == 0, 0, w / np.where(total == 0, 1, total))
    v = np.where((places >= 0)[:, :, None], z.astype(np.float64)[np.clip(places, 0, len(z) - 1)], 0)
    v[places >= len(z)] = np.nan
    terms = np.where((places >= 0)[:, :, None], w[:, :, None] * v, 0)
    size = np.abs(terms).sum(axis=1)
    return terms.sum(axis=1), size * ((each + 1) * 2.0 ** -24 + (0 if kind == "plain" else 2.0 ** -16)) + 2.0 ** -130
