"""The 8-bit floating point inner products, the quantizer in front of them and the log probabilities behind them, as cases that can be timed.

A program that answers with large inner products keeps their weights as e4m3 codes with one float32 scale for each block of 128 x 128,
quantizes its rows as they come (one scale for each 128 values of a row), and reads log probabilities off the last product:

* ``quantize`` -- float32 or half rows to codes and scales,
* ``product``  -- rows times weights, with a bias, as float32 or half,
* ``gated``    -- a feed-forward block's two projections, the activation of the first and their product, as half or as codes for the next product,
* ``logprob``  -- log probabilities of given classes, the entropy, and the largest classes with theirs.

``own`` chooses between the plain forms and the library's entry points; operands are torch's device memory in both.
"""
import functools
import math

import torch

own = False

BLOCK = 128          # values that share a scale
LARGEST = 448.0      # of e4m3
LEAST_SCALE = 2.0 ** -100
GATES = ("silu", "gelu", "sigmoid", "relu")


def listed():
    return [
        # one row in front of a serving step's product: launch latency
        dict(name="quantize-f16-1x4096", op="quantize", dtype="f16", m=1, k=4096, pad=0),
        # a prompt's activations, as a float32 network leaves them, in rows of a wider tensor
        dict(name="quantize-f32-8192x5000", op="quantize", dtype="f32", m=8192, k=5000, pad=24),
        # one row: reading the weights is all of it
        dict(name="product-f16-1x4096x4096", op="product", m=1, n=4096, k=4096, pad=0, bias=False, out="f16"),
        # a small batch of images through a classifier head of ragged sizes, float32 answers
        dict(name="product-f32-33x1000x2200", op="product", m=33, n=1000, k=2200, pad=16, bias=True, out="f32"),
        # a few hundred rows with no size a multiple of anything
        dict(name="product-f32-777x5003x1531", op="product", m=777, n=5003, k=1531, pad=0, bias=True, out="f32"),
        # a prompt through a large layer: the matrix cores are all of it
        dict(name="product-f16-8192x8192x4096", op="product", m=8192, n=8192, k=4096, pad=0, bias=False, out="f16"),
        # the feed-forward block for one row
        dict(name="gated-f16-1x11264x4096", op="gated", m=1, n=11264, k=4096, pad=0, gate="silu", bias=False, out="f16"),
        # a serving batch of ragged sizes, with biases
        dict(name="gated-f16-130x1500x1000", op="gated", m=130, n=1500, k=1000, pad=0, gate="gelu", bias=True, out="f16"),
        # a prompt, its result quantized for the projection behind it
        dict(name="gated-f8-4096x8192x4096", op="gated", m=4096, n=8192, k=4096, pad=0, gate="silu", bias=False, out="f8"),
        # one step of serving: one class was taken, twenty are shown
        dict(name="logprob-f32-1x131072", op="logprob", dtype="f32", m=1, c=131072, pad=0, ids=1, top=20, masked=0.0),
        # a prompt is scored: the classes are given
        dict(name="logprob-f16-4096x32000", op="logprob", dtype="f16", m=4096, c=32000, pad=0, ids=1, top=0, masked=0.0),
        # a batch with a grammar's mask, an odd number of classes, several candidates scored
        dict(name="logprob-f16-300x100003", op="logprob", dtype="f16", m=300, c=100003, pad=1, ids=4, top=8, masked=0.4),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _rows(rng, most):
    return 1 if rng.random() < 0.2 else _log(rng, 1, max(1, min(8192, most)))


def draw(rng):
    op = rng.choice(("quantize", "product", "product", "gated", "gated", "logprob", "logprob"))
    if op == "quantize":
        k = _log(rng, 64, 16384)
        return dict(op=op, dtype=rng.choice(("f16", "f32")), m=_rows(rng, 8192 * 5000 // k), k=k, pad=rng.choice((0, 0, rng.randint(1, 40))))
    if op == "logprob":
        c = _log(rng, 100, 262144)
        m = _rows(rng, 4096 * 32000 // c)
        # where alternatives are asked, the plain form sorts
        top = rng.choice((0, rng.randint(1, 32))) if m * c > 32 * 1024 * 1024 else rng.randint(0, 32)
        return dict(op=op, dtype=rng.choice(("f16", "f32")) if m * c <= 64 * 1024 * 1024 else "f16", m=m, c=c, pad=rng.choice((0, 0, rng.randint(1, 9))),
                    ids=rng.choice((0, 1, 1, rng.randint(2, 8))), top=top if m * c <= 32 * 1024 * 1024 else 0, masked=rng.choice((0.0, 0.0, rng.uniform(0.1, 0.9))))
    n, k = _log(rng, 64, 16384), _log(rng, 64, 16384)
    if n * k > 8192 * 8192:
        n = 8192 * 8192 // k
    most = (8192 * 8192 * 4096 if op == "product" else 4096 * 8192 * 4096) // (n * k)
    case = dict(op=op, m=_rows(rng, min(most, 2 ** 26 // n)), n=n, k=k, pad=16 * rng.choice((0, 0, rng.randint(1, 4))), bias=rng.random() < 0.5)
    if op == "product":
        return dict(case, out=rng.choice(("f16", "f32")))
    return dict(case, gate=rng.choice(GATES), out=rng.choice(("f16", "f8")))


def work(case):
    m, op = case["m"], case["op"]
    if op == "quantize":
        k, blocks = case["k"], -(-case["k"] // BLOCK)
        return dict(bytes=m * (k * ((2 if case["dtype"] == "f16" else 4) + 1) + 4 * blocks), flops=2 * m * k)
    if op == "logprob":
        values = m * case["c"]
        return dict(bytes=values * (2 if case["dtype"] == "f16" else 4) + m * (8 * case["ids"] + 8 * case["top"] + 4), flops=5 * values)
    n, k = case["n"], case["k"]
    blocks_n, blocks_k, sides = -(-n // BLOCK), -(-k // BLOCK), 2 if op == "gated" else 1
    result = n * dict(f16=2, f32=4, f8=1)[case["out"]] + (4 * blocks_n if case["out"] == "f8" else 0)
    return dict(bytes=m * k + 4 * m * blocks_k + sides * (n * k + 4 * blocks_n * blocks_k + (4 * n if case["bias"] else 0)) + m * result, flops=2 * sides * m * n * k)


# ---- plain forms: float32 whatever the operands' type, one rounding at the end ----
def _f8(x):
    return x.to(torch.float8_e4m3fn)


def _blocks(x):
    """[m][k] as [m][blocks][128], zeros behind the last value."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    return torch.nn.functional.pad(x, (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)


def _quantize_rows(x):
    """float32 [m][k] to e4m3 [m][k] and scales [blocks][m]."""
    b = _blocks(x)
    scale = (b.abs().amax(2) / LARGEST).clamp_min(LEAST_SCALE)
    codes = _f8(b * (1.0 / scale)[:, :, None])
    return codes.view(x.shape[0], -1)[:, :x.shape[1]], scale.t().contiguous()


def _quantize_weights(w):
    """float32 [n][k] to e4m3 [n][k] and scales [n blocks][k blocks]."""
    n, k = w.shape
    bn, bk = -(-n // BLOCK), -(-k // BLOCK)
    b = torch.nn.functional.pad(w, (0, bk * BLOCK - k, 0, bn * BLOCK - n)).view(bn, BLOCK, bk, BLOCK)
    scale = (b.abs().amax((1, 3)) / LARGEST).clamp_min(LEAST_SCALE)
    codes = _f8(b * (1.0 / scale)[:, None, :, None]).view(bn * BLOCK, bk * BLOCK)
    return codes[:n, :k].contiguous(), scale


def _rows_of(codes, scale, dtype=torch.float32):
    """What codes [m][k] with scales [blocks][m] stand for."""
    return codes.to(dtype) * scale.to(dtype).t().repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _weights_of(codes, scale, dtype=torch.float32):
    n, k = codes.shape
    return codes.to(dtype) * scale.to(dtype).repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _gate(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return torch.sigmoid(g) if name == "sigmoid" else torch.where(g > 0, g, torch.zeros_like(g))


def _log_probabilities(x, ids, top):
    """Of rows x: (log probabilities of ids, entropy, the `top` largest classes, their log probabilities)."""
    most = x.amax(1, keepdim=True)
    empty = most == -math.inf
    t = torch.where(empty, -math.inf, x - torch.where(empty, 0.0, most))
    e = torch.exp(t)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = torch.where(empty, 0.0, log_total - torch.where(e > 0, e * t, 0.0).sum(1, keepdim=True) / total)[:, 0]
    asked = torch.where(ids < 0, 0.0, t.gather(1, ids.clamp_min(0).long()) - torch.where(empty, 0.0, log_total))
    if not top:
        return asked, entropy, None, None
    values, order = torch.sort(x, dim=1, descending=True, stable=True)
    best = order[:, :top]
    return asked, entropy, best.to(torch.int32), t.gather(1, best) - torch.where(empty, 0.0, log_total)


# ---- what a program has in hand ----
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(m, k, g):
    """Rows of different size, a few channels far larger than the others."""
    x = torch.randn(m, k, generator=g, device="cuda")
    x *= torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    x *= torch.where(torch.rand(1, k, generator=g, device="cuda") < 0.01, 20.0, 1.0)
    return x


def _strided(m, width, stride, dtype):
    """[m][width] inside rows of `stride`."""
    return torch.zeros(m, stride, dtype=dtype, device="cuda")[:, :width]


def _inputs(case, seed):
    g = _generator(seed)
    m, op = case["m"], case["op"]
    if op == "quantize":
        x = _strided(m, case["k"], case["k"] + case["pad"], torch.float16 if case["dtype"] == "f16" else torch.float32)
        x.copy_(_activations(m, case["k"], g))
        return dict(x=x)
    if op == "logprob":
        c = case["c"]
        x = _strided(m, c, c + case["pad"], torch.float16 if case["dtype"] == "f16" else torch.float32)
        logits = torch.randn(m, c, generator=g, device="cuda") * 2.5
        # some rows are nearly sure of one class
        sure = torch.rand(m, 1, generator=g, device="cuda") * 20.0
        logits.scatter_add_(1, torch.randint(c, (m, 1), generator=g, device="cuda"), sure)
        if case["masked"]:
            logits.masked_fill_(torch.rand(m, c, generator=g, device="cuda") < case["masked"], -math.inf)
            # padding rows: nothing is left of the last one in 16
            logits[15::16] = -math.inf
        x.copy_(logits)
        ids = torch.randint(c, (m, case["ids"]), generator=g, device="cuda", dtype=torch.int32)
        if case["masked"]:
            ids[15::16] = -1
        return dict(x=x, ids=ids)
    n, k = case["n"], case["k"]
    codes, x_scale = _quantize_rows(_activations(m, k, g))
    x = _strided(m, k, -(-k // 16) * 16 + case["pad"], torch.float8_e4m3fn)
    x.view(torch.uint8).copy_(codes.view(torch.uint8))
    s = dict(x=x, x_scale=x_scale)
    for side in ("gate", "up") if op == "gated" else ("w",):
        s[side], s[side + "_scale"] = _quantize_weights(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k))
        s[side + "_bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
    return s


@functools.lru_cache(maxsize=None)
def _ctx():
    from excalibur_amd import hip
    return hip.Ctx(0)


def _view(t, dtype=None):
    """torch's memory as the library's Python face takes it: rows with their stride."""
    if t is None:
        return None
    import numpy as np
    if dtype is None:
        dtype = {torch.float32: np.float32, torch.float16: np.uint16, torch.int32: np.int32}.get(t.dtype, np.uint8)
    shape = (t.shape[0], t.stride(0)) if t.dim() == 2 and t.shape[0] > 1 else tuple(t.shape)
    return _ctx().view(t.data_ptr(), shape, dtype)


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        _lay_out(state)
    return state


def _lay_out(s):
    """What a program sets up once: the weights' layout, the results' memory and the workspace."""
    case, ctx = s["case"], _ctx()
    m, op = case["m"], case["op"]
    empty = functools.partial(torch.empty, device="cuda")
    if op == "quantize":
        k = case["k"]
        s["y"] = empty(m, -(-k // 16) * 16, dtype=torch.uint8)
        s["scale"] = empty(-(-k // BLOCK), m)
        s["args"] = dict(x=_view(s["x"]), k=k, y=_view(s["y"]), scale=_view(s["scale"]))
        s["out"] = dict(codes=s["y"][:, :k].view(torch.float8_e4m3fn), scale=s["scale"])
    elif op == "logprob":
        c, ids, top = case["c"], case["ids"], case["top"]
        s["work"] = empty(max(1, ctx.log_probabilities_workspace(m, c, top)), dtype=torch.uint8)
        out = dict(entropy=empty(m))
        if ids:
            out["log_p"] = empty(m, ids)
        if top:
            out.update(top_ids=empty(m, top, dtype=torch.int32), top_log_p=empty(m, top))
        s["out"] = out
        s["args"] = dict(x=_view(s["x"]), c=c, ids=_view(s["ids"]) if ids else None, top=top, workspace=_view(s["work"]), **{name: _view(t) for name, t in out.items()})
    else:
        n, k = case["n"], case["k"]
        s["d"] = ctx.f8_desc(m, n, k, x_stride=s["x"].stride(0) if m > 1 else None, y_stride=-(-n // 16) * 16 if case["out"] == "f8" else n)
        sides = ("gate", "up") if op == "gated" else ("w",)
        s["packed"] = empty(ctx.f8_packed_bytes(n, k, gated=op == "gated"), dtype=torch.uint8)
        ctx.pack_f8_weights(n, k, *[_view(s[side]) for side in sides], packed=_view(s["packed"]))
        args = dict(x=_view(s["x"]), x_scale=_view(s["x_scale"]), w=_view(s["packed"]))
        if op == "product":
            args.update(w_scale=_view(s["w_scale"]), bias=_view(s["w_bias"]))
        else:
            args.update(gate=case["gate"], w_scale_gate=_view(s["gate_scale"]), w_scale_up=_view(s["up_scale"]), bias_gate=_view(s["gate_bias"]), bias_up=_view(s["up_bias"]))
        if case["out"] == "f8":
            codes, scale = empty(m, -(-n // 16) * 16, dtype=torch.uint8), empty(-(-n // BLOCK), m)
            args.update(y_f8=_view(codes), y_scale=_view(scale))
            s["out"] = dict(codes=codes[:, :n].view(torch.float8_e4m3fn), scale=scale)
        else:
            y = empty(m, n, dtype=torch.float16 if case["out"] == "f16" else torch.float32)
            args["y_" + case["out"]] = _view(y)
            s["out"] = dict(y=y)
        s["args"] = args


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        ctx = _ctx()
        if op == "quantize":
            ctx.quantize_rows_f8(**s["args"])
        elif op == "product":
            ctx.innerproduct_f8(s["d"], **s["args"])
        elif op == "gated":
            ctx.innerproduct_gated_f8(s["d"], **s["args"])
        else:
            ctx.log_probabilities(**s["args"])
        return s["out"]
    if op == "quantize":
        codes, scale = _quantize_rows(s["x"].float())
        return dict(codes=codes, scale=scale)
    if op == "logprob":
        asked, entropy, best, best_p = _log_probabilities(s["x"].float(), s["ids"], case["top"])
        out = dict(entropy=entropy)
        if case["ids"]:
            out["log_p"] = asked
        if case["top"]:
            out.update(top_ids=best, top_log_p=best_p)
        return out
    x = _rows_of(s["x"], s["x_scale"])
    if op == "product":
        y = x @ _weights_of(s["w"], s["w_scale"]).t()
        if s["w_bias"] is not None:
            y = y + s["w_bias"]
        return dict(y=y.half() if case["out"] == "f16" else y)
    g, u = x @ _weights_of(s["gate"], s["gate_scale"]).t(), x @ _weights_of(s["up"], s["up_scale"]).t()
    if s["gate_bias"] is not None:
        g, u = g + s["gate_bias"], u + s["up_bias"]
    h = _gate(case["gate"], g) * u
    if case["out"] == "f16":
        return dict(y=h.half())
    codes, scale = _quantize_rows(h)
    return dict(codes=codes, scale=scale)


# ---- the definitions in 64 bits ----
def _round_e4m3(v):
    """To the nearest of e4m3's values, ties to the even one: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def _exact_rows(h):
    m, k = h.shape
    blocks = -(-k // BLOCK)
    wide = torch.zeros(m, blocks * BLOCK, dtype=torch.float64, device=h.device)
    wide[:, :k] = h
    wide = wide.view(m, blocks, BLOCK)
    scale = torch.maximum(wide.abs().max(2).values / LARGEST, torch.full((), LEAST_SCALE, dtype=torch.float64, device=h.device))
    return dict(codes=_round_e4m3(wide / scale.unsqueeze(2)).reshape(m, -1)[:, :k], scale=scale.t().contiguous())


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_rows(s["x"].double())
    if op == "logprob":
        x, ids = s["x"].double(), s["ids"].long()
        empty = torch.isinf(x).all(1)
        x[empty] = 0.0
        log_p = x - torch.logsumexp(x, 1, keepdim=True)
        log_p[empty] = -math.inf
        entropy = torch.special.entr(torch.exp(log_p)).sum(1)
        out = dict(entropy=entropy)
        if case["ids"]:
            out["log_p"] = torch.where(ids < 0, 0.0, log_p.gather(1, ids.clamp(min=0)))
        if case["top"]:
            out.update(top_ids=None, top_log_p=torch.topk(log_p, case["top"], dim=1).values)
        return out
    x = _rows_of(s["x"], s["x_scale"], torch.float64)
    sides = [torch.nn.functional.linear(x, _weights_of(s[side], s[side + "_scale"], torch.float64), None if s[side + "_bias"] is None else s[side + "_bias"].double())
             for side in (("w",) if op == "product" else ("gate", "up"))]
    if op == "product":
        return dict(y=sides[0])
    g, u = sides
    act = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, sigmoid=torch.sigmoid, relu=torch.relu)[case["gate"]]
    return dict(y=act(g) * u) if case["out"] == "f16" else _exact_rows(act(g) * u)
