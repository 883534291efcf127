"""Inner products in 8-bit integers with a scale for each row and each output, alone and by experts, as cases that can be timed.

A program that answers with large inner products keeps their weights as 8-bit integers with one float32 scale for each output and quantizes its rows as
they come, one scale a row. Where each row goes to a few of many experts, rows are put in order by expert, multiplied by their expert's weights, and what
the experts of a row answer is added up with the router's weights:

* ``quantize`` -- float32 or half rows to codes and scales,
* ``product``  -- rows times weights, with a bias, or (``gate``) both projections of a feed-forward block with the activation and their product,
* ``grouped``  -- the same with the weights of each row's expert,
* ``group``    -- the experts that were chosen for each row to the rows in order by expert,
* ``combine``  -- the weighted sum of what the experts of each row answered.

``own`` chooses between the plain forms and the library's entry points; operands are torch's device memory in both.
"""
import functools
import math

import torch

own = False

LARGEST = 127.0      # of the codes
LEAST_SCALE = 2.0 ** -100
GATES = ("silu", "gelu", "sigmoid", "relu")
WEIGHTS = ("plain", "log", "log_normalized")


def listed():
    return [
        # one row in front of a serving step's product: launch latency
        dict(name="quantize-f16-1x4096", op="quantize", dtype="f16", m=1, k=4096, pad=0),
        # a prompt's activations, as a float32 network leaves them, in rows of odd length that begin anywhere
        dict(name="quantize-f32-8000x5001", op="quantize", dtype="f32", m=8000, k=5001, pad=8),
        # one row: reading the weights is all of it
        dict(name="product-f16-1x4096x4096", op="product", m=1, n=4096, k=4096, pad=0, gate="", bias=False, out="f16"),
        # a serving batch through a feed-forward block of ragged sizes, with biases
        dict(name="gated-f16-257x1003x2200", op="product", m=257, n=1003, k=2200, pad=16, gate="gelu", bias=True, out="f16"),
        # a prompt through a large layer: the matrix cores are all of it
        dict(name="product-f16-8192x8192x4096", op="product", m=8192, n=8192, k=4096, pad=0, gate="", bias=False, out="f16"),
        # one row's experts: their weights are read for it alone
        dict(name="grouped-gated-f16-1x8of64x1536x2048", op="grouped", tokens=1, each=8, experts=64, n=1536, k=2048, pad=0, gather=True, gate="silu", bias=False, out="f16"),
        # a small batch, few experts of ragged sizes, some of them without rows, float32 answers
        dict(name="grouped-f32-150x3of20x1000x1530", op="grouped", tokens=150, each=3, experts=20, n=1000, k=1530, pad=16, gather=False, gate="", bias=True, out="f32"),
        # a prompt through the first half of its experts, some of them chosen far more often than others
        dict(name="grouped-gated-f16-4096x8of64x1536x2048", op="grouped", tokens=4096, each=8, experts=64, n=1536, k=2048, pad=0, gather=True, gate="silu", bias=False, out="f16"),
        # a serving step's batch put in order
        dict(name="group-16x8of64", op="group", tokens=16, each=8, experts=64, dropped=0.0),
        # a prompt put in order, a few choices dropped
        dict(name="group-8191x8of256", op="group", tokens=8191, each=8, experts=256, dropped=0.02),
        # one row's answer
        dict(name="combine-f16-1x8x4096", op="combine", tokens=1, each=8, n=4096, pad=0, out="f16", weights="log_normalized", dropped=0.0),
        # a prompt's answers, in rows of odd length, a few choices dropped
        dict(name="combine-f32-8191x6x4099", op="combine", tokens=8191, each=6, n=4099, pad=5, out="f32", weights="plain", dropped=0.02),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _rows(rng, most):
    return 1 if rng.random() < 0.2 else _log(rng, 1, max(1, min(8192, most)))


def draw(rng):
    op = rng.choice(("quantize", "product", "product", "grouped", "grouped", "group", "combine"))
    if op == "quantize":
        k = _log(rng, 16, 16384)
        return dict(op=op, dtype=rng.choice(("f16", "f32")), m=_rows(rng, 8000 * 5001 // k), k=k, pad=rng.choice((0, 0, rng.randint(1, 40))))
    if op in ("group", "combine"):
        each = rng.randint(1, 8)
        case = dict(op=op, tokens=_rows(rng, 8191), each=each, dropped=rng.choice((0.0, 0.0, rng.uniform(0.01, 0.5))))
        if op == "group":
            return dict(case, experts=_log(rng, max(2, each), 256))
        n = _log(rng, 16, 16384)
        case["tokens"] = min(case["tokens"], 8191 * 4099 * 7 // (n * (each + 1)))
        return dict(case, n=n, pad=rng.choice((0, 0, rng.randint(1, 9))), out=rng.choice(("f16", "f32")), weights=rng.choice(WEIGHTS))
    gate = rng.choice(("", "", *GATES))
    sides = 2 if gate else 1
    case = dict(op=op, gate=gate, pad=16 * rng.choice((0, 0, rng.randint(1, 4))), bias=rng.random() < 0.5, out=rng.choice(("f16", "f32")))
    if op == "product":
        n, k = _log(rng, 64, 16384), _log(rng, 64, 16384)
        if n * k * sides > 8192 * 8192:
            n = 8192 * 8192 // (k * sides)
        return dict(case, m=_rows(rng, min(8192 * 8192 * 4096 // (n * k * sides), 2 ** 26 // n)), n=n, k=k)
    n, k, each = _log(rng, 64, 8192), _log(rng, 64, 8192), rng.randint(1, 8)
    experts = _log(rng, max(2, each), max(each, 2, min(128, 64 * 2 * 1536 * 2048 // (n * k * sides))))
    tokens = _rows(rng, min(4096 * 8 * 2 * 1536 * 2048 // (n * k * sides * each), 2 ** 25 // (max(n, k) * each)))
    return dict(case, tokens=tokens, each=each, experts=experts, n=n, k=k, gather=rng.random() < 0.5)


def _popularity(experts):
    """How often each expert is chosen: the first four times as often as the last."""
    p = [4.0 ** (-e / max(1, experts - 1)) for e in range(experts)]
    return [v / sum(p) for v in p]


def work(case):
    op = case["op"]
    if op == "quantize":
        m, k = case["m"], case["k"]
        return dict(bytes=m * (k * ((2 if case["dtype"] == "f16" else 4) + 1) + 4), flops=2 * m * k)
    if op == "group":
        choices = case["tokens"] * case["each"]
        return dict(bytes=choices * 12 + 4 * (case["experts"] + 1), flops=choices)
    out = 2 if case["out"] == "f16" else 4
    if op == "combine":
        choices = case["tokens"] * case["each"]
        return dict(bytes=choices * (2 * case["n"] * (1.0 - case["dropped"]) + 8) + case["tokens"] * case["n"] * out, flops=2 * choices * case["n"])
    n, k, sides = case["n"], case["k"], 2 if case["gate"] else 1
    if op == "product":
        m = source = case["m"]
        present = 1.0
    else:
        m = case["tokens"] * case["each"]
        source = case["tokens"] if case["gather"] else m
        present = sum(1.0 - (1.0 - min(1.0, case["each"] * p)) ** case["tokens"] for p in _popularity(case["experts"]))
    weights = sides * (n * k + 4 * n + (4 * n if case["bias"] else 0))
    return dict(bytes=source * (k + 4) + present * weights + m * n * out, flops=2 * sides * m * n * k)


# ---- plain forms: float32 whatever the operands' type, one rounding at the end ----
def _quantize(x):
    """float32 [m][k] to codes [m][k] and scales [m]. Codes are the whole numbers nearest to x / scale, so the quotient is taken in 64 bits."""
    most = x.abs().amax(1).double()
    scale = (most / torch.full_like(most, LARGEST)).clamp_min(LEAST_SCALE).float()
    return torch.round(x.double() / scale.double()[:, None]).to(torch.int8), scale


def _gate(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return torch.sigmoid(g) if name == "sigmoid" else torch.where(g > 0, g, torch.zeros_like(g))


def _finish(case, sums, scales, biases):
    """The sums of codes, their scales and biases as the result: of each projection [..][n], scales of the rows [..][1]."""
    row, outputs = scales
    sides = [s * row * w if b is None else s * row * w + b for s, w, b in zip(sums, outputs, biases)]
    y = _gate(case["gate"], sides[0]) * sides[1] if case["gate"] else sides[0]
    return y.half() if case["out"] == "f16" else y


def _plain_product(s):
    case, x = s["case"], s["x"].float()
    sides = range(2 if case["gate"] else 1)
    return _finish(case, [x @ s["w"][i].float().t() for i in sides], (s["x_scale"][:, None], [s["w_scale"][i] for i in sides]), [s["bias"][i] for i in sides])


def _plain_grouped(s):
    """Each expert's rows as far as the most that one has, zeros behind them; or, for a few rows, each row with its expert's weights."""
    case, sides = s["case"], range(2 if s["case"]["gate"] else 1)
    m = case["tokens"] * case["each"]
    at = torch.arange(m, device="cuda", dtype=torch.int32)
    expert = torch.searchsorted(s["offsets"][1:].contiguous(), at, right=True)
    x, row = s["x"].float(), s["x_scale"]
    if case["gather"]:
        x, row = x[s["rows"].long()], row[s["rows"].long()]
    if m <= case["experts"]:
        sums = [(x[:, None, :] * s["w"][i][expert].float()).sum(2) for i in sides]
    else:
        within = (at - s["offsets"][expert]).long()
        wide = torch.zeros(case["experts"], s["most"], x.shape[1], device="cuda")
        wide[expert, within] = x
        sums = [torch.bmm(wide, s["w"][i].float().transpose(1, 2).contiguous())[expert, within] for i in sides]
    return _finish(case, sums, (row[:, None], [s["w_scale"][i][expert] for i in sides]), [None if s["bias"][i] is None else s["bias"][i][expert] for i in sides])


def _plain_group(s):
    ids, experts = s["ids"], s["case"]["experts"]
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    ordered, choice = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(experts + 1, device="cuda"))
    place = torch.empty_like(flat)
    place[choice] = torch.arange(flat.numel(), device="cuda")
    rows = torch.where(ordered < experts, choice // ids.shape[1], -1)
    return dict(offsets=offsets.int(), rows=rows.int(), places=torch.where(key < experts, place, -1).int().view(ids.shape))


def _plain_combine(s):
    case, places, w = s["case"], s["places"].long(), s["weights"]
    if case["weights"] != "plain":
        top = w.amax(1, keepdim=True) if case["weights"] == "log_normalized" else torch.zeros_like(w[:, :1])
        w = torch.exp(w - top)
        if case["weights"] == "log_normalized":
            w = w / w.sum(1, keepdim=True)
    z = torch.where((places >= 0)[:, :, None], s["z"].float()[places.clamp_min(0)], 0.0)
    y = (z * w[:, :, None]).sum(1)
    return dict(y=y.half() if case["out"] == "f16" else y)


# ---- what a program has in hand ----
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(m, k, g):
    """Rows of different size, a few channels far larger than the others."""
    x = torch.randn(m, k, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=g, device="cuda"))
    x *= torch.where(torch.rand(1, k, generator=g, device="cuda") < 0.01, 20.0, 1.0)
    return x


def _strided(m, width, stride, dtype):
    """[m][width] inside rows of `stride`."""
    return torch.zeros(m, stride, dtype=dtype, device="cuda")[:, :width]


def _chosen(case, g):
    """Different experts for each row, by their popularity: int32 [tokens][each]."""
    p = torch.tensor(_popularity(case["experts"]), device="cuda")
    noise = -torch.log(-torch.log(torch.rand(case["tokens"], case["experts"], generator=g, device="cuda").clamp(1e-9, 1.0 - 1e-7)))
    return torch.sort(torch.log(p) + noise, dim=1, descending=True).indices[:, :case["each"]].to(torch.int32).contiguous()


def _inputs(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "quantize":
        x = _strided(case["m"], case["k"], case["k"] + case["pad"], torch.float16 if case["dtype"] == "f16" else torch.float32)
        x.copy_(_activations(case["m"], case["k"], g))
        return dict(x=x)
    if op == "group":
        ids = _chosen(case, g)
        ids[torch.rand(ids.shape, generator=g, device="cuda") < case["dropped"]] = -1
        return dict(ids=ids)
    if op == "combine":
        tokens, each, n = case["tokens"], case["each"], case["n"]
        z = _strided(tokens * each, n, n + case["pad"], torch.float16)
        z.copy_(torch.randn(tokens * each, n, generator=g, device="cuda"))
        # the choices in an order of their own, as experts put them
        places = torch.randperm(tokens * each, generator=g, device="cuda").to(torch.int32).view(tokens, each)
        places[torch.rand(tokens, each, generator=g, device="cuda") < case["dropped"]] = -1
        weights = torch.log_softmax(torch.randn(tokens, each + 8, generator=g, device="cuda") * 1.5, 1)[:, :each].contiguous()
        return dict(z=z, places=places, weights=torch.exp(weights) if case["weights"] == "plain" else weights)
    n, k, experts = case["n"], case["k"], case.get("experts", 0)
    s = {}
    if op == "grouped":
        ids = _chosen(case, g)
        key, choice = torch.sort(ids.reshape(-1), stable=True)
        counts = torch.bincount(key, minlength=experts)
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.cumsum(0)]).to(torch.int32)
        s["rows"] = (choice // case["each"]).to(torch.int32) if case["gather"] else None
        s["most"] = int(counts.max())
        m = case["tokens"] if case["gather"] else case["tokens"] * case["each"]
    else:
        m = case["m"]
    codes, s["x_scale"] = _quantize(_activations(m, k, g))
    s["x"] = _strided(m, k, -(-k // 16) * 16 + case["pad"], torch.int8)
    s["x"].copy_(codes)
    s["w"], s["w_scale"], s["bias"] = [], [], []
    for _ in range(2 if case["gate"] else 1):
        some = max(1, experts)
        w, scale = _quantize(torch.randn(some * n, k, generator=g, device="cuda") / math.sqrt(k))
        bias = torch.randn(some, n, generator=g, device="cuda") if case["bias"] else None
        lead = (some,) if experts else ()
        s["w"].append(w.view(*lead, n, k))
        s["w_scale"].append(scale.view(*lead, n))
        s["bias"].append(None if bias is None else bias.view(*lead, n))
    return s


@functools.lru_cache(maxsize=None)
def _ctx():
    from excalibur_amd import hip
    return hip.Ctx(0)


def _view(t):
    """torch's memory as the library's Python face takes it: rows with their stride."""
    if t is None:
        return None
    import numpy as np
    dtype = {torch.float32: np.float32, torch.float16: np.uint16, torch.int32: np.int32, torch.int8: np.int8}.get(t.dtype, np.uint8)
    shape = (t.shape[0], t.stride(0)) if t.dim() == 2 and t.shape[0] > 1 else tuple(t.shape)
    return _ctx().view(t.data_ptr(), shape, dtype)


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        _lay_out(state)
    return state


def _lay_out(s):
    """What a program sets up once: the weights' layout and the results' memory."""
    case, ctx = s["case"], _ctx()
    op = case["op"]
    empty = functools.partial(torch.empty, device="cuda")
    if op == "quantize":
        m, k = case["m"], case["k"]
        codes, scale = empty(m, -(-k // 16) * 16, dtype=torch.int8), empty(m)
        s["args"] = dict(x=_view(s["x"]), k=k, y=_view(codes), scale=_view(scale))
        s["out"] = dict(codes=codes[:, :k], scale=scale)
    elif op == "group":
        choices = case["tokens"] * case["each"]
        s["out"] = dict(offsets=empty(case["experts"] + 1, dtype=torch.int32), rows=empty(choices, dtype=torch.int32), places=empty(case["tokens"], case["each"], dtype=torch.int32))
        s["args"] = dict(ids=_view(s["ids"]), experts=case["experts"], **{name: _view(t) for name, t in s["out"].items()})
    elif op == "combine":
        y = empty(case["tokens"], case["n"], dtype=torch.float16 if case["out"] == "f16" else torch.float32)
        s["args"] = dict(z=_view(s["z"]), n=case["n"], places=_view(s["places"]), weights=_view(s["weights"]), kind=case["weights"])
        s["args"]["y_" + case["out"]] = _view(y)
        s["out"] = dict(y=y)
    else:
        n, k, experts, gated = case["n"], case["k"], case.get("experts", 0), bool(case["gate"])
        m = case["tokens"] * case["each"] if experts else case["m"]
        s["d"] = ctx.i8_desc(m, n, k, x_stride=s["x"].stride(0) if s["x"].shape[0] > 1 else None)
        s["packed"] = empty(ctx.i8_packed_bytes(n, k, gated=gated, experts=max(1, experts)), dtype=torch.uint8)
        ctx.pack_i8_weights(n, k, *[_view(w.view(-1)) for w in s["w"]], packed=_view(s["packed"]), experts=max(1, experts))
        args = dict(x=_view(s["x"]), x_scale=_view(s["x_scale"]), w=_view(s["packed"]))
        if gated:
            args.update(gate=case["gate"], w_scale_gate=_view(s["w_scale"][0].view(-1)), w_scale_up=_view(s["w_scale"][1].view(-1)))
            if case["bias"]:
                args.update(bias_gate=_view(s["bias"][0].view(-1)), bias_up=_view(s["bias"][1].view(-1)))
        else:
            args.update(w_scale=_view(s["w_scale"][0].view(-1)), bias=_view(s["bias"][0].view(-1)) if case["bias"] else None)
        if experts:
            args.update(experts=experts, offsets=_view(s["offsets"]))
            if case["gather"]:
                args.update(rows=_view(s["rows"]), x_rows=case["tokens"])
        y = empty(m, n, dtype=torch.float16 if case["out"] == "f16" else torch.float32)
        args["y_" + case["out"]] = _view(y)
        s["args"], s["out"] = args, dict(y=y)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        ctx = _ctx()
        if op == "quantize":
            ctx.quantize_rows_i8(**s["args"])
        elif op == "group":
            ctx.group_rows(**s["args"])
        elif op == "combine":
            ctx.combine_rows(**s["args"])
        elif op == "grouped":
            (ctx.innerproduct_grouped_gated_i8 if case["gate"] else ctx.innerproduct_grouped_i8)(s["d"], **s["args"])
        else:
            (ctx.innerproduct_gated_i8 if case["gate"] else ctx.innerproduct_i8)(s["d"], **s["args"])
        return s["out"]
    if op == "quantize":
        codes, scale = _quantize(s["x"].float())
        return dict(codes=codes, scale=scale)
    if op == "group":
        return _plain_group(s)
    if op == "combine":
        return _plain_combine(s)
    return dict(y=_plain_grouped(s) if op == "grouped" else _plain_product(s))


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].to(torch.float64)
        scale = torch.maximum(torch.linalg.vector_norm(x, ord=math.inf, dim=1) / LARGEST, torch.full((), LEAST_SCALE, dtype=torch.float64, device="cuda"))
        # the codes are those of the scale that is stored
        return dict(codes=torch.special.round(torch.true_divide(x, scale.to(torch.float32).to(torch.float64).unsqueeze(1))).to(torch.int8), scale=scale)
    if op == "group":
        ids = s["ids"].reshape(-1).cpu()
        of = [(ids == e).nonzero()[:, 0] for e in range(case["experts"])]
        order, ends = torch.cat(of), [0]
        for each in of:
            ends.append(ends[-1] + len(each))
        rows, places = torch.full_like(ids, -1), torch.full_like(ids, -1)
        rows[:len(order)] = (order // case["each"]).to(torch.int32)
        places[order] = torch.arange(len(order), dtype=torch.int32)
        return dict(offsets=torch.tensor(ends, dtype=torch.int32), rows=rows, places=places.view(case["tokens"], case["each"]))
    if op == "combine":
        w = s["weights"].double()
        if case["weights"] == "log_normalized":
            w = torch.softmax(w, 1)
        elif case["weights"] == "log":
            w = w.exp()
        y = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device="cuda")
        for j in range(case["each"]):
            here = s["places"][:, j] >= 0
            y[here] += w[here, j].unsqueeze(1) * s["z"][s["places"][here, j].long()].double()
        return dict(y=y)
    act = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, sigmoid=torch.sigmoid, relu=torch.relu)

    def rows_through(x, expert):
        of = lambda t: t if expert is None else t[expert]  # noqa: E731
        sides = []
        for w, scale, bias in zip(s["w"], s["w_scale"], s["bias"]):
            sides.append(torch.nn.functional.linear(x, of(w).double() * of(scale).double().unsqueeze(1), None if bias is None else of(bias).double()))
        return act[case["gate"]](sides[0]) * sides[1] if case["gate"] else sides[0]

    x = s["x"].double() * s["x_scale"].double().unsqueeze(1)
    if op == "product":
        return dict(y=rows_through(x, None))
    if case["gather"]:
        x = x[s["rows"].long()]
    ends = s["offsets"].tolist()
    return dict(y=torch.cat([rows_through(x[ends[e]:ends[e + 1]], e) for e in range(case["experts"])]))
