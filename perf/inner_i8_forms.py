"""What every form of the products in 8-bit integers takes, and the figures that the choice among the forms goes by (excalibur_amd/csrc/inner_i8.hip: kPlain, kGrouped).

    python3 perf/inner_i8_forms.py time PART/PARTS > FILE        on the GPU: the shapes of the table anew, every PARTS-th of them, for instance 1/3
    python3 perf/inner_i8_forms.py table FILE ...                the table from what `time` wrote for all its parts
    python3 perf/inner_i8_forms.py check                         how much longer the form that the figures choose takes than the fastest, section by section
    python3 perf/inner_i8_forms.py fit products|experts [SEED]   other figures for a list, from its section (some seconds; seeds differ, the best of some is taken)

The table is profiles/inner_i8_forms.txt, and its lines are the shapes: for others, add lines with no times to it.
"""
import collections
import ctypes
import math
import os
import re
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
TABLE = os.path.join(ROOT, "profiles", "inner_i8_forms.txt")
CUS = 256
# (name, by experts, whether its shapes are those that the figures are fitted to)
SECTIONS = (("products", False, True), ("products by experts", True, True), ("products that the figures were not fitted to", False, False),
            ("products by experts that the figures were not fitted to", True, False), ("products outside the sizes that the figures were fitted to", False, False),
            ("products by experts outside the sizes that the figures were fitted to", True, False))
HEAD = """What every form of the products in 8-bit integers takes, beside the one that the rule takes (inner_i8.hip: the lists kPlain and kGrouped behind run_best)
made by perf/inner_i8_forms.py: launches recorded eight at a time (exhip_graph_begin .. exhip_graph_end) with the option i8_form, as many replays between a pair of HIP events as take 3 ms, the middle of three such
times, the forms of a shape one after the other; us a launch; random codes; up to 1024 rows the weights in as many copies, up to eight, as 600 MB hold, used in turn; results in halves, f32: in float32; by experts each
row's experts are drawn, the last of them a fourth as likely as the first
kernel sources %s (comments apart, those that were timed)
rows x outputs x inputs (g: gated, silu; e: experts:choices a row, where rows are then those before the choice), the form that the rule takes and the time of a call that leaves the choice to it, then the forms in the order
of the list; -: not timed, at least six times the fastest by its figures
rows<times 16 outputs a wave, times 16 rows, waves that share the blocks, blocks under way, gated, by experts>; wide<times 32 outputs a wave, times 32 rows a wave, waves along the outputs, along the rows, buffers in LDS, blocks of weights under way, gated, by experts>
"""

Shape = collections.namedtuple("Shape", "rows n k gated f32 experts each")
Form = collections.namedtuple("Form", "name halves rows at_once split figures")


def forms(by_experts):
    """The list in the source; `halves` of a product without and with an activation."""
    with open(os.path.join(ROOT, "excalibur_amd", "csrc", "inner_i8.hip")) as f:
        body = f.read().split("constexpr Form %s[] = {" % ("kGrouped" if by_experts else "kPlain"))[1].split("};")[0]
    found = []
    for name, rest in re.findall(r"\{run_(\w+<[^>]*>), (.*)\},", body):
        halves, rows, at_once, split, *figures = rest.split(", ")
        both = re.match(r"GATED \? (\d+) : (\d+)", halves)
        halves = (int(both[2]), int(both[1])) if both else (int(halves),) * 2
        found.append(Form(name.replace("GATED ? 2 : 1", "2 with g, 1 without").replace("GATED", "g"), halves, int(rows), int(at_once), int(split), [float(v.rstrip("f")) for v in figures]))
    return found


def features(f, s):
    """What a launch's time depends on: groups, blocks of a wave, bytes of weights, whether there is an activation, bytes that groups read beside the weights once."""
    m = s.rows * s.each
    experts = s.experts * (1.0 - math.exp(-m / s.experts)) if s.experts else 1.0
    tiles, blocks = -(-s.n // (16 if s.gated else 32)), -(-s.k // 128)
    tiles_m = max(experts, m / f.rows + 0.5 * experts if m > 0.25 * f.rows * experts else 0.0) if s.experts else -(-m // f.rows)
    halves = f.halves[s.gated]
    groups_n = -(-2 * tiles // halves)
    groups, weights = groups_n * tiles_m, experts * tiles * blocks * 4096
    return groups, -(-blocks // f.split), weights, float(s.gated), max(0.0, blocks * (groups * halves * 2048 + groups_n * m * 128) - weights)


def time_of(figures, at_once, groups, blocks, weights, gated, again):
    """As time_of() of inner_i8.hip, of one launch or arrays of them."""
    start, around, alone, share, memory, gate, l2 = figures
    times = np.ceil(groups / CUS - 1e-9)
    full = np.floor(times / at_once)
    rest = times - full * at_once
    us = start + full * (around + blocks * np.maximum(alone, at_once * share)) + gate * gated * times
    us = us + np.where(rest > 0, around + blocks * np.maximum(alone, rest * share), 0.0)
    return np.maximum(us, start + 1.0 + gate * gated + weights / memory + again / l2)


def chosen(listed, s):
    us = [float(time_of(f.figures, f.at_once, *features(f, s))) for f in listed]
    return us.index(min(us)), us


def text_of(s):
    return "%6d x %6d x %6d%s%s%s" % (s.rows, s.n, s.k, " g" if s.gated else "", " f32" if s.f32 else "", " e%d:%d" % (s.experts, s.each) if s.experts else "")


def read(path=TABLE):
    """[(section's index, shape, the rule's time or None, times of the forms or None where not timed)]"""
    names, at, found = {name: i for i, (name, _, _) in enumerate(SECTIONS)}, None, []
    with open(path) as f:
        for line in f:
            shape = re.match(r"\s*(\d+) x\s+(\d+) x\s+(\d+)((?: \S+)*?)(?:\s+\(\d+\)(.*))?$", line.rstrip())
            if shape is None:
                at = names.get(line.split(": ")[0].split(";")[0], at)
                continue
            flags = shape[4].split()
            e = [v[1:].split(":") for v in flags if re.match(r"e\d+:", v)]
            times = [None if v == "-" else float(v) for v in (shape[5] or "").split()]
            s = Shape(*(int(shape[i]) for i in (1, 2, 3)), "g" in flags, "f32" in flags, *(map(int, e[0]) if e else (0, 1)))
            found.append((at, s, times[0] if times else None, times[1:]))
    return found


# ---- on the GPU ----
def timer(ctx, hip):
    events = hip.Event(), hip.Event()

    def between(step, repeats):
        events[0].record(ctx)
        for _ in range(repeats):
            step()
        events[1].record(ctx)
        return events[0].elapsed_ms(events[1]) * 1e3 / repeats

    def timed(call, copies):
        """us of call(copy), recorded; each copy in turn."""
        graph, count = ctypes.c_void_p(), copies * max(1, 8 // copies)
        call(0)
        ctx.sync()
        hip._check(hip.lib().exhip_graph_begin(ctx.h))
        try:
            for i in range(count):
                call(i % copies)
        finally:
            hip._check(hip.lib().exhip_graph_end(ctx.h, ctypes.byref(graph)))
        replay = lambda: hip._check(hip.lib().exhip_graph_launch(ctx.h, graph))  # noqa: E731
        replay()
        once = between(replay, 1)
        us = sorted(between(replay, max(2, min(400, int(3000 / once)))) for _ in range(3))[1] / count
        hip._check(hip.lib().exhip_graph_destroy(graph))
        return us

    return timed


def operands(ctx, torch, s):
    """A call of the shape's product that takes the number of a copy of the weights, and how many copies there are."""
    def view(t, dtype=np.uint8):
        return ctx.view(t.data_ptr(), tuple(t.shape), dtype)

    def codes(*shape):
        return torch.randint(-128, 128, shape, dtype=torch.int8, device="cuda")

    experts, sides, m, stride = max(1, s.experts), 2 if s.gated else 1, s.rows * s.each, -(-s.k // 16) * 16
    copies = max(1, min(8, int(600e6 / (experts * s.n * s.k * sides)))) if m <= 1024 else 1
    packed = []
    for _ in range(copies):
        w = [codes(experts * s.n, s.k) for _ in range(sides)]
        packed.append(torch.empty(ctx.i8_packed_bytes(s.n, s.k, gated=s.gated, experts=experts), dtype=torch.uint8, device="cuda"))
        ctx.pack_i8_weights(s.n, s.k, *[view(a) for a in w], packed=view(packed[-1]), experts=experts)
        ctx.sync()
    x, x_scale, w_scale = codes(s.rows, stride), torch.rand(s.rows, device="cuda") * 0.01, torch.rand(experts * s.n, device="cuda") * 0.01
    y = torch.empty(m, s.n, dtype=torch.float32 if s.f32 else torch.float16, device="cuda")
    args = dict(x=view(x), x_scale=view(x_scale, np.float32))
    args["y_f32" if s.f32 else "y_f16"] = view(y, np.float32 if s.f32 else np.uint16)
    args.update({name: view(w_scale, np.float32) for name in (("w_scale_gate", "w_scale_up") if s.gated else ("w_scale",))})
    kept = [x, x_scale, w_scale, y, packed]
    if s.experts:
        likely = -math.log(4.0) / max(1, experts - 1) * torch.arange(experts, device="cuda")
        noise = -torch.log(-torch.log(torch.rand(s.rows, experts, device="cuda").clamp(1e-9, 1.0 - 1e-7)))
        key, choice = torch.sort(torch.topk(likely + noise, s.each, dim=1).indices.reshape(-1), stable=True)
        counts = torch.bincount(key, minlength=experts).cumsum(0)
        offsets, source = torch.cat([torch.zeros_like(counts[:1]), counts]).int(), (choice // s.each).int()
        args.update(experts=experts, offsets=view(offsets, np.int32), rows=view(source, np.int32), x_rows=s.rows)
        kept += [offsets, source]
    product = getattr(ctx, "innerproduct" + ("_grouped" if s.experts else "") + ("_gated" if s.gated else "") + "_i8")
    d, views = ctx.i8_desc(m, s.n, s.k, x_stride=stride), [view(p) for p in packed]
    torch.cuda.synchronize()
    return lambda copy, _=kept: product(d, w=views[copy], **args), copies


def time_all(part, parts):
    import torch

    import bench
    from excalibur_amd import hip
    ctx = hip.Ctx(0)
    timed = timer(ctx, hip)
    lists = forms(False), forms(True)
    print("kernel sources", bench.csrc_digest())
    for i, (at, s, _, _) in enumerate(read()):
        if i % parts != part - 1:
            continue
        listed = lists[SECTIONS[at][1]]
        best, guess = chosen(listed, s)
        call, copies = operands(ctx, torch, s)
        us = ["     -"] * (len(listed) + 1)
        for form in (*range(1, len(listed) + 1), 0):  # (the first of a shape's times may be longer: clocks, address translation)
            if form == 0 or guess[form - 1] <= 6.0 * min(guess):
                hip.set_option("i8_form", form)
                us[form] = "%6.1f" % timed(call, copies)
        print("%d|%d|%s  (%d) %s" % (at, i, text_of(s), best + 1, " ".join(us)), flush=True)


# ---- the table and its figures ----
def table(paths):
    lines, digests = {}, set()
    for path in paths:
        with open(path) as f:
            for line in f:
                if line.startswith("kernel sources"):
                    digests.add(line.split()[2])
                elif "|" in line:
                    at, i, text = line.rstrip("\n").split("|")
                    lines.setdefault(int(at), {})[int(i)] = text
    if len(digests) != 1 or sum(map(len, lines.values())) != len(read()):
        sys.exit("the parts are not those of one table: kernel sources %s, %d of %d shapes" % (digests, sum(map(len, lines.values())), len(read())))
    out = [HEAD % digests.pop()]
    for at, (name, by_experts, _) in enumerate(SECTIONS):
        out += ["%s: %s" % (name, ", ".join("%d %s" % (i + 1, f.name) for i, f in enumerate(forms(by_experts)))), *(lines.get(at, {})[i] for i in sorted(lines.get(at, {}))), ""]
    with open(TABLE, "w") as f:
        f.write("\n".join(out))


def timed_shapes(at):
    """Of a section: shapes and times of all forms, those not timed as three times the longest."""
    rows = [(s, times) for where, s, _, times in read() if where == at and times]
    longest = [max(t for t in times if t is not None) for _, times in rows]
    return [s for s, _ in rows], np.array([[3 * most if t is None else t for t in times] for (_, times), most in zip(rows, longest)])


def check():
    for at, (name, by_experts, _) in enumerate(SECTIONS):
        shapes, us = timed_shapes(at)
        if not shapes:
            continue
        listed, best = forms(by_experts), us.min(1)
        longer = np.array([us[i, chosen(listed, s)[0]] for i, s in enumerate(shapes)]) / best - 1
        print("%s: %d shapes, the choice takes %.1f %% longer on average, %.0f %% at most (%s)" % (name, len(shapes), 100 * longer.mean(), 100 * longer.max(), text_of(shapes[longer.argmax()]).strip()))
        if SECTIONS[at][2]:
            without = [100 * (np.delete(us, i, 1).min(1) / best - 1).max() for i in range(len(listed))]
            print("    without a form some product would take longer by %s %%" % ", ".join("%.0f" % w for w in without))


def fit(which, seed):
    """Figures near each form's own times first, then a walk by what the choice costs: on average, those of at most 64 rows twice, and the worst twenty."""
    from scipy.optimize import least_squares
    by_experts = which == "experts"
    listed, rng = forms(by_experts), np.random.default_rng(seed)
    shapes, us = timed_shapes(1 if by_experts else 0)
    best, counted = us.min(1), np.array([2.0 if s.rows * s.each <= 64 else 1.0 for s in shapes])
    features_of = [np.array([features(f, s) for s in shapes], float).T for f in listed]
    scale = np.array([1, 1, 1, 1, 1e6, 1, 1e6])
    low, high = np.array([0.5, 0.02, 0.02, 0.02, 2.5, 0.0, 4.0]), np.array([7.0, 8.0, 4.0, 4.0, 16.0, 8.0, 200.0])

    def predicted(i, figures):
        return time_of(figures * scale, listed[i].at_once, *features_of[i])

    def near(i):
        weight, found = np.sqrt(np.exp(-2 * (us[:, i] / best - 1)) + 0.02), None
        for _ in range(8):
            first = np.clip(np.array([2, 1.5, 0.3, 0.2, 5, 0.3, 20]) * np.exp(0.4 * rng.standard_normal(7)), low * 1.03 + 0.01, high * 0.99)
            got = least_squares(lambda v, i=i: weight * np.log(predicted(i, v) / us[:, i]), first, bounds=(low, high), loss="soft_l1", f_scale=0.1)
            if found is None or got.cost < found.cost:
                found = got
        return found.x

    def cost(all_us):
        longer = us[np.arange(len(shapes)), all_us.argmin(0)] / best - 1
        return (counted * longer).mean() + 0.05 * np.sort(longer)[-20:].mean()

    figures = [near(i) for i in range(len(listed))]
    now = np.array([predicted(i, v) for i, v in enumerate(figures)])
    least = cost(now)
    for _ in range(60000):
        i, some = rng.integers(len(listed)), rng.integers(7, size=rng.integers(1, 3))
        tried = figures[i].copy()
        tried[some] = np.clip(tried[some] * np.exp(0.12 * rng.standard_normal(len(some))), low[some], high[some])
        was, now[i] = now[i].copy(), predicted(i, tried)
        c = cost(now)
        if c <= least:
            least, figures[i] = c, tried
        else:
            now[i] = was
    rounded = [np.round(v, 2) for v in figures]
    longer = us[np.arange(len(shapes)), np.array([predicted(i, v) for i, v in enumerate(rounded)]).argmin(0)] / best - 1
    print("%.2f %% longer on average, %.0f %% at most" % (100 * longer.mean(), 100 * longer.max()))
    for f, v in zip(listed, rounded):
        print("%-40s %s" % (f.name, ", ".join("%gf" % x if i not in (4, 6) else "%ge6f" % x for i, x in enumerate(v))))


if __name__ == "__main__":
    what = sys.argv[1] if len(sys.argv) > 1 else ""
    if what == "time":
        time_all(*map(int, sys.argv[2].split("/")))
    elif what == "table":
        table(sys.argv[2:])
    elif what == "check":
        check()
    elif what == "fit":
        fit(sys.argv[2], int(sys.argv[3]) if len(sys.argv) > 3 else 0)
    else:
        sys.exit(__doc__)
