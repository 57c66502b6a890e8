"""Measured cases of the expert feed-forward operators: routing, grouped products, the weighted
sum of experts' outputs, and the norms around a block.

`run` computes a case in plain torch operations, or, where `own` is true, with the calls that a
user of this framework makes.  Sizes are those of encoder feed-forward blocks with experts: few
rows (one request), ordinary batches, and the largest packed batches.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
ACTS = {"identity": 0, "gelu": 1, "swiglu": 4}
NORMS = {"none": 0, "layer": 1, "rms": 2}
SCORES = {"softmax": 0, "sigmoid": 1}
EPS = 1e-5


def size_of(dtype):
    return 4 if dtype == "f32" else 2


# ---------------------------------------------------------------- cases
def route(name, rows, experts, k, dtype, score="softmax", normalise=True, masked=0.0):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "k": k, "dtype": dtype, "score": score,
            "normalise": normalise, "masked": masked}


def grouped(name, rows, experts, k, inner, outer, act, dtype, bias=False, skew=0.5):
    """`outer`: output columns after the activation.  k > 1 or unsorted rows: the rows are tokens,
    gathered by their choices."""
    return {"name": name, "op": "grouped", "rows": rows, "experts": experts, "k": k, "inner": inner, "outer": outer,
            "act": act, "dtype": dtype, "bias": bias, "skew": skew}


def combine(name, rows, experts, k, cols, dtype, norm="layer"):
    return {"name": name, "op": "combine", "rows": rows, "experts": experts, "k": k, "cols": cols, "dtype": dtype,
            "norm": norm}


def blocknorm(name, rows, cols, dtype, post, pre, gate, residual_scale=1.0):
    return {"name": name, "op": "blocknorm", "rows": rows, "cols": cols, "dtype": dtype, "post": post, "pre": pre,
            "gate": gate, "residual_scale": residual_scale}


def layer(name, rows, experts, k, hidden, inner, act, dtype, skew=0.5):
    return {"name": name, "op": "layer", "rows": rows, "experts": experts, "k": k, "hidden": hidden, "inner": inner,
            "act": act, "dtype": dtype, "skew": skew}


def listed():
    return [
        # one row of a single request through a small router: latency only
        route("route_one_row", 1, 8, 2, "f32"),
        # the largest packed batch through a wide router
        route("route_batch", 65536, 64, 6, "bf16", "softmax", False),
        # one token through two of eight experts: the weights' bytes are the work
        grouped("up_one_token", 1, 8, 2, 768, 2048, "swiglu", "bf16"),
        # a handful of short queries over many narrow experts: nearly every expert has a few rows
        grouped("up_few_rows", 48, 64, 4, 1024, 704, "swiglu", "bf16"),
        # ragged groups and odd widths of an adapter per language, with a bias, float16
        grouped("adapter_ragged", 1531, 12, 1, 776, 1000, "gelu", "f16", True, 1.0),
        # a full packed batch, every token through two experts
        grouped("up_batch", 32768, 8, 2, 768, 2048, "swiglu", "bf16"),
        # the parity type, at a width that no vector size divides
        grouped("parity_f32", 509, 5, 1, 129, 130, "gelu", "f32", True),
        # a query's rows: sum of the experts, residual and LayerNorm
        combine("combine_query", 24, 8, 2, 768, "bf16"),
        # the same for a full packed batch
        combine("combine_batch", 32768, 8, 2, 768, "bf16"),
        # norms around a block over a long packed batch, gated per channel
        blocknorm("norms_batch", 49152, 1024, "bf16", "rms", "rms", "channel"),
        # the same block for one row, with a gate of its own and a scaled residual
        blocknorm("norms_one_row", 1, 1024, "f16", "layer", "layer", "element", 0.5),
        # the whole block of an ordinary batch: route, up, down, combine
        layer("experts_batch", 4096, 8, 2, 768, 2048, "swiglu", "bf16"),
    ]


def log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "grouped", "grouped", "combine", "blocknorm", "layer"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "route":
        experts = log_between(rng, 3, 200)
        return _unnamed(route("", log_between(rng, 1, 65536), experts, rng.randint(1, min(8, experts)), dtype,
                              rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, rng.choice([0.0, 0.02])))
    if op == "combine":
        experts = log_between(rng, 2, 64)
        k = rng.randint(1, min(4, experts))
        cols = rng.choice([log_between(rng, 16, 2048), 8 * log_between(rng, 4, 256)])
        rows = min(log_between(rng, 1, 32768), 50_000_000 // (cols * k))
        return _unnamed(combine("", rows, experts, k, cols, dtype, rng.choice(["none", "layer", "rms"])))
    if op == "blocknorm":
        cols = rng.choice([log_between(rng, 16, 8192), 8 * log_between(rng, 4, 1024)])
        rows = min(log_between(rng, 1, 49152), 25_000_000 // cols)
        return _unnamed(blocknorm("", rows, cols, dtype, rng.choice(["none", "layer", "rms"]),
                                  rng.choice(["layer", "rms"]), rng.choice(["none", "channel", "element"]),
                                  rng.choice([1.0, 0.5, 2.25])))
    if op == "layer":
        dtype = rng.choice(["bf16", "f16"])
        experts = log_between(rng, 2, 64)
        k = rng.randint(1, min(6, experts))
        hidden, inner = 64 * rng.randint(2, 20), 64 * rng.randint(1, 24)
        rows = min(log_between(rng, 1, 8192), int(8e10 / (k * hidden * inner * 6)))
        return _unnamed(layer("", rows, experts, k, hidden, inner, rng.choice(["gelu", "swiglu"]), dtype,
                              rng.choice([0.0, 0.5, 1.0])))
    experts = log_between(rng, 2, 64)
    k = rng.randint(1, min(6, experts))
    odd = dtype == "f32" or rng.random() < 0.15
    inner, outer = ((rng.randint(20, 700), rng.randint(20, 700)) if odd
                    else (8 * log_between(rng, 8, 256), 8 * log_between(rng, 8, 256)))
    act = rng.choice(["identity", "gelu", "swiglu"])
    wide = 2 if act == "swiglu" else 1
    rows = min(log_between(rng, 1, 32768), int((2e9 if odd else 1.5e11) / (k * inner * outer * wide)))
    return _unnamed(grouped("", max(1, rows), experts, k, inner, outer, act, dtype, rng.random() < 0.5,
                            rng.choice([0.0, 0.5, 1.0])))


def _unnamed(c):
    del c["name"]
    return c


def work(c):
    s = size_of(c["dtype"])
    if c["op"] == "route":
        pairs = c["rows"] * c["k"]
        return {"bytes": c["rows"] * c["experts"] * s + pairs * 16 + 4 * c["experts"], "flops": c["rows"] * c["experts"] * 4}
    if c["op"] == "blocknorm":
        n = c["rows"] * c["cols"]
        gate = {"none": 0, "channel": c["cols"], "element": n}[c["gate"]]
        return {"bytes": (4 * n + gate) * s + 16 * c["cols"], "flops": 20 * n}
    pairs = c["rows"] * c["k"]
    if c["op"] == "combine":
        n = c["rows"] * c["cols"]
        extra = 0 if c["norm"] == "none" else n
        return {"bytes": (pairs * c["cols"] + n + extra) * s + 8 * pairs, "flops": 2 * pairs * c["cols"] + 10 * n}
    touched = c["experts"] * (1.0 - (1.0 - c["k"] / c["experts"]) ** c["rows"])  # experts that get a row, evenly drawn
    wide = 2 if c["act"] == "swiglu" else 1
    if c["op"] == "grouped":
        return {"bytes": (c["rows"] * c["inner"] + touched * c["inner"] * c["outer"] * wide + pairs * c["outer"]) * s,
                "flops": 2 * pairs * c["inner"] * c["outer"] * wide}
    one = c["hidden"] * c["inner"] * (wide + 1)
    return {"bytes": (3 * c["rows"] * c["hidden"] + touched * one) * s + c["rows"] * c["experts"] * s, "flops": 2 * pairs * one}


# ---------------------------------------------------------------- inputs
def _logits(c, g, skew):
    """Router logits: unit normal rows with experts of uneven popularity."""
    z = torch.randn(c["rows"], c["experts"], generator=g, device="cuda")
    return z + skew * torch.randn(1, c["experts"], generator=g, device="cuda")


def prepare(c, seed):
    if own:
        _fletcher()  # from here on its stream is torch's
    s = _inputs(c, seed)
    if own:
        s["handles"] = _handles(s)
    return s


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[c["dtype"]]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = {"case": c}
    rows = c["rows"]
    if c["op"] == "route":
        z = 2.0 * _logits(c, g, 0.5)
        if c["masked"]:  # experts that are off, and rows with none
            z = z.masked_fill(torch.rand(rows, c["experts"], generator=g, device="cuda") < c["masked"], -math.inf)
            z = z.masked_fill(torch.rand(rows, 1, generator=g, device="cuda") < c["masked"], -math.inf)
        s["logits"] = z.to(t)
        return s
    if c["op"] == "blocknorm":
        n = c["cols"]
        s["y"], s["residual"] = normal(rows, n), normal(rows, n, scale=3.0)
        s["gate"] = {"none": None, "channel": normal(1, n), "element": normal(rows, n)}[c["gate"]]
        for name in ("post_gamma", "pre_gamma"):
            s[name] = 1.0 + normal(1, n, scale=0.1, dtype=torch.float32)
        for name in ("post_beta", "pre_beta"):
            s[name] = normal(1, n, scale=0.1, dtype=torch.float32)
        s["out"], s["out_norm"] = torch.empty_like(s["y"]), torch.empty_like(s["y"])
        return s
    pairs, experts, k = rows * c["k"], c["experts"], c["k"]
    z = _logits(c, g, c.get("skew", 0.5))
    if c["op"] == "layer":
        s["logits"] = z.to(t)
        hidden, inner = c["hidden"], c["inner"]
        s["x"] = normal(rows, hidden)
        s["up"] = normal(experts * hidden, inner * (2 if c["act"] == "swiglu" else 1), scale=hidden ** -0.5)
        s["down"] = normal(experts * inner, hidden, scale=2.0 * inner ** -0.5)
        s["gamma"], s["beta"] = 1.0 + normal(1, hidden, scale=0.1, dtype=torch.float32), normal(1, hidden, scale=0.1, dtype=torch.float32)
        s["out"] = torch.empty_like(s["x"])
        return s
    # the choices and their weights, as a router made them before
    top, ids = torch.topk(z, k, dim=1)
    s["ids"], s["weights"] = ids.to(torch.int32).contiguous(), torch.softmax(top, 1).contiguous()
    if c["op"] == "combine":
        n = c["cols"]
        s["y"], s["residual"] = normal(pairs, n), normal(rows, n)
        s["gamma"], s["beta"] = 1.0 + normal(1, n, scale=0.1, dtype=torch.float32), normal(1, n, scale=0.1, dtype=torch.float32)
        s["out"] = torch.empty_like(s["residual"])
        return s
    inner, outer = c["inner"], c["outer"]
    wide = outer * (2 if c["act"] == "swiglu" else 1)
    s["x"] = normal(rows, inner)
    s["w"] = normal(experts * inner, wide, scale=inner ** -0.5)
    s["bias"] = normal(experts, wide, scale=0.1) if c["bias"] else None
    s["out"] = torch.empty(pairs, outer, dtype=t, device="cuda")
    return s


# ---------------------------------------------------------------- the plain form
def _plain_route(logits, k, score, normalise):
    z = logits.float()
    key = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    top, ids = torch.sort(key, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    chosen = top > -math.inf
    if score == "softmax":
        m = top[:, :1]
        e = torch.where(top == m, torch.ones_like(top), torch.exp(top - m))
        total = torch.where(key == m, torch.ones_like(key), torch.exp(key - m)).sum(1, keepdim=True)
        w = e / total
    else:
        w = 1.0 / (1.0 + torch.exp(-top))
    w = torch.where(chosen, w, torch.zeros_like(w))
    if normalise:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return torch.where(chosen, ids, torch.full_like(ids, -1)).to(torch.int32), w


def _plain_group(ids, experts):
    """offsets [experts+1], slot of each choice (-1: none): choices ordered by expert, then row."""
    flat = ids.reshape(-1).long()
    order_key = torch.where(flat < 0, torch.full_like(flat, experts), flat)
    order = torch.sort(order_key, stable=True)[1]
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    slots = torch.where(flat < 0, torch.full_like(slots, -1), slots)
    counts = (order_key[None, :] == torch.arange(experts, device=flat.device)[:, None]).sum(1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=flat.device), counts.cumsum(0)])
    return offsets, slots.view_as(ids)


def _plain_act(y, act):
    if act == "swiglu":
        a, b = y.chunk(2, dim=-1)
        return a / (1.0 + torch.exp(-a)) * b
    if act == "gelu":  # the framework's GELU: tanh by its Pade form, cut at 4
        u = 0.7978846 * (y + 0.044715 * y * y * y)
        t = u * (27.0 + u * u) / (27.0 + 9.0 * u * u)
        t = torch.where(u > 4.0, torch.ones_like(u), torch.where(u < -4.0, -torch.ones_like(u), t))
        return 0.5 * y * (1.0 + t)
    return y


def _plain_grouped(x, ids, w, bias, act, experts, slot_rows=None):
    """The grouped product in slot order, as one batched product over groups padded to the largest.
    slot_rows: x is already in slot order."""
    offsets, slots = _plain_group(ids, experts)
    flat, slots = ids.reshape(-1).long(), slots.reshape(-1)
    most = int((offsets[1:] - offsets[:-1]).max())
    place = flat * most + slots - offsets[flat]  # of each choice in the padded layout
    rows = torch.arange(flat.numel(), device=x.device) // ids.shape[1]
    inner = x.shape[1]
    padded = torch.zeros(experts * most, inner, dtype=torch.float32, device=x.device)
    padded[place] = x.float()[rows] if slot_rows is None else x.float()[slots]
    y = torch.bmm(padded.view(experts, most, inner), w.float().view(experts, inner, -1))
    if bias is not None:
        y = y + bias.float()[:, None, :]
    y = _plain_act(y, act)
    out = torch.empty(flat.numel(), y.shape[2], dtype=torch.float32, device=x.device)
    out[slots] = y.reshape(experts * most, -1)[place]
    return out, slots


def _plain_norm(x, kind, gamma, beta, eps):
    if kind == "layer":
        d = x - x.mean(1, keepdim=True)
        return d / torch.sqrt((d * d).mean(1, keepdim=True) + eps) * gamma + beta
    if kind == "rms":
        return x / torch.sqrt((x * x).mean(1, keepdim=True) + eps) * gamma
    return x


def _plain_combine(y, slots, weights, k):
    return (y.float()[slots].view(-1, k, y.shape[1]) * weights.view(-1, k, 1)).sum(1)


def _plain(s):
    c = s["case"]
    t = DTYPES[c["dtype"]]
    if c["op"] == "route":
        ids, w = _plain_route(s["logits"], c["k"], c["score"], c["normalise"])
        offsets, slots = _plain_group(ids, c["experts"])
        return ids, w, offsets.to(torch.int32), slots.to(torch.int32)
    if c["op"] == "blocknorm":
        y = _plain_norm(s["y"].float(), c["post"], s["post_gamma"], s["post_beta"], EPS)
        if s["gate"] is not None:
            y = y * s["gate"].float()
        u = c["residual_scale"] * s["residual"].float() + y
        return u.to(t), _plain_norm(u, c["pre"], s["pre_gamma"], s["pre_beta"], EPS).to(t)
    if c["op"] == "combine":
        slots = _plain_group(s["ids"], c["experts"])[1]
        y = _plain_combine(s["y"], slots.reshape(-1), s["weights"], c["k"])
        if c["norm"] != "none":
            y = _plain_norm(s["residual"].float() + y, c["norm"], s["gamma"], s["beta"], EPS)
        return y.to(t)
    if c["op"] == "grouped":
        return _plain_grouped(s["x"], s["ids"], s["w"], s["bias"], c["act"], c["experts"])[0].to(t)
    ids, w = _plain_route(s["logits"], c["k"], "softmax", True)
    h, slots = _plain_grouped(s["x"], ids, s["up"], None, c["act"], c["experts"])
    y, _ = _plain_grouped(h, ids, s["down"], None, "identity", c["experts"], slots)
    y = s["x"].float() + _plain_combine(y, slots, w, c["k"])
    return _plain_norm(y, "layer", s["gamma"], s["beta"], EPS).to(t)


# ---------------------------------------------------------------- the framework's calls
_backend = None


def _fletcher():
    """The framework's host module and one backend for all cases."""
    global _backend
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "longbow-fletcher_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import fletcher
    if _backend is None:
        _backend = fletcher.Backend(0)
        # The program works on the framework's stream: what torch computes before a call and after it is ordered
        # with it, and nothing waits for that.
        stream = torch.cuda.ExternalStream(_backend.stream())
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
    return fletcher, _backend


class _DeviceArray:
    """Device memory of the framework, for torch.as_tensor; keeps its owner alive."""

    def __init__(self, owner, ptr, shape, kind):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "typestr": kind, "version": 3}


def _handles(s):
    """What a program keeps beside its buffers: their framework tensors, and the routing.  In the grouped and the
    combine cases the routing was made before, by a router or by the program's own choice (a language's adapter),
    and serves every product until the next one: it is the plan of these ids and weights, and the tensors stay."""
    fl, be = _fletcher()
    c = s["case"]
    dt = CODES[c["dtype"]]
    h = {}

    def wrap(name):
        x = s.get(name)
        h[name] = None if x is None else be.wrap(x.data_ptr(), x.shape[0], x.shape[1], 0 if x.dtype == torch.float32 else dt)

    for name in ("logits", "x", "w", "bias", "up", "down", "y", "residual", "gate", "out", "out_norm", "gamma", "beta",
                 "post_gamma", "post_beta", "pre_gamma", "pre_beta"):
        wrap(name)
    if c["op"] != "blocknorm":
        r = h["routing"] = be.routing(c["rows"], c["experts"], c["k"])
        if "ids" in s:
            r.assign(s["ids"].cpu().numpy(), s["weights"].cpu().numpy())
        if c["op"] == "route":
            p = r.device_pointers()
            h["result"] = tuple(torch.as_tensor(_DeviceArray(r, p[n], shape, kind), device="cuda")
                                for n, shape, kind in (("experts", (c["rows"], c["k"]), "<i4"),
                                                       ("weights", (c["rows"], c["k"]), "<f4"),
                                                       ("offsets", (c["experts"] + 1,), "<i4"),
                                                       ("slots", (c["rows"], c["k"]), "<i4")))
    if c["op"] == "layer":
        pairs = c["rows"] * c["k"]
        h["mid"] = be.new_tensor(pairs, c["inner"], None, dt)
        h["expert_out"] = be.new_tensor(pairs, c["hidden"], None, fl.F32)  # summed before they are rounded
    if c["op"] == "blocknorm":
        h["norm"] = fl.BlockNorm(post=NORMS[c["post"]], pre=NORMS[c["pre"]], eps=EPS, residual=h["residual"],
                                 gate=h["gate"], residual_scale=c["residual_scale"],
                                 post_gamma=h["post_gamma"] if c["post"] != "none" else None,
                                 post_beta=h["post_beta"] if c["post"] == "layer" else None, pre_gamma=h["pre_gamma"],
                                 pre_beta=h["pre_beta"] if c["pre"] == "layer" else None)
    elif c["op"] == "layer" or c.get("norm", "none") != "none":
        kind = c.get("norm", "layer")
        h["norm"] = fl.BlockNorm(pre=NORMS[kind], eps=EPS, residual=h["x"] if c["op"] == "layer" else h["residual"],
                                 pre_gamma=h["gamma"], pre_beta=h["beta"] if kind == "layer" else None)
    return h


def _own(s):
    h = s.get("handles")
    if h is None:  # a state of the plain form
        h = s["handles"] = _handles(s)
    c = s["case"]
    op = c["op"]
    if op == "route":
        h["routing"].route(h["logits"], SCORES[c["score"]], c["normalise"])
        return h["result"]
    if op == "blocknorm":
        h["y"].block_norm(h["norm"], out=h["out"], out_norm=h["out_norm"])
        return s["out"], s["out_norm"]
    r = h["routing"]
    if op == "combine":
        if c["norm"] == "none":
            r.combine(h["y"], out=h["out"])
        else:
            r.combine(h["y"], h["norm"], out_norm=h["out"])
        return s["out"]
    if op == "grouped":
        r.linear(h["x"], h["w"], h["bias"], ACTS[c["act"]], out=h["out"])
        return s["out"]
    r.route(h["logits"])
    r.linear(h["x"], h["up"], None, ACTS[c["act"]], out=h["mid"])
    r.linear(h["mid"], h["down"], None, grouped_input=True, out=h["expert_out"])
    r.combine(h["expert_out"], h["norm"], out_norm=h["out"])
    return s["out"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_route(z, k, score, normalise):
    z = z.double()
    off = torch.isnan(z) | torch.isneginf(z)
    p = torch.softmax(z.masked_fill(off, -math.inf), 1) if score == "softmax" else torch.sigmoid(z)
    left = z.masked_fill(off, -math.inf).clone()
    ids, ws = [], []
    at = torch.arange(z.shape[1], device=z.device)
    for _ in range(k):  # the largest that is left, the first of equals
        best = left.max(1, keepdim=True)[0]
        i = torch.where(left == best, at, z.shape[1]).min(1, keepdim=True)[0]
        none = torch.isneginf(best)
        ids.append(torch.where(none, -1, i))
        ws.append(torch.where(none, 0.0, p.gather(1, i)))
        left.scatter_(1, i, -math.inf)
    ids, w = torch.cat(ids, 1), torch.cat(ws, 1)
    if normalise:
        w = torch.nan_to_num(w / w.sum(1, keepdim=True), nan=0.0)
    return ids, w


def _exact_linear(x, w, bias, act):
    y = x @ w
    if bias is not None:
        y += bias
    if act == "swiglu":
        n = y.shape[1] // 2
        return y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
    if act == "gelu":
        u = 0.7978846 * (y + 0.044715 * y ** 3)
        t = u * (27 + u ** 2) / (27 + 9 * u ** 2)
        return 0.5 * y * (1 + torch.where(u.abs() > 4, torch.sign(u), t))
    return y


def _exact_norm(u, kind, gamma, beta):
    if kind == "none":
        return u
    if kind == "layer":
        return (u - u.mean(1, keepdim=True)) * torch.rsqrt(u.var(1, unbiased=False, keepdim=True) + EPS) * gamma.double() + beta.double()
    return u * torch.rsqrt(u.pow(2).mean(1, keepdim=True) + EPS) * gamma.double()


def exact(c, seed):
    s = _inputs(c, seed)
    if c["op"] == "route":
        _, w = _exact_route(s["logits"], c["k"], c["score"], c["normalise"])
        return None, w, None, None
    if c["op"] == "blocknorm":
        y = _exact_norm(s["y"].double(), c["post"], s["post_gamma"], s["post_beta"])
        u = c["residual_scale"] * s["residual"].double() + (y if s["gate"] is None else s["gate"].double() * y)
        return u, _exact_norm(u, c["pre"], s["pre_gamma"], s["pre_beta"])
    experts, k = c["experts"], c["k"]
    ids, w = (_exact_route(s["logits"], k, "softmax", True) if c["op"] == "layer" else (s["ids"].long(), s["weights"].double()))
    token = torch.arange(c["rows"], device="cuda")[:, None].expand(-1, k)
    groups = [(ids == e).nonzero(as_tuple=True) for e in range(experts)]  # (row, choice) of each expert, rows ascending
    if c["op"] == "combine":
        y = torch.zeros(c["rows"], c["cols"], dtype=torch.float64, device="cuda")
        at = 0
        for r, j in groups:
            y[r] += w[r, j][:, None] * s["y"][at:at + r.numel()].double()
            at += r.numel()
        return y if c["norm"] == "none" else _exact_norm(y + s["residual"].double(), c["norm"], s["gamma"], s["beta"])
    if c["op"] == "grouped":
        ws = s["w"].view(experts, c["inner"], -1)
        return torch.cat([_exact_linear(s["x"][token[r, j]].double(), ws[e].double(),
                                        None if s["bias"] is None else s["bias"][e].double(), c["act"])
                          for e, (r, j) in enumerate(groups)])
    up, down = s["up"].view(experts, c["hidden"], -1), s["down"].view(experts, c["inner"], -1)
    y = s["x"].double()
    for e, (r, j) in enumerate(groups):
        h = _exact_linear(s["x"][r].double(), up[e].double(), None, c["act"])
        y[r] += w[r, j][:, None] * (h @ down[e].double())
    return _exact_norm(y, "layer", s["gamma"], s["beta"])
