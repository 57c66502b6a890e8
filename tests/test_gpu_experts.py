"""GPU tests of the expert feed-forward operators (Cuda_Routing_*, Cuda_Linear_Grouped,
Cuda_Combine_Grouped, Cuda_BlockNorm) against plain 64-bit numpy.

Tolerances count roundings: an output of type T is off by at most eps_T / 2 relative (bf16 2^-8 of
its 8-bit significand's last place halved: 2^-9 is written u = eps/2 below), plus fp32 arithmetic
on the way, bounded by n * 2^-24 times the sum of the terms' absolute values for a sum of n terms.
"""
import ctypes

import numpy as np
import pytest

from helpers import bf16_round

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # eps / 2
TINY = {"f32": 1e-38, "f16": 2.0 ** -24, "bf16": 1e-38}  # spacing of the smallest values, rounded up
E24 = 2.0 ** -24


@pytest.fixture(scope="module")
def fl():
    import build
    build.build()
    import fletcher
    return fletcher


@pytest.fixture(scope="module")
def be(fl):
    b = fl.Backend(0)
    b.set_half_conversion(fl.HALF_RNE)  # fp16 inputs and results cross as IEEE values
    return b


def quantise(x, dtype):
    x = np.asarray(x, np.float32)
    if dtype == "bf16":
        return bf16_round(x)
    return x.astype(np.float16).astype(np.float32) if dtype == "f16" else x


def tensor(fl, be, x, dtype):
    x = np.asarray(x, np.float32)
    return be.new_tensor(x.shape[0], x.shape[1], x, fl.DTYPES[dtype])


# ---------------------------------------------------------------- references
def route_ref(z, k, score="softmax", normalise=True, scale=1.0):
    z = np.asarray(z, np.float64)
    rows, experts = z.shape
    key = np.where(np.isnan(z), -np.inf, z) + 0.0
    order = np.argsort(-key, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(key, order, 1)
    ok = top > -np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        if score == "softmax":
            m = top[:, :1]
            e = np.where(top == m, 1.0, np.exp(top - m))
            w = e / np.where(key == m, 1.0, np.exp(key - m)).sum(1, keepdims=True)
        else:
            w = 1.0 / (1.0 + np.exp(-top))
        w = np.where(ok, w, 0.0)
        if normalise:
            t = w.sum(1, keepdims=True)
            w = np.where(t > 0, w / np.where(t > 0, t, 1.0), 0.0)
    return np.where(ok, order, -1).astype(np.int32), w * scale


def group_ref(ids, experts):
    flat = ids.reshape(-1)
    order = np.argsort(np.where(flat < 0, experts, flat), kind="stable")
    n = int((flat >= 0).sum())
    slots = np.full(flat.size, -1, np.int32)
    slots[order[:n]] = np.arange(n)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=experts))]).astype(np.int32)
    return slots.reshape(ids.shape), offsets, order[:n]


def act_ref(y, act):
    """(act(y), a factor that bounds how much it amplifies an error, values near GELU's cut)"""
    near = np.zeros(y.shape, bool)
    if act == 4:
        a, b = np.split(y, 2, axis=1)
        with np.errstate(over="ignore"):
            return a / (1 + np.exp(-a)) * b, None, np.zeros(a.shape, bool)
    if act == 1:
        u = 0.7978846 * (y + 0.044715 * y ** 3)
        t = np.where(np.abs(u) > 4, np.sign(u), u * (27 + u * u) / (27 + 9 * u * u))
        return 0.5 * y * (1 + t), 1.2, np.abs(np.abs(u) - 4) < 1e-3
    if act == 2:
        t = np.where(np.abs(y) > 4, np.sign(y), y * (27 + y * y) / (27 + 9 * y * y))
        return t, 1.0, np.abs(np.abs(y) - 4) < 1e-3
    return y, 1.0, near


def grouped_ref(x, w, b, ids, experts, act, grouped_input):
    """Exact result in slot order and its tolerance before the last rounding."""
    slots, offsets, order = group_ref(ids, experts)
    K = x.shape[1]
    w3 = w.reshape(experts, K, -1).astype(np.float64)
    n_out = w3.shape[2] // (2 if act == 4 else 1)
    out, tol = np.zeros((order.size, n_out)), np.zeros((order.size, n_out))
    skip = np.zeros((order.size, n_out), bool)
    for e in range(experts):
        lo, hi = offsets[e], offsets[e + 1]
        if lo == hi:
            continue
        rows = np.arange(lo, hi) if grouped_input else order[lo:hi] // ids.shape[1]
        xe = x[rows].astype(np.float64)
        y = xe @ w3[e]
        mag = np.abs(xe) @ np.abs(w3[e])
        if b is not None:
            y = y + b[e]
            mag = mag + np.abs(b[e])
        err = (K + 4) * E24 * mag
        v, gain, near = act_ref(y, act)
        if act == 4:
            a, u = np.split(y, 2, axis=1)
            ea, eu = np.split(err, 2, axis=1)
            silu = np.abs(a / (1 + np.exp(-a)))
            # |silu'| <= 1.1; the exponential and the division add a few fp32 roundings, the
            # exponent's argument one of |a| * 2^-23
            err = 1.1 * ea * np.abs(u) + silu * eu + (8 + 4 * np.abs(a)) * E24 * np.abs(v)
        else:
            # the polynomial's few roundings, on values of up to |y| before cancellation
            err = gain * err + (16 * E24 * np.abs(y) if act else 0)
        out[lo:hi], tol[lo:hi], skip[lo:hi] = v, err, near
    return out, tol, skip


def norm_ref(x, kind, gamma, beta, eps):
    if kind == 0:
        return x
    if kind == 1:
        d = x - x.mean(1, keepdims=True)
        y = d / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    else:
        y = x / np.sqrt((x * x).mean(1, keepdims=True) + eps)
    return y * (1.0 if gamma is None else gamma) + (0.0 if beta is None else beta)


def check(got, want, tol, dtype, what=""):
    bound = np.abs(want) * U[dtype] * (1 + 1e-6) + tol * (1 + 2 * U[dtype]) + TINY[dtype]
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, worst "
                           f"{np.max((np.abs(got - want) / bound)[bad])} of the bound at {np.argwhere(bad)[0]}")


# ---------------------------------------------------------------- routing
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,experts,k", [(1, 8, 2), (0, 8, 2), (1, 1, 1), (7, 3, 3), (300, 9, 1), (513, 17, 16),
                                            (1000, 64, 6), (2049, 33, 5), (4099, 128, 8), (700, 256, 16), (9001, 200, 3), (1, 256, 16), (40, 200, 5), (128, 65, 2)])
def test_routing(fl, be, rows, experts, k, dtype):
    rng = np.random.default_rng(rows * 1000 + experts)
    z = quantise(2 * rng.standard_normal((rows, experts)), dtype)
    if dtype != "f32" or rows % 2:  # many equal logits, zeros of both signs
        z = np.round(z * 4) / 4
        z[rng.random(z.shape) < 0.1] = -0.0
    z = z.astype(np.float32)
    t = tensor(fl, be, z, dtype)
    r = be.routing(rows + 3, experts, k)
    for score, normalise, scale in ((0, True, 1.0), (0, False, 1.0), (1, True, 2.5), (1, False, 0.5)):
        r.route(t, score, normalise, scale)
        got = r.read()
        ids, w = route_ref(z, k, ["softmax", "sigmoid"][score], normalise, scale)
        assert (got["experts"] == ids).all()
        # expf is good to 2 roundings, its argument x - m to one of |x - m| <= 32, sums to 256 terms
        assert np.allclose(got["weights"], w, rtol=(300 + 64) * E24, atol=1e-37)
        slots, offsets, _ = group_ref(ids, experts)
        assert (got["slots"] == slots).all() and (got["offsets"] == offsets).all()


@pytest.mark.parametrize("rows,experts,k,dtype", [(300000, 16, 8, "bf16"), (200003, 5, 1, "f32")])
def test_routing_many_rows(fl, be, rows, experts, k, dtype):
    """More pairs a block than it ranks at once, and as many blocks as there are."""
    rng = np.random.default_rng(rows)
    z = quantise(rng.standard_normal((rows, experts)) + np.linspace(0, 2, experts), dtype)
    r = be.routing(rows, experts, k)
    r.route(tensor(fl, be, z, dtype))
    got = r.read()
    ids, _ = route_ref(z, k)
    slots, offsets, _ = group_ref(ids, experts)
    assert (got["experts"] == ids).all() and (got["slots"] == slots).all() and (got["offsets"] == offsets).all()


def test_routing_masks(fl, be):
    inf, nan, low = np.inf, np.nan, float(np.finfo(np.float32).min)
    z = np.array([[-inf] * 4, [nan] * 4, [0, -inf, nan, -inf], [inf, 1, inf, 0], [low] * 4, [low, 0, low, -inf],
                  [inf, nan, -inf, low], [1, 1, 1, 1]], np.float32)
    for score in ("softmax", "sigmoid"):
        for normalise in (True, False):
            r = be.routing(8, 4, 3)
            r.route(tensor(fl, be, z, "f32"), ["softmax", "sigmoid"].index(score), normalise)
            got = r.read()
            ids, w = route_ref(z, 3, score, normalise)
            assert (got["experts"] == ids).all(), (score, got["experts"], ids)
            assert np.allclose(got["weights"], w, rtol=1e-5, atol=0)
            slots, offsets, _ = group_ref(ids, 4)
            assert (got["slots"] == slots).all() and (got["offsets"] == offsets).all()


@pytest.mark.parametrize("rows,experts,k", [(5, 4, 2), (3000, 7, 3), (20000, 256, 2)])
def test_routing_assign(fl, be, rows, experts, k):
    rng = np.random.default_rng(rows)
    ids = rng.integers(-1, experts, (rows, k)).astype(np.int32)  # an expert may come twice in a row
    ids[rng.random(rows) < 0.3] = experts - 1
    w = rng.random((rows, k)).astype(np.float32)
    r = be.routing(rows, experts, k)
    for weights in (w, None):
        r.assign(ids, weights)
        got = r.read()
        slots, offsets, _ = group_ref(ids, experts)
        assert (got["experts"] == ids).all() and (got["slots"] == slots).all() and (got["offsets"] == offsets).all()
        assert (got["weights"] == (1.0 if weights is None else w)).all()


# ---------------------------------------------------------------- grouped products
def run_grouped(fl, be, rows, experts, k, K, N, act, dtype, bias, grouped_input, ids=None, seed=0, out=None):
    out = out or dtype
    rng = np.random.default_rng(seed + rows + 7 * K + 13 * N)
    if ids is None:
        ids = np.argsort(rng.random((rows, experts)) + np.linspace(0, 1, experts), 1)[:, :k].astype(np.int32)
    pairs = ids.size
    x = quantise(rng.standard_normal((pairs if grouped_input else rows, K)), dtype)
    w = quantise(rng.standard_normal((experts * K, N)) / np.sqrt(K), dtype)
    b = quantise(rng.standard_normal((experts, N)) * 0.5, dtype) if bias else None
    r = be.routing(rows + 5, experts, k)
    r.assign(ids)
    n_out = N // 2 if act == 4 else N
    before = quantise(rng.standard_normal((pairs + 2, n_out)), out)  # rows behind the last stay
    y = tensor(fl, be, before, out)
    r.linear(tensor(fl, be, x, dtype), tensor(fl, be, w, dtype), None if b is None else tensor(fl, be, b, dtype), act,
             grouped_input, out=y)
    got = y.to_host()
    be.synchronize()
    want, tol, skip = grouped_ref(x, w, b, ids, experts, act, grouped_input)
    n = want.shape[0]
    assert (got[n:] == before[n:]).all(), "rows behind the last slot were written"
    check(np.where(skip, want, got[:n]), want, tol, out, f"{rows} {experts} {k} {K} {N} {act} {dtype}")


SHAPES = [  # rows, experts, k, K, N
    (1, 8, 2, 64, 128), (1, 1, 1, 8, 16), (3, 4, 1, 72, 40), (16, 64, 4, 256, 192), (33, 5, 2, 200, 264),
    (130, 3, 2, 136, 512), (257, 2, 1, 64, 256), (500, 12, 3, 320, 384), (1031, 4, 2, 128, 1032),
    (1, 8, 2, 768, 1536), (2, 4, 1, 2048, 136), (20, 2, 1, 1000, 72), (40, 2, 2, 520, 64)]


@pytest.mark.parametrize("rows,experts,k,K,N", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("act", [0, 1, 4])
def test_linear_grouped(fl, be, rows, experts, k, K, N, act, dtype):
    run_grouped(fl, be, rows, experts, k, K, N, act, dtype, act != 0, False)
    run_grouped(fl, be, rows, experts, k, K, N, act, dtype, act == 0, True)


@pytest.mark.parametrize("rows,experts,k,K,N", [SHAPES[i] for i in (0, 3, 4, 7, 8, 9)] + [(70, 3, 2, 17, 66), (2100, 3, 1, 64, 776)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_linear_grouped_f32_result(fl, be, rows, experts, k, K, N, dtype):
    """16-bit operands, the sums kept in fp32."""
    for act in (0, 1, 4):
        run_grouped(fl, be, rows, experts, k, K, N, act, dtype, act == 1, act == 0, out="f32")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,experts,k,K,N", [(5, 2, 1, 1, 2), (70, 3, 2, 17, 66), (9, 4, 2, 129, 130), (64, 2, 1, 64, 2)])
def test_linear_grouped_odd_widths(fl, be, rows, experts, k, K, N, dtype):
    for act in (0, 1, 2, 4):
        run_grouped(fl, be, rows, experts, k, K, N, act, dtype, True, False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pattern", ["one_expert", "first_and_last", "none", "holes", "twice"])
@pytest.mark.parametrize("rows", [2, 300])
def test_linear_grouped_uneven(fl, be, pattern, rows, dtype):
    """All rows with one expert, experts without rows, rows without experts, an expert twice in a row."""
    E, k = 9, 2
    ids = np.full((rows, k), -1, np.int32)
    if pattern == "one_expert":
        ids[:, 0] = 4
    elif pattern == "first_and_last":
        ids[:, 0], ids[:, 1] = 0, E - 1
    elif pattern == "holes":
        ids[::3, 1] = 7
        ids[1::3] = [2, 5]
    elif pattern == "twice":
        ids[:] = 3
    for grouped_input in (False, True):
        run_grouped(fl, be, rows, E, k, 128, 256, 4, dtype, True, grouped_input, ids=ids)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [4, 400])
def test_linear_grouped_nonfinite(fl, be, dtype, rows):
    """A NaN or inf in one row reaches that row alone, one in an expert's weights that expert alone,
    also where a row length that no tile divides makes tiles reach into their neighbours."""
    E, K, N = 3, 72, 136
    rng = np.random.default_rng(1)
    ids = (np.arange(rows) % 3).astype(np.int32)[:, None]
    x = quantise(rng.standard_normal((rows, K)), dtype)
    w = quantise(rng.standard_normal((E * K, N)) / 8, dtype)
    x[1] = np.nan
    w[K] = np.inf  # expert 1's first row
    w[2 * K - 1] = np.nan  # and its last
    r = be.routing(rows, E, 1)
    r.assign(ids)
    y = r.linear(tensor(fl, be, x, dtype), tensor(fl, be, w, dtype)).to_host()
    _, offsets, order = group_ref(ids, E)
    finite = np.isfinite(y).all(1)
    assert (finite == (ids[order, 0] != 1)).all()


# ---------------------------------------------------------------- norms and combine
def norm_case(rng, rows, cols, dtype, post, pre, gate, residual):
    q = lambda *s: quantise(rng.standard_normal(s), dtype)  # noqa: E731
    c = dict(y=q(rows, cols), residual=3 * q(rows, cols) if residual else None,
             gate={0: None, 1: q(1, cols), 2: q(rows, cols)}[gate])
    c["residual"] = None if c["residual"] is None else quantise(c["residual"], dtype)
    for n, kind in (("post", post), ("pre", pre)):
        c[n + "_gamma"] = (1 + 0.2 * rng.standard_normal((1, cols))).astype(np.float32) if kind else None
        c[n + "_beta"] = (0.2 * rng.standard_normal((1, cols))).astype(np.float32) if kind == 1 else None
    return c


def norm_expect(c, y, post, pre, eps, rs, bs):
    """(u, h) in 64 bits and bounds of their fp32 errors."""
    n = y.shape[1]
    v = norm_ref(y, post, c["post_gamma"], c["post_beta"], eps)
    ev = (n + 16) * E24 * (np.abs(v) + (1.0 if post else 0.0) * np.abs(norm_ref(y, post, c["post_gamma"], None, eps)))
    g = 1.0 if c["gate"] is None else c["gate"].astype(np.float64)
    u = bs * g * v
    eu = np.abs(bs * g) * ev
    if c["residual"] is not None:
        u = u + rs * c["residual"].astype(np.float64)
        eu = eu + 4 * E24 * (np.abs(u) + np.abs(rs * c["residual"]))
    eu = eu + 4 * E24 * np.abs(u)
    h = norm_ref(u, pre, c["pre_gamma"], c["pre_beta"], eps)
    # an error of u moves the row's statistics too: its norm over the row's spread, twice
    d = u - u.mean(1, keepdims=True) if pre == 1 else u
    spread = np.sqrt((d * d).mean(1, keepdims=True) + eps) + 1e-300
    big = np.sqrt((eu * eu).mean(1, keepdims=True)) + 2 * E24 * np.abs(u).max(1, keepdims=True)
    gam = 1.0 if c["pre_gamma"] is None else np.abs(c["pre_gamma"])
    z = np.abs(d) / spread
    eh = gam * (eu + big * (1 + z)) / spread + (n + 16) * E24 * (gam * z + np.abs(h))
    return u, h, eu, eh


def make_norm(fl, be, c, dtype, post, pre, eps, rs, bs):
    t = {k: None if v is None else tensor(fl, be, v, "f32" if "gamma" in k or "beta" in k else dtype)
         for k, v in c.items() if k != "y"}
    return fl.BlockNorm(post=post, pre=pre, eps=eps, residual_scale=rs, branch_scale=bs, **t), t


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1024), (5, 8), (3, 100), (2, 1), (70, 768), (33, 1000), (9, 2056), (4, 4096),
                                       (3, 8192), (2, 9001), (2000, 136), (1, 49152)])
def test_block_norm(fl, be, rows, cols, dtype):
    rng = np.random.default_rng(rows + cols)
    for post, pre, gate, residual, rs, bs in ((0, 1, 0, True, 1.0, 1.0), (1, 2, 1, True, 0.5, 1.0), (2, 0, 2, True, 2.0, -0.25),
                                              (0, 0, 1, False, 1.0, 3.0), (2, 2, 0, True, 1.0, 1.0), (1, 1, 2, False, 1.0, 1.0)):
        eps = 1e-5
        c = norm_case(rng, rows, cols, dtype, post, pre, gate, residual)
        u, h, eu, eh = norm_expect(c, c["y"].astype(np.float64), post, pre, eps, rs, bs)
        norm, _ = make_norm(fl, be, c, dtype, post, pre, eps, rs, bs)
        gu, gh = tensor(fl, be, c["y"], dtype).block_norm(norm)
        check(gu.to_host(), u, eu, dtype, f"u {post} {pre} {gate}")
        assert (gh is None) == (pre == 0)
        if pre:
            check(gh.to_host(), h, eh, dtype, f"h {post} {pre} {gate}")
            only = tensor(fl, be, np.zeros((rows, cols)), dtype)  # the norm alone
            assert tensor(fl, be, c["y"], dtype).block_norm(norm, out_norm=only)[0] is None
            assert (only.to_host() == gh.to_host()).all()


@pytest.mark.parametrize("dtype,cols", [("bf16", 768), ("f32", 768), ("f16", 77), ("bf16", 4104)])
def test_block_norm_in_place(fl, be, dtype, cols):
    rng = np.random.default_rng(cols)
    rows = 50
    c = norm_case(rng, rows, cols, dtype, 2, 1, 2, True)
    norm, t = make_norm(fl, be, c, dtype, 2, 1, 1e-6, 1.0, 1.0)
    wu, wh = (x.to_host() for x in tensor(fl, be, c["y"], dtype).block_norm(norm))
    for u_over, h_over in (("residual", "y"), ("y", "gate"), ("gate", "residual")):
        norm, t = make_norm(fl, be, c, dtype, 2, 1, 1e-6, 1.0, 1.0)
        t["y"] = tensor(fl, be, c["y"], dtype)
        t["y"].block_norm(norm, out=t[u_over], out_norm=t[h_over])
        assert (t[u_over].to_host() == wu).all() and (t[h_over].to_host() == wh).all()


@pytest.mark.parametrize("dtype,slots_dtype", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows,experts,k,cols", [(1, 8, 2, 768), (40, 4, 1, 8), (257, 16, 5, 100), (600, 8, 2, 1536),
                                                 (33, 3, 3, 2049), (5, 4, 4, 8192)])
def test_combine(fl, be, rows, experts, k, cols, dtype, slots_dtype):
    rng = np.random.default_rng(rows + cols)
    ids = rng.integers(-1, experts, (rows, k)).astype(np.int32)
    w = rng.standard_normal((rows, k)).astype(np.float32)
    r = be.routing(rows, experts, k)
    r.assign(ids, w)
    slots = group_ref(ids, experts)[0]
    g = quantise(rng.standard_normal((rows * k, cols)), slots_dtype)
    tg = tensor(fl, be, g, slots_dtype)
    terms = np.where(slots[..., None] >= 0, w[..., None] * g.astype(np.float64)[np.maximum(slots, 0)], 0.0)
    y, mag = terms.sum(1), np.abs(terms).sum(1)
    plain = be.new_tensor(rows, cols, None, fl.DTYPES[dtype])
    check(r.combine(tg, out=plain).to_host(), y, (k + 1) * E24 * mag, dtype)
    c = norm_case(rng, rows, cols, dtype, 0, 1, 1, True)
    norm, t = make_norm(fl, be, c, dtype, 0, 1, 1e-5, 1.0, 1.0)
    u, h, eu, eh = norm_expect(c, y, 0, 1, 1e-5, 1.0, 1.0)
    eu = eu + (k + 1) * E24 * mag * np.abs(c["gate"])
    d = u - u.mean(1, keepdims=True)
    spread = np.sqrt((d * d).mean(1, keepdims=True) + 1e-5)
    eh = eh + np.abs(c["pre_gamma"]) * 3 * (np.abs(d) / spread + 1) * (k + 1) * E24 * (mag * np.abs(c["gate"])).max(1, keepdims=True) / spread
    gu, gh = r.combine(tg, norm)
    check(gu.to_host(), u, eu, dtype)
    check(gh.to_host(), h, eh, dtype)
    _, over = r.combine(tg, norm, out_norm=t["residual"])  # the stream's own buffer
    assert (over.to_host() == gh.to_host()).all()


def test_combine_skips_stale_rows(fl, be):
    """NaN in the rows behind the last slot, and in no chosen row, reaches nothing."""
    r = be.routing(4, 2, 2)
    r.assign(np.array([[0, -1], [-1, -1], [1, 0], [-1, 1]], np.int32))
    g = np.full((8, 16), np.nan, np.float32)
    g[:4] = np.arange(4)[:, None] + 1
    got = r.combine(tensor(fl, be, g, "f32")).to_host()
    assert (got[:, 0] == [1, 0, 2 + 3, 4]).all()


# ---------------------------------------------------------------- the block, captures, order
def block(be, fl, r, t, mid, out2, out, act):
    r.route(t["logits"])
    r.linear(t["x"], t["up"], None, act, out=mid)
    r.linear(mid, t["down"], None, grouped_input=True, out=out2)
    r.combine(out2, t["norm"], out_norm=out)


@pytest.mark.parametrize("rows,experts,k,H,I,act,dtype", [(1, 8, 2, 128, 256, 4, "bf16"), (50, 16, 4, 192, 128, 1, "f16"),
                                                        (900, 8, 2, 256, 320, 4, "bf16"), (77, 4, 2, 65, 33, 1, "f32")])
def test_expert_block(fl, be, rows, experts, k, H, I, act, dtype):
    """route -> up -> down -> combine with residual and LayerNorm, against 64 bits throughout."""
    rng = np.random.default_rng(rows)
    wide = 2 if act == 4 else 1
    q = lambda s, *d: quantise(s * rng.standard_normal(d), dtype)  # noqa: E731
    a = dict(logits=q(1.0, rows, experts), x=q(1.0, rows, H), up=q(H ** -0.5, experts * H, I * wide),
             down=q(I ** -0.5, experts * I, H))
    t = {n: tensor(fl, be, v, dtype) for n, v in a.items()}
    t["norm"] = fl.BlockNorm(pre=fl.NORM_LAYER, eps=1e-5, residual=t["x"])
    r = be.routing(rows, experts, k)
    dt = fl.DTYPES[dtype]
    mid, out2, out = (be.new_tensor(n, m, None, d) for n, m, d in ((rows * k, I, dt), (rows * k, H, fl.F32), (rows, H, dt)))
    block(be, fl, r, t, mid, out2, out, act)
    got = out.to_host()
    ids, w = route_ref(a["logits"], k)
    slots, _, _ = group_ref(ids, experts)
    h, _, _ = grouped_ref(a["x"], a["up"], None, ids, experts, act, False)
    g, _, _ = grouped_ref(h, a["down"], None, ids, experts, 0, True)
    want = norm_ref(a["x"] + (w[..., None] * g[slots]).sum(1), 1, None, None, 1e-5)
    # Two roundings to T meet (h and the result; the experts' outputs stay fp32), each of relative size u
    # on values whose rows have a norm of at most a few times the result's: 6 u of a row's norm.
    err = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
    assert err.max() <= (6 * U[dtype] if dtype != "f32" else 2e-5), err.max()


def test_expert_block_captured(fl, be):
    """The block captured into two graphs over two routings, replayed in turn on new inputs."""
    import torch
    rng = np.random.default_rng(3)
    rows, E, k, H, I = 200, 8, 2, 128, 192
    stream = torch.cuda.ExternalStream(be.stream())
    sides = []
    for _ in range(2):
        a = dict(logits=rng.standard_normal((rows, E)), x=rng.standard_normal((rows, H)),
                 up=rng.standard_normal((E * H, 2 * I)) * 0.1, down=rng.standard_normal((E * I, H)) * 0.1)
        t = {n: tensor(fl, be, v, "bf16") for n, v in a.items()}
        t["norm"] = fl.BlockNorm(pre=fl.NORM_LAYER, eps=1e-5, residual=t["x"])
        r = be.routing(rows, E, k)
        bufs = [be.new_tensor(n, m, None, fl.BF16) for n, m in ((rows * k, I), (rows * k, H), (rows, H))]
        block(be, fl, r, t, *bufs, 4)
        be.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            block(be, fl, r, t, *bufs, 4)
        sides.append((g, t, r, bufs))
    for step in range(3):
        new = [(rng.standard_normal((rows, E)), rng.standard_normal((rows, H))) for _ in sides]
        for (g, t, r, bufs), (z, x) in zip(sides, new):
            t["logits"].copy_from_float32(z)
            t["x"].copy_from_float32(x)
        with torch.cuda.stream(stream):
            for g, *_ in sides:
                g.replay()
        be.synchronize()
        got = [bufs[2].to_host() for _, _, _, bufs in sides]
        for (g, t, r, bufs), y in zip(sides, got):
            block(be, fl, r, t, *bufs, 4)
            assert (bufs[2].to_host() == y).all()
    del sides


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_rows(fl, be, dtype):
    new = lambda r, c: be.new_tensor(r, c, None, fl.DTYPES[dtype])  # noqa: E731
    r = be.routing(0, 4, 2)
    r.route(new(0, 4))
    got = r.read()
    assert got["experts"].shape == (0, 2) and (got["offsets"] == 0).all()
    h = r.linear(new(0, 64), new(4 * 64, 128), None, 4)
    assert h.dims() == (0, 64)
    u, n = r.combine(r.linear(h, new(4 * 64, 32), grouped_input=True), fl.BlockNorm(pre=1, residual=new(0, 32)))
    assert u.dims() == n.dims() == (0, 32)
    assert new(0, 32).block_norm(fl.BlockNorm(pre=2, gate=new(1, 32)))[1].dims() == (0, 32)
    be.synchronize()


def test_past_32_bits(fl, be):
    """Outputs and slots of more than 2^31 elements: the last rows against torch."""
    import torch
    rows, k, K, N, E = 140000, 2, 64, 8192, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, K, generator=g, device="cuda").bfloat16()
    w = (torch.randn(E * K, N, generator=g, device="cuda") / 8).bfloat16()
    y = torch.empty(rows * k, N, device="cuda", dtype=torch.bfloat16)
    out = torch.empty(rows, N, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    wrap = lambda t: be.wrap(t.data_ptr(), *t.shape, fl.BF16)  # noqa: E731
    r = be.routing(rows, E, k)
    ids = np.stack([np.arange(rows) % 3, (np.arange(rows) + 1) % 3], 1).astype(np.int32)
    r.assign(ids)
    r.linear(wrap(x), wrap(w), out=wrap(y))
    r.combine(wrap(y), out=wrap(out))
    slots = torch.from_numpy(r.read()["slots"]).cuda().long()
    pick = torch.tensor([0, 1, 2, rows // 2, rows - 2, rows - 1], device="cuda")
    e = torch.from_numpy(ids).cuda()[pick].long()
    want = torch.einsum("rk,rjkn->rjn", x[pick].double(), w.view(E, K, N)[e].double())
    mag = torch.einsum("rk,rjkn->rjn", x[pick].double().abs(), w.view(E, K, N)[e].double().abs())
    got = y[slots[pick]].double()
    assert ((got - want).abs() <= want.abs() * U["bf16"] + (K + 4) * E24 * mag + 1e-30).all()
    total = got.sum(1)
    assert ((out[pick].double() - total).abs() <= total.abs() * U["bf16"] + 4 * E24 * got.abs().sum(1) + 1e-30).all()
    norm = fl.BlockNorm(pre=fl.NORM_RMS, eps=0.0)
    wrap(y).block_norm(norm, out_norm=wrap(y))  # in place over 2.3e9 elements
    be.synchronize()
    rms = (got * got).mean(2, keepdim=True).sqrt()
    normed = got / rms
    assert ((y[slots[pick]].double() - normed).abs() <= normed.abs() * (U["bf16"] + (N + 16) * E24)).all()


def test_memory_is_kept_and_returned(fl, be):
    """A routing's workspace grows on first use only, also across smaller calls, and goes with the routing."""
    before = be.vram_usage()[0]
    r = be.routing(512, 4, 2)
    x, w, y = (be.new_tensor(n, m, None, fl.BF16) for n, m in ((512, 256), (4 * 256, 128), (1024, 128)))
    small = be.new_tensor(100, 256, None, fl.BF16)
    r.assign(np.tile([0, 3], (512, 1)))
    r.linear(x, w, out=y)
    held = be.vram_usage()[0]
    r.linear(x, w, out=y)
    r.assign(np.tile([1, 2], (100, 1)))
    r.linear(small, w, out=y)
    assert be.vram_usage()[0] == held
    del r, x, w, y, small
    assert be.vram_usage()[0] == before


def test_growing_workspace_is_refused_in_a_capture(fl, be):
    import torch
    r = be.routing(512, 4, 2)
    x, w, y = (be.new_tensor(n, m, None, fl.BF16) for n, m in ((512, 256), (4 * 256, 128), (1024, 128)))
    w2, y2 = be.new_tensor(4 * 128, 64, None, fl.BF16), be.new_tensor(1024, 64, None, fl.BF16)
    r.assign(np.tile([0, 3], (512, 1)))
    be.synchronize()
    g, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(be.stream())
    with torch.cuda.graph(g, stream=stream):
        refuses(fl, be, lambda: r.linear(x, w, out=y), "before capturing")
        r.linear(y, w2, grouped_input=True, out=y2)  # needs none
    be.synchronize()


def test_two_contexts_at_once(fl, be):
    """Two contexts on one device, each in a thread of its own, give what each gives alone."""
    import threading
    results, errors = {}, []

    def work(name, rounds, seed):
        try:
            b = fl.Backend(0)
            rng = np.random.default_rng(seed)
            rows, E, k, H, I = (300, 8, 2, 128, 192) if seed else (20, 16, 4, 192, 128)
            t = {n: tensor(fl, b, rng.standard_normal(s) * f, "bf16") for n, s, f in (
                ("logits", (rows, E), 1.0), ("x", (rows, H), 1.0), ("up", (E * H, 2 * I), 0.1), ("down", (E * I, H), 0.1))}
            t["norm"] = fl.BlockNorm(pre=fl.NORM_LAYER, eps=1e-5, residual=t["x"])
            r = b.routing(rows, E, k)
            bufs = [b.new_tensor(n, m, None, fl.BF16) for n, m in ((rows * k, I), (rows * k, H), (rows, H))]
            for _ in range(rounds):
                block(b, fl, r, t, *bufs, 4)
            results[name] = bufs[2].to_host()
            b.synchronize()
            del r, t, bufs
            b.close()
        except Exception as e:  # seen by the test's own thread
            errors.append(e)

    for seed in (0, 1):
        work(("alone", seed), 1, seed)
    threads = [threading.Thread(target=work, args=(("both", seed), 200, seed)) for seed in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for seed in (0, 1):
        assert (results["both", seed] == results["alone", seed]).all()


def test_calls_are_repeatable(fl, be):
    """The same bits from call to call, between other calls of other sizes."""
    rng = np.random.default_rng(8)
    out = []
    for n in (700, 3, 700):
        z = np.random.default_rng(n).standard_normal((n, 32))
        x = np.random.default_rng(n + 1).standard_normal((n, 128))
        w = np.random.default_rng(2).standard_normal((32 * 128, 256)) * 0.1
        r = be.routing(1000, 32, 4)
        r.route(tensor(fl, be, z, "bf16"))
        y = r.linear(tensor(fl, be, x, "bf16"), tensor(fl, be, w, "bf16"), None, 4)
        out.append((r.read(), y.to_host()))
    for key in out[0][0]:
        assert (out[0][0][key] == out[2][0][key]).all()
    assert (out[0][1] == out[2][1]).all()


# ---------------------------------------------------------------- refusals
def refuses(fl, be, call, text):
    with pytest.raises(fl.FletcherError) as e:
        call()
    assert text in str(e.value), str(e.value)


def test_refusals(fl, be):
    L = fl.lib()
    new = lambda r, c, dt="bf16": be.new_tensor(r, c, None, fl.DTYPES[dt])  # noqa: E731
    for rows, experts, k in ((-1, 8, 2), (4, 0, 1), (4, 257, 1), (4, 8, 0), (4, 8, 9), (4, 64, 17), ((1 << 29) + 1, 8, 2)):
        refuses(fl, be, lambda: be.routing(rows, experts, k), "Routing")
    r = be.routing(8, 4, 2)
    refuses(fl, be, lambda: r.linear(new(8, 16), new(64, 16)), "nothing routed")
    refuses(fl, be, lambda: r.combine(new(16, 16), out=new(8, 16)), "nothing routed")
    refuses(fl, be, lambda: r.read(), "nothing routed")
    refuses(fl, be, lambda: r.route(new(9, 4)), "rows outside")
    refuses(fl, be, lambda: r.route(new(8, 5)), "columns")
    refuses(fl, be, lambda: r.route(new(8, 4), 7), "scoring")
    refuses(fl, be, lambda: r.assign(np.full((8, 2), 4)), "outside")
    refuses(fl, be, lambda: r.assign(np.full((8, 2), -2)), "outside")
    refuses(fl, be, lambda: r.assign(np.zeros((9, 2))), "rows outside")
    r.route(new(8, 4))
    x, w, y = new(8, 16), new(64, 32), new(16, 32)
    refuses(fl, be, lambda: r.linear(new(7, 16), w, out=y), "input must hold")
    refuses(fl, be, lambda: r.linear(new(15, 16), w, grouped_input=True, out=y), "input must hold")
    refuses(fl, be, lambda: r.linear(x, w, out=new(15, 32)), "result must hold")
    refuses(fl, be, lambda: r.linear(x, w, new(3, 32), out=y), "bias must hold")
    refuses(fl, be, lambda: r.linear(x, w, out=new(16, 32, "f16")), "dtype")
    refuses(fl, be, lambda: r.linear(x, w, None, fl.ACT_SOFTMAX, out=y), "activation")
    refuses(fl, be, lambda: r.linear(x, new(64, 33), None, fl.ACT_SWIGLU, out=new(16, 33)), "even")
    refuses(fl, be, lambda: r.linear(new(16, 16), new(64, 16), grouped_input=True, out=new(2, 2)), "result must hold")
    g = new(16, 16)
    refuses(fl, be, lambda: r.linear(g, new(64, 16), grouped_input=True, out=g), "overlaps")
    assert L.Cuda_Linear_Grouped(r.h, x.buf, 2, 16, w.buf, 32, None, y.buf, 0) == 1
    assert L.Cuda_Linear_Grouped(r.h, x.buf, 0, 0, w.buf, 32, None, y.buf, 0) == 1
    assert L.Cuda_Linear_Grouped(r.h, x.buf, 0, 1 << 40, w.buf, 32, None, y.buf, 0) == 1
    assert L.Cuda_Linear_Grouped(r.h, None, 0, 16, w.buf, 32, None, y.buf, 0) == 1
    assert L.Cuda_Linear_Grouped(None, x.buf, 0, 16, w.buf, 32, None, y.buf, 0) == 1
    refuses(fl, be, lambda: r.combine(g, out=g), "overlaps")
    refuses(fl, be, lambda: r.combine(g, out=new(8, 16, "f16")), "dtype")
    refuses(fl, be, lambda: new(8, 16, "f32").block_norm(fl.BlockNorm(), out=new(8, 16)), "dtype")
    refuses(fl, be, lambda: r.combine(g, out=new(7, 16)), "outputs must be")
    refuses(fl, be, lambda: r.combine(new(15, 16), out=new(8, 16)), "input must hold")

    f = lambda c: new(1, c, "f32")  # noqa: E731
    a = new(8, 16)
    bad = [(dict(pre=3), {}, "unknown norm"), (dict(pre=1, eps=-1.0), {}, "eps"), (dict(pre=1, eps=float("nan")), {}, "eps"),
           (dict(pre=1, pre_gamma=new(1, 16)), {}, "f32"), (dict(pre=1, pre_gamma=f(15)), {}, "f32"),
           (dict(pre=2, pre_beta=f(16)), {}, "no beta"), (dict(post_gamma=f(16)), {}, "without its norm"),
           (dict(residual=new(8, 15)), {}, "residual must be"), (dict(residual=new(8, 16, "f16")), {}, "residual must be"),
           (dict(gate=new(2, 16)), {}, "gate_rows"), (dict(gate=new(1, 15)), {}, "gate must be"),
           (dict(pre=1), dict(out=new(8, 16)), "exactly when"), (dict(), dict(out_norm=new(8, 16)), "exactly when"),
           (dict(pre=1), dict(out=a, out_norm=a), "outputs overlap"), (dict(), dict(out=new(7, 16)), "outputs must be")]
    for kw, outs, text in bad:
        refuses(fl, be, lambda: new(8, 16).block_norm(fl.BlockNorm(**kw), **outs), text)
    gate = new(1, 16)
    refuses(fl, be, lambda: new(1, 16).block_norm(fl.BlockNorm(gate=new(1, 16, "f32"))), "gate must be")
    wide = new(16, 16)
    part = be.wrap(wide.ptr() + 32, 8, 16, fl.BF16)
    refuses(fl, be, lambda: be.wrap(wide.ptr(), 8, 16, fl.BF16).block_norm(fl.BlockNorm(), out=part), "overlaps")
    assert L.Cuda_BlockNorm(be.ctx, a.buf, 8, 16, None, a.buf, None) == 1
    assert L.Cuda_BlockNorm(be.ctx, a.buf, 8, 0, fl.BlockNorm()._p, a.buf, None) == 1
    assert L.Cuda_BlockNorm(be.ctx, a.buf, -1, 16, fl.BlockNorm()._p, a.buf, None) == 1
    refuses(fl, be, lambda: new(2, 49153, "f32").block_norm(fl.BlockNorm()), "columns outside")

    refuses(fl, be, lambda: be.wrap(0, 2, 2, fl.F32), "device memory")
    host = np.zeros(16, np.float32)
    refuses(fl, be, lambda: be.wrap(host.ctypes.data, 2, 2, fl.F32), "device memory")
    refuses(fl, be, lambda: be.wrap(wide.ptr() + 16, 2, 2, fl.BF16), "aligned")
    full = be.routing(8, 4, 4)
    own = be.wrap(full.device_pointers()["weights"], 8, 4, fl.F32)
    refuses(fl, be, lambda: full.route(own), "overlap")
    refuses(fl, be, lambda: be.wrap(wide.ptr(), -1, 2, fl.BF16), "shape")
    refuses(fl, be, lambda: be.wrap(wide.ptr(), 2, 2, 3), "dtype")
    be.synchronize()


def test_wrapped_weight_follows_its_memory(fl, be):
    """Linear on a wrapped weight uses what the memory holds now, not an earlier layout of it."""
    import torch
    w = torch.ones(64, 128, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    t = be.wrap(w.data_ptr(), 64, 128, fl.BF16)
    x = tensor(fl, be, np.ones((4, 64)), "bf16")
    assert (x.linear(x, t, None).to_host() == 64).all()
    w.fill_(2.0)
    torch.cuda.synchronize()
    assert (x.linear(x, t, None).to_host() == 128).all()
    y = be.new_tensor(4, 128, None, fl.BF16)
    call = lambda: be.check(fl.lib().Cuda_Linear_Fused(be.ctx, x.buf, 4, 64, t.buf, 128, None, y.buf, 0))  # noqa: E731
    g, stream = torch.cuda.CUDAGraph(), torch.cuda.ExternalStream(be.stream())
    call()
    be.synchronize()
    with torch.cuda.graph(g, stream=stream):
        call()
    w.fill_(3.0)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        g.replay()
    be.synchronize()
    assert (y.to_host() == 192).all()
