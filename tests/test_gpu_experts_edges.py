"""GPU tests of the expert feed-forward operators where calls meet in unusual ways: routings that a
graph has captured or replayed, and the kernels of the largest products."""
import numpy as np
import pytest

from test_gpu_experts import E24, U, be, fl, group_ref, grouped_ref, quantise, refuses, route_ref, run_grouped, tensor  # noqa: F401

pytestmark = pytest.mark.gpu


def graph_of(be, calls):
    import torch
    be.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(be.stream())):
        calls()
    return g


def replay(be, g):
    import torch
    with torch.cuda.stream(torch.cuda.ExternalStream(be.stream())):
        g.replay()
    be.synchronize()


@pytest.mark.parametrize("rows,N,K,dtype", [(2, 136, 64, "bf16"), (20, 136, 64, "bf16"), (60, 136, 64, "f16"), (900, 2080, 64, "bf16"),
                                            (60, 136, 64, "f32"), (300, 70, 33, "bf16")])
def test_rows_of_another_routing_stay_out(fl, be, rows, N, K, dtype):  # noqa: F811
    """The device holds the routing of many rows while the last one called, of few, is only captured:
    products and sums neither read nor write past the few."""
    many, E, k = 2000, 4, 2
    rng = np.random.default_rng(rows)
    z = rng.standard_normal((many, E))
    r = be.routing(many, E, k)
    x, y = np.full((many, K), np.nan), np.full((many * k, N), 7.0)
    x[:rows] = quantise(rng.standard_normal((rows, K)), dtype)
    w = quantise(rng.standard_normal((E * K, N)) / 8, dtype)
    tx, ty, tw = tensor(fl, be, x, dtype), tensor(fl, be, y, dtype), tensor(fl, be, w, dtype)
    few, out = tensor(fl, be, z[:rows], "f32"), be.new_tensor(many, N, np.full((many, N), 7.0), fl.DTYPES[dtype])
    r.route(few)
    r.linear(tx, tw, out=ty)  # the workspace grows outside of the capture
    r.route(tensor(fl, be, z, "f32"))
    g = graph_of(be, lambda: r.route(few))
    ty.copy_from_float32(y)
    r.linear(tx, tw, out=ty)
    got = ty.to_host()
    assert np.isfinite(got).all() and (got[rows * k:] == 7.0).all()
    y[:rows * k], y[rows * k:] = 1.0, np.nan
    ty.copy_from_float32(y)
    r.combine(ty, out=out)
    got = out.to_host()
    assert np.isfinite(got).all() and (got[rows:] == 7.0).all()
    replay(be, g)  # the device holds the few rows' routing
    r.linear(tx, tw, out=ty)
    ids, _ = route_ref(np.float32(z[:rows]), k)
    want, _, _ = grouped_ref(x[:rows], w, None, ids, E, 0, False)
    got = ty.to_host()
    assert (np.abs(got[:rows * k] - want) <= np.abs(want) * U[dtype] * 1.01 + (K + 4) * E24 * 64).all()
    assert np.isnan(got[rows * k:]).all()
    del g


def test_what_cannot_be_captured_is_refused(fl, be):  # noqa: F811
    """Create, Assign and Read fail during a capture, which goes on, and so does the routing."""
    r = be.routing(4, 4, 2)
    z = np.array([[0, 1, 2, 3], [3, 2, 1, 0]], np.float32)
    t = tensor(fl, be, z, "f32")
    r.assign(np.array([[1, 0], [2, 3], [0, 1]]))

    def calls():
        refuses(fl, be, lambda: be.routing(4, 4, 2), "captured")
        refuses(fl, be, lambda: r.assign(np.array([[1, 0]])), "captured")
        refuses(fl, be, lambda: r.read(), "captured")
        r.route(t)

    g = graph_of(be, calls)
    for _ in range(2):
        r.assign(np.array([[0, 1], [2, 3]]))
        assert (r.read()["experts"] == [[0, 1], [2, 3]]).all()
        replay(be, g)
        assert (r.read()["experts"] == [[3, 2], [0, 1]]).all()
    del g


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,experts,k", [(3000, 8, 2), (3000, 8, 8), (5000, 40, 2), (100, 96, 8), (4000, 64, 12)])
def test_routing_weights_are_fp32(fl, be, rows, experts, k, dtype):  # noqa: F811
    """Weights far below the row's largest are as good as it.  Logits are multiples of 1/4, so that their
    differences are exact and an exponential is off by expf's own error alone: one place, 2 u."""
    rng = np.random.default_rng(experts)
    z = np.round(rng.uniform(-16, 16, (rows, experts)) * 4) / 4  # exact in each type: at most 7 significant bits
    t = tensor(fl, be, z, dtype)
    r = be.routing(rows, experts, k)
    for score, normalise in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        r.route(t, ["softmax", "sigmoid"].index(score), normalise, 2.0)
        _, want = route_ref(np.float64(z), k, score, normalise, 2.0)
        one = 2 if score == "softmax" else 4  # exponential; sigmoid also an addition and a division
        if normalise:  # the chosen are added up and divided by
            u = one + (one + k - 1) + 1
        elif score == "softmax":  # so are all, and each chunk of a lane's may scale the sum so far (3: factor, product)
            u = one + (one + experts - 1 + 3 * (experts // 8 + 1)) + 1
        else:
            u = one
        off = np.abs(r.read()["weights"] - want) / want
        assert off.max() <= u * E24 * (1 + 1e-5), (score, normalise, off.max() / E24, u)


# Shapes of the 256-column products: pairs of SMs gated (2 x 776) and not (1552), single SMs gated (2 x 520) and not (1040).
WIDE = [(2100, 3, 1, 64, 1552), (1000, 32, 2, 72, 1040)]


@pytest.mark.parametrize("rows,experts,k,K,N", WIDE)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", [0, 1, 4])
@pytest.mark.parametrize("bias", [True, False])
def test_widest_products(fl, be, rows, experts, k, K, N, act, dtype, bias):  # noqa: F811
    for grouped_input in (False, True):
        for out in (dtype, "f32"):
            run_grouped(fl, be, rows, experts, k, K, N, act, dtype, bias, grouped_input, out=out)


@pytest.mark.parametrize("rows,experts,k,dtype", [(3000, 40, 12, "bf16"), (2500, 64, 16, "f32"), (5000, 17, 2, "bf16"), (9001, 8, 2, "f16"),
                                                  (20000, 8, 8, "f32"), (2100, 256, 16, "f16")])
def test_routing_in_two_launches(fl, be, rows, experts, k, dtype):  # noqa: F811
    """Every count of choices kept and of lanes a row, where one cluster cannot hold the pairs."""
    rng = np.random.default_rng(rows)
    z = quantise(np.round(8 * rng.standard_normal((rows, experts))) / 4, dtype)
    r = be.routing(rows, experts, k)
    for _ in range(2):  # the counts are cleared for the next call
        r.route(tensor(fl, be, z, dtype))
        got = r.read()
        ids, w = route_ref(z, k)
        slots, offsets, _ = group_ref(ids, experts)
        assert (got["experts"] == ids).all() and (got["slots"] == slots).all() and (got["offsets"] == offsets).all()
        assert np.allclose(got["weights"], w, rtol=64 * E24, atol=0)


def test_graph_outlives_a_growing_workspace(fl, be):  # noqa: F811
    """A captured product of token rows replays right after a larger one has outgrown its workspace."""
    rng = np.random.default_rng(5)
    E, k, K, N = 4, 2, 128, 64
    small, large = 100, 3000
    r = be.routing(large, E, k)
    w = quantise(rng.standard_normal((E * K, N)) / 8, "bf16")
    tw, z = tensor(fl, be, w, "bf16"), tensor(fl, be, rng.standard_normal((small, E)), "f32")
    tx, ty = be.new_tensor(small, K, None, fl.BF16), be.new_tensor(small * k, N, None, fl.BF16)

    def calls():
        r.route(z)
        r.linear(tx, tw, out=ty)

    calls()
    g = graph_of(be, calls)
    held = be.vram_usage()[0]
    big, out = tensor(fl, be, rng.standard_normal((large, K)), "bf16"), be.new_tensor(large * k, N, None, fl.BF16)
    r.route(tensor(fl, be, rng.standard_normal((large, E)), "f32"))
    r.linear(big, tw, out=out)
    assert be.vram_usage()[0] >= held + large * k * K * 2 + (large * K + large * k * N) * 2
    for step in range(2):
        x = quantise(rng.standard_normal((small, K)), "bf16")
        tx.copy_from_float32(x)
        big.copy_from_float32(np.zeros((large, K)))
        replay(be, g)
        got = ty.to_host()
        calls()
        assert (ty.to_host() == got).all()
        ids = r.read()["experts"]
        want, tol, _ = grouped_ref(x, w, None, ids, E, 0, False)
        assert (np.abs(got - want) <= np.abs(want) * U["bf16"] * (1 + 1e-6) + tol * 1.01 + 1e-37).all()
    del g


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,experts,K,N,act", [(6, 3, 72, 136, 0), (40, 3, 72, 136, 4), (400, 3, 72, 136, 0), (2100, 3, 72, 1552, 0),
                                                  (2100, 3, 72, 1552, 4), (2000, 32, 72, 1040, 0), (2000, 32, 72, 1040, 4)])
@pytest.mark.parametrize("grouped_input", [False, True])
def test_nonfinite_row_stays_alone(fl, be, rows, experts, K, N, act, dtype, grouped_input):  # noqa: F811
    """A NaN row and an inf row, among finite weights, reach their own slots alone, and an expert's inf and NaN
    weights that expert's slots alone."""
    rng = np.random.default_rng(rows)
    ids = (np.arange(rows) % experts).astype(np.int32)[:, None]
    order = group_ref(ids, experts)[2]
    x = quantise(rng.standard_normal((rows, K)), dtype)
    x[0, :] = np.nan  # of expert 0
    x[experts + 2, 3] = np.inf  # of expert 2
    w = quantise(rng.standard_normal((experts * K, N)) / 8, dtype)
    w[K, 0], w[2 * K - 1, N - 1] = np.inf, np.nan  # expert 1's first and last element
    bad = np.zeros((rows, N), bool)
    bad[0] = bad[experts + 2] = True
    bad[ids[:, 0] == 1, 0] = bad[ids[:, 0] == 1, N - 1] = True
    if act == 4:
        bad = bad[:, :N // 2] | bad[:, N // 2:]
    r = be.routing(rows, experts, 1)
    r.assign(ids)
    y = r.linear(tensor(fl, be, x[order] if grouped_input else x, dtype), tensor(fl, be, w, dtype), None, act, grouped_input).to_host()
    seen = ~np.isfinite(y)
    assert not (seen & ~bad[order]).any()
    must = bad.copy()  # silu(-inf) and 0 * inf aside, what is not finite shows
    if act == 4:
        must[experts + 2] = False
        must[ids[:, 0] == 1, 0] = False
    assert seen[must[order]].all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,experts,k,K,half", [(2, 8, 2, 64, 64), (40, 4, 2, 64, 72), (300, 4, 1, 64, 72), (1000, 32, 2, 72, 520),
                                                   (2100, 3, 1, 64, 776), (300, 3, 1, 65, 66)])
def test_f32_swiglu_of_16_bit_operands(fl, be, rows, experts, k, K, half, dtype):  # noqa: F811
    """An fp32 result is fp32 through the activation.  Each row picks one row of weights, so that gate and up
    are exact; what is off is expf (2 u), an addition, a division and a product (u each)."""
    rng = np.random.default_rng(rows + K)
    ids = np.argsort(rng.random((rows, experts)), 1)[:, :k].astype(np.int32)
    x = np.zeros((rows, K), np.float32)
    x[np.arange(rows), np.arange(rows) % K] = 1.0
    w = np.concatenate([quantise(rng.uniform(-30, 10, (experts * K, half)), dtype), quantise(rng.uniform(1, 2, (experts * K, half)), dtype)], 1)
    r = be.routing(rows, experts, k)
    r.assign(ids)
    got = r.linear(tensor(fl, be, x, dtype), tensor(fl, be, w, dtype), None, fl.ACT_SWIGLU, dtype=fl.F32).to_host()
    order = group_ref(ids, experts)[2]
    picked = w[ids.reshape(-1)[order] * K + (order // k) % K].astype(np.float64)
    want = picked[:, :half] / (1.0 + np.exp(-picked[:, :half])) * picked[:, half:]
    off = np.abs(got - want) / np.maximum(np.abs(want), 1e-30)
    assert off.max() <= 5 * E24 * (1 + 1e-5), off.max() / E24


@pytest.mark.parametrize("rows", [0, 1, 5])
def test_taller_gate(fl, be, rows):  # noqa: F811
    """A gate with more rows than the call has serves like a residual with more rows, in place too."""
    rng = np.random.default_rng(rows)
    y, gate = (rng.standard_normal((n, 24)).astype(np.float32) for n in (rows, 9))
    ty, tg = tensor(fl, be, y, "f32"), tensor(fl, be, gate, "f32")
    got, _ = ty.block_norm(fl.BlockNorm(gate=tg))
    assert (got.to_host() == y * gate[:rows]).all()
    r = be.routing(9, 2, 1)
    r.assign(np.zeros((rows, 1)))
    got, _ = r.combine(ty, fl.BlockNorm(gate=tg))
    assert (got.to_host() == y * gate[:rows]).all()
    ty.block_norm(fl.BlockNorm(gate=tg), out=tg)
    assert (tg.to_host() == np.concatenate([y * gate[:rows], gate[rows:]])).all()
    refuses(fl, be, lambda: tensor(fl, be, np.ones((10, 24)), "f32").block_norm(fl.BlockNorm(gate=tg)), "gate_rows")


def test_other_widths_are_refused(fl, be):  # noqa: F811
    """A tensor that is large enough, but whose rows have another width, is not read or written at the wrong stride."""
    new = lambda r, c: be.new_tensor(r, c, None, fl.BF16)  # noqa: E731
    r = be.routing(8, 4, 2)
    r.route(new(8, 4))
    x, w, g = new(8, 16), new(64, 32), new(16, 32)
    refuses(fl, be, lambda: r.linear(x, w, out=new(16, 40)), "result must hold")
    refuses(fl, be, lambda: r.linear(x, w, None, fl.ACT_SWIGLU, out=new(16, 32)), "result must hold")
    refuses(fl, be, lambda: r.linear(x, w, new(4, 40)), "bias must hold")
    refuses(fl, be, lambda: r.combine(g, out=new(8, 40)), "outputs must be")
    for kw, text in ((dict(residual=new(8, 40)), "residual must be"), (dict(gate=new(8, 40)), "gate must be"), (dict(gate=new(1, 40)), "gate must be")):
        refuses(fl, be, lambda: r.combine(g, fl.BlockNorm(**kw)), text)
        refuses(fl, be, lambda: new(8, 32).block_norm(fl.BlockNorm(**kw)), text)
    refuses(fl, be, lambda: new(8, 32).block_norm(fl.BlockNorm(), out=new(8, 40)), "outputs must be")
    refuses(fl, be, lambda: new(8, 32).block_norm(fl.BlockNorm(pre=1), out_norm=new(8, 40)), "outputs must be")
    assert r.linear(x, w, new(1, 4 * 32), out=new(1, 16 * 32)).dims() == (1, 512)  # flat buffers hold the same rows
    r.combine(g, out=new(1, 8 * 32))
    be.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [127, 128, 129])
@pytest.mark.parametrize("experts,k", [(64, 16), (65, 1), (256, 16), (200, 9), (8, 8), (8, 3), (9, 9)])
def test_routing_between_lane_counts(fl, be, rows, experts, k, dtype):  # noqa: F811
    """One, four and 32 lanes a row, on both sides of where they change."""
    rng = np.random.default_rng(rows + experts)
    z = quantise(np.round(8 * rng.standard_normal((rows, experts))) / 4, dtype)
    r = be.routing(rows, experts, k)
    r.route(tensor(fl, be, z, dtype))
    got = r.read()
    ids, w = route_ref(z, k)
    slots, offsets, _ = group_ref(ids, experts)
    assert (got["experts"] == ids).all() and (got["slots"] == slots).all() and (got["offsets"] == offsets).all()
    assert np.allclose(got["weights"], w, rtol=64 * E24, atol=0)


def test_workspace_bound(fl, be):  # noqa: F811
    """However the needs grow, a routing holds less than four times the largest; the largest first, just that."""
    E, k, K, N = 2, 2, 256, 64
    w = be.new_tensor(E * K, N, None, fl.BF16)
    for needs, most in (((400, 404, 804, 1612), 4), ((1612, 400, 804), 1)):
        r = be.routing(2000, E, k)
        x, y = be.new_tensor(2000, K, None, fl.BF16), be.new_tensor(2000 * k, N, None, fl.BF16)
        before = be.vram_usage()[0]
        for rows in needs:
            r.assign(np.tile([0, 1], (rows, 1)))
            r.linear(x, w, out=y)
        held = be.vram_usage()[0] - before
        assert max(needs) * k * K * 2 <= held <= most * max(needs) * k * K * 2, held
        be.synchronize()
        del r, x, y


def test_weight_read_in_two_shapes(fl, be):  # noqa: F811
    """One weight buffer as (256, 512) and then as (512, 256): the same bytes, but not the same layout."""
    rng = np.random.default_rng(6)
    w = quantise(rng.standard_normal(256 * 512) / 16, "bf16")
    tw = tensor(fl, be, w.reshape(256, 512), "bf16")
    for K in (256, 512, 256):
        x = quantise(rng.standard_normal((40, K)), "bf16")
        N = w.size // K
        ty = be.new_tensor(40, N, None, fl.BF16)
        tx = tensor(fl, be, x, "bf16")  # kept: the call takes its handle
        be.check(fl.lib().Cuda_Linear_Fused(be.ctx, tx.buf, 40, K, tw.buf, N, None, ty.buf, 0))
        want = x.astype(np.float64) @ w.reshape(K, N)
        mag = np.abs(x.astype(np.float64)) @ np.abs(w.reshape(K, N))
        assert (np.abs(ty.to_host() - want) <= np.abs(want) * U["bf16"] * 1.01 + (K + 4) * E24 * mag).all()
