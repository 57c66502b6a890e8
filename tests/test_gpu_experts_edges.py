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
