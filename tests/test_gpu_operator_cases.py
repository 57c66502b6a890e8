"""GPU test of how the measured cases of the expert operators (perf/operators.py) call the framework."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


@pytest.fixture(scope="module")
def cases():
    import torch

    import build
    build.build()
    spec = importlib.util.spec_from_file_location("operator_cases", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    before = torch.cuda.current_stream()
    m.own = True
    yield m
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)


@pytest.mark.parametrize("name,changed", [("norms_one_row", "y"), ("route_one_row", "logits"), ("up_few_rows", "x"),
                                          ("combine_query", "residual"), ("experts_batch", "x")])
def test_calls_are_in_order_with_torch(cases, name, changed):
    """An input that torch is still to write is written before the call reads it, and torch reads the output
    after the call has: nothing waits on the host in between."""
    import torch
    case = next(c for c in cases.listed() if c["name"] == name)
    state, other = cases.prepare(case, 1), cases.prepare(case, 2)
    cases.run(state), cases.run(other)
    torch.cuda.synchronize()
    a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    for _ in range(20):  # some 15 ms of work in front of the copy
        a = a @ a * 1e-2
    state[changed].copy_(other[changed])
    got = cases.run(state)
    got = [g.clone() for g in (got if isinstance(got, tuple) else (got,))]
    torch.cuda.synchronize()
    want = cases.run(state)
    torch.cuda.synchronize()
    for g, w in zip(got, want if isinstance(want, tuple) else (want,)):
        assert torch.equal(g, w)
