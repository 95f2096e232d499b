"""The measured cases' calls of the library, used from torch: inputs that torch still writes and results that
torch reads at once, without a synchronisation by the host."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
LONG = 40_000_000  # cycles: some 20 ms, the calls take microseconds


@pytest.fixture
def cases():
    import torch
    spec = importlib.util.spec_from_file_location("operators_under_test", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    with torch.cuda.stream(torch.cuda.current_stream()):  # the current stream is put back at the end
        yield m
        torch.cuda.synchronize()
    m._dev().close()


def test_calls_wait_for_torch_and_torch_for_them(cases):
    import torch
    M = cases
    torch.cuda._sleep(LONG)
    fresh = torch.randn(64, 1024, device="cuda")  # pending work of the stream that torch had before
    s = M.prepare({"op": "norm", "rows": 64, "cols": 1024}, 1)
    s["x"].copy_(fresh)
    first = M.run(s)["h"].clone()
    torch.cuda._sleep(LONG)
    s["x"].zero_()
    second = M.run(s)["h"].clone()  # the input is still to be written, the result to be computed
    torch.cuda.synchronize()
    assert torch.equal(first, fresh + s["res"])
    assert torch.equal(second, s["res"])


def test_passes_of_two_states_that_nothing_waits_between(cases):
    import torch
    M = cases
    case = {"op": "quantize", "rows": 700, "cols": 900, "block": False, "transpose": True}
    a, b = (M.prepare(case, seed) for seed in (1, 2))
    got = []
    for s in (a, b, a):
        torch.cuda._sleep(LONG // 8)
        s["x"].mul_(2.0)
        got.append({n: v.clone() for n, v in M.run(s).items()})
    torch.cuda.synchronize()
    for s, g, scale in ((a, got[0], 0.5), (b, got[1], 1.0), (a, got[2], 1.0)):
        want = M._plain({**s, "x": s["x"] * scale})
        assert torch.equal(g["q"].view(torch.uint8), want["q"].view(torch.uint8))
        assert torch.equal(g["q_scale"], want["q_scale"])
