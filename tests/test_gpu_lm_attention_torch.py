"""The attention operators used from torch: inputs that torch still writes and results that torch reads at once, without a
synchronisation by the host; a layer's calls one after another."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
LONG = 40_000_000  # cycles: some 20 ms, the calls take microseconds


@pytest.fixture
def cases():
    import torch
    spec = importlib.util.spec_from_file_location("more_operators_under_test", os.path.join(ROOT, "perf", "more_operators.py"))
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
    fresh = torch.randn(64, 4, 128, device="cuda")  # pending work of the stream that torch had before
    s = M.prepare({"op": "heads", "rows": 64, "heads": 4, "dim": 128, "rot": 0, "pairs": False, "norm": False}, 1)
    s["x"].copy_(fresh)
    first = M.run(s)["y"].clone()
    torch.cuda._sleep(LONG)
    s["x"].zero_()
    second = M.run(s)["y"].clone()  # the input is still to be written, the result to be computed
    torch.cuda.synchronize()
    assert torch.equal(first, fresh)  # neither norm nor rotation: bit for bit
    assert not second.any()


@pytest.mark.parametrize("new", [1, 70])
def test_a_write_and_the_attention_that_reads_it(cases, new):
    """Keys and values go into the pages that the next call reads, while torch still writes the projection."""
    import torch
    M = cases
    case = {"op": "attention", "seqs": 3, "new": new, "length": 500, "q_heads": 8, "heads": 2, "dim": 64, "page": 16, "window": 0}
    s = M.prepare(case, 1)
    w = M.prepare({"op": "write", "rows": s["rows"], "q_heads": 8, "heads": 2, "dim": 64, "page": 16, "rot": 64, "pairs": False, "norm": True}, 2)
    at = [length - n + i for n, length in s["sequences"] for i in range(n)]
    seq = [i for i, (n, _) in enumerate(s["sequences"]) for _ in range(n)]
    slot = s["table"][torch.tensor(seq), torch.tensor(at) // 16].cpu() * 16 + torch.tensor(at, dtype=torch.int32) % 16
    w["slot"].copy_(slot)
    w["pos"].copy_(torch.tensor(at, dtype=torch.int32))
    for n in ("k", "k_scale", "v", "v_scale"):
        w[n] = s[n]
    w["cache"], s["q"] = s["cache"], w["q_out"]
    torch.cuda._sleep(LONG)
    w["qkv"].mul_(0.5)
    M.run(w)
    got = {n: t.clone() for n, t in M.run(s).items()}
    torch.cuda.synchronize()
    # the plain form over what the cache holds now: its sums of up to 500 terms in 32 bits, of values below 16
    want = M._plain(s)
    assert (got["out"] - want["out"]).abs().max() <= 2 * 500 * 2.0 ** -24 * 16
    assert (got["lse"] - want["lse"]).abs().max() <= 500 * 2.0 ** -24 * want["lse"].abs().max()
    # and the write's own plain form: the scales of the rows that were written
    page, slot = 16, w["slot"].long()
    v = w["v_in"].abs().amax(-1) / M.E4M3_MAX
    assert ((s["v_scale"][slot // page, :, slot % page] - v).abs() <= 2.0 ** -22 * v).all()
