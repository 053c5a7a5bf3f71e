"""The measured calls of the paged cache (perf/operators.py) run in the order of the
caller's stream: inputs that it is still to write are waited for, and what it does with
the results waits for them."""
import importlib.util
import os

import pytest

from tests.conftest import ROOT, step

pytestmark = pytest.mark.gpu


@pytest.fixture
def cases():
    import torch

    spec = importlib.util.spec_from_file_location("paged_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    before = torch.cuda.current_stream()
    yield m
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    if m._engine:
        m._engine[0].Close()
        m._engine.clear()


@pytest.mark.parametrize("own_stream", [False, True])
def test_calls_follow_the_callers_stream(cases, own_stream):
    import torch

    case = {"kind": "attention", "req": 40, "new_lo": 1, "new_hi": 1, "many": 0, "kv_lo": 100, "kv_hi": 4000, "pad": 0, "heads": 16, "kv": 8,
            "dim": 64, "page": 16, "cache": "bf16", "mix": 7}
    x = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    s = cases.prepare(case, 1)
    q = s["q"].clone()
    torch.cuda.synchronize()
    want = cases.run(s)["out"]
    torch.cuda.synchronize()
    want = want.clone()
    s["q"].zero_()
    s["out"].fill_(7.0)
    torch.cuda.synchronize()
    step(f"attention behind slow work of the caller's stream, one of its own: {own_stream}")
    with torch.cuda.stream(torch.cuda.Stream() if own_stream else torch.cuda.current_stream()):
        for _ in range(10):  # milliseconds of work before the queries are there
            x = x @ x
        s["q"].copy_(q)
        got = cases.run(s)["out"].clone()
        torch.cuda.current_stream().synchronize()
    assert want.abs().sum() > 0 and torch.equal(got, want)
