"""The measured calls of the drafted trees and the log probabilities (perf/more_operators.py)
run in the order of the caller's stream, and give what their plain forms give."""
import importlib.util
import os

import pytest

from tests.conftest import ROOT, step

pytestmark = pytest.mark.gpu

CASES = {
    "plan": {"req": 9, "n_lo": 1, "n_hi": 33, "runs": 1, "kv_lo": 50, "kv_hi": 900, "words": 2, "pad": 3, "mix": 4},
    "attention": {"req": 20, "n_lo": 1, "n_hi": 20, "runs": 1, "kv_lo": 100, "kv_hi": 3000, "words": 1, "pad": 2, "heads": 16, "kv": 8, "dim": 64, "page": 16,
                  "cache": "bf16", "mix": 7},
    "logprobs": {"rows": 7, "vocab": 50021, "top": 5, "tokens": 2, "entropy": 1, "logits": "bf16", "allowed": 1.0, "mix": 3},
    "commit": {"req": 9, "n_lo": 4, "n_hi": 20, "runs": 1, "kv_lo": 50, "kv_hi": 900, "words": 1, "pad": 3, "kv": 2, "dim": 64, "page": 8, "cache": "f16",
               "mix": 5},
}


@pytest.fixture
def cases():
    import torch

    spec = importlib.util.spec_from_file_location("tree_cases", os.path.join(ROOT, "perf", "more_operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    before = torch.cuda.current_stream()
    yield m
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    if m._engine:
        m._engine[0].Close()
        m._engine.clear()


def run(m, own, state):
    import torch

    m.own = own
    out = {k: v.clone() for k, v in m.run(state).items()}
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("kind", CASES)
def test_calls_give_what_the_plain_forms_give(cases, kind):
    """Whole numbers and moved keys equal; 16-bit results a rounding of both apart, log
    probabilities some roundings of their sums'."""
    import torch

    case = dict(CASES[kind], kind=kind, name=kind)
    step(f"measured {kind} and its plain form")
    plain = run(cases, False, cases.prepare(case, 1))
    got = run(cases, True, cases.prepare(case, 1))
    assert set(got) == set(plain)
    for k, want in plain.items():
        if kind in ("plan", "commit") or not want.is_floating_point():
            assert torch.equal(got[k].to(want.dtype), want), k
        else:
            d = (got[k].double() - want.double()).abs().max().item()
            # attention: values of size below 8 rounded to bf16 on both sides, and the plain form's
            # probabilities and products in fp32; else: fp32 sums of 50021 terms around ln V < 11
            assert d <= (2 * 2 ** -8 * want.double().abs().max().item() if kind == "attention" else 64 * 2 ** -24 * 16), (k, d)


@pytest.mark.parametrize("own_stream", [False, True])
@pytest.mark.parametrize("kind,name,out", [("attention", "q", "out"), ("logprobs", "logits", "entropy")])
def test_calls_follow_the_callers_stream(cases, kind, name, out, own_stream):
    import torch

    cases.own = True
    x = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    s = cases.prepare(dict(CASES[kind], kind=kind, name=kind), 1)
    real = s[name].clone()
    want = run(cases, True, s)[out]
    if kind == "attention":
        want[-CASES[kind]["pad"]:] = 7.0  # rows that nobody has stay as they were
    s[name].zero_()
    s[out].fill_(7.0)
    torch.cuda.synchronize()
    step(f"{kind} behind slow work of the caller's stream, one of its own: {own_stream}")
    with torch.cuda.stream(torch.cuda.Stream() if own_stream else torch.cuda.current_stream()):
        for _ in range(10):  # milliseconds of work before the inputs are there
            x = x @ x
        s[name].copy_(real)
        got = cases.run(s)[out].clone()
        torch.cuda.current_stream().synchronize()
    assert want.abs().sum() > 0 and torch.equal(got, want)
