"""The operators' cases as a program on torch's stream calls them: the calls
run on the context's stream, ordered after the inputs and before the reader."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SMALL = [
    dict(op="rotary", tokens=4096, heads=8, dim=64, dtype="bf16", axes=2, interleaved=False, inverse=False),
    dict(op="norm", rows=4096, width=1024, residual="f32", dtype="bf16", cond="bf16", per_cond=7, post="rms", pre="rms",
         gate=True, modulate=True, residual_scale=True, out_norm=False),
    dict(op="attention", sequences=16, new=1, length=3000, prefix=0, heads=8, kv_heads=8, dim=64, page=64, dtype="bf16",
         storage="same", window=0, sinks=0, frame=1),
    dict(op="append", sequences=64, new=30, length=60, heads=8, kv_heads=8, dim=64, page=16, dtype="bf16",
         storage="e4m3", axes=1, interleaved=False),
]
INPUT = dict(rotary="x", norm="y", attention="q", append="qkv")


@pytest.fixture(scope="module")
def operators():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    with torch.cuda.stream(torch.cuda.current_stream()):  # it makes its context's stream the current one
        yield m


def tensors(out):
    return [t.clone() for t in (out.values() if isinstance(out, dict) else [out])]


@pytest.mark.parametrize("case", SMALL, ids=lambda c: c["op"])
@pytest.mark.parametrize("on", ["context", "default", "side"])
def test_calls_are_ordered_with_torchs_stream(operators, case, on):
    """An input that is written late is the one that is used, and its result is what torch reads next; no waiting
    in between."""
    state, name = operators.prepare(case, 1), INPUT[case["op"]]
    operators.run(state)
    torch.cuda.synchronize()
    late = operators.prepare(case, 2)[name]
    last = torch.zeros_like(late)
    torch.cuda.synchronize()
    stream = {"context": torch.cuda.current_stream, "default": torch.cuda.default_stream, "side": torch.cuda.Stream}[on]()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)  # some 10 ms
        state[name].copy_(late)
        got = tensors(operators.run(state))
        torch.cuda._sleep(20_000_000)
        state[name].copy_(last)
        operators.run(state)
    torch.cuda.synchronize()
    state[name].copy_(late)
    torch.cuda.synchronize()
    want = operators.run(state)
    torch.cuda.synchronize()
    for a, b in zip(got, tensors(want)):
        assert torch.equal(a, b)
