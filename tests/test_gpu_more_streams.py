"""Shared-prefix attention, linear attention and token sampling as a program
on torch's stream calls them: the calls run on the context's stream, ordered
after the inputs and before the reader."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ATTENTION = dict(op="shared", groups=2, candidates=60, prefix=3000, tail=20, new=1, heads=8, kv_heads=8, dim=64, page=16,
                 dtype="bf16", storage="same", window=0, sinks=0, frame=1)
LINEAR = dict(op="linear", sequences=20, new=1, heads=8, kv_heads=8, dim=64, dtype="bf16", fork=False)
CASES = {"shared": ATTENTION, "shared, few rows": dict(ATTENTION, groups=1, candidates=3, prefix=50),
         "shared, long tails": dict(ATTENTION, tail=400), "linear": LINEAR,
         "linear, chunks": dict(LINEAR, new=300, dtype="f16"), "linear, histories": dict(LINEAR, new=500, dim=128),
         "linear, cut along time": dict(LINEAR, sequences=1, new=6000),
         "draw": dict(op="draw", rows=64, vocab=5000, dtype="f32", temperature=0.8, top_k=0, top_p=0.9, min_p=0.0)}
INPUT = dict(shared="q", linear="v", draw="logits")


@pytest.fixture(scope="module")
def operators():
    spec = importlib.util.spec_from_file_location("more_operator_cases", os.path.join(ROOT, "perf", "more_operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    with torch.cuda.stream(torch.cuda.current_stream()):  # it makes its context's stream the current one
        yield m


def tensors(out):
    return [t.clone() for t in (out.values() if isinstance(out, dict) else [out])]


def late_input(state):
    return state["qkv"][:, -1] if state["case"]["op"] == "linear" else state[INPUT[state["case"]["op"]]]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("on", ["context", "default", "side"])
def test_calls_are_ordered_with_torchs_stream(operators, case, on):
    """An input that is written late is the one that is used, and its result is what torch reads next; no waiting
    in between."""
    state = operators.prepare(CASES[case], 1)
    operators.run(state)
    torch.cuda.synchronize()
    into = late_input(state)
    late = late_input(operators.prepare(CASES[case], 2)).clone()
    last = torch.zeros_like(late)
    torch.cuda.synchronize()
    stream = {"context": torch.cuda.current_stream, "default": torch.cuda.default_stream, "side": torch.cuda.Stream}[on]()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)  # some 10 ms
        into.copy_(late)
        got = tensors(operators.run(state))
        torch.cuda._sleep(20_000_000)
        into.copy_(last)
        operators.run(state)
    torch.cuda.synchronize()
    into.copy_(late)
    torch.cuda.synchronize()
    want = operators.run(state)
    torch.cuda.synchronize()
    for a, b in zip(got, tensors(want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_two_contexts_at_once(operators, ctx, case):
    """Calls of two contexts in flight together, each with a workspace of its own: the same results as one by one."""
    import lewm_b200 as L
    first, second = operators.prepare(CASES[case], 3), operators.prepare(CASES[case], 4)
    want = [[t.clone() for t in tensors(operators.run(s))] for s in (first, second)]
    torch.cuda.synchronize()
    other = L.Context(0)
    inputs = [late_input(s).clone() for s in (first, second)]
    for s in (first, second):
        late_input(s).copy_(inputs[0] * 0)
        operators.run(s)
    torch.cuda.synchronize()
    for s, x in zip((first, second), inputs):
        late_input(s).copy_(x)
    torch.cuda.synchronize()
    plans = [s["plan"] for s in (first, second)]
    got = []
    for _ in range(10):
        got = [operators._call(L, c, s, p) for c, s, p in ((ctx, first, plans[0]), (other, second, plans[1]))]
    ctx.synchronize()
    other.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(tensors(a), b):
            assert torch.equal(x, y)
