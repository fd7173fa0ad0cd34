"""Linear attention, token sampling and shared-prefix attention without a GPU:
the calls that are refused before any device work."""
import ctypes as C

import pytest

import lewm_b200 as L

torch = pytest.importorskip("torch")

P = 1 << 20  # an aligned address that is never read: every call below is refused first
NAN = float("nan")


def _message():
    return L.lib.lwm_last_error().decode()


def _states(**kw):
    d = dict(states=P, starts=P, source=None, target=None, slots=2, heads=4, head_dim=64, sequences=2, tokens=6, max_new=4)
    d.update(kw)
    return L._StateBatch(**d)


def _linear(**kw):
    d = dict(q=P, k=P, v=P, out=P, q_token_stride=256, q_head_stride=64, k_token_stride=128, k_head_stride=64,
             v_token_stride=128, v_head_stride=64, out_token_stride=256, out_head_stride=64, log_decay=P, kv_heads=2,
             dtype=1, scale=0.125)
    d.update(kw)
    return L._LinearAttentionArgs(**d)


@pytest.mark.parametrize("batch,args,message", [
    ({}, dict(dtype=0), "linear attention dtype must be bf16 or f16"),
    (dict(head_dim=96), {}, "state head_dim 96 is not 32, 64 or 128"),
    (dict(heads=0), {}, "state heads must be 1 to 65535"),
    (dict(heads=3), {}, "state heads 3 must be a positive multiple of kv_heads 2"),
    ({}, dict(kv_heads=0), "state heads 4 must be a positive multiple of kv_heads 0"),
    ({}, dict(scale=NAN), "attention scale must be finite"),
    (dict(slots=1 << 31), {}, "state slots out of range"),
    (dict(max_new=7), {}, "batch sizes out of range (max_new 7, tokens 6)"),
    (dict(tokens=1 << 31), {}, f"batch sizes out of range (max_new 4, tokens {1 << 31})"),
    (dict(sequences=1 << 26, heads=4, source=P, target=P), {}, "batch is too large for one call"),
    (dict(states=None), {}, "states are null"),
    (dict(states=P + 8), {}, "states are not 16-byte aligned"),
    (dict(starts=None), {}, "batch arrays are null"),
    (dict(target=P + 1), {}, "batch arrays are not 4-byte aligned"),
    (dict(slots=1), {}, "sequences 2 need as many state slots, or source and target"),
    (dict(slots=1, source=P), {}, "sequences 2 need as many state slots, or source and target"),
    ({}, dict(log_decay=None), "log_decay is null"),
    ({}, dict(log_decay=P + 2), "log_decay is not 4-byte aligned"),
    ({}, dict(q=None), "q is null"),
    ({}, dict(k=P + 2), "k is not 16-byte aligned"),
    ({}, dict(v_head_stride=63), "v strides must be multiples of 8 elements"),
    ({}, dict(out=None), "out is null"),
    ({}, {}, "null context"),
    (dict(slots=1, source=P, target=P), {}, "null context"),
    (dict(sequences=0, states=None, starts=None), {}, "null context"),
])
def test_linear_attention_refusals(batch, args, message):
    assert L.lib.lwm_linear_attention_device(None, C.byref(_states(**batch)), C.byref(_linear(**args))) != 0
    assert _message() == message


def _sample(**kw):
    d = dict(logits=P, stride=100, uniform=P, tokens=P, log_probs=None, temperatures=None, top_ks=None, top_ps=None,
             min_ps=None, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0, rows=3, vocab=100, dtype=1)
    d.update(kw)
    return L._SampleTokensArgs(**d)


@pytest.mark.parametrize("kw,message", [
    (dict(dtype=3), "unknown dtype"),
    (dict(vocab=0), "vocabulary must be greater than zero"),
    (dict(vocab=(1 << 18) + 1), "vocabulary 262145 is above 262144"),
    (dict(rows=1 << 27), "rows out of range"),
    (dict(temperature=-0.5), "temperature must be finite and non-negative"),
    (dict(temperature=NAN), "temperature must be finite and non-negative"),
    (dict(top_p=0.0), "top_p must be above 0 and at most 1"),
    (dict(top_p=1.01), "top_p must be above 0 and at most 1"),
    (dict(top_p=NAN), "top_p must be above 0 and at most 1"),
    (dict(min_p=-0.1), "min_p must be 0 to 1"),
    (dict(min_p=NAN), "min_p must be 0 to 1"),
    (dict(logits=None), "logits are null"),
    (dict(logits=P + 1), "logits must be aligned to their element size"),
    (dict(logits=P + 2, dtype=0), "logits must be aligned to their element size"),
    (dict(uniform=None), "uniform or tokens are null"),
    (dict(tokens=None), "uniform or tokens are null"),
    (dict(log_probs=P + 2), "row arrays must be aligned to 4 bytes"),
    (dict(top_ps=P + 1, top_p=NAN), "row arrays must be aligned to 4 bytes"),
    (dict(temperatures=P, temperature=NAN), "null context"),
    (dict(rows=0, logits=None), "null context"),
    (dict(), "null context"),
])
def test_sampling_refusals(kw, message):
    assert L.lib.lwm_sample_tokens_device(None, C.byref(_sample(**kw))) != 0
    assert _message() == message


def test_null_arguments():
    assert L.lib.lwm_linear_attention_device(None, None, None) != 0 and _message() == "null argument"
    assert L.lib.lwm_sample_tokens_device(None, None) != 0 and _message() == "null argument"


class _Context:
    handle, device = None, 0


def _refused(message, f, *args, **kw):
    with pytest.raises(L.LwmError) as e:
        f(*args, **kw)
    assert e.value.message == message


def test_python_checks_shapes_types_and_devices():
    states, starts = torch.zeros(2, 4, 32, 32), torch.zeros(3, dtype=torch.int32)
    _refused("states must be a [slots, heads, head_dim, head_dim] float32 tensor", L.StateBatch, states[..., :16], starts, 5)
    _refused("states must be a [slots, heads, head_dim, head_dim] float32 tensor", L.StateBatch, states.half(), starts, 5)
    _refused("states must be contiguous", L.StateBatch, states.transpose(0, 1), starts, 5)
    _refused("starts must be [sequences + 1]", L.StateBatch, states, starts[:0], 5)
    _refused("source must be a contiguous int32 tensor [2], got torch.int32 [3]", L.StateBatch, states, starts, 5, source=starts)
    _refused("max_new must be 0 to 2^32 - 1, got -1", L.StateBatch, states, starts, 5, -1)
    b = L.StateBatch(states, starts, 5)
    q = torch.zeros(5, 4, 32, dtype=torch.bfloat16)
    _refused("states must be on cuda:0, got cpu", L.linear_attention_device, _Context, b, q, q, q, q, torch.zeros(4))
    logits, u, tokens = torch.zeros(3, 10), torch.zeros(3), torch.zeros(3, dtype=torch.int32)
    _refused("logits must be [rows, vocab], got [10]", L.sample_tokens_device, _Context, logits[0], u, tokens)
    _refused("logits need contiguous rows", L.sample_tokens_device, _Context, logits.t()[:3], u, tokens)
    _refused("uniform must be a contiguous float32 tensor [3], got torch.float64 [3]", L.sample_tokens_device, _Context,
             logits, u.double(), tokens)
    _refused("uniform must be on cuda:0, got cpu", L.sample_tokens_device, _Context, logits, u, tokens)
