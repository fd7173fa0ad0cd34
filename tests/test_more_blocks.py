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


def _cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, pages=4, kv_heads=2, page_tokens=16, head_dim=64, dtype=1, storage=1)
    d.update(kw)
    return L._PagedCache(**d)


def _batch(**kw):
    d = dict(table=P, lengths=P, starts=P, sequences=64, table_stride=4000, tokens=64, max_new=1, max_length=0)
    d.update(kw)
    return L._CacheBatch(**d)


def _prefix(**kw):
    d = dict(groups=P, lengths=P, count=1, max_tokens=64, max_length=50000, max_tail=30)
    d.update(kw)
    return L._SharedPrefix(**d)


def _attention(**kw):
    d = dict(q=P, out=P, q_token_stride=256, q_head_stride=64, out_token_stride=256, out_head_stride=64, heads=4,
             scale=0.125, causal=1, window=0, sinks=0, frame_tokens=1)
    d.update(kw)
    return L._CacheAttentionArgs(**d)


def _bytes(cache, batch, prefix, args):
    n = C.c_uint64(99)
    status = L.lib.lwm_cache_attention_shared_workspace(C.byref(cache), C.byref(batch), C.byref(prefix), C.byref(args), C.byref(n))
    return status, n.value


def test_shared_attention_says_what_workspace_it_needs():
    status, n = _bytes(_cache(), _batch(), _prefix(), _attention(q=None, out=None))
    assert status == 0 and n > 0 and n % (64 * 4 * 65 * 4) == 0  # [splits, tokens, heads, head_dim + 1] f32
    for batch, prefix in ((dict(sequences=0, tokens=0, max_new=0), dict(count=0, max_tokens=0)), ({}, dict(count=0)),
                          (dict(sequences=2, tokens=2, table_stride=4), dict(max_tokens=2, max_length=40))):
        assert _bytes(_cache(), _batch(**batch), _prefix(**prefix), _attention()) == (0, 0)


@pytest.mark.parametrize("batch,prefix,args,work,message", [
    ({}, dict(count=65), {}, {}, "groups 65 are more than the sequences"),
    ({}, dict(groups=None), {}, {}, "group arrays are null"),
    ({}, dict(lengths=P + 2), {}, {}, "group arrays are not 4-byte aligned"),
    ({}, dict(max_tokens=65), {}, {}, "max_tokens 65 is above the batch's tokens 64"),
    (dict(max_new=65), {}, {}, {}, "batch sizes out of range (max_new 65, tokens 64)"),
    ({}, {}, dict(heads=3), {}, "query heads 3 must be a positive multiple of kv_heads 2"),
    ({}, {}, dict(q=None), {}, "q is null"),
    ({}, {}, dict(out_head_stride=63), {}, "out strides must be multiples of 8 elements"),
    ({}, {}, {}, dict(workspace=None), "workspace is null"),
    ({}, {}, {}, dict(workspace=P + 8), "workspace is not 16-byte aligned"),
    ({}, {}, {}, {}, "null context"),
])
def test_shared_attention_refusals(batch, prefix, args, work, message):
    c, b, p, a = _cache(), _batch(**batch), _prefix(**prefix), _attention(**args)
    at, size = work.get("workspace", P), work.get("size", 1 << 40)
    assert L.lib.lwm_cache_attention_shared_device(None, C.byref(c), C.byref(b), C.byref(p), C.byref(a), at, size) != 0
    assert _message() == message


def test_shared_attention_refuses_a_small_workspace():
    c, b, p, a = _cache(), _batch(), _prefix(), _attention()
    _, n = _bytes(c, b, p, a)
    assert L.lib.lwm_cache_attention_shared_device(None, C.byref(c), C.byref(b), C.byref(p), C.byref(a), P, n - 1) != 0
    assert _message() == f"workspace has {n - 1} bytes, the call needs {n}"
    assert L.lib.lwm_cache_attention_shared_device(None, C.byref(c), C.byref(b), C.byref(p), C.byref(a), P, n) != 0
    assert _message() == "null context"


def test_null_arguments():
    assert L.lib.lwm_cache_attention_shared_device(None, C.byref(_cache()), C.byref(_batch()), None, C.byref(_attention()), P, 0) != 0
    assert _message() == "null argument"
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
