"""The transformer blocks without a GPU: rotary frequencies, and the calls
that lwm_rotary_device, lwm_cache_*_device and lwm_gated_norm_device refuse
before any device work."""
import ctypes as C
import math

import pytest

import lewm_b200 as L

torch = pytest.importorskip("torch")

P = 1 << 20  # an aligned address that is never read: every call below is refused first


def _message():
    return L.lib.lwm_last_error().decode()


@pytest.mark.parametrize("dims,bases", [([64], [10000.0]), ([32, 16, 16], [10000.0, 100.0, 100.0]),
                                        ([16, 16], [0.5, 1e6]), ([128], [500000.0])])
def test_rotary_frequencies_are_exact_fractions_of_a_turn(dims, bases):
    r = L.Rotary.make(dims, bases)
    p = 0
    for n, base in zip(dims, bases):
        for i in range(n // 2):
            want = base ** (-2.0 * i / n) / (2.0 * math.pi) % 1.0
            got = int(r.turn[p]) / 2.0 ** 64
            # the double has 53 bits, the table 64
            assert abs(got - want) <= 4 * 2.0 ** -53 * max(1.0, base ** (-2.0 * i / n)), (n, i)
            p += 1


@pytest.mark.parametrize("dims,bases,interleaved,message", [
    ([], [], False, "rotary axes must be 1 to 4"),
    ([16] * 5, [1e4] * 5, False, "rotary axes must be 1 to 4"),
    ([24], [1e4], False, "rotary dims[0]=24 must be a positive multiple of 16"),
    ([16, 0], [1e4] * 2, False, "rotary dims[1]=0 must be a positive multiple of 16"),
    ([12], [1e4], True, "rotary dims[0]=12 must be a positive multiple of 8"),
    ([64, 64, 16], [1e4] * 3, False, "rotary dims exceed 128 channels"),
    ([64], [0.0], False, "rotary base 0 must be finite and greater than zero"),
    ([64], [float("nan")], False, "rotary base 0 must be finite and greater than zero"),
    ([64], [1e4, 1e4], False, "rotary has 1 axes and 2 bases"),
])
def test_rotary_refusals(dims, bases, interleaved, message):
    with pytest.raises(L.LwmError) as e:
        L.Rotary.make(dims, bases, interleaved)
    assert e.value.message == message


def _rotary_args(**kw):
    d = dict(x=P, out=P, x_token_stride=128, x_head_stride=64, out_token_stride=128, out_head_stride=64, positions=P,
             tokens=3, heads=2, head_dim=64, dtype=1, inverse=0)
    d.update(kw)
    return L._RotaryArgs(**d)


@pytest.mark.parametrize("kw,message", [
    (dict(head_dim=32), "rotary dims (64 channels) exceed head_dim 32"),
    (dict(head_dim=264), "rotary head_dim 264 must be a multiple of 8 up to 256"),
    (dict(head_dim=68), "rotary head_dim 68 must be a multiple of 8 up to 256"),
    (dict(heads=0), "rotary heads must be greater than zero"),
    (dict(dtype=3), "unknown dtype"),
    (dict(tokens=1 << 31), "rotary tokens or heads out of range"),
    (dict(x=P + 8), "x is not 16-byte aligned"),
    (dict(out=None), "out is null"),
    (dict(x_head_stride=68), "x strides must be multiples of 8 elements"),
    (dict(positions=None), "positions are null"),
    (dict(positions=P + 1), "positions are not 4-byte aligned"),
    (dict(), "null context"),
])
def test_rotary_call_refusals(kw, message):
    r = L.Rotary.make([64], [1e4])
    assert L.lib.lwm_rotary_device(None, C.byref(r), C.byref(_rotary_args(**kw))) != 0
    assert _message() == message


def _cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, pages=4, kv_heads=2, page_tokens=16, head_dim=64, dtype=1, storage=1)
    d.update(kw)
    return L._PagedCache(**d)


def _batch(**kw):
    d = dict(table=P, lengths=P, starts=P, sequences=2, table_stride=2, tokens=6, max_new=4, max_length=0)
    d.update(kw)
    return L._CacheBatch(**d)


def _append(**kw):
    d = dict(q=P, q_out=P, k=P, v=P, q_token_stride=256, q_head_stride=64, q_out_token_stride=256,
             q_out_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64,
             positions=None, heads=4)
    d.update(kw)
    return L._CacheAppendArgs(**d)


def _gather(**kw):
    d = dict(k_out=P, v_out=P, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64)
    d.update(kw)
    return L._CacheGatherArgs(**d)


def _attention(**kw):
    d = dict(q=P, out=P, q_token_stride=256, q_head_stride=64, out_token_stride=256, out_head_stride=64, heads=4,
             scale=0.125, causal=1, window=0, sinks=0, frame_tokens=1)
    d.update(kw)
    return L._CacheAttentionArgs(**d)


CACHE_REFUSALS = [
    (dict(dtype=0), {}, "cache dtype must be bf16 or f16"),
    (dict(storage=2), {}, "unknown cache storage"),
    (dict(head_dim=96), {}, "cache head_dim 96 is not 32, 64 or 128"),
    (dict(page_tokens=24), {}, "cache page_tokens 24 is not 16, 32, 64 or 128"),
    (dict(kv_heads=0), {}, "cache kv_heads must be greater than zero"),
    (dict(pages=1 << 31), {}, "cache pages or kv_heads out of range"),
    (dict(pages=0), {}, "cache pages must be greater than zero"),
    (dict(v=None), {}, "cache pools are null"),
    (dict(k=P + 4), {}, "cache pools are not 16-byte aligned"),
    (dict(k_scale=None), {}, "an 8-bit cache needs its scales"),
    (dict(v_scale=P + 2), {}, "cache scales are not 4-byte aligned"),
    ({}, dict(table=None), "batch arrays are null"),
    ({}, dict(lengths=P + 1), "batch arrays are not 4-byte aligned"),
    ({}, dict(table_stride=0), "batch table_stride must be greater than zero"),
    ({}, dict(max_new=7), "batch sizes out of range (max_new 7, tokens 6)"),
    ({}, {}, "null context"),
    ({}, dict(sequences=0, tokens=0, max_new=0), "null context"),
]


@pytest.mark.parametrize("cache,batch,message", CACHE_REFUSALS)
@pytest.mark.parametrize("call", ["append", "gather", "attention"])
def test_cache_refusals(call, cache, batch, message):
    c, b = _cache(**cache), _batch(**batch)
    if call == "append":
        status = L.lib.lwm_cache_append_device(None, C.byref(c), C.byref(b), None, C.byref(_append()))
    elif call == "gather":
        status = L.lib.lwm_cache_gather_device(None, C.byref(c), C.byref(b), C.byref(_gather()))
    else:
        status = L.lib.lwm_cache_attention_device(None, C.byref(c), C.byref(b), C.byref(_attention()))
    assert status != 0 and _message() == message


@pytest.mark.parametrize("kw,message", [
    (dict(heads=0), "query heads must be greater than zero"),
    (dict(k=None), "k is null"),
    (dict(v=P + 2), "v is not 16-byte aligned"),
    (dict(k_token_stride=100), "k strides must be multiples of 8 elements"),
    (dict(q_out=None), "q_out is null"),
    (dict(positions=P + 2), "positions are not 4-byte aligned"),
    (dict(q=None, q_out=None, heads=0), "null context"),
])
def test_append_refusals(kw, message):
    status = L.lib.lwm_cache_append_device(None, C.byref(_cache()), C.byref(_batch()), None, C.byref(_append(**kw)))
    assert status != 0 and _message() == message


def test_append_refuses_a_rotary_wider_than_the_head():
    r = L.Rotary.make([64, 16], [1e4] * 2)
    status = L.lib.lwm_cache_append_device(None, C.byref(_cache()), C.byref(_batch()), C.byref(r), C.byref(_append()))
    assert status != 0 and _message() == "rotary dims (80 channels) exceed head_dim 64"


@pytest.mark.parametrize("kw,batch,message", [
    (dict(heads=3), {}, "query heads 3 must be a positive multiple of kv_heads 2"),
    (dict(heads=0), {}, "query heads 0 must be a positive multiple of kv_heads 2"),
    (dict(scale=float("inf")), {}, "attention scale must be finite"),
    (dict(frame_tokens=(1 << 30) + 1), {}, "frame_tokens out of range"),
    (dict(q=None), {}, "q is null"),
    (dict(out=P + 8), {}, "out is not 16-byte aligned"),
    (dict(out_token_stride=12), {}, "out strides must be multiples of 8 elements"),
    (dict(), dict(tokens=0x7fffffff, max_new=0x7fffffff), "batch is too large for one call"),
])
def test_attention_refusals(kw, batch, message):
    status = L.lib.lwm_cache_attention_device(None, C.byref(_cache()), C.byref(_batch(**batch)),
                                              C.byref(_attention(**kw)))
    assert status != 0 and _message() == message


def _norm(**kw):
    d = dict(x=P, y=P, x_out=P, h=P, x_stride=192, y_stride=192, x_out_stride=192, h_stride=192, rows=5, width=192,
             residual_dtype=0, dtype=1, cond_dtype=0, gate=P, shift=None, scale=None, cond_stride=192,
             rows_per_cond=1, residual_scale=None, post_kind=2, pre_kind=1, post_eps=1e-6, pre_eps=1e-6, out_eps=1e-5)
    d.update(kw)
    return L._GatedNormArgs(**d)


@pytest.mark.parametrize("kw,message", [
    (dict(dtype=4), "unknown dtype"),
    (dict(cond_dtype=-1), "unknown conditioning dtype"),
    (dict(width=0), "gated norm width 0 must be 1 to 8192"),
    (dict(width=8193), "gated norm width 8193 must be 1 to 8192"),
    (dict(rows=1 << 31), "gated norm rows out of range"),
    (dict(pre_kind=0), "gated norm kinds are layer, rms or none"),
    (dict(pre_eps=-1.0), "gated norm eps must be finite and non-negative"),
    (dict(post_kind=3, post_eps=float("nan")), "gated norm eps must be finite and non-negative"),
    (dict(out_bias=P), "out_bias needs out_weight"),
    (dict(rows_per_cond=0), "rows_per_cond must be greater than zero"),
    (dict(x_out=None, h=None), "gated norm has no output"),
    (dict(x=None), "x is null"),
    (dict(x=P + 2), "gated norm tensors must be aligned to their element size"),
    (dict(pre_weight=P + 1), "gated norm weights must be aligned to 4 bytes"),
    (dict(), "null context"),
    (dict(rows=0), "null context"),
    (dict(rows=0, x=None, y=None, x_out=None, h=None), "null context"),
])
def test_gated_norm_refusals(kw, message):
    assert L.lib.lwm_gated_norm_device(None, C.byref(_norm(**kw))) != 0
    assert _message() == message


def test_python_checks_name_the_tensor():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    cache = L.PagedCache(k, k.clone())
    assert (cache.pages, cache.kv_heads, cache.page_tokens, cache.head_dim) == (4, 2, 16, 64)
    with pytest.raises(L.LwmError, match="needs k_scale"):
        L.PagedCache(k.to(torch.float8_e4m3fn), k.to(torch.float8_e4m3fn))
    with pytest.raises(L.LwmError, match="must be two"):
        L.PagedCache(k, k[:, :1])
    with pytest.raises(L.LwmError, match="contiguous"):
        L.PagedCache(k.transpose(1, 2), k.transpose(1, 2))
    with pytest.raises(L.LwmError, match="bfloat16 or float16"):
        L.PagedCache(k.float(), k.float())
    table = torch.zeros(2, 3, dtype=torch.int32)
    starts, lengths = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    L.CacheBatch(table, starts, lengths, 0)
    with pytest.raises(L.LwmError, match="starts must be"):
        L.CacheBatch(table, lengths, lengths, 0)
    with pytest.raises(L.LwmError, match="page table must be"):
        L.CacheBatch(table[:, :2], starts, lengths, 0)
    with pytest.raises(L.LwmError, match="lengths must be"):
        L.CacheBatch(table, starts, lengths.long(), 0)
    with pytest.raises(L.LwmError, match="max_new must be 0 to"):
        L.CacheBatch(table, starts, lengths, 4, max_new=-1)
    with pytest.raises(L.LwmError, match="max_length must be 0 to"):
        L.CacheBatch(table, starts, lengths, 4, max_length=1 << 32)
    with pytest.raises(L.LwmError, match="kinds"):
        L.GatedNorm(pre="batch")
    with pytest.raises(L.LwmError, match="float32"):
        L.GatedNorm(pre_weight=torch.ones(8, dtype=torch.bfloat16))
    with pytest.raises(L.LwmError, match="width or device"):
        L.GatedNorm(pre_weight=torch.ones(8), pre_bias=torch.ones(9))
    assert L.GatedNorm(pre_weight=torch.ones(8)).width == 8


def _huge(*shape, dtype=torch.bfloat16):
    """A tensor of any shape without memory; its device counts as -1, which is what the context below says."""
    return torch.empty(shape, device="meta", dtype=dtype)


class _NoContext:
    device, handle = -1, None


TOO_MANY = (1 << 32) + 1  # one, when cut to 32 bits


@pytest.mark.parametrize("rows_per_cond", [TOO_MANY, 1 << 32, 1 << 63, -1, 0])
def test_rows_per_cond_is_not_cut_to_32_bits(rows_per_cond):
    """Cut, it would be 1, and row r would read conditioning row r of a table with one row."""
    x = torch.zeros(4, 8)
    with pytest.raises(L.LwmError, match="rows_per_cond must be 0 to" if rows_per_cond else "gate must be"):
        L.gated_norm_device(_NoContext, L.GatedNorm(), x, h=x, gate=torch.zeros(1, 8), rows_per_cond=rows_per_cond)


def test_sizes_are_not_cut_to_32_bits():
    r, n = L.Rotary.make([64], [1e4]), TOO_MANY
    cache = L.PagedCache(_huge(4, 2, 16, 64), _huge(4, 2, 16, 64))
    i32 = torch.int32
    batch = L.CacheBatch(torch.zeros(1, 2, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32), 1)
    pos, q, kv, x = _huge(1, 1, dtype=i32), _huge(1, n, 64), _huge(1, 2, 64), _huge(n, 1, 64)
    for name, call in (
            ("x", lambda: L.rotary_device(_NoContext, r, x, x, _huge(n, 1, dtype=i32))),
            ("x", lambda: L.rotary_device(_NoContext, r, q, q, pos)),
            ("x", lambda: L.rotary_device(_NoContext, r, _huge(1, 1, n), _huge(1, 1, n), pos)),
            ("q", lambda: L.cache_append_device(_NoContext, cache, batch, kv, kv, q=q, q_out=q)),
            ("q", lambda: L.cache_attention_device(_NoContext, cache, batch, q, q)),
            ("x", lambda: L.gated_norm_device(_NoContext, L.GatedNorm(), x[:, 0], h=x[:, 0])),
            ("x", lambda: L.gated_norm_device(_NoContext, L.GatedNorm(), q[:, :, 0], h=q[:, :, 0])),
            ("page table", lambda: L.CacheBatch(_huge(n, 2, dtype=i32), _huge(n + 1, dtype=i32), _huge(n, dtype=i32), 1)),
            ("page table", lambda: L.CacheBatch(_huge(1, n, dtype=i32), _huge(2, dtype=i32), _huge(1, dtype=i32), 1))):
        with pytest.raises(L.LwmError, match=f"{name} must have sizes below"):
            call()


def test_append_refuses_an_output_without_its_queries():
    status = L.lib.lwm_cache_append_device(None, C.byref(_cache()), C.byref(_batch()), None, C.byref(_append(q=None)))
    assert status != 0 and _message() == "q_out needs q"
    cache = L.PagedCache(_huge(4, 2, 16, 64), _huge(4, 2, 16, 64))
    i32 = torch.int32
    batch = L.CacheBatch(torch.zeros(1, 2, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32), 1)
    with pytest.raises(L.LwmError, match="q_out needs q"):
        L.cache_append_device(_NoContext, cache, batch, _huge(1, 2, 64), _huge(1, 2, 64), q_out=_huge(1, 4, 64))
