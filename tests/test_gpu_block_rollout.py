"""A candidate rollout on 8-bit caches, checked at every step: each append's
scales and codes against the keys and values that went in, each attention
against 64 bits over the tokens that the pages then stand for, so that a stale
scale, a wrong window or page shows at once, not only in a score."""
import os

import numpy as np
import pytest

import lewm_b200 as L
from test_gpu_block_scales import tolerance
from test_gpu_blocks import (BF16, F8, WorldModel, attention_64, attention_tolerance, close, gen, ints, mask_of, need_scale,  # noqa: F401
                             on_context_stream, randn, turned)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Mirror:
    """What one pool (keys or values) of an 8-bit cache holds, as far as it has been checked."""

    def __init__(self, pool, scale, exact):
        self.pool, self.scale, self.exact = pool, scale, exact
        self.take()

    def take(self):
        self.codes, self.scales = self.pool.double(), self.scale.clone()

    def appended(self, table, lens, news, x, mag):
        """x [tokens, kv, d] in 64 bits went in (keys: turned, `mag` what their rounding is relative to)."""
        page, t = self.pool.shape[2], 0
        for s, (length, n) in enumerate(zip(lens, news)):
            i = length - n
            while i < length:
                slot, count = i % page, min(page - i % page, length - i)
                p = int(table[s, i // page])
                part, m = x[t:t + count].transpose(0, 1), mag[t:t + count].transpose(0, 1)
                got = self.scale[p]
                for h, top in enumerate(part.abs().amax((1, 2)).tolist()):
                    low = float(self.scales[p, h]) if slot else 0.0
                    allowed = {max(need_scale(top * (1 + e)), low) for e in ((0.0,) if self.exact else (0.0, 2.0 ** -20, -2.0 ** -20))}
                    assert float(got[h]) in allowed, (s, i, h, float(got[h]), allowed)
                y = part / got[:, None, None].double()
                new = self.pool[p, :, slot:slot + count].double()
                # half a step of a code, 2^-10 below the smallest normal; keys were turned in 32 bits
                close(new, y, (y.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * 1.001 + m / got[:, None, None] * 2.0 ** -20)
                if slot:
                    again = self.codes[p, :, :slot] * (self.scales[p] / got)[:, None, None].double()
                    assert torch.equal(self.pool[p, :, :slot].double(), again.float().to(F8).double())
                i, t = i + count, t + count
        written = {int(table[s, j // page]) for s, (length, n) in enumerate(zip(lens, news)) for j in range(length - n, length)}
        rest = torch.tensor([p for p in range(self.pool.shape[0]) if p not in written], device="cuda", dtype=torch.int64)
        assert torch.equal(self.pool[rest].double(), self.codes[rest]) and torch.equal(self.scale[rest], self.scales[rest])
        self.take()

    def dense(self, table, s, length):
        rows = torch.tensor(np.asarray(table[s]), device="cuda", dtype=torch.int64)
        x = self.codes[rows] * self.scales[rows].double()[:, :, None, None]
        each = self.scales[rows].double().repeat_interleave(self.pool.shape[2], 0)
        return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:length], each[:length]


@pytest.mark.parametrize("H,windows", [(21, (16, 2, 1)), (40, (7, 0, 1)), (33, (2, 5, 6)), (31, (0, 0, 1))])
def test_8_bit_rollout_step_by_step(ctx, H, windows):
    m = WorldModel(300)
    B, S, T, A = 2, 5, 4, 2  # vehicles, candidates, horizon, action dims
    d, h, kv, w, page = m.D, m.HEADS, m.KV, m.DIM, m.PAGE
    g = gen(301)
    full, per, n = H // page, -(-(H + T) // page), B * S
    pages = B * per + n * (per - full)
    own = np.arange(B * per).reshape(B, per)
    table = np.zeros((n, per), np.int32)
    table[:, :full] = np.repeat(own[:, :full], S, 0)
    table[:, full:] = B * per + np.arange(n * (per - full)).reshape(n, -1)
    pools, mirrors = [], []
    for _ in range(m.LAYERS):
        k = torch.zeros(pages, kv, page, w, device="cuda").to(F8)
        args = (k, k.clone(), torch.full((pages, kv), 2.0 ** 50, device="cuda"), torch.full((pages, kv), 2.0 ** 50, device="cuda"))
        pools.append((args, L.PagedCache(*args, dtype=BF16)))
        mirrors.append((Mirror(args[0], args[2], False), Mirror(args[1], args[3], True)))
    rotary = L.Rotary.make(m.dims, m.bases)

    def forward(x, actions, pos, where, lens, news):
        rows = x.shape[0]
        starts = np.concatenate([[0], np.cumsum(news)])
        batch = L.CacheBatch(ints(where), ints(starts), ints(lens), rows, max_new=max(news), max_length=H + T)
        u = torch.empty(rows, d, device="cuda", dtype=BF16)
        for i, ly in enumerate(m.layers):
            ada = actions @ ly["ada"]
            L.gated_norm_device(ctx, L.GatedNorm(pre="layer", pre_weight=ly["pre"]), x, h=u, shift=ada[:, d:2 * d],
                                scale=ada[:, 2 * d:])
            qkv = (u @ ly["qkv"]).view(rows, h + 2 * kv, w)
            # sizes that change from step to step: pages keep, raise and restart their scales
            qkv[:, h:] *= 2.0 ** int(torch.randint(-3, 4, (1,), generator=g, device="cuda"))
            before = qkv.clone()
            q, out = qkv[:, :h], torch.full((rows, h, w), 5.0, device="cuda", dtype=BF16)
            L.cache_append_device(ctx, pools[i][1], batch, qkv[:, h:h + kv], qkv[:, h + kv:], rotary=rotary,
                                  positions=pos, q=q, q_out=q)
            L.cache_attention_device(ctx, pools[i][1], batch, q, out, window=windows[0], sinks=windows[1],
                                     frame_tokens=windows[2])
            wk, mk = turned(before[:, h:h + kv], pos, m.dims, m.bases, False)
            mirrors[i][0].appended(where, lens, news, wk, mk)
            mirrors[i][1].appended(where, lens, news, before[:, h + kv:].double(), torch.zeros_like(mk))
            for s, (length, count) in enumerate(zip(lens, news)):
                a, z = int(starts[s]), int(starts[s + 1])
                (k, _), (v, vs) = mirrors[i][0].dense(where, s, length), mirrors[i][1].dense(where, s, length)
                seen = mask_of(length, count, True, *windows)
                parts = attention_64(q[a:z].double(), k, v, seen, w ** -0.5)
                close(out[a:z], parts[0], tolerance(parts, q[a:z].double(), k, vs, seen, w ** -0.5, BF16))
            y = out.view(rows, h * w) @ ly["out"]
            L.gated_norm_device(ctx, L.GatedNorm(post="rms", post_weight=ly["post"]), x, y, x, gate=ada[:, :d])
        return x

    x = randn(g, B * H, d)
    last = forward(x, randn(g, B * H, A), m.positions(range(H), B), own, [H] * B, [H] * B).view(B, H, d)[:, -1]
    if H % page:  # the partly filled page of the history, copied for each candidate with its scales
        for args, pair in zip((a for a, _ in pools), mirrors):
            for t in args:
                flat = t.view(torch.uint8) if t.element_size() == 1 else t
                flat[table[:, full].astype(np.int64)] = flat[np.repeat(own[:, full], S).astype(np.int64)]
            for mirror in pair:
                mirror.take()
    x, acts = last.repeat_interleave(S, 0), randn(g, n, T, A)
    for t in range(T):
        x = x + acts[:, t] @ m.embed
        x = forward(x.clone(), acts[:, t].contiguous(), m.positions([H + t], n), table, [H + t + 1] * n, [1] * n)
    assert torch.isfinite(x).all()


def test_the_guides_example(ctx):
    """The integration guide's program, and its last attention against 64 bits."""
    guide = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    program = [b.split("```")[0] for b in guide.split("```python\n")[1:] if "PagedCache" in b.split("```")[0]]
    assert len(program) == 1
    names = dict(ctx=ctx, L=L)
    exec(program[0], names)
    q, out, dim, S = names["q"], names["out"], names["dim"], names["S"]
    k, v = (p[[0, 1]].double() for p in names["pool"])
    for s in range(S):
        dense = [torch.cat([whole, p[3 + s][None].double()]).transpose(1, 2).reshape(-1, names["kv"], dim)[:41]
                 for whole, p in zip((k, v), names["pool"])]
        parts = attention_64(q[s:s + 1].double(), *dense, mask_of(41, 1, True, 0, 0, 1), dim ** -0.5)
        close(out[s:s + 1], parts[0], attention_tolerance(*parts, dim, BF16, False, 0.0))
