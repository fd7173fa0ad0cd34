"""Candidates of several vehicles drawn token by token, with every operator of
such a rollout: each layer's keys appended to a paged cache, attention that
reads a vehicle's history once for its candidates, linear attention whose
states fork from the vehicle's, and the next token drawn from the logits.
Every step of it is checked against 64 bits on what it read, and a graph of one
step replays to the same rollout."""
import os

import numpy as np
import pytest

import lewm_b200 as L
from test_gpu_blocks import Paged, attention_64, attention_tolerance, close, gen, ints, mask_of, randn
from test_gpu_linear import recurrence, tolerances
from test_gpu_sample import definition

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def on_context_stream(ctx):
    with torch.cuda.stream(ctx.torch_stream()):
        yield
    ctx.synchronize()


class Rollout:
    """A layer of attention, a layer of linear attention and a head, over `vehicles` histories of `history` tokens."""

    HEADS, KV, DIM, D, VOCAB, PAGE = 4, 2, 64, 128, 1000, 16

    def __init__(self, ctx, dtype, codes, vehicles, candidates, history, horizon, window=0, sinks=0):
        self.ctx, self.dtype, self.codes, self.mask = ctx, dtype, codes, dict(window=window, sinks=sinks)
        self.V, self.S, self.H, self.T = vehicles, candidates, history, horizon
        h, kv, w, d, page, n = self.HEADS, self.KV, self.DIM, self.D, self.PAGE, vehicles * candidates
        g = gen(900)
        self.embed = randn(g, self.VOCAB, d, dtype=dtype)
        self.qkv = [randn(g, d, (h + 2 * kv) * w, dtype=dtype) / d ** 0.5 for _ in "ab"]
        self.back = [randn(g, h * w, d, dtype=dtype) / (h * w) ** 0.5 for _ in "ab"]
        self.head = randn(g, d, self.VOCAB, dtype=dtype) / 4
        self.norm = L.GatedNorm(pre="rms")
        self.decay = torch.tensor([-0.02, -0.2, 0.0, -1.0], device="cuda")
        self.rotary = L.Rotary.make([w], 1e4)
        self.c = Paged(901, [history + horizon] * n, page, kv, w, dtype, codes)
        whole = history // page
        for s in range(n):
            self.c.table[s, :whole] = self.c.table[s - s % candidates, :whole]
        self.leads = [v * candidates for v in range(vehicles)]
        self.states = torch.zeros(vehicles + n, h, w, w, device="cuda")
        self.own = ints(np.arange(n) + vehicles)  # slots: the vehicles', then the candidates'
        # what the steps read and move on
        self.tokens, self.lengths, self.source = ints([0] * n), ints([0] * n), ints([0] * n)
        self.uniform, self.score = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        bound = history + horizon
        self.batch = L.CacheBatch(ints(self.c.table), ints(np.arange(n + 1)), self.lengths, n, 1, bound)
        self.prefix = L.SharedPrefix(ints(self.leads + [n]), ints([history] * vehicles), candidates, history, horizon)
        size = L.shared_attention_workspace(self.c.cache, self.batch, self.prefix, h, **self.mask)
        self.shared = size > 0  # the history is read once for its candidates; few of them read it by themselves
        self.work = torch.empty(size, device="cuda", dtype=torch.uint8)
        self.linear = L.StateBatch(self.states, ints(np.arange(n + 1)), n, 1, source=self.source, target=self.own)

    def projected(self, x, i):
        u = torch.empty_like(x)
        L.gated_norm_device(self.ctx, self.norm, x, h=u)
        y = (u @ self.qkv[i]).view(len(x), -1, self.DIM)
        return y[:, :self.HEADS], y[:, self.HEADS:self.HEADS + self.KV], y[:, self.HEADS + self.KV:]

    def observe(self, tokens):
        """The vehicles' histories [vehicles, history]: the cache and the vehicles' states."""
        v, n = self.V, self.V * self.H
        x = self.embed[tokens.flatten()]
        starts = ints(np.arange(v + 1) * self.H)
        q, k, val = self.projected(x, 0)
        out = torch.empty_like(q)
        batch = L.CacheBatch(ints(self.c.table[self.leads]), starts, ints([self.H] * v), n, self.H, self.H)
        L.cache_append_device(self.ctx, self.c.cache, batch, k, val, rotary=self.rotary, q=q, q_out=q)
        L.cache_attention_device(self.ctx, self.c.cache, batch, q, out, **self.mask)
        x = x + out.reshape(n, -1) @ self.back[0]
        q, k, val = self.projected(x, 1)
        out = torch.empty(q.shape, device="cuda", dtype=self.dtype)
        slots = ints(np.arange(v))
        L.linear_attention_device(self.ctx, L.StateBatch(self.states, starts, n, self.H, source=ints([-1] * v), target=slots),
                                  q, k, val, out, self.decay)
        want, mag, after, sizes = recurrence(q, k, val, self.decay, [self.H] * v, torch.zeros_like(self.states[:v]), self.DIM ** -0.5)
        tol, state_tol = tolerances(self.dtype, self.DIM, self.H, self.decay, want, mag, sizes, False)
        close(out, want, tol)
        close(self.states[:v], after, state_tol)
        rest = self.H % self.PAGE
        if rest:  # the page that the history ends in, for each candidate
            at = self.c.table[:, self.H // self.PAGE]
            lead = at[np.repeat(self.leads, self.S)]
            for t in (self.c.k, self.c.v, self.c.ks, self.c.vs):
                if t is not None:
                    flat = t.view(torch.uint8) if t.element_size() == 1 else t
                    flat[at] = flat[lead]

    def start(self, seed):
        g = gen(seed)
        self.tokens.copy_(torch.randint(0, self.VOCAB, self.tokens.shape, generator=g, device="cuda"))
        self.lengths.fill_(self.H + 1)
        self.source.copy_(ints(np.repeat(np.arange(self.V), self.S)))
        self.score.zero_()
        return torch.rand(self.T, len(self.tokens), generator=g, device="cuda")

    def step(self):
        """A token for each candidate; nothing here depends on which step it is."""
        c, n = self.c, len(self.tokens)
        x = self.embed[self.tokens.long()]
        q, k, v = self.projected(x, 0)
        out = torch.empty(q.shape, device="cuda", dtype=self.dtype)
        L.cache_append_device(self.ctx, c.cache, self.batch, k, v, rotary=self.rotary, q=q, q_out=q)
        L.cache_attention_shared_device(self.ctx, c.cache, self.batch, self.prefix, q, out, self.work, **self.mask)
        x = x + out.reshape(n, -1) @ self.back[0]
        lq, lk, lv = self.projected(x, 1)
        lout = torch.empty(lq.shape, device="cuda", dtype=self.dtype)
        L.linear_attention_device(self.ctx, self.linear, lq, lk, lv, lout, self.decay)
        x = x + lout.reshape(n, -1) @ self.back[1]
        logits, logs = x @ self.head, torch.empty_like(self.score)
        drawn = torch.empty_like(self.tokens)
        L.sample_tokens_device(self.ctx, logits, self.uniform, drawn, logs, temperature=0.9, top_k=200, top_p=0.95)
        self.score += logs
        self.tokens.copy_(drawn)
        self.lengths += 1
        self.source.copy_(self.own)
        return dict(q=q, out=out, linear=(lq, lk, lv, lout), logits=logits, logs=logs)

    def rollout(self, seed, step, after=None):
        u, tokens = self.start(seed), []
        for t in range(self.T):
            self.uniform.copy_(u[t])
            before = self.states.clone()
            source = self.source.long()
            got = step()
            tokens.append(self.tokens.clone())
            if after:
                after(t, before[source], got)
        return torch.stack(tokens), self.score.clone(), self.states.clone()

    def check(self, t, states, got):
        """Step t on what it read: the cache as it is, the states before."""
        c, n = self.c, len(self.tokens)
        c.lengths = [self.H + t + 1] * n
        for s in range(n):
            parts = attention_64(got["q"][s:s + 1].double(), c.dense("k", s), c.dense("v", s),
                                 mask_of(self.H + t + 1, 1, True, self.mask["window"], self.mask["sinks"], 1), self.DIM ** -0.5)
            vs = float(c.vs[c.table[s, :-(-c.lengths[s] // c.page)]].max()) if c.codes else 0.0
            close(got["out"][s:s + 1], parts[0],
                  attention_tolerance(*parts, self.DIM, self.dtype, c.codes, vs) + parts[1] * 2.0 ** -15)
        q, k, v, out = got["linear"]
        want, mag, after, sizes = recurrence(q, k, v, self.decay, [1] * n, states, self.DIM ** -0.5)
        tol, state_tol = tolerances(self.dtype, self.DIM, 1, self.decay, want, mag, sizes, True)
        close(out, want, tol)
        close(self.states[self.own.long()], after, state_tol)
        logits, u = got["logits"].double().cpu().numpy(), self.uniform.double().cpu().numpy()
        for s in range(n):
            token, log = definition(logits[s], u[s], 0.9, 200, 0.95, 0.0)
            assert int(self.tokens[s]) == token, s
            assert abs(float(got["logs"][s]) - log) <= 2.0 ** -24 * abs(log) * 1.01 + 2.0 ** -22


@pytest.mark.parametrize("dtype,codes", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("vehicles,candidates,history,window,shared", [
    (2, 40, 2050, 0, True), (1, 96, 1600, 0, False), (3, 64, 4100, 1500, True)])
def test_tokens_drawn_step_by_step(ctx, dtype, codes, vehicles, candidates, history, window, shared):
    r = Rollout(ctx, dtype, codes, vehicles, candidates, history, 4, window, 4 if window else 0)
    assert r.shared == shared
    r.observe(torch.randint(0, r.VOCAB, (vehicles, history), generator=gen(7), device="cuda"))
    history_states = r.states[:vehicles].clone()
    tokens, score, states = r.rollout(11, r.step, r.check)
    assert torch.equal(states[:vehicles], history_states)  # the vehicles' own states are not the candidates'
    # the next control step starts from the same history: other candidates, then these again
    other = r.rollout(12, r.step)[0]
    assert not torch.equal(other, tokens)
    again = r.rollout(11, r.step)
    for a, b in zip((tokens, score, states), again):
        assert torch.equal(a, b)
    # a graph of one step, replayed for each token
    graph = torch.cuda.CUDAGraph()
    r.start(13)
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        r.step()
    again = r.rollout(11, graph.replay)
    for a, b in zip((tokens, score, states), again):
        assert torch.equal(a, b)
    ctx.synchronize()
    del graph


def test_the_guides_program_goes_on(ctx):
    """The integration guide's second program after its first one, each result against 64 bits."""
    guide = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    programs = [b.split("```")[0] for b in guide.split("```python\n")[1:] if "PagedCache" in b.split("```")[0] or "SharedPrefix" in b.split("```")[0]]
    assert len(programs) == 2
    names = dict(ctx=ctx, L=L)
    exec(programs[0], names)
    before = names["out"].clone()
    names["out"].fill_(7.0)
    exec(programs[1], names)
    h, kv, d, S = names["heads"], names["kv"], names["dim"], names["S"]
    assert torch.equal(names["out"], before)  # so few run by themselves
    split = lambda x: (x[:, :h], x[:, h:h + kv], x[:, h + kv:])
    states = torch.zeros(1, h, d, d, device="cuda")
    for x, out, news, starts_from, kept in ((names["x"], names["seen"], [40], states, names["states"][:1]),
                                            (names["y"], names["went"], [1] * S, names["states"][:1].expand(S, -1, -1, -1), names["states"][1:])):
        want, mag, after, sizes = recurrence(*split(x), names["decay"], news, starts_from, d ** -0.5)
        tol, state_tol = tolerances(BF16, d, max(news), names["decay"], want, mag, sizes, max(news) <= 8)
        close(out, want, tol)
        close(kept, after, state_tol)
    x, u = names["logits"].double().cpu().numpy(), names["uniform"].double().cpu().numpy()
    assert [definition(x[s], u[s], 0.9, 200, 0.95, 0.0)[0] for s in range(S)] == names["tokens"].tolist()
