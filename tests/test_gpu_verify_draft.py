"""kvmem_hip_verify_draft against the definition in float64, row by row: types, odd
vocabularies and row strides, drafts with and without probabilities, temperatures (0
too), ragged requests, masks of every kind, numbers at the ends of their ranges."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from recurrent_helpers import DT, TYPE, ints, kv, ptr

pytestmark = pytest.mark.gpu

FILL = -77


def draw(w, u):
    """The lowest id whose running sum passes u times the total, by exact sums; the last positive one if none does."""
    total = math.fsum(w)
    c = np.cumsum(w.astype(np.longdouble))
    over = np.flatnonzero((c > np.longdouble(u) * np.longdouble(total)) & (w > 0))
    return int(over[0]) if over.size else int(np.flatnonzero(w > 0)[-1])


def probabilities(x, t):
    """p of a row of logits, or None where nothing is above -inf."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return None
    if t <= 0 or top == np.inf:
        return (np.arange(x.size) == np.argmax(x)).astype(np.float64)
    e = np.exp((x - top) / t)
    return e / math.fsum(e)


def expected(logits, probs, tokens, starts, t, ua, us, most):
    """(tokens, accepted, keep) of every request."""
    out = []
    for s in range(len(starts) - 1):
        a, b = starts[s], min(starts[s + 1], len(logits), starts[s] + most + 1)
        got, n = [], max(0, b - a)
        for r in range(a, b):
            x, tt = logits[r], 1.0 if t is None else float(t[s])
            p = probabilities(x, tt)
            if p is None:
                got.append(-1)
                break
            sure = tt <= 0 or np.nanmax(x) == np.inf
            if r + 1 < b:
                d = int(tokens[r + 1])
                known = 0 <= d < x.size
                q = None if probs is None or sure else probs[r]
                if known and float(ua[r]) * (1.0 if q is None else float(q[d])) < p[d]:
                    got.append(d)
                    continue
                w = p.copy()
                if q is not None:
                    w = np.maximum(p - q, 0.0)
                elif known:
                    w[d] = 0.0
                p = w if w.sum() > 0 else p
            got.append(draw(p, float(us[s])))
            break
        keep = len(got)
        out.append((got + [-1] * (most + 1 - len(got)), max(0, keep - 1), keep if n else 0))
    return out


class Verify:
    def __init__(self, ctx, rows, V, type_="f32", probs=None, temps=None, seed=0, pad=0, most=None, noise=0.4, spread=3.0,
                 tail=0):
        self.ctx, self.V, self.type, self.probs_type = ctx, V, type_, probs
        g = np.random.default_rng(seed)
        S = len(rows)
        self.S, self.most = S, max([1, *rows]) - 1 if most is None else most
        self.starts = [0, *np.cumsum(rows).tolist()]
        N = self.N = self.starts[-1] + tail
        x = spread * g.standard_normal((max(1, N), V + pad))
        x[:, :V][np.arange(max(1, N))[:, None], g.integers(0, V, (max(1, N), 3))] += 4.0 * spread * g.random((max(1, N), 3))
        self.logits = torch.tensor(x).to(DT[type_]).cuda()
        t = [(1.0, 0.7, 0.0, 1.5)[(s + seed) % 4] for s in range(S)] if temps is None else temps
        self.temps = None if temps is False else torch.tensor(t, dtype=torch.float32).cuda()
        guess = x[:, :V] + noise * g.standard_normal((max(1, N), V))
        guess = np.exp(guess - guess.max(1, keepdims=True))
        guess /= guess.sum(1, keepdims=True)
        self.probs = None if probs is None else torch.tensor(np.pad(guess, ((0, 0), (0, pad)))).to(DT[probs]).cuda()
        picks = [int(g.choice(V, p=r / r.sum())) for r in guess]
        self.tokens = ints([0, *picks[:-1]])
        self.ua = torch.tensor(g.random(max(1, N)), dtype=torch.float32).cuda()
        self.us = torch.tensor(g.random(S), dtype=torch.float32).cuda()
        self.kv_len = ints([100 + 7 * s + n for s, n in enumerate(rows)])
        f = lambda *n: torch.full(n, FILL, dtype=torch.int32, device="cuda")  # noqa: E731
        self.o = dict(tokens=f(S, self.most + 1), n_accepted=f(S), n_keep=f(S), kv_len=f(S))
        self.q_start = ints(self.starts)

    def args(self, **over):
        e = self.logits.element_size()
        a = dict(logits=ptr(self.logits), type=TYPE[self.type], logits_nb=self.logits.stride(0) * e, probs=ptr(self.probs),
                 probs_type=TYPE[self.probs_type or "f32"],
                 probs_nb=0 if self.probs is None else self.probs.stride(0) * self.probs.element_size(), n_vocab=self.V,
                 n_rows=self.N, n_seq=self.S, max_draft=self.most, q_start=ptr(self.q_start), tokens=ptr(self.tokens),
                 temperature=ptr(self.temps), u_accept=ptr(self.ua), u_sample=ptr(self.us), kv_len=ptr(self.kv_len),
                 tokens_out=ptr(self.o["tokens"]), n_accepted=ptr(self.o["n_accepted"]), n_keep=ptr(self.o["n_keep"]),
                 kv_len_out=ptr(self.o["kv_len"]))
        return kv.VerifyArgs(**{**a, **over})

    def run(self, **over):
        torch.cuda.synchronize()
        self.ctx.verify_draft(self.args(**over))
        self.ctx.sync()

    def check(self, **over):
        f = lambda t: None if t is None else t.double().cpu().numpy()[:, :self.V]  # noqa: E731
        starts = over.get("starts", self.starts)
        want = expected(f(self.logits)[:self.N], f(self.probs), self.tokens.cpu().numpy(), starts,
                        None if self.temps is None else self.temps.cpu().numpy(), self.ua.cpu().numpy(),
                        self.us.cpu().numpy(), self.most)
        got = {k: v.cpu().numpy() for k, v in self.o.items()}
        kv_len = self.kv_len.cpu().numpy()
        for s, (tokens, accepted, keep) in enumerate(want):
            assert got["tokens"][s].tolist() == tokens, (s, got["tokens"][s], tokens)
            assert (got["n_accepted"][s], got["n_keep"][s]) == (accepted, keep), s
            assert got["kv_len"][s] == kv_len[s] - (starts[s + 1] - starts[s]) + keep, s


@pytest.mark.parametrize("type_,probs", [("f32", None), ("bf16", None), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f16"),
                                         ("f32", "f32"), ("f16", None), ("bf16", "f32")])
@pytest.mark.parametrize("V,pad", [(1, 0), (2, 6), (7, 0), (255, 1), (2048, 0), (2049, 7), (5003, 0), (8192, 8)])
def test_vocabularies_and_types(ctx, V, pad, type_, probs):
    print(f"[verify] V={V} pad={pad} {type_} {probs}", flush=True)
    for seed in range(2):
        c = Verify(ctx, [4, 1, 0, 6, 2, 3, 1, 5], V, type_, probs, pad=pad, seed=seed, tail=1)
        c.run()
        c.check()


@pytest.mark.parametrize("probs", [None, "f32"])
def test_large_vocabularies_and_many_rows(ctx, probs):
    for rows, V, type_ in (([6], 131072, "bf16"), ([3] * 40, 50001, "f32"), ([8] * 20, 120000, "bf16"),
                           ([1], 3000001, "f32")):
        print(f"[verify] {len(rows)} x {rows[0]} x {V}", flush=True)
        c = Verify(ctx, rows, V, type_, probs, seed=V)
        c.run()
        c.check()


@pytest.mark.parametrize("type_,probs", [("bf16", None), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16")])
def test_the_largest_vocabularies(ctx, type_, probs):
    """Rows of more than a thousand parts, several to a thread: odd ends, drafts that stay and that do not."""
    for V, pad in ((2097153, 0), (2100008, 8)):
        print(f"[verify] {V} {type_} {probs}", flush=True)
        c = Verify(ctx, [3, 2], V, type_, probs, pad=pad, seed=V)
        c.run()
        c.check()


@pytest.mark.parametrize("probs", [None, "f32"])
@pytest.mark.parametrize("noise", [0.0, 0.05, 5.0])
def test_drafts_from_equal_to_unlike(ctx, probs, noise):
    """Drafts that all stay, mostly stay and hardly stay; long runs of drafts."""
    for rows in ([128] * 2, [17, 5, 9, 1, 128, 33]):
        c = Verify(ctx, rows, 300, "f32", probs, noise=noise, seed=len(rows), temps=[1.0] * len(rows))
        c.run()
        c.check()


def test_every_place_of_the_draw(ctx):
    """u at 0, at the largest below 1, and between the borders of every id of a few likely ones over parts' ends."""
    V = 5000
    for probs in (None, "f32"):
        for u in (0.0, 0.25, 0.5, 0.999, 1.0 - 2.0 ** -24):
            c = Verify(ctx, [1, 2, 1, 3], V, "f32", probs, seed=3, temps=[1.0, 1.0, 0.5, 2.0])
            c.logits.fill_(-30.0)
            c.logits[:, [0, 1, 7, 8, 2047, 2048, 4095, 4096, 4999]] = 3.0
            c.us.fill_(u)
            c.run()
            c.check()


def test_masks_infinities_and_nan(ctx):
    for probs in (None, "f32"):
        for type_ in ("f32", "bf16"):
            c = Verify(ctx, [3, 3, 3, 3, 3, 3, 3, 2], 4100, type_, probs, seed=1, temps=[1.0, 0.0, 1.0, 1.0, 0.0, 1.0, 1.0, 0.8])
            inf, nan = float("inf"), float("nan")
            c.logits[0:3] = -inf                    # nothing left: nothing stays, -1
            c.logits[3:6] = -inf
            c.logits[6] = nan
            c.logits[9, ::2] = -inf                 # masks
            c.logits[10, 5:] = -inf
            c.logits[11] = torch.finfo(DT[type_]).min
            c.logits[12, 3:4000] = nan
            c.logits[15, [4099, 77, 2050]] = inf    # the lowest of several
            c.logits[18, 4000] = inf
            c.tokens[16] = 77
            c.tokens[19] = 4000
            c.run()
            c.check()


def test_drafts_outside_the_vocabulary_and_ties(ctx):
    for probs in (None, "f32"):
        for temps in ([1.0] * 4, [0.0] * 4):
            c = Verify(ctx, [3, 3, 3, 3], 3000, "f32", probs, seed=2, temps=temps, noise=0.0)
            c.tokens[[1, 4]] = ints([-1, 3000])
            c.tokens[7] = 0x7fffffff
            c.logits[9] = 1.5  # all equal: the lowest at temperature 0
            c.tokens[10] = 0
            c.run()
            c.check()


def test_a_draft_that_was_all_there_is(ctx):
    """The refused draft had all the probability: the draw is from p itself (u = 1 is not in the range, but ends too)."""
    c = Verify(ctx, [2, 2], 100, "f32", None, temps=[1.0, 1.0])
    c.logits.fill_(-1e4)
    c.logits[[0, 2], [5, 99]] = 0.0
    c.tokens[[1, 3]] = ints([5, 99])
    c.ua.fill_(1.0)
    c.run()
    assert c.o["tokens"].tolist() == [[5, -1], [99, -1]] and c.o["n_accepted"].tolist() == [0, 0]
    c = Verify(ctx, [2], 100, "f32", "f32", temps=[1.0])
    c.probs.fill_(1.0)  # nothing of p is above q
    c.ua.fill_(1.0)
    c.run()
    x = c.logits[0].double().cpu().numpy()
    assert c.o["tokens"][0, 0] == draw(probabilities(x, 1.0), float(c.us[0]))


def test_optional_arrays_and_bounds(ctx):
    c = Verify(ctx, [4, 4, 4], 600, "f32", "f32", temps=False, most=3, seed=5)
    c.run(q_start=None)
    c.check()
    n_keep = c.o["n_keep"].clone()
    c.o["n_keep"].fill_(FILL), c.o["kv_len"].fill_(FILL)
    c.run(n_keep=None, kv_len=None, kv_len_out=None)
    assert (c.o["n_keep"] == FILL).all() and (c.o["kv_len"] == FILL).all()
    # in place
    lens = c.kv_len.clone()
    c.run(kv_len_out=ptr(c.kv_len))
    assert torch.equal(c.kv_len, lens - 4 + n_keep)
    # more rows than drafts are looked at; starts beyond the rows
    c = Verify(ctx, [9, 5], 600, "f32", None, most=3, seed=6)
    c.run()
    c.check()
    c.q_start = torch.tensor([10, 0x7fffffff, -1], dtype=torch.int32, device="cuda")
    c.run()
    assert c.o["n_keep"].tolist()[1] == 0 and c.o["tokens"][1].tolist() == [-1] * 4


def test_captured_and_replayed(ctx):
    c = Verify(ctx, [4, 1, 6, 3], 5003, "bf16", "f32", seed=9)
    need = ctx.verify_draft_workspace(c.args())
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(g, stream=stream):
            ctx.verify_draft(c.args(workspace=ptr(ws), workspace_bytes=need))
    finally:
        ctx.set_stream(None)
    for i in range(4):
        gen = torch.Generator(device="cuda").manual_seed(i)
        c.ua.copy_(torch.rand(c.ua.shape, generator=gen, device="cuda"))
        c.us.copy_(torch.rand(c.us.shape, generator=gen, device="cuda"))
        c.tokens.copy_(c.tokens.roll(1))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        stream.synchronize()
        c.check()
        c.run()
        c.check()
