"""kvmem_hip_conv_rows against float64 (recurrent_helpers): widths, types, channel
counts and alignments, norms of every run, requests from no token to many, tokens
that take no part, states in place, zero and missing, rows no request owns."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from recurrent_helpers import DT, FILL, TYPE, Requests, close, conv_reference, half_step, kv, ptr

pytestmark = pytest.mark.gpu


class Conv:
    def __init__(self, ctx, rq, C, W, type_="bf16", silu=True, bias=True, norm=0, norm_dim=0, eps=1e-6, seed=0, state=True,
                 offset=0, pad=8, scale=1.0):
        self.ctx, self.rq, self.C, self.W, self.type = ctx, rq, C, W, type_
        self.opts = (silu, norm, norm_dim, eps)
        g = torch.Generator().manual_seed(seed)
        dt = DT[type_]
        self.raw = (scale * torch.randn((rq.N, C + pad + offset), generator=g)).to(dt).cuda()
        self.x = self.raw[:, offset:offset + C]
        self.w = (torch.randn((C, W), generator=g) / W ** 0.5).cuda()
        self.b = (0.2 * torch.randn(C, generator=g)).cuda() if bias else None
        self.state = (scale * torch.randn((rq.n_slots, W - 1, C), generator=g)).to(dt).cuda() if state else None
        self.out = torch.full((rq.N, C), FILL, dtype=dt, device="cuda")
        self.state_out = torch.full((rq.n_slots, W - 1, C), FILL, dtype=dt, device="cuda")

    def args(self, max_q=None, **over):
        silu, norm, norm_dim, eps = self.opts
        a = dict(x=ptr(self.x), type=TYPE[self.type], x_nb=self.x.stride(0) * self.x.element_size(), n_channels=self.C,
                 width=self.W, weight=ptr(self.w), bias=ptr(self.b), silu=int(silu), norm_channels=norm,
                 norm_dim=norm_dim, eps=eps, state=ptr(self.state), state_out=ptr(self.state_out), out=ptr(self.out),
                 **self.rq.args(max_q))
        return kv.ConvArgs(**{**a, **over})

    def run(self, max_q=None, **over):
        torch.cuda.synchronize()
        self.ctx.conv_rows(self.args(max_q, **over))
        self.ctx.sync()

    def check(self, out=True, stored=True, before=None):
        rq = self.rq
        f = lambda t: t.double().cpu().numpy()  # noqa: E731
        x, w, got, state = f(self.x), f(self.w), f(self.out), f(self.state_out)
        before = before if before is not None else None if self.state is None else f(self.state)
        bias = None if self.b is None else f(self.b)
        written, touched = np.zeros(rq.N, bool), np.zeros(rq.n_slots, bool)
        for s in range(rq.S):
            a, n, slot = rq.starts[s], rq.use[s], rq.slots[s]
            old = before[slot] if before is not None and slot < rq.n_slots else np.zeros((self.W - 1, self.C))
            y, e, new = conv_reference(x[a:a + n], old, w, bias, *self.opts)
            if out:
                close(got[a:a + n], y, e + half_step(y, self.type), f"rows of request {s}")
                written[a:a + n] = True
            if stored and slot < rq.n_slots:
                assert np.array_equal(state[slot], new), f"state of request {s}"
                touched[slot] = True
        assert (got[~written] == FILL).all() and (state[~touched] == FILL).all()


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("W", range(2, 9))
def test_widths_and_types(ctx, W, type_):
    print(f"[conv_rows] W={W} {type_}", flush=True)
    # none, one, W-2, W-1, W tokens; a tile's border; several tiles
    rq = Requests([0, 1, W - 2, W - 1, W, 16, 17, 50], slots=[3, 9, 0, 5, 1, 2, 8, 4], n_slots=10, tail=3)
    c = Conv(ctx, rq, 520, W, type_, norm=384, norm_dim=128, seed=W)
    c.run()
    c.check()


@pytest.mark.parametrize("C,norm,norm_dim,offset", [(1, 0, 0, 0), (7, 0, 0, 0), (96, 64, 32, 0), (72, 64, 64, 1),
                                                    (513, 512, 512, 0), (1030, 256, 256, 3), (1536, 1024, 512, 8),
                                                    (2056, 2048, 128, 0), (640, 640, 64, 0)])
@pytest.mark.parametrize("type_", ["bf16", "f32"])
def test_channels_runs_and_alignments(ctx, C, norm, norm_dim, offset, type_):
    print(f"[conv_rows] C={C} norm={norm}/{norm_dim} offset={offset} {type_}", flush=True)
    rq = Requests([5, 1, 20])
    c = Conv(ctx, rq, C, 4, type_, norm=norm, norm_dim=norm_dim, offset=offset, pad=offset % 8, seed=C)
    c.run()
    c.check()


@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("bias", [True, False])
def test_without_silu_bias_state(ctx, silu, bias):
    rq = Requests([3, 40])
    for state in (True, False):
        c = Conv(ctx, rq, 256, 4, "f16", silu=silu, bias=bias, state=state)
        c.run()
        c.check()


def test_tokens_that_take_part(ctx):
    """n_use below, at and beyond a request's tokens; slots that name no state; one token a request without starts."""
    rq = Requests([6, 6, 6, 33, 2], use=[0, 1, 6, 20, 99], slots=[1, 0xffffffff, 0, 5, 2], n_slots=5)
    for out, stored in ((True, True), (True, False), (False, True)):
        c = Conv(ctx, rq, 264, 4, "bf16", norm=256, norm_dim=256, seed=2)
        c.run(**({} if out else dict(out=None)), **({} if stored else dict(state_out=None)))
        c.check(out, stored)
    rq = Requests([1, 1, 1], slots=[2, 0, 1])
    c = Conv(ctx, rq, 64, 3)
    c.run(q_start=None)
    c.check()


def test_states_in_place_and_a_prompt_in_pieces(ctx):
    """A prompt in pieces of every length, the state updated in place, gives the rows of one call."""
    N, C, W = 70, 520, 4
    whole = Conv(ctx, Requests([N], n_slots=1), C, W, norm=512, norm_dim=128, seed=4)
    whole.run()
    whole.check()
    state, at = whole.state.clone(), 0
    out = torch.full_like(whole.out, FILL)
    for n in (1, 1, 2, 3, 0, 5, 17, 1, 40):
        rq = Requests([n], n_slots=1)
        piece = whole.args(**rq.args(), x=ptr(whole.x[at:]) if n else ptr(whole.x), out=ptr(out[at:]) if n else ptr(out),
                           state=ptr(state), state_out=ptr(state))
        torch.cuda.synchronize()
        ctx.conv_rows(piece)
        ctx.sync()
        at += n
    assert at == N and torch.equal(out, whole.out) and torch.equal(state, whole.state_out)


def test_lengths_beyond_every_bound(ctx):
    """Starts, uses and rows beyond n_tokens and max_q stay in range."""
    rq = Requests([9, 30, 7])
    c = Conv(ctx, rq, 128, 4, "f32")
    rq.dev["q_start"] = torch.tensor([0, 9, 39, 0x7fffffff], dtype=torch.int32, device="cuda")
    rq.use = [8, 8, 7]  # max_q
    c.run(max_q=8)
    c.check()
    c.out.fill_(FILL), c.state_out.fill_(FILL)
    rq.dev["q_start"] = torch.tensor([50, 40, -1, -1], dtype=torch.int32, device="cuda")
    rq.starts, rq.use = [0, 40, 0, 0], [0, 6, 0]  # of the second request what rows there are
    c.run()
    c.check()


def test_numbers_that_are_not_finite_and_extremes(ctx):
    """NaN and infinities stay in their channel (and run) and behind their token; runs whose squares leave fp32,
    runs of zeros."""
    rq = Requests([12], n_slots=1)
    c = Conv(ctx, rq, 256, 4, "f32", silu=False, bias=False, norm=128, norm_dim=32, seed=1)
    c.raw[5, 40] = float("nan")
    c.raw[5, 200] = float("inf")
    c.run()
    got = c.out.cpu().numpy()
    odd = ~np.isfinite(got)
    want = np.zeros_like(odd)
    want[5:9, 32:64] = True
    want[5:9, 200] = True
    assert (odd == want).all()
    for scale, eps in ((1e25, 1e-6), (1e-25, 0.0), (1e-30, 1e-38), (0.0, 0.0)):
        c = Conv(ctx, rq, 256, 4, "f32", silu=False, bias=False, norm=256, norm_dim=128, eps=eps, scale=scale, seed=3)
        c.run()
        c.check()


def test_captured_and_replayed(ctx):
    rq = Requests([4, 0, 19], use=[2, 0, 19])
    c = Conv(ctx, rq, 640, 4, norm=512, norm_dim=128, seed=6)
    c.run()
    first, state = c.out.clone(), c.state_out.clone()
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    ctx.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(g, stream=stream):
            ctx.conv_rows(c.args())
    finally:
        ctx.set_stream(None)
    for i in range(3):
        c.out.fill_(FILL), c.state_out.fill_(FILL)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        stream.synchronize()
        assert torch.equal(c.out, first) and torch.equal(c.state_out, state)
        ctx.conv_rows(c.args())
        ctx.sync()
