"""kvmem_hip_linear_attention against the float64 recurrence and the bounds of
recurrent_helpers: token by token and by chunks, with and without the delta rule,
decays per token, per head and none, head sizes, types, ragged requests, tokens that
take no part, states in place, zero and missing, numbers that are not finite."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from recurrent_helpers import FILL, Linear, Requests, close, kv, ptr

pytestmark = pytest.mark.gpu

HEADS = [(1, 1, 64, 32), (2, 4, 64, 64), (1, 3, 128, 128), (2, 2, 128, 96), (1, 2, 256, 64), (1, 1, 256, 256),
         (1, 2, 64, 512)]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("type_,out", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32"),
                                       ("f32", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("heads", HEADS)
def test_heads_and_types(ctx, heads, type_, out, delta):
    print(f"[linear] {heads} {type_} {out} delta={delta}", flush=True)
    few = Requests([1, 0, 3, 7], slots=[2, 0, 5, 1], n_slots=6, tail=2)
    many = Requests([70, 1, 0, 64, 129], slots=[4, 1, 0, 2, 6], n_slots=7, tail=2)
    for rq in (few, many):
        c = Linear(ctx, rq, *heads, type_, out, delta, seed=sum(heads))
        c.run()
        c.check()


@pytest.mark.parametrize("decay", ["token", "head", "none"])
@pytest.mark.parametrize("n", [1, 2, 23, 24, 63, 64, 65, 128, 191, 200])
def test_lengths_and_decays(ctx, n, decay):
    print(f"[linear] n={n} decay={decay}", flush=True)
    for rate in (1.0, 30.0):
        c = Linear(ctx, Requests([n]), 1, 2, 64, 64, decay=decay, seed=n, rate=rate)
        c.run()
        c.check()


@pytest.mark.parametrize("lengths", [[5, 5, 5, 6, 2], [40, 64, 70, 100, 26]])
def test_tokens_that_take_part(ctx, lengths):
    """n_use below, at and beyond a request's tokens, slots that name no state; without an out, without storing,
    without a state."""
    use = [0, 1, lengths[2], lengths[3] - 3, 1000]
    for out, stored, state in ((True, True, True), (True, False, True), (False, True, True), (True, True, False)):
        rq = Requests(lengths, use=use, slots=[1, 0xffffffff, 0, 5, 2], n_slots=5)
        c = Linear(ctx, rq, 2, 4, 64, 64, seed=3, state=state)
        c.run(**({} if out else dict(out=None, q=None)), **({} if stored else dict(state_out=None)))
        c.check(out=out, stored=stored)


def test_one_token_a_request_without_starts(ctx):
    c = Linear(ctx, Requests([1, 1, 1, 1], slots=[3, 0, 2, 1]), 1, 2, 128, 64, "f16", "f32", scale=0.37)
    c.run(q_start=None)
    c.check()


@pytest.mark.parametrize("type_", ["bf16", "f32"])
def test_a_prompt_in_pieces_in_place(ctx, type_):
    """Pieces of every kind, the state updated in place: each piece within its own bounds of the recurrence that
    starts from the state the piece before left."""
    n = [1, 64, 3, 100, 24, 1, 7]
    whole = Linear(ctx, Requests([sum(n)], n_slots=1), 1, 2, 128, 64, type_, "f32", seed=8)
    state, at = whole.state.clone(), 0
    for m in n:
        old = state.double().cpu().numpy()[0]
        part = {x: ptr(getattr(whole, x)[at:]) for x in "qkv"}
        torch.cuda.synchronize()
        rq = Requests([m], n_slots=1)
        ctx.linear_attention(whole.args(**rq.args(), **part, out=ptr(whole.out[at:]),
                                        log_decay=ptr(whole.decay[at:]), beta=ptr(whole.beta[at:]), state=ptr(state),
                                        state_out=ptr(state)))
        ctx.sync()
        sub = Requests([m])
        sub.starts, sub.N = [at, at + m], whole.rq.N
        keep, whole.rq = whole.rq, sub
        o, b, S, bs = whole.want(0, m >= 24, old)
        whole.rq = keep
        close(whole.out[at:at + m].double().cpu().numpy(), o, b, f"piece at {at}")
        close(state.double().cpu().numpy()[0], S, bs, f"state behind {at + m}")
        at += m


def test_chunks_and_tokens_agree_with_growing_states(ctx):
    """Keys that are not normalized, decays of one and above, values of other magnitudes: chunks against the
    float64 recurrence, column by column."""
    for scale_k, scale_v, up in ((3.0, 1e4, 0.0), (0.01, 1e-6, 0.0), (0.5, 1.0, 0.02)):
        c = Linear(ctx, Requests([150]), 1, 2, 64, 64, "f32", "f32", delta=False, seed=5)
        c.k.mul_(scale_k), c.v.mul_(scale_v)
        c.decay.mul_(0.1).add_(up)
        c.v[:, :, 3] = 0.0
        c.state[:, :, :, 3] = 0.0
        c.v[:, :, 5] *= 1e-20
        c.state[:, :, :, 5] *= 1e-20
        c.run()
        c.check()


def test_decays_that_clear_the_state(ctx):
    """-inf clears the state: what was before is gone, exactly; also decays far below fp32's exponents."""
    for n, at in ((5, 3), (140, 90)):
        for low in (-float("inf"), -1e30, -200.0):
            c = Linear(ctx, Requests([n]), 1, 2, 64, 64, "bf16", "f32", seed=n)
            c.decay[at] = low
            c.decay[at // 2, 1] = low
            c.run()
            c.check()
            d = Linear(ctx, Requests([n]), 1, 2, 64, 64, "bf16", "f32", seed=n)
            d.decay[at] = low
            d.rows[:at // 2] = d.rows[:at // 2].flip(0)
            d.state.mul_(1e3)
            d.run()
            if n < 24:
                assert torch.equal(c.out[at:], d.out[at:])
            else:
                # the chunk that clears it cuts its columns 2^-39 below their largest (below 2^11), times at
                # most 64 rows of (1 + A)^-1; every number a few units of 22 bits
                assert torch.allclose(c.out[at:], d.out[at:], rtol=2.0 ** -18, atol=2.0 ** -22)


@pytest.mark.parametrize("delta", [True, False])
def test_numbers_that_are_not_finite(ctx, delta):
    """A value that is not finite reaches no earlier token and only its own dim; a key, query or gate no earlier
    token and no other head; requests beside stay as they are."""
    rq = Requests([150, 100])
    clean = Linear(ctx, rq, 2, 2, 64, 64, "bf16", "f32", delta, seed=4)
    clean.run()
    for t in (0, 70, 149):
        for x in (float("nan"), float("inf")):
            c = Linear(ctx, rq, 2, 2, 64, 64, "bf16", "f32", delta, seed=4)
            c.v[t, 1, 9] = x
            c.run()
            ok = torch.isfinite(c.out)
            want = torch.ones_like(ok)
            want[t:150, 1, 9] = False
            assert torch.equal(ok, want)
            assert torch.allclose(torch.where(ok, c.out, 0), torch.where(ok, clean.out, 0), rtol=1e-4, atol=1e-5)
            state = torch.isfinite(c.state_out[0])
            assert not state[1, :, 9].any() and state[1, :, :9].all() and state[0].all()
            for which in ("k", "q", "decay") + (("beta",) if delta else ()):
                c = Linear(ctx, rq, 2, 2, 64, 64, "bf16", "f32", delta, seed=4)
                if which in "kq":
                    getattr(c, which)[t, 1, 11] = x
                else:
                    getattr(c, which)[t, 1] = x
                c.run()
                ok = torch.isfinite(c.out)
                assert ok[:t].all() and ok[:, 0].all() and ok[150:].all(), which
                assert not ok[t, 1].any(), which
                if which == "q":
                    assert ok[t + 1:].all() and torch.isfinite(c.state_out[:2]).all()
                else:
                    assert not ok[t:150, 1].any(-1).any(), which


def test_rows_behind_the_last_request_may_hold_anything(ctx):
    rq = Requests([30, 90], tail=80)
    c = Linear(ctx, rq, 1, 2, 128, 64, seed=2)
    for x in (c.rows, c.decay, c.beta):
        x[120:] = float("nan")
    c.state[2:] = float("nan")
    c.run()
    c.check()


def test_lengths_beyond_every_bound(ctx):
    for top, most in ((20, 8), (100, 64), (100, 70)):
        rq = Requests([top, top // 2, 7])
        c = Linear(ctx, rq, 1, 1, 64, 32, "f32", "f32", seed=1)
        a, b = rq.starts[1], rq.starts[2]
        rq.dev["q_start"] = torch.tensor([0, a, b, 0x7fffffff], dtype=torch.int32, device="cuda")
        rq.use = [min(most, n) for n in rq.lengths]
        c.run(max_q=most)
        c.check(chunked=most >= 24)
        c.out.fill_(FILL), c.state_out.fill_(FILL)
        rq.dev["q_start"] = torch.tensor([0x7ffffff0, 0x7ffffff1, -3, -1], dtype=torch.int32, device="cuda")
        rq.use = [0, 0, 0]
        c.run()
        c.check()


def test_many_requests_and_heads(ctx):
    g = np.random.default_rng(3)
    for most in (4, 90):
        lengths = [int(x) for x in g.integers(0, most, 40)]
        slots = [int(x) for x in g.permutation(42)[:40]]
        c = Linear(ctx, Requests(lengths, slots=slots), 3, 9, 64, 64, seed=most)
        c.run()
        c.check(chunked=max(lengths) >= 24)


@pytest.mark.parametrize("n,type_", [(24, "bf16"), (55, "bf16"), (56, "bf16"), (255, "f32"), (256, "f32")])
def test_calls_of_many_states(ctx, n, type_):
    """Calls whose states fill the card go by chunks from longer requests on: either way within its bounds."""
    rq = Requests([n, 1, n - 1] + [2] * 29)
    c = Linear(ctx, rq, 4, 8, 64, 512, type_, "f32", seed=n)
    chunked = n >= (256 if type_ == "f32" else 56)
    assert (ctx.linear_attention_workspace(c.args()) > 0) == chunked
    c.run()
    c.check(chunked=chunked)


@pytest.mark.parametrize("n,type_", [(47, "f32"), (48, "f32"), (23, "f16"), (24, "f16")])
def test_calls_of_some_states(ctx, n, type_):
    rq = Requests([n, 1, n - 1] + [2] * 5)
    c = Linear(ctx, rq, 4, 8, 64, 512, type_, "f32", seed=n)
    chunked = n >= (48 if type_ == "f32" else 24)
    assert (ctx.linear_attention_workspace(c.args()) > 0) == chunked
    c.run()
    c.check(chunked=chunked)


@pytest.mark.parametrize("type_,out,dims", [("f16", "f16", (64, 64)), ("bf16", "bf16", (128, 96)), ("f32", "f32", (64, 32)),
                                            ("bf16", "f32", (256, 64))])
def test_long_requests_without_the_delta_rule(ctx, type_, out, dims):
    """Requests in segments: long, short, empty and cut ones, of every kind of decay, states stored in place, missing
    and not wanted, without an out."""
    for decay, rate in (("token", 1.0), ("head", 1.0), ("none", 1.0), ("token", 100.0)):
        rq = Requests([1100, 1, 64, 320, 0, 129, 640], slots=[3, 0, 5, 9, 1, 2, 4], n_slots=6,
                      use=[1090, 1, 64, 400, 0, 65, 128], tail=1)
        c = Linear(ctx, rq, 1, 2, *dims, type_, out, delta=False, decay=decay, seed=sum(dims), rate=rate)
        c.run()
        c.check()
        # in place, and without an out
        want, states = c.out.clone(), c.state_out.clone()
        for state, more in ((c.state.clone(), {}), (c.state.clone(), dict(out=None, q=None))):
            before = state.clone()
            c.out.fill_(FILL)
            torch.cuda.synchronize()
            ctx.linear_attention(c.args(state=ptr(state), state_out=ptr(state), **more))
            ctx.sync()
            assert torch.equal(c.out, torch.full_like(c.out, FILL) if more else want)
            for s, slot in enumerate(rq.slots):
                if slot < rq.n_slots:
                    assert torch.equal(state[slot], states[slot]), (s, slot)
            kept = [x for x in range(rq.n_slots) if x not in rq.slots]
            assert all(torch.equal(state[x], before[x]) for x in kept)


def test_segments_with_numbers_that_are_not_finite(ctx):
    """As in one piece: values stay in their dim, clearing decays clear, gates and keys stay in their head, and no
    earlier token changes."""
    n = 1000
    clean = Linear(ctx, Requests([n]), 2, 2, 64, 64, "bf16", "f32", delta=False, seed=4)
    clean.run()
    for t in (0, 130, 700, 999):
        for what in ("v", "k", "decay"):
            for x in (float("nan"), float("inf")):
                c = Linear(ctx, Requests([n]), 2, 2, 64, 64, "bf16", "f32", delta=False, seed=4)
                if what == "decay":
                    c.decay[t, 1] = x
                else:
                    getattr(c, what)[t, 1, 9] = x
                c.run()
                ok = torch.isfinite(c.out)
                assert ok[:t].all() and ok[:, 0].all() and not ok[t:, 1, 9].any()
                if what == "v":
                    assert ok[:, 1, :9].all() and ok[:, 1, 10:].all()
                assert torch.allclose(torch.where(ok, c.out, 0), torch.where(ok, clean.out, 0), rtol=1e-4, atol=1e-5)
    c = Linear(ctx, Requests([n]), 2, 2, 64, 64, "bf16", "f32", delta=False, seed=4)
    c.decay[130] = -float("inf")
    c.decay[700, 1] = -float("inf")
    c.run()
    c.check()


def test_own_workspace_streams_and_replays(ctx):
    """A captured call brings its workspace; two graphs with one each replay at once; results are the eager ones."""
    calls = [Linear(ctx, Requests([100, 30]), 1, 2, 128, 128, seed=i) for i in range(2)]
    need = ctx.linear_attention_workspace(calls[0].args())
    assert need > 0 and ctx.linear_attention_workspace(Linear(ctx, Requests([5]), 1, 2, 128, 128).args()) == 0
    want, graphs, streams, keep = [], [], [], []
    for c in calls:
        c.run()
        want.append((c.out.clone(), c.state_out.clone()))
        st, g, ws = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        ctx.set_stream(st.cuda_stream)
        try:
            with torch.cuda.graph(g, stream=st):
                ctx.linear_attention(c.args(workspace=ptr(ws), workspace_bytes=need))
            # the context's own workspace is no captured call's
            g2 = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g2, stream=st):
                with pytest.raises(kv.KvMemError) as e:
                    ctx.linear_attention(c.args())
                assert e.value.code == kv.ERR_INVALID and "workspace" in str(e.value)
        finally:
            ctx.set_stream(None)
        graphs.append(g), streams.append(st), keep.append(ws)
    for _ in range(3):
        for c in calls:
            c.out.fill_(FILL), c.state_out.fill_(FILL)
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for c, w in zip(calls, want):
            assert torch.equal(c.out, w[0]) and torch.equal(c.state_out, w[1])
        calls[0].run()


def test_segments_replayed_in_place(ctx):
    """A captured call in segments that updates its state: every replay is the eager call's next one."""
    c = Linear(ctx, Requests([1100, 300, 64]), 1, 2, 64, 64, "f16", "f32", delta=False, seed=6)
    need = ctx.linear_attention_workspace(c.args())
    st, g, ws = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    eager, state = c.state.clone(), c.state.clone()
    torch.cuda.synchronize()
    ctx.set_stream(st.cuda_stream)
    try:
        with torch.cuda.graph(g, stream=st):
            ctx.linear_attention(c.args(workspace=ptr(ws), workspace_bytes=need, state=ptr(state), state_out=ptr(state)))
    finally:
        ctx.set_stream(None)
    for _ in range(4):
        ctx.linear_attention(c.args(state=ptr(eager), state_out=ptr(eager)))
        ctx.sync()
        want = c.out.clone()
        c.out.fill_(FILL)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, want) and torch.equal(state, eager)


def test_segments_cut_by_the_call(ctx):
    """max_q, n_use and n_tokens cut requests inside a segment; requests behind the last token have none."""
    for most in (1000, 513, 512, 511, 130):
        rq = Requests([1100, 700, 3])
        c = Linear(ctx, rq, 1, 1, 64, 64, "f16", "f32", delta=False, seed=2)
        rq.use = [min(most, n) for n in rq.lengths]
        c.run(max_q=most)
        c.check(chunked=True)
    rq = Requests([1100, 700, 3])
    c = Linear(ctx, rq, 1, 1, 64, 64, "f16", "f32", delta=False, seed=2)
    rq.use = [1100, 1200 - 1100, 0]
    c.run(n_tokens=1200)
    c.check()


@pytest.mark.parametrize("S", [2, 63, 64, 65, 90])
def test_requests_of_every_order(ctx, S):
    """Chunked requests in and out of order of their lengths, equal and empty ones, around a wave's lanes of them."""
    g = np.random.default_rng(S)
    for lengths in (sorted(int(x) for x in g.integers(0, 140, S)), [70] * S, [int(x) for x in g.integers(0, 3, S) * 65]):
        c = Linear(ctx, Requests(lengths, slots=[int(x) for x in g.permutation(S)], tail=1), 1, 1, 64, 32, "f16", "f32", seed=S)
        c.run(max_q=140)
        c.check(chunked=True)


def test_two_contexts_at_once(ctx):
    other = kv.Context(0)
    try:
        a, b = Linear(ctx, Requests([200]), 1, 2, 64, 64, seed=1), Linear(other, Requests([200]), 1, 2, 64, 64, seed=2)
        torch.cuda.synchronize()
        for _ in range(5):
            ctx.linear_attention(a.args())
            other.linear_attention(b.args())
        ctx.sync(), other.sync()
        a.check(), b.check()
    finally:
        other.close()
