"""Linear attention by chunks with a bf16 out: the output is the fp32 result rounded
once, so it errs by an f32 out's bound (recurrent_helpers) and half a step of bf16, also
where large terms leave a small output."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from recurrent_helpers import FILL, Linear, Requests, close, half_step

pytestmark = pytest.mark.gpu

# by a 22-bit factor each comes out nearly exact; rounded to 11 bits one goes down, the other up
A, B = 1.0 + 0.49 * 2.0 ** -10, 1.0 + 0.51 * 2.0 ** -10


def check(c):
    got = c.out.double().cpu().numpy()
    c.out_type = "f32"
    for s in range(c.rq.S):
        o, b, _, _ = c.want(s, chunked=True)
        a = c.rq.starts[s]
        close(got[a:a + c.rq.use[s]], o, b + half_step(np.abs(o) + b, "bf16"), f"out of request {s}")


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads", [(1, 2, 64, 64), (2, 2, 128, 128), (1, 3, 128, 96), (1, 1, 256, 128), (1, 2, 64, 32)])
def test_rounded_once(ctx, heads, type_, delta):
    print(f"[linear] {heads} {type_} delta={delta}", flush=True)
    for decay in ("token", "none"):
        c = Linear(ctx, Requests([150, 24, 64]), *heads, type_, "bf16", delta, decay=decay, seed=sum(heads), rate=0.1)
        c.run()
        check(c)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (256, 64)])
def test_states_that_cancel(ctx, dims, type_):
    """A column of A, -B, A, -B, ... and equal queries."""
    c = Linear(ctx, Requests([64, 100]), 1, 2, *dims, type_, "bf16", delta=False, decay="none", seed=1)
    c.state[:, :, 0::2], c.state[:, :, 1::2] = A, -B
    c.q.fill_(0.125)
    c.v.zero_()
    c.run()
    check(c)


@pytest.mark.parametrize("which", ["values", "scores"])
@pytest.mark.parametrize("dims", [(64, 64), (128, 128)])
def test_values_and_scores_that_cancel(ctx, dims, which):
    """Equal scores of values A, -B, A, -B, ..., and values of 1, -1, ... under scores of A, B, ..."""
    c = Linear(ctx, Requests([64, 130]), 1, 2, *dims, "f32", "bf16", delta=False, decay="none", seed=1, state=False)
    up = torch.where(torch.arange(c.rq.N, device="cuda") % 2 == 0, A, B)[:, None, None]
    sign = torch.where(torch.arange(c.rq.N, device="cuda") % 2 == 0, 1.0, -1.0)[:, None, None]
    c.q.fill_(0.125), c.k.fill_(0.125), c.v.copy_(sign.expand_as(c.v))
    if which == "values":
        c.v.mul_(up)
    else:
        c.k.mul_(up)
    c.run()
    check(c)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads", [(1, 2, 64, 64), (2, 2, 128, 128), (1, 3, 128, 96), (1, 1, 256, 128), (1, 2, 64, 32)])
def test_the_state_alone(ctx, heads, type_, delta):
    """Without an out (and without queries) the state is the one that the call with an out stores, bit for bit."""
    print(f"[linear] {heads} {type_} delta={delta}", flush=True)
    c = Linear(ctx, Requests([150, 24, 64], use=[130, 24, 9], tail=1), *heads, type_, "f32", delta, seed=sum(heads))
    c.run()
    c.check()
    want = c.state_out.clone()
    c.out.fill_(FILL), c.state_out.fill_(FILL)
    c.run(out=None, q=None)
    c.check(out=False)
    assert torch.equal(c.state_out, want)
