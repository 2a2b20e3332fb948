"""Linear attention by chunks over the whole range of its numbers, against the float64
recurrence: prompts that start from a state of zeros, or from columns of zeros and of
next to nothing beside others, with values far beyond one -- what is finite by the
formula and fits the output's type comes out finite and within the bounds of
recurrent_helpers."""
from __future__ import annotations

import pytest
import torch

from recurrent_helpers import Linear, Requests

pytestmark = pytest.mark.gpu

# rows, outputs, the values' magnitude: results below fp16's 65504 where the output is fp16
MAGNITUDES = [("bf16", "bf16", 1e3), ("bf16", "bf16", 1e5), ("bf16", "f32", 1e8), ("bf16", "f16", 1e3),
              ("f16", "f16", 1e3), ("f16", "f32", 1e4), ("f16", "bf16", 1e4), ("f32", "f32", 1e3), ("f32", "f32", 1e5),
              ("f32", "bf16", 1e8), ("f32", "f16", 1e3)]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("type_,out,size", MAGNITUDES)
def test_prompts_from_a_state_of_zeros(ctx, type_, out, size, delta):
    """No state, a slot that names none, a state of zeros, columns of zeros and of 1e-30 beside others."""
    print(f"[linear] {type_} {out} {size} delta={delta}", flush=True)
    for dims in ((64, 64), (128, 96)):
        rq = Requests([150, 64, 30], slots=[0, 7, 2], n_slots=3)
        for state in ("none", "zeros", "columns"):
            c = Linear(ctx, rq, 1, 2, *dims, type_, out, delta, seed=dims[0], state=state != "none")
            c.v.mul_(size)
            if state == "zeros":
                c.state.zero_()
            elif state == "columns":
                c.state[..., 5] = 0.0
                c.state[..., 17] *= 1e-30
            c.run()
            assert torch.isfinite(c.out[:rq.starts[-1]]).all()
            c.check()


@pytest.mark.parametrize("type_,size", [("bf16", 1e5), ("f16", 1e4), ("f32", 1e5)])
def test_equal_keys_and_small_queries(ctx, type_, size):
    """Without decay and the delta rule the values of all tokens add up; queries down to 2^-10."""
    for small in (1.0, 2.0 ** -10):
        c = Linear(ctx, Requests([64, 100]), 1, 2, 128, 64, type_, "f32", delta=False, decay="none", seed=1, state=False)
        c.k.copy_(c.k[:1].expand_as(c.k))
        c.q.copy_(c.k * small)
        c.v.copy_(c.v.abs() * size)
        c.run()
        c.check()


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("type_,size", [("bf16", 1e5), ("f16", 1e4), ("f32", 1e5)])
def test_states_cleared_before_a_chunk(ctx, type_, size, delta):
    """A decay of -inf at a chunk's last token, whose value is zero, leaves the next chunk a state of zeros."""
    for low in (-float("inf"), -300.0):
        c = Linear(ctx, Requests([200]), 1, 2, 64, 64, type_, "f32", delta, seed=9)
        c.v.mul_(size)
        c.v[63], c.v[127, 1] = 0.0, 0.0
        c.decay[63], c.decay[127, 1] = low, low
        c.run()
        c.check()


@pytest.mark.parametrize("type_,out,size", [("f16", "f16", 1e3), ("bf16", "f32", 1e6), ("f32", "bf16", 1e6)])
def test_segments_from_a_state_of_zeros(ctx, type_, out, size):
    """Long requests without the delta rule: every segment but the first begins with zeros in the first pass."""
    rq = Requests([1100, 320, 64], slots=[1, 9, 0], n_slots=2)
    for state in (True, False):
        c = Linear(ctx, rq, 1, 2, 64, 64, type_, out, delta=False, seed=2, state=state)
        c.v.mul_(size)
        if state:
            c.state.zero_()
        c.run()
        c.check()


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("type_,out", [("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("what", ["states", "values", "keys", "queries"])
def test_numbers_near_the_smallest(ctx, what, type_, out, delta):
    """A factor of a few steps above fp32's smallest normal number keeps its digits, whatever it meets."""
    tiny, huge = 2.0 ** -118, 2.0 ** 100
    c = Linear(ctx, Requests([150]), 1, 2, 64, 64, type_, out, delta, seed=6, rate=0.1)
    if what == "states":
        c.state.mul_(tiny), c.v.mul_(tiny)
    elif what == "values":
        c.v.mul_(tiny), c.state.zero_()
    else:
        (c.k if what == "keys" else c.q).mul_(tiny), c.v.mul_(huge), c.state.mul_(huge)
    if what in ("states", "values"):
        c.q.mul_(huge)
    c.run()
    c.check()
