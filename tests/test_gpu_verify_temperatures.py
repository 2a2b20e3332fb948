"""kvmem_hip_verify_draft at temperatures down to fp32's smallest and logits up to its
largest: the definition subtracts the row's largest logit before it divides, so equal
largest logits share the probability however small the temperature."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_verify_draft import Verify

pytestmark = pytest.mark.gpu

TEMPERATURES = [1e-3, 1e-6, 1e-10, 1e-12, 1e-14, 1e-18, 1e-20, 1e-38, 1e-45]


def ties(c, top):
    """The largest logits: four equal ones in three parts, and one a step below."""
    near = torch.full_like(c.logits, top)
    c.logits[:, [3, 900, 2049, 4600]] = near[:, :4]
    if c.type == "f32":
        c.logits[:, 4100] = torch.nextafter(near, torch.zeros_like(near))[:, 0]
    c.tokens[1::2] = 900


@pytest.mark.parametrize("type_,probs", [("f32", None), ("f32", "f32"), ("bf16", None), ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("t", TEMPERATURES)
def test_small_temperatures(ctx, t, type_, probs):
    for seed in range(4):
        c = Verify(ctx, [3, 1, 2, 4, 2, 3, 2, 2], 5003, type_, probs, seed=seed, temps=[t] * 8)
        if seed:
            ties(c, 20.3125 + 3.0 * seed)
        if probs and seed > 1:
            c.probs.zero_()
            c.probs[:, 3], c.probs[:, 900] = 0.75, 0.25
        c.run()
        c.check()
        assert (c.o["tokens"][:, 0] >= 0).all()


@pytest.mark.parametrize("probs", [None, "f32"])
@pytest.mark.parametrize("type_,top", [("f32", 1e20), ("f32", 3e38), ("bf16", 1e20), ("f16", 6e4), ("f32", -1e20)])
def test_large_logits(ctx, type_, top, probs):
    for seed in range(3):
        for t in (0.7, 1e-3, 50.0):
            c = Verify(ctx, [3, 1, 2, 4, 2, 3, 2, 2], 5003, type_, probs, seed=seed, temps=[t] * 8)
            if top < 0:
                c.logits.add_(top).mul_(1.5)
            ties(c, top)
            c.run()
            c.check()


def test_a_draw_at_every_border_of_a_small_temperature(ctx):
    """Steps of fp32 below the largest logit are e^-1.9 of it at 1e-6: u in the middle of each id's range and next
    to its ends."""
    for probs in (None, "f32"):
        c = Verify(ctx, [2] * 40, 5003, "f32", probs, seed=3, temps=[1e-6] * 40)
        at = [3, 900, 2049, 4100, 4600]
        x = torch.tensor(20.3125)
        for i in at:
            c.logits[:, i] = x
            x = torch.nextafter(x, torch.tensor(0.0))
        c.tokens.fill_(7)
        c.ua.fill_(0.5)
        if probs:
            c.probs.zero_()
            c.probs[:, 7] = 1.0
        w = np.exp((c.logits[0, at].double().cpu().numpy() - 20.3125) / float(np.float32(1e-6)))
        ends = np.concatenate([[0.0], np.cumsum(w)]) / w.sum()
        us = [v for a, b in zip(ends, ends[1:]) for v in (a + 1e-7, (a + b) / 2, b - 1e-7)]
        c.us[:len(us)] = torch.tensor([min(max(v, 0.0), 1.0 - 2.0 ** -24) for v in us], dtype=torch.float32).cuda()
        c.run()
        c.check()
