"""kvmem_hip_attention with device lengths and starts beyond every bound of the call:
the keys and rows that the bounds leave, each element within the float64
reference's own bound and lse too (attention_helpers) -- a key attended too many or
too few is far outside it."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
from attention_helpers import Case  # noqa: E402


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("m", [1, 2, 60])
def test_lengths_and_starts_past_the_call(ctx, oracle, m, D, causal):
    """Lengths of 2^32 - 1 and a last start far behind the tokens: 90 keys and m rows a request are left."""
    print(f"[bounds] {m} {D} {causal}", flush=True)
    c = Case(ctx, oracle, [300, 90], [m, m], 4, 1, D, 32, causal=causal, seed=401)
    c.dev["lens"].fill_(-1)
    c.dev["starts"].copy_(torch.tensor([0, m, 2 ** 31 - 1], dtype=torch.int32))
    c.args.max_kv = 90
    c.run()
    c.causal = False  # every row's last key lies behind the bound
    c.check(lens=[90, 90], m=[m, m])


def test_one_key_more_or_less_is_seen(ctx, oracle):
    """The reference itself: a call over 89 or 91 keys is outside the bounds of 90."""
    for m in (2, 60):
        for keys in (89, 91):
            c = Case(ctx, oracle, [300, 300], [m, m], 4, 1, 64, 32, causal=False, max_kv=keys, seed=402)
            c.run()
            c.args.max_kv = 90
            with pytest.raises(AssertionError):
                c.check()
