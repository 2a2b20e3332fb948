"""Linear attention by chunks over requests that lie in any order: starts that descend
(a request whose next start is below its own is empty) give every other request its
own rows, chunks of both sides included."""
from __future__ import annotations

import pytest
import torch

from recurrent_helpers import FILL, Linear, Requests, ints

pytestmark = pytest.mark.gpu

# starts, rows: what lies between two requests out of order is an empty request
ORDERS = [([128, 256, 0, 128], 256), ([64, 200, 0, 64], 200), ([300, 431, 100, 300, 0, 100], 431),
          ([33, 97, 0, 33], 97), ([640, 1400, 0, 640], 1400), ([90, 120, 30, 90, 0, 30], 130)]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("type_,out,dims", [("bf16", "bf16", (64, 64)), ("f32", "f32", (128, 32)), ("f32", "f32", (256, 64)),
                                            ("f16", "f32", (128, 128))])
@pytest.mark.parametrize("starts,n", ORDERS)
def test_requests_in_any_order(ctx, starts, n, type_, out, dims, delta):
    print(f"[linear] {starts} {type_} {out} {dims} delta={delta}", flush=True)
    lengths = [max(0, b - a) for a, b in zip(starts, starts[1:])]
    for cut in (False, True):
        use = [max(0, x - 5 * s) for s, x in enumerate(lengths)] if cut else None
        rq = Requests(lengths, use=use, slots=list(reversed(range(len(lengths)))))
        rq.starts, rq.N = starts, n
        rq.dev["q_start"] = ints(starts)
        c = Linear(ctx, rq, 2, 4, *dims, type_, out, delta, seed=n)
        need = ctx.linear_attention_workspace(c.args())
        assert need > 0
        ws = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
        for _ in range(3):
            c.out.fill_(FILL), c.state_out.fill_(FILL)
            c.run(workspace=ws.data_ptr(), workspace_bytes=need)
            c.check(chunked=True)
            assert (ws[need:] == 255).all()
