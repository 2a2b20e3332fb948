"""The recurrent layers' calls and the verification of drafts together, as a program
makes them: a small model of two recurrent layers decodes requests with drafted tokens --
kvmem_hip_conv_rows and kvmem_hip_linear_attention over the step's tokens without storing
their states, kvmem_hip_verify_draft, then both again to fold the tokens that stay into
the states -- and token by token without drafts.  Both go through the same arithmetic
per token, so the tokens and the states are the same, bit for bit; with prompts first,
requests that end at other places, the calls captured and replayed."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from recurrent_helpers import kv, ptr

pytestmark = pytest.mark.gpu

V, E = 509, 64
HK, H, DK, DV, W = 2, 4, 64, 64, 4
C = 2 * HK * DK + H * DV
LAYERS, DRAFTS, STEPS = 2, 4, 9


class Model:
    """Weights, and the states of `S` requests."""

    def __init__(self, ctx, S, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
        self.ctx, self.S = ctx, S
        self.embed = r(V, E).double()
        self.w_in = [(r(E, C) / E ** 0.5).double() for _ in range(LAYERS)]
        self.w_gate = [(r(E, 2 * H) / E ** 0.5).double() for _ in range(LAYERS)]
        self.w_out = [(r(H * DV, E) / 8).double() for _ in range(LAYERS)]
        self.head = (3.0 * r(E, V) / E ** 0.5).double()
        self.conv_w = [r(C, W) / 2 for _ in range(LAYERS)]
        self.slots = torch.randperm(S + 1, generator=g, device="cuda")[:S].to(torch.int32)
        self.conv = [torch.zeros((S + 1, W - 1, C), dtype=torch.bfloat16, device="cuda") for _ in range(LAYERS)]
        self.lin = [torch.zeros((S + 1, H, DK, DV), device="cuda") for _ in range(LAYERS)]

    def conv_args(self, layer, b, store):
        return kv.ConvArgs(x=ptr(b["x"][layer]), type=kv.TYPE_BF16, silu=1, x_nb=2 * C, n_channels=C, width=W,
                           n_slots=self.S + 1, norm_channels=2 * HK * DK, norm_dim=DK, eps=1e-6,
                           weight=ptr(self.conv_w[layer]), state=ptr(self.conv[layer]),
                           state_out=ptr(self.conv[layer]) if store else None,
                           out=None if store == "fold" else ptr(b["y"][layer]), **b["batch"],
                           **({"n_use": ptr(b["keep"])} if store == "fold" else {}))

    def linear_args(self, layer, b, store):
        at = ptr(b["y"][layer])
        return kv.LinearArgs(q=None if store == "fold" else at, k=at + 2 * HK * DK, v=at + 4 * HK * DK,
                             type=kv.TYPE_BF16, out_type=kv.TYPE_F32, **{f"{n}_nb1": 2 * DK for n in "qk"},
                             v_nb1=2 * DV, **{f"{n}_nb2": 2 * C for n in "qkv"}, n_head_k=HK, n_head=H, head_dim_k=DK,
                             head_dim_v=DV, n_slots=self.S + 1, log_decay=ptr(b["decay"][layer]), decay_nb=4 * H,
                             beta=ptr(b["beta"][layer]), beta_nb=4 * H, state=ptr(self.lin[layer]),
                             state_out=ptr(self.lin[layer]) if store else None,
                             out=None if store == "fold" else ptr(b["o"][layer]), **b["batch"],
                             **({"n_use": ptr(b["keep"])} if store == "fold" else {}))

    def batch(self, lengths):
        N = sum(lengths)
        starts = torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32, device="cuda")
        e = lambda *n, dt=torch.bfloat16: [torch.zeros(n, dtype=dt, device="cuda") for _ in range(LAYERS)]  # noqa: E731
        return dict(x=e(N, C), y=e(N, C), o=e(N, H, DV, dt=torch.float32), decay=e(N, H, dt=torch.float32),
                    beta=e(N, H, dt=torch.float32), keep=torch.zeros(len(lengths), dtype=torch.int32, device="cuda"),
                    starts=starts, batch=dict(n_tokens=N, n_seq=len(lengths), max_q=max(lengths), q_start=ptr(starts),
                                              slots=ptr(self.slots)))

    def forward(self, b, tokens, store):
        """Logits of the batch's tokens; float64 products, so that a row does not depend on the rows beside it."""
        h = self.embed[tokens.long()]
        for i in range(LAYERS):
            b["x"][i].copy_(h @ self.w_in[i])
            gates = h @ self.w_gate[i]
            b["decay"][i].copy_(-0.3 * torch.nn.functional.softplus(gates[:, :H]))
            b["beta"][i].copy_(torch.sigmoid(gates[:, H:]))
            torch.cuda.synchronize()
            self.ctx.conv_rows(self.conv_args(i, b, store))
            self.ctx.linear_attention(self.linear_args(i, b, store))
            self.ctx.sync()
            h = h + torch.tanh(b["o"][i].double().flatten(1)) @ self.w_out[i]
        return (h @ self.head).float()

    def prompt(self, lengths, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        tokens = torch.randint(0, V, (sum(lengths),), generator=g, device="cuda")
        b = self.batch(lengths)
        logits = self.forward(b, tokens, "store")
        return logits[b["starts"][1:].long() - 1].argmax(-1).tolist()

    def states(self):
        return [t[self.slots.long()].clone() for t in (*self.conv, *self.lin)]


def plain(model, first, n):
    """n tokens of every request, one a step; the states behind every step."""
    S = model.S
    b = model.batch([1] * S)
    streams, states, last = [[t] for t in first], [model.states()], torch.tensor(first, device="cuda")
    for _ in range(n):
        last = model.forward(b, last, "store").argmax(-1)
        for s in range(S):
            streams[s].append(int(last[s]))
        states.append(model.states())
    return streams, states


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("prompts", [[3, 30, 1, 90, 17], [2, 5, 9, 1, 7]])
def test_drafts_give_the_tokens_and_states_of_plain_decoding(ctx, prompts, captured):
    S = len(prompts)
    rng = np.random.default_rng(sum(prompts))
    reference = Model(ctx, S)
    first = reference.prompt(prompts, 5)
    n = STEPS * (DRAFTS + 1)
    want, states = plain(reference, first, n + DRAFTS + 1)

    model = Model(ctx, S)
    assert model.prompt(prompts, 5) == first
    # ragged steps: up to DRAFTS drafts, none for some requests
    lengths = [DRAFTS + 1, 1, DRAFTS + 1, 3, 2]
    b = model.batch(lengths)
    N = sum(lengths)
    tokens = torch.zeros(N, dtype=torch.int32, device="cuda")
    logits = torch.zeros((N, V), device="cuda")
    u = torch.full((N,), 0.5, device="cuda")
    out = torch.zeros((S, DRAFTS + 1), dtype=torch.int32, device="cuda")
    accepted = torch.zeros(S, dtype=torch.int32, device="cuda")
    kv_len = torch.zeros(S, dtype=torch.int32, device="cuda")
    zero = torch.zeros(S, device="cuda")
    verify = kv.VerifyArgs(logits=ptr(logits), type=kv.TYPE_F32, logits_nb=4 * V, n_vocab=V, n_rows=N, n_seq=S,
                           max_draft=DRAFTS, q_start=ptr(b["starts"]), tokens=ptr(tokens), temperature=ptr(zero),
                           u_accept=ptr(u), u_sample=ptr(u), kv_len=ptr(kv_len), kv_len_out=ptr(kv_len),
                           tokens_out=ptr(out), n_accepted=ptr(accepted), n_keep=ptr(b["keep"]))
    ws = torch.empty(ctx.verify_draft_workspace(verify), dtype=torch.uint8, device="cuda")
    verify.workspace, verify.workspace_bytes = ptr(ws), ws.numel()

    def decide():
        ctx.verify_draft(verify)
        for i in range(LAYERS):
            ctx.conv_rows(model.conv_args(i, b, "fold"))
            ctx.linear_attention(model.linear_args(i, b, "fold"))

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    if captured:
        torch.cuda.synchronize()
        ctx.set_stream(stream.cuda_stream)
        try:
            with torch.cuda.graph(graph, stream=stream):
                decide()
        finally:
            ctx.set_stream(None)
    at = [0] * S  # tokens behind the first
    counts = set()
    for step in range(STEPS):
        rows = []
        for s in range(S):
            guess = want[s][at[s]:at[s] + lengths[s]]
            wrong = int(rng.integers(1, lengths[s] + 1))
            rows += [t if i < wrong else (t + 1 + step) % V for i, t in enumerate(guess)]
        tokens.copy_(torch.tensor(rows, dtype=torch.int32))
        before = kv_len.clone()
        kv_len += torch.tensor(lengths, dtype=torch.int32, device="cuda")
        logits.copy_(model.forward(b, tokens, None))
        torch.cuda.synchronize()
        if captured:
            with torch.cuda.stream(stream):
                graph.replay()
            stream.synchronize()
        else:
            decide()
            ctx.sync()
        keep = b["keep"].tolist()
        assert keep == [x + 1 for x in accepted.tolist()] and kv_len.tolist() == (before + b["keep"]).tolist()
        for s in range(S):
            got = out[s].tolist()
            assert got[:keep[s]] == want[s][at[s] + 1:at[s] + 1 + keep[s]] and set(got[keep[s]:]) <= {-1}, (step, s)
            at[s] += keep[s]
            counts.add(keep[s])
        now = model.states()
        for s in range(S):
            for x, y in zip(now, states[at[s]]):
                assert torch.equal(x[s], y[s]), f"state of request {s} behind step {step}"
    assert counts >= {1, 2, 3, DRAFTS + 1}
