"""Timed cases of the operators of recurrent layers and of drafted tokens, from
one decoded token to long prompts.

A case is a dict of plain values; its "kind" says which call it makes:

  conv    kvmem_hip_conv_rows: short causal convolution of a recurrent layer's
          projections with its state, SiLU, L2 norm of the query and key heads
  linear  kvmem_hip_linear_attention: attention through a decaying state per head
          (with the delta rule where the case has "delta"), token by token for few
          tokens a request, in chunks for prompts
  verify  kvmem_hip_verify_draft: drafted tokens accepted or refused against the
          target's probabilities, and the next token, from given random numbers

`own` False computes the same in elementary torch operations.
"""
from __future__ import annotations

import functools
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1.0e-6
CHUNK = 64
# (key heads, value heads, key head size, value head size) of a recurrent layer
HEADS = [(16, 48, 128, 128), (16, 48, 128, 128), (16, 32, 128, 128), (8, 8, 64, 64), (4, 16, 128, 64),
         (4, 8, 256, 256), (2, 6, 64, 128), (1, 5, 128, 256)]


def listed() -> list[dict]:
    return [
        # one decoded token behind the fused projection of 16 + 16 + 48 heads of 128
        dict(name="conv_decode_1", kind="conv", seqs=1, tokens=1, keep=False, channels=10240, width=4, norm=4096,
             norm_dim=128, silu=True, bias=False, type="bf16", stored=True),
        # six tokens (one sampled, five drafted) of 32 requests, the accepted ones kept
        dict(name="conv_draft_32x6", kind="conv", seqs=32, tokens=6, keep=True, channels=10240, width=4, norm=4096,
             norm_dim=128, silu=True, bias=True, type="f16", stored=True),
        # a prompt of the same layer
        dict(name="conv_prompt_8k", kind="conv", seqs=1, tokens=8191, keep=False, channels=10240, width=4, norm=4096,
             norm_dim=128, silu=True, bias=False, type="bf16", stored=True),
        # one decoded token: 48 states of 128 x 128
        dict(name="linear_decode_1", kind="linear", seqs=1, tokens=1, keep=False, heads_k=16, heads=48, dim_k=128,
             dim_v=128, delta=True, decay="token", type="bf16", out="bf16"),
        # a decode batch of 64 requests
        dict(name="linear_decode_64", kind="linear", seqs=64, tokens=1, keep=False, heads_k=16, heads=48, dim_k=128,
             dim_v=128, delta=True, decay="token", type="bf16", out="bf16"),
        # the sampled and five drafted tokens of eight requests, the accepted ones folded in
        dict(name="linear_draft_8x6", kind="linear", seqs=8, tokens=6, keep=True, heads_k=16, heads=48, dim_k=128,
             dim_v=128, delta=True, decay="token", type="bf16", out="f32"),
        # a user's turn, ragged over four requests: heads of 64 keys, decay alone
        dict(name="linear_turn_4x1k", kind="linear", seqs=4, tokens=1021, keep=False, heads_k=8, heads=8, dim_k=64,
             dim_v=64, delta=False, decay="head", type="f16", out="f16"),
        # a prompt through one layer of the delta rule
        dict(name="linear_prompt_8k", kind="linear", seqs=1, tokens=8192, keep=False, heads_k=16, heads=48, dim_k=128,
             dim_v=128, delta=True, decay="token", type="bf16", out="bf16"),
        # a prefill batch of eight ragged prompts
        dict(name="linear_prompt_8x4k", kind="linear", seqs=8, tokens=4096, keep=False, heads_k=16, heads=32,
             dim_k=128, dim_v=128, delta=True, decay="token", type="bf16", out="bf16"),
        # five drafts of one request, drawn without probabilities (a lookup in the text so far)
        dict(name="verify_1x5", kind="verify", seqs=1, drafts=5, vocab=131072, type="bf16", probs=False),
        # three drafts of 16 requests with the drafter's probabilities, rows of an odd vocabulary
        dict(name="verify_16x3", kind="verify", seqs=16, drafts=3, vocab=50001, type="f32", probs=True),
        # a large batch, seven drafts each
        dict(name="verify_64x7", kind="verify", seqs=64, drafts=7, vocab=152000, type="bf16", probs=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["conv", "conv", "linear", "linear", "linear", "linear", "verify", "verify"])
    if kind == "conv":
        while True:
            heads_k, heads, dim_k, dim_v = rng.choice(HEADS)
            seqs, tokens = _log_int(rng, 1, 256), rng.choice([1, rng.randrange(2, 10), _log_int(rng, 10, 8192)])
            channels = 2 * heads_k * dim_k + heads * dim_v
            if seqs * tokens * channels <= 8191 * 10240:
                break
        norm = rng.random() < 0.8
        return dict(kind=kind, seqs=seqs, tokens=tokens, keep=tokens > 1 and rng.random() < 0.3, channels=channels,
                    width=rng.choice([4, 4, 4, 2, 3, 5, 8]), norm=2 * heads_k * dim_k if norm else 0,
                    norm_dim=dim_k if norm else 0, silu=rng.random() < 0.9, bias=rng.random() < 0.4,
                    type=rng.choice(["bf16", "bf16", "f16", "f32"]), stored=rng.random() < 0.9)
    if kind == "linear":
        while True:
            heads_k, heads, dim_k, dim_v = rng.choice(HEADS)
            seqs = _log_int(rng, 1, 128)
            tokens = rng.choice([1, 1, rng.randrange(2, 20), _log_int(rng, 20, 16384), _log_int(rng, 20, 16384)])
            if seqs * tokens * heads * dim_k * dim_v <= 8192 * 48 * 128 * 128 and \
                    seqs * heads * dim_k * dim_v <= 64 * 48 * 128 * 128:
                break
        type_ = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
        return dict(kind=kind, seqs=seqs, tokens=tokens, keep=tokens > 1 and rng.random() < 0.3, heads_k=heads_k,
                    heads=heads, dim_k=dim_k, dim_v=dim_v, delta=rng.random() < 0.7,
                    decay=rng.choice(["token", "token", "token", "head", "none"]), type=type_,
                    out=rng.choice([type_, type_, "f32"]))
    while True:
        seqs, drafts, vocab = _log_int(rng, 1, 128), rng.choice([0, 1, 3, 5, rng.randrange(2, 13)]), \
            _log_int(rng, 1000, 260000)
        if seqs * (drafts + 1) * vocab <= 64 * 8 * 152000:
            break
    return dict(kind=kind, seqs=seqs, drafts=drafts, vocab=vocab, type=rng.choice(["bf16", "bf16", "f16", "f32"]),
                probs=rng.random() < 0.6)


# ------------------------------------------------------------------ shapes
def _spread(n: int, most: int, least: int) -> list[int]:
    """n ragged lengths up to `most`, the first the largest: most times the
    fractional parts of golden-ratio steps."""
    return [most if i == 0 else max(least, int(most * ((i * 0.6180339887498949) % 1.0))) for i in range(n)]


def _lengths(case) -> tuple[list[int], list[int]]:
    """(tokens, tokens that take part) of every request."""
    m = _spread(case["seqs"], case["tokens"], 1) if case["tokens"] > 9 else [case["tokens"]] * case["seqs"]
    use = [1 + (5 * i + 2) % n for i, n in enumerate(m)] if case["keep"] else m
    return m, use


def work(case) -> dict:
    if case["kind"] == "conv":
        e, C, W = SIZES[case["type"]], case["channels"], case["width"]
        n = sum(_lengths(case)[1])
        state = 2 * case["seqs"] * (W - 1) * C * e if case["stored"] else 0
        return {"bytes": 2 * n * C * e + state + 4 * C * W, "flops": n * C * (2 * W + (4 if case["silu"] else 0))}
    if case["kind"] == "linear":
        e, n = SIZES[case["type"]], sum(_lengths(case)[1])
        Hk, H, Dk, Dv = case["heads_k"], case["heads"], case["dim_k"], case["dim_v"]
        gates = 4 * H * ((case["decay"] == "token") + case["delta"])
        bytes_ = n * (2 * Hk * Dk * e + H * Dv * (e + SIZES[case["out"]]) + gates) + 8 * case["seqs"] * H * Dk * Dv
        return {"bytes": bytes_, "flops": n * H * Dk * Dv * (6 if case["delta"] else 4)}
    e, S, rows = SIZES[case["type"]], case["seqs"], case["seqs"] * (case["drafts"] + 1)
    # every logit once; a refusing row's draft probabilities (all of them where drafts are as good as here)
    more = 4 * case["vocab"] * (S // 2 if case["probs"] and case["drafts"] else 0)
    return {"bytes": rows * case["vocab"] * e + more + 8 * rows + 8 * S, "flops": 4 * rows * case["vocab"]}


# ------------------------------------------------------------------ inputs
def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _batch(case, g) -> dict:
    """Starts, used tokens and state slots (in no order, two of them unused) of a batch."""
    m, use = _lengths(case)
    starts = [0]
    for k in m:
        starts.append(starts[-1] + k)
    S = case["seqs"]
    return dict(S=S, N=starts[-1], max_q=max(m), n_slots=S + 2, q_start=_int32(starts),
                n_use=_int32(use) if case["keep"] else None,
                slots=torch.randperm(S + 2, generator=g, device="cuda")[:S].to(torch.int32))


def _conv_state(case, g) -> dict:
    b, C, W, dt = _batch(case, g), case["channels"], case["width"], DTYPES[case["type"]]
    # the projection's rows hold the layer's other projections behind the convolved channels
    x = torch.randn((b["N"], C + 64), generator=g, device="cuda").to(dt)
    state = torch.randn((b["n_slots"], W - 1, C), generator=g, device="cuda").to(dt) if case["stored"] else None
    out = dict(out=torch.zeros((b["N"], C), dtype=dt, device="cuda"))
    if case["stored"]:
        out["state"] = torch.zeros_like(state)
    return dict(kind="conv", **b, C=C, W=W, type=case["type"], norm=case["norm"], norm_dim=case["norm_dim"],
                silu=case["silu"], x=x, state=state, out=out,
                weight=torch.randn((C, W), generator=g, device="cuda") / math.sqrt(W),
                bias=0.1 * torch.randn(C, generator=g, device="cuda") if case["bias"] else None)


def _linear_state(case, g) -> dict:
    b, dt = _batch(case, g), DTYPES[case["type"]]
    N, Hk, H, Dk, Dv = b["N"], case["heads_k"], case["heads"], case["dim_k"], case["dim_v"]

    def unit(x):
        return (x / x.norm(dim=-1, keepdim=True)).to(dt)

    # a token's queries, keys and values side by side; a head's keys share a direction
    rows = torch.empty((N, 2 * Hk * Dk + H * Dv), dtype=dt, device="cuda")
    q, k, v = (t.view(N, -1, d) for t, d in zip(rows.split([Hk * Dk, Hk * Dk, H * Dv], 1), (Dk, Dk, Dv)))
    q.copy_(unit(torch.randn(q.shape, generator=g, device="cuda")))
    k.copy_(unit(torch.randn(k.shape, generator=g, device="cuda") +
                 0.7 * torch.randn((1, Hk, Dk), generator=g, device="cuda")))
    v.copy_(torch.randn(v.shape, generator=g, device="cuda").to(dt))
    decay = beta = None
    rate = 16.0 * torch.rand(H, generator=g, device="cuda") ** 3 + 0.001
    if case["decay"] == "token":
        x = torch.randn((N, H), generator=g, device="cuda") - 3.0
        decay = -rate * torch.log1p(torch.exp(x))
    elif case["decay"] == "head":
        decay = -0.05 * rate
    if case["delta"]:
        beta = torch.sigmoid(torch.randn((N, H), generator=g, device="cuda"))
    state = 0.3 * torch.randn((b["n_slots"], H, Dk, Dv), generator=g, device="cuda")
    return dict(kind="linear", **b, Hk=Hk, H=H, Dk=Dk, Dv=Dv, type=case["type"], out_type=case["out"], q=q, k=k, v=v,
                decay=decay, beta=beta, state=state,
                out=dict(out=torch.zeros((N, H, Dv), dtype=DTYPES[case["out"]], device="cuda"),
                         state=torch.zeros_like(state)))


def _verify_state(case, g) -> dict:
    S, M, V, dt = case["seqs"], case["drafts"], case["vocab"], DTYPES[case["type"]]
    rows = S * (M + 1)
    # a few likely tokens over a long tail; the drafter is nearly the target
    logits = 2.0 * torch.randn((rows, V), generator=g, device="cuda")
    logits.scatter_add_(1, torch.randint(0, V, (rows, 8), generator=g, device="cuda"),
                        16.0 * torch.rand((rows, 8), generator=g, device="cuda"))
    guess = logits + 0.3 * torch.randn((rows, V), generator=g, device="cuda")
    temperature = torch.tensor([(1.0, 0.7, 0.0, 1.3)[i % 4] for i in range(S)], device="cuda")
    drafted = torch.softmax(guess / temperature.clamp_min(0.25).repeat_interleave(M + 1)[:, None], -1)
    picks = torch.multinomial(drafted, 1, generator=g)[:, 0]
    tokens = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), picks[:-1]]).to(torch.int32)
    n = dict(n_accepted=torch.empty(S, dtype=torch.int32, device="cuda"),
             n_keep=torch.empty(S, dtype=torch.int32, device="cuda"),
             tokens=torch.empty((S, M + 1), dtype=torch.int32, device="cuda"))
    return dict(kind="verify", S=S, M=M, V=V, type=case["type"], logits=logits.to(dt),
                probs=drafted if case["probs"] else None, tokens=tokens, temperature=temperature,
                q_start=_int32([i * (M + 1) for i in range(S + 1)]),
                u_accept=torch.rand(rows, generator=g, device="cuda"),
                u_sample=torch.rand(S, generator=g, device="cuda"), out=n)


def prepare(case, seed) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"conv": _conv_state, "linear": _linear_state, "verify": _verify_state}[case["kind"]](case, g)


# -------------------------------------------------------------- plain forms
def _padded(s):
    """Row index and whether it takes part, [requests, longest], and the requests' counts."""
    start = s["q_start"].long()
    n = start[1:] - start[:-1]
    use = n if s["n_use"] is None else torch.minimum(n, s["n_use"].long())
    i = torch.arange(s["max_q"], device="cuda")
    live = i < use[:, None]
    return torch.where(live, start[:-1, None] + i, 0), live, use


def _plain_conv(s):
    W, C, out = s["W"], s["C"], s["out"]
    at, live, use = _padded(s)
    slots = s["slots"].long()
    x = torch.where(live[..., None], s["x"][at, :C].float(), 0.0)
    before = torch.zeros((s["S"], W - 1, C), device="cuda") if s["state"] is None else s["state"][slots].float()
    x = torch.cat([before, x], 1)
    y = sum(x[:, j:j + s["max_q"]] * s["weight"][:, j] for j in range(W))
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["silu"]:
        y = y / (1.0 + torch.exp(-y))
    if s["norm"]:
        heads = y[..., :s["norm"]].unflatten(-1, (-1, s["norm_dim"]))
        heads = heads * torch.rsqrt((heads * heads).sum(-1, keepdim=True) + EPS)
        y = torch.cat([heads.flatten(-2), y[..., s["norm"]:]], -1)
    out["out"][at[live]] = y[live].to(out["out"].dtype)
    if s["state"] is not None:
        last = use[:, None] + torch.arange(W - 1, device="cuda")
        out["state"][slots] = x.gather(1, last[..., None].expand(-1, -1, C)).to(out["state"].dtype)
    return out


def _plain_linear(s):
    S, H, Dk, Dv, out = s["S"], s["H"], s["Dk"], s["Dv"], s["out"]
    at, live, _ = _padded(s)
    C = min(CHUNK, s["max_q"])
    n = -(-s["max_q"] // C)

    def chunks(x, fill=0.0):  # [tokens, heads, ...] -> [chunks, requests * heads, C, ...]
        x = torch.where(live.view(*live.shape, *([1] * (x.ndim - 1))), x[at], fill)
        x = torch.nn.functional.pad(x, [0, 0] * (x.ndim - 2) + [0, n * C - x.shape[1]])
        x = x.unflatten(1, (n, C)).movedim(1, 0).movedim(3, 2)
        return x.repeat_interleave(H // x.shape[2], 2).flatten(1, 2).contiguous()

    q, k, v = (chunks(s[x].float()) for x in "qkv")
    zero = torch.zeros((s["N"], H), dtype=torch.float64, device="cuda")
    g = zero if s["decay"] is None else zero + s["decay"].double()
    G = chunks(g).cumsum(-1)
    later = torch.ones((C, C), dtype=torch.bool, device="cuda").triu(1)
    decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(later, -math.inf)).float()
    from_first, to_last = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None]
    whole = torch.exp(G[..., -1]).float()[..., None, None]
    scores = q @ k.mT.contiguous() * decay
    kd, solve, beta = (k * to_last).mT.contiguous(), None, None
    if s["beta"] is not None:
        beta = chunks(s["beta"])[..., None]
        A = k @ k.mT.contiguous() * decay * beta
        solve = torch.eye(C, device="cuda").expand_as(A).contiguous()
        for i in range(1, C):
            solve[..., i, :i] = -(A[..., i, None, :i] @ solve[..., :i, :i])[..., 0, :]
    slots = s["slots"].long()
    state, o = s["state"][slots].flatten(0, 1), []
    for c in range(n):
        d = v[c]
        if solve is not None:
            d = solve[c] @ (beta[c] * (d - from_first[c] * (k[c] @ state)))
        o.append(from_first[c] * (q[c] @ state) + scores[c] @ d)
        state = whole[c] * state + kd[c] @ d
    o = torch.cat(o, 1).view(S, H, n * C, Dv)[:, :, :s["max_q"]].movedim(1, 2) / math.sqrt(Dk)
    out["out"][at[live]] = o[live].to(out["out"].dtype)
    out["state"][slots] = state.view(S, H, Dk, Dv)
    return out


def _plain_verify(s):
    S, M, V, out = s["S"], s["M"], s["V"], s["out"]
    x, t = s["logits"].view(S, M + 1, V).double(), s["temperature"].double()
    # a temperature of 0 leaves the largest logit alone (the lowest index of equal ones)
    best = x == x.amax(-1, keepdim=True)
    best = best & (torch.arange(V, device="cuda") == best.int().argmax(-1, keepdim=True))
    greedy = (t == 0.0)[:, None, None]
    p = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(t == 0.0, 1.0, t)[:, None, None])
    p = torch.where(greedy, best.double(), p / p.sum(-1, keepdim=True))
    draft = s["tokens"].view(S, M + 1).long()[:, 1:]
    p_draft = p[:, :M].gather(2, draft[..., None])[..., 0]
    q_draft = torch.ones_like(p_draft)
    if s["probs"] is not None:
        probs = s["probs"].view(S, M + 1, V).double()
        q_draft = torch.where(greedy[..., 0], q_draft, probs[:, :M].gather(2, draft[..., None])[..., 0])
    ok = s["u_accept"].view(S, M + 1)[:, :M].double() * q_draft < p_draft
    count = ok.int().cumprod(-1).sum(-1)
    r = torch.arange(S, device="cuda")
    w, refused = p[r, count], count < M
    if M:
        at = draft[r, count.clamp(max=M - 1)]
        alone = (torch.arange(V, device="cuda") == at[:, None]).double()
        if s["probs"] is not None:
            alone = torch.where(greedy[:, 0], alone, probs[r, count])
        rest = torch.where(alone == 1.0, 0.0, (w - alone).clamp_min(0.0)) if s["probs"] is None else \
            (w - alone).clamp_min(0.0)
        w = torch.where((refused & (rest.sum(-1) > 0.0))[:, None], rest, w)
    c = w.cumsum(-1)
    beyond = (c > s["u_sample"].double()[:, None] * c[:, -1:]) & (w > 0.0)
    token = beyond.int().argmax(-1)
    i = torch.arange(M + 1, device="cuda")
    drafts = torch.nn.functional.pad(draft, (0, 1))
    got = torch.where(i < count[:, None], drafts, torch.where(i == count[:, None], token[:, None], -1))
    out["tokens"].copy_(got)
    out["n_accepted"].copy_(count)
    out["n_keep"].copy_(count + 1)
    return out


# ----------------------------------------------------------- the framework's
@functools.lru_cache(maxsize=None)
def _framework():
    """The package and one context, which every state's calls run on."""
    if "kvmem_amd" not in sys.modules:
        pkg = ROOT / "kvmem-llama.cpp_amd"
        spec = importlib.util.spec_from_file_location("kvmem_amd", pkg / "__init__.py",
                                                      submodule_search_locations=[str(pkg)])
        sys.modules["kvmem_amd"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["kvmem_amd"])
    kv = sys.modules["kvmem_amd"]
    return kv, kv.Context(0)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _type(kv, name):
    return {"f32": kv.TYPE_F32, "f16": kv.TYPE_F16, "bf16": kv.TYPE_BF16}[name]


def _own_conv(s):
    kv, ctx = _framework()
    o = s["out"]
    args = kv.ConvArgs(x=s["x"].data_ptr(), type=_type(kv, s["type"]), x_nb=s["x"].stride(0) * s["x"].element_size(),
                       n_tokens=s["N"], n_seq=s["S"], max_q=s["max_q"], n_channels=s["C"], width=s["W"],
                       n_slots=s["n_slots"], weight=s["weight"].data_ptr(), bias=_ptr(s["bias"]), silu=int(s["silu"]),
                       norm_channels=s["norm"], norm_dim=s["norm_dim"], eps=EPS, q_start=s["q_start"].data_ptr(),
                       n_use=_ptr(s["n_use"]), slots=s["slots"].data_ptr(), state=_ptr(s["state"]),
                       state_out=_ptr(o.get("state")), out=o["out"].data_ptr())
    return functools.partial(ctx.conv_rows, args), o


def _own_linear(s):
    kv, ctx = _framework()
    o, e = s["out"], s["q"].element_size()
    args = kv.LinearArgs(type=_type(kv, s["type"]), out_type=_type(kv, s["out_type"]), n_tokens=s["N"], n_seq=s["S"],
                         max_q=s["max_q"], n_head_k=s["Hk"], n_head=s["H"], head_dim_k=s["Dk"], head_dim_v=s["Dv"],
                         n_slots=s["n_slots"], log_decay=_ptr(s["decay"]),
                         decay_nb=0 if s["decay"] is None or s["decay"].ndim == 1 else 4 * s["H"],
                         beta=_ptr(s["beta"]), beta_nb=0 if s["beta"] is None else 4 * s["H"],
                         q_start=s["q_start"].data_ptr(), n_use=_ptr(s["n_use"]), slots=s["slots"].data_ptr(),
                         state=s["state"].data_ptr(), state_out=o["state"].data_ptr(), out=o["out"].data_ptr(),
                         **{n: s[n].data_ptr() for n in "qkv"},
                         **{f"{n}_nb{d}": e * s[n].stride(2 - d) for n in "qkv" for d in (1, 2)})
    return functools.partial(ctx.linear_attention, args), o


def _own_verify(s):
    kv, ctx = _framework()
    o = s["out"]
    args = kv.VerifyArgs(logits=s["logits"].data_ptr(), type=_type(kv, s["type"]),
                         logits_nb=s["logits"].stride(0) * s["logits"].element_size(),
                         probs=_ptr(s["probs"]), probs_type=kv.TYPE_F32, probs_nb=4 * s["V"], n_vocab=s["V"],
                         n_rows=s["S"] * (s["M"] + 1), n_seq=s["S"], max_draft=s["M"],
                         q_start=s["q_start"].data_ptr(), tokens=s["tokens"].data_ptr(),
                         temperature=s["temperature"].data_ptr(), u_accept=s["u_accept"].data_ptr(),
                         u_sample=s["u_sample"].data_ptr(), tokens_out=o["tokens"].data_ptr(),
                         n_accepted=o["n_accepted"].data_ptr(), n_keep=o["n_keep"].data_ptr())
    return functools.partial(ctx.verify_draft, args), o


def run(state):
    if own:
        if "call" not in state:  # the argument block a program builds once for its buffers
            state["call"] = {"conv": _own_conv, "linear": _own_linear, "verify": _own_verify}[state["kind"]](state)
        call, out = state["call"]
        call()
        return out
    return {"conv": _plain_conv, "linear": _plain_linear, "verify": _plain_verify}[state["kind"]](state)


# -------------------------------------------------------------------- exact
def exact(case, seed):
    """What run() returns, in float64 from the definitions: the convolution request by
    request and tap by tap, the linear attention's state token by token."""
    if case["kind"] == "verify":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_conv(s) if case["kind"] == "conv" else _exact_linear(s)


def _exact_conv(s):
    out = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for n, t in s["out"].items()}
    starts, slots = s["q_start"].tolist(), s["slots"].tolist()
    use = [b - a for a, b in zip(starts, starts[1:])] if s["n_use"] is None else s["n_use"].tolist()
    for r in range(s["S"]):
        a, n = starts[r], use[r]
        rows = [torch.zeros((s["W"] - 1, s["C"]), dtype=torch.float64, device="cuda") if s["state"] is None
                else s["state"][slots[r]].double(), s["x"][a:a + n, :s["C"]].double()]
        x = torch.cat(rows)
        y = torch.zeros((n, s["C"]), dtype=torch.float64, device="cuda")
        if s["bias"] is not None:
            y += s["bias"].double()
        for tap in range(s["W"]):
            y.addcmul_(x[tap:tap + n], s["weight"][:, tap].double().expand(n, -1))
        if s["silu"]:
            y *= torch.sigmoid(y)
        for h in range(0, s["norm"], s["norm_dim"] or 1):
            head = y[:, h:h + s["norm_dim"]]
            head /= (torch.linalg.vector_norm(head, dim=1, keepdim=True) ** 2 + EPS).sqrt()
        out["out"][a:a + n] = y
        if s["state"] is not None:
            out["state"][slots[r]] = x[n:]
    return out


def _exact_linear(s):
    S, H, grp = s["S"], s["H"], s["H"] // s["Hk"]
    out = {n: torch.zeros(t.shape, dtype=torch.float64, device="cuda") for n, t in s["out"].items()}
    start, slots = s["q_start"][:-1].long(), s["slots"].long()
    n = s["q_start"][1:].long() - start
    use = n if s["n_use"] is None else s["n_use"].long()
    state = s["state"][slots].double()
    head = torch.arange(H, device="cuda") // grp
    for t in range(int(use.max())):
        on = torch.nonzero(use > t)[:, 0]
        at, all_on = start[on] + t, on.numel() == S
        q, k, v = s["q"][at][:, head].double(), s["k"][at][:, head].double(), s["v"][at].double()
        now = state if all_on else state[on]
        if s["decay"] is not None:
            g = s["decay"][at] if s["decay"].ndim == 2 else s["decay"][None]
            now = now * torch.exp(g.double())[..., None, None]
        if s["beta"] is not None:
            v = s["beta"][at].double()[..., None] * (v - torch.matmul(k[..., None, :], now)[..., 0, :])
        now = now + k[..., None] * v[..., None, :]
        out["out"][at] = torch.matmul(q[..., None, :], now)[..., 0, :] / s["Dk"] ** 0.5
        if all_on:
            state = now
        else:
            state[on] = now
    out["state"][slots] = state
    return out
