"""Timed cases of the operators that write new tokens into the KV window and
attend over it, from one decoded token to long prompts.

A case is a dict of plain values; its "kind" says which call it makes:

  slots      kvmem_hip_slot_map: block tables, cells and positions of the new
             tokens of a batch of requests, from their lengths
  rows       kvmem_hip_qkv_rows: per-head RMS norm of queries and keys, RoPE and
             Walsh-Hadamard rotation, keys and values into the cache
  attention  kvmem_hip_attention: new queries over the cached blocks of their
             requests (q4_0, q5_0, q8_0 or f16 rows)

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
GROUP_BYTES = {"q8_0": 34, "q5_0": 22, "q4_0": 18, "f16": 64}
FREQ_BASE = 1.0e6
EPS = 1.0e-6
# (query heads, KV heads, head size): the reselect workloads' heads, the timed cases'
# other geometries, narrow heads, and one KV head
GEOMETRIES = [(24, 4, 256), (24, 4, 256), (32, 8, 128), (8, 2, 128), (16, 4, 256), (16, 2, 128), (16, 2, 64),
              (7, 1, 128)]


def listed() -> list[dict]:
    return [
        # one decode step of a small batch: one new token each
        dict(name="slots_decode_8", kind="slots", seqs=8, new=1, kv=32768, block_tokens=128),
        # a prefill batch of many ragged prompts, finer blocks
        dict(name="slots_prefill_256", kind="slots", seqs=256, new=509, kv=8000, block_tokens=32),
        # one decoded token behind a fused projection; the rows also feed the query window
        # and the raw history
        dict(name="rows_decode_1", kind="rows", tokens=1, heads=24, kv_heads=4, head_dim=256, n_rot=64, type="bf16",
             norm=True, hadamard=False, capture=True, max_pos=262144),
        # a decode batch of 96 requests, 128-wide heads rotated over their whole width
        dict(name="rows_batch_96", kind="rows", tokens=96, heads=32, kv_heads=8, head_dim=128, n_rot=128,
             type="f16", norm=True, hadamard=False, capture=False, max_pos=131072),
        # a prefill batch of the reselect workloads' heads
        dict(name="rows_prefill_8k", kind="rows", tokens=8191, heads=24, kv_heads=4, head_dim=256, n_rot=64,
             type="bf16", norm=True, hadamard=False, capture=False, max_pos=1048576),
        # an agent's first turns: one token over a short window
        dict(name="decode_2k", kind="attention", seqs=1, q_tokens=1, kv=2011, heads=24, kv_heads=4, head_dim=256,
             block_tokens=128, type_k="q4_0", type_v="q4_0", q_type="bf16", hadamard=True),
        # one token over the full 256-block window
        dict(name="decode_32k", kind="attention", seqs=1, q_tokens=1, kv=32768, heads=24, kv_heads=4, head_dim=256,
             block_tokens=128, type_k="q4_0", type_v="q4_0", q_type="bf16", hadamard=True),
        # a decode batch of ragged requests, 128-wide heads in smaller blocks
        dict(name="decode_batch_32", kind="attention", seqs=32, q_tokens=1, kv=16384, heads=32, kv_heads=8,
             head_dim=128, block_tokens=64, type_k="q4_0", type_v="q4_0", q_type="f16", hadamard=False),
        # one token over the 512-block budget of a 1M-token session, mixed-precision cache
        dict(name="decode_mixed_64k", kind="attention", seqs=1, q_tokens=1, kv=65500, heads=24, kv_heads=4,
             head_dim=256, block_tokens=128, type_k="q8_0", type_v="q4_0", q_type="bf16", hadamard=True),
        # five drafted tokens of eight requests checked in one call, 64-wide heads
        dict(name="draft_5", kind="attention", seqs=8, q_tokens=5, kv=8192, heads=16, kv_heads=2, head_dim=64,
             block_tokens=32, type_k="q5_0", type_v="q5_0", q_type="bf16", hadamard=False),
        # a user's turn of 512 tokens over the full window
        dict(name="prefill_512_32k", kind="attention", seqs=1, q_tokens=512, kv=32768, heads=24, kv_heads=4,
             head_dim=256, block_tokens=128, type_k="q4_0", type_v="q4_0", q_type="bf16", hadamard=True),
        # prompts from their first token: four ragged requests into an empty f16 window
        dict(name="prompt_4x2k", kind="attention", seqs=4, q_tokens=2048, kv=2048, heads=32, kv_heads=8,
             head_dim=128, block_tokens=128, type_k="f16", type_v="f16", q_type="bf16", hadamard=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["slots", "rows", "rows", "attention", "attention", "attention", "attention"])
    heads, kv_heads, head_dim = rng.choice(GEOMETRIES)
    if kind == "slots":
        seqs = _log_int(rng, 1, 512)
        return dict(kind=kind, seqs=seqs, new=rng.choice([1, 1, _log_int(rng, 2, 130000 // seqs)]),
                    kv=_log_int(rng, 1, min(131072, 2048000 // seqs)), block_tokens=rng.choice([128, 128, 64, 32, 16, 80]))
    if kind == "rows":
        return dict(kind=kind, tokens=_log_int(rng, 1, 6000), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    n_rot=rng.choice([0, 32, 64, head_dim, head_dim]), type=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    norm=rng.random() < 0.8, hadamard=rng.random() < 0.3, capture=rng.random() < 0.3,
                    max_pos=_log_int(rng, 4096, 1048576))
    q_tokens = rng.choice([1, 1, 1, 1, rng.randrange(2, 9), _log_int(rng, 16, 1024)])
    while True:
        seqs, length = _log_int(rng, 1, 64), max(q_tokens, _log_int(rng, 1, 65536))
        small = seqs * length * kv_heads * head_dim <= 2 ** 27
        if small and q_tokens * heads * seqs * length * head_dim <= 512 * 24 * 32768 * 256:
            break
    type_k, type_v = rng.choice([("q4_0", "q4_0"), ("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q5_0", "q5_0"),
                                 ("q8_0", "q8_0"), ("f16", "f16")])
    return dict(kind=kind, seqs=seqs, q_tokens=q_tokens, kv=length, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, block_tokens=rng.choice([128, 128, 64, 32, 16, 80]), type_k=type_k, type_v=type_v,
                q_type=rng.choice(["bf16", "bf16", "f16"]) if q_tokens == 1 else "bf16",
                hadamard=type_k != "f16" and rng.random() < 0.6)


# ------------------------------------------------------------------ shapes
def _spread(n: int, most: int, least: int) -> list[int]:
    """n ragged lengths up to `most`, the first the largest: most times the
    fractional parts of golden-ratio steps."""
    return [most if i == 0 else max(least, int(most * ((i * 0.6180339887498949) % 1.0))) for i in range(n)]


def _lengths(case) -> tuple[list[int], list[int]]:
    """(keys, query tokens) of every request; the keys include the new tokens."""
    m = _spread(case["seqs"], case["q_tokens"], 1)
    return [max(k, q) for k, q in zip(_spread(case["seqs"], case["kv"], 1), m)], m


def _theta(n_rot: int) -> torch.Tensor:
    i = torch.arange(n_rot // 2, dtype=torch.float64)
    return torch.pow(torch.tensor(FREQ_BASE, dtype=torch.float64), -2.0 * i / max(1, n_rot)).to(torch.float32)


def _hadamard(width: int, dtype) -> torch.Tensor:
    h = torch.ones((1, 1), dtype=dtype, device="cuda")
    while h.shape[0] < width:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(width)


def work(case) -> dict:
    if case["kind"] == "slots":
        n, m = _slot_lengths(case)
        T = case["block_tokens"]
        blocks = sum(-(-(a + b) // T) - -(-a // T) for a, b in zip(n, m))
        # lengths, new counts and first positions in, new lengths and starts out; the free
        # slots in, the table entries out; a position and a cell a token
        return {"bytes": 4 * (5 * case["seqs"] + 2 * blocks + 2 * sum(m)), "flops": 0}
    D, Hq, Hkv = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "rows":
        e = 4 if case["type"] == "f32" else 2
        q, k = case["tokens"] * Hq * D, case["tokens"] * Hkv * D
        more = e * (q + k) if case["capture"] else 0
        return {"bytes": e * (q + 2 * k) + e * q + 4 * k + more + 8 * case["tokens"], "flops": 10 * (q + k)}
    lens, m = _lengths(case)
    row = Hkv * D // 32 * (GROUP_BYTES[case["type_k"]] + GROUP_BYTES[case["type_v"]])
    pairs = sum(sum(L - k + i + 1 for i in range(k)) for L, k in zip(lens, m))
    return {"bytes": sum(lens) * row + sum(m) * Hq * D * 4, "flops": 4 * D * Hq * pairs}


def _slot_lengths(case) -> tuple[list[int], list[int]]:
    """(cached, new) tokens of every request; some have nothing cached, some bring nothing."""
    n = [0 if i % 7 == 3 else v for i, v in enumerate(_spread(case["seqs"], case["kv"], 0))]
    m = [0 if i % 11 == 5 else v for i, v in enumerate(_spread(case["seqs"], case["new"], 1))]
    return n, m


# ------------------------------------------------------------------ inputs
def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantize(x: torch.Tensor, type_: str) -> torch.Tensor:
    """Rows of f32 values [..., n] as the cache holds them: uint8 [..., bytes], ggml's formats."""
    if type_ == "f16":
        return x.half().view(torch.uint8)
    g = x.view(*x.shape[:-1], -1, 32)
    if type_ == "q8_0":
        d = g.abs().amax(-1, keepdim=True) / 127.0
        c = torch.round(g / d.clamp_min(1e-30)).to(torch.int8).view(torch.uint8)
        out = torch.cat([d.half().view(torch.uint8), c], -1)
    else:
        half = 8 if type_ == "q4_0" else 16
        d = g.gather(-1, g.abs().argmax(-1, keepdim=True)) / -half
        inv = torch.where(d == 0, d, 1.0 / d)
        c = (g * inv + (half + 0.5)).to(torch.int32).clamp_(0, 2 * half - 1)
        qs = (c[..., :16] & 15) | ((c[..., 16:] & 15) << 4)
        parts = [d.half().view(torch.uint8)]
        if type_ == "q5_0":
            bits = (c >> 4).view(*c.shape[:-1], 4, 8) << torch.arange(8, device="cuda")
            parts.append(bits.sum(-1).to(torch.uint8))
        out = torch.cat([*parts, qs.to(torch.uint8)], -1)
    return out.flatten(-2)


def _slot_state(case, g) -> dict:
    n, m = _slot_lengths(case)
    T, S = case["block_tokens"], case["seqs"]
    held = [-(-a // T) for a in n]
    need = [-(-(a + b) // T) for a, b in zip(n, m)]
    stride = max(1, max(need) + 2)
    n_slots = sum(need) + 7
    order = torch.randperm(n_slots, generator=g, device="cuda").to(torch.int32)
    host = order.cpu()
    table = torch.full((S, stride), -1, dtype=torch.int32)
    at = 0
    for s in range(S):
        table[s, :held[s]] = host[at:at + held[s]]
        at += held[s]
    return dict(kind="slots", T=T, S=S, stride=stride, n_slots=n_slots, max_tokens=sum(m) + 5,
                n_new=_int32(m), kv_len=_int32(n), pos0=_int32([3 * a for a in n]), table=table.cuda(),
                free=order[at - 2 if at >= 2 else 0:].contiguous(), used=_int32([2 if at >= 2 else 0]),
                out=dict(kv_len=torch.empty(S, dtype=torch.int32, device="cuda"),
                         q_start=torch.empty(S + 1, dtype=torch.int32, device="cuda"),
                         positions=torch.empty(sum(m) + 5, dtype=torch.int32, device="cuda"),
                         cells=torch.empty(sum(m) + 5, dtype=torch.int32, device="cuda"),
                         used=torch.empty(1, dtype=torch.int32, device="cuda"),
                         missing=torch.empty(1, dtype=torch.int32, device="cuda")))


def _row_state(case, g) -> dict:
    N, Hq, Hkv, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    dt, T = DTYPES[case["type"]], 128
    # one projection's output holds a token's queries, keys and values side by side
    proj = torch.randn((N, (Hq + 2 * Hkv) * D), generator=g, device="cuda")
    proj[:, Hq * D::61] *= 8.0
    proj = proj.to(dt)
    q, k, v = (t.view(N, -1, D) for t in proj.split([Hq * D, Hkv * D, Hkv * D], 1))
    n_slots = -(-N // T) + 1
    cells = torch.randperm(n_slots * T, generator=g, device="cuda")[:N].to(torch.int32)
    cells[N - 1:] = cells[N - 1:] if N == 1 else -1  # the batch's last token is padding
    s = dict(kind="rows", q=q, k=k, v=v, n_slots=n_slots, T=T, n_rot=case["n_rot"], type=case["type"],
             theta=_theta(case["n_rot"]), theta_dev=_theta(case["n_rot"]).cuda(),
             had=D if case["hadamard"] else 0, had_v=64 if case["hadamard"] else 0, cells=cells,
             positions=torch.randint(0, case["max_pos"], (N,), generator=g, device="cuda", dtype=torch.int32),
             wq=1.0 + 0.1 * torch.randn(D, generator=g, device="cuda") if case["norm"] else None,
             wk=1.0 + 0.1 * torch.randn(D, generator=g, device="cuda") if case["norm"] else None)
    out = dict(q=torch.empty((N, Hq, D), dtype=dt, device="cuda"),
               pool_k=torch.zeros((n_slots * T, Hkv * D), dtype=torch.float16, device="cuda"),
               pool_v=torch.zeros((n_slots * T, Hkv * D), dtype=torch.float16, device="cuda"))
    if case["capture"]:
        out["q_norm"] = torch.empty((N, Hq, D), dtype=dt, device="cuda")
        out["k_norm"] = torch.empty((N, Hkv, D), dtype=dt, device="cuda")
    return {**s, "out": out}


def _attention_state(case, g) -> dict:
    lens, m = _lengths(case)
    T, S, Hq, Hkv, D = case["block_tokens"], case["seqs"], case["heads"], case["kv_heads"], case["head_dim"]
    held = [-(-a // T) for a in lens]
    n_slots, stride = sum(held) + 3, max(held) + 1
    slots = torch.randperm(n_slots, generator=g, device="cuda").to(torch.int32)
    host = slots.cpu()
    table = torch.full((S, stride), -1, dtype=torch.int32)
    at = 0
    for s in range(S):
        table[s, :held[s]] = host[at:at + held[s]]
        at += held[s]
    if max(held) > 8:
        table[0, 5] = -1  # a block the request has dropped
    pools = {}
    # the rows behind a request's last token, and the slots nobody holds, are all ones: NaN scales
    live = torch.zeros(n_slots * T, dtype=torch.bool)
    for s in range(S):
        for_s = torch.arange(lens[s])
        live[table[s, for_s // T].long() * T + for_s % T] = True
    live = live.cuda()
    for which, type_ in (("k", case["type_k"]), ("v", case["type_v"])):
        row = Hkv * D // 32 * GROUP_BYTES[type_]
        pool = torch.full((n_slots * T, row), 255, dtype=torch.uint8, device="cuda")
        step = max(1, 2 ** 24 // (Hkv * D))
        offset = 0.3 * torch.randn(Hkv * D, generator=g, device="cuda") if which == "k" else 0.0
        for c in range(0, n_slots * T, step):
            x = torch.randn((min(step, n_slots * T - c), Hkv * D), generator=g, device="cuda") + offset
            pool[c:c + step] = torch.where(live[c:c + step, None], _quantize(x, type_), pool[c:c + step])
        pools[which] = pool
    dt, N = DTYPES[case["q_type"]], sum(m)
    starts = [0]
    for k in m:
        starts.append(starts[-1] + k)
    return dict(kind="attention", S=S, N=N, T=T, Hq=Hq, Hkv=Hkv, D=D, n_slots=n_slots, stride=stride,
                max_q=max(m), max_kv=max(lens), type_k=case["type_k"], type_v=case["type_v"],
                q_type=case["q_type"], had_v=64 if case["hadamard"] else 0, k=pools["k"], v=pools["v"],
                table=table.cuda(), kv_len=_int32(lens), q_start=_int32(starts),
                q=(2.0 * torch.randn((N, Hq, D), generator=g, device="cuda")).to(dt),
                out=torch.empty((N, Hq, D), dtype=dt, device="cuda"))


def prepare(case, seed) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"slots": _slot_state, "rows": _row_state, "attention": _attention_state}[case["kind"]](case, g)


# -------------------------------------------------------------- plain forms
def _plain_slots(s) -> dict:
    T, stride, out = s["T"], s["stride"], s["out"]
    n, m, table = s["kv_len"].long(), s["n_new"].long(), s["table"].long()
    start = torch.cumsum(m, 0)
    b0, b1 = (n + T - 1) // T, (n + m + T - 1) // T
    need = b1.clamp(max=stride) - b0.clamp(max=stride)
    first = s["used"].long() + torch.cumsum(need, 0) - need
    j = torch.arange(stride, device="cuda")
    at = first[:, None] + j - b0[:, None]
    n_free = s["free"].numel()
    taken = torch.where(at < n_free, s["free"].long()[at.clamp(0, n_free - 1)], -1)
    table = torch.where((j >= b0[:, None]) & (j < b1[:, None]), taken, table)
    s["table"].copy_(table)
    t = torch.arange(s["max_tokens"], device="cuda")
    r = torch.searchsorted(start, t, right=True).clamp(max=s["S"] - 1)
    i = t - (start - m)[r]
    p = n[r] + i
    slot = torch.where(p // T < stride, table[r, (p // T).clamp(max=stride - 1)], -1)
    live = t < start[-1]
    out["kv_len"].copy_(n + m)
    out["q_start"].copy_(torch.cat([torch.zeros_like(start[:1]), start]))
    out["positions"].copy_(torch.where(live, s["pos0"].long()[r] + i, 0))
    out["cells"].copy_(torch.where(live & (slot >= 0), slot * T + p % T, -1))
    used = (s["used"].long() + need.sum()).clamp(max=n_free)
    out["used"].copy_(used)
    out["missing"].copy_((b1 - b0).sum() - (used - s["used"]))
    return {"table": s["table"], **out}


def _plain_norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_rope(x, positions, theta, n_rot):
    if n_rot == 0:
        return x
    # the cache's rows are rotated by the float32 product of position and frequency
    a = (positions.float()[:, None] * theta).double()
    c, sn, h = a.cos().float()[:, None], a.sin().float()[:, None], n_rot // 2
    x0, x1 = x[..., :h], x[..., h:n_rot]
    return torch.cat([x0 * c - x1 * sn, x0 * sn + x1 * c, x[..., n_rot:]], -1)


def _plain_walsh(x, width):
    if width == 0:
        return x
    return (x.unflatten(-1, (-1, width)) @ _hadamard(width, x.dtype)).flatten(-2)


def _plain_rows(s) -> dict:
    out = s["out"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    q, k = _plain_norm(q, s["wq"]), _plain_norm(k, s["wk"])
    if "q_norm" in out:
        out["q_norm"].copy_(q)
        out["k_norm"].copy_(k)
    q, k = (_plain_walsh(_plain_rope(x, s["positions"], s["theta_dev"], s["n_rot"]), s["had"]) for x in (q, k))
    v = _plain_walsh(v, s["had_v"])
    out["q"].copy_(q)
    # a token without a cell goes to a row of its own behind the cache
    n = s["n_slots"] * s["T"]
    cell = torch.where(s["cells"] >= 0, s["cells"], n).long()
    for name, x in (("pool_k", k), ("pool_v", v)):
        wide = torch.cat([out[name], out[name][:1]])
        wide[cell] = x.flatten(1).half()
        out[name].copy_(wide[:n])
    return out


def _plain_dequant(b, type_: str):
    """uint8 [..., bytes] -> f32 [..., n] (the formats' own definition)."""
    g = b.unflatten(-1, (-1, GROUP_BYTES[type_]))
    if type_ == "f16":
        return g.contiguous().view(torch.float16).float().flatten(-2)
    d = g[..., :2].contiguous().view(torch.float16).float()
    if type_ == "q8_0":
        return (g[..., 2:].contiguous().view(torch.int8).float() * d).flatten(-2)
    qs = g[..., -16:]
    c = torch.cat([qs & 15, qs >> 4], -1).float()
    if type_ == "q5_0":
        bit = (g[..., 2:6, None] >> torch.arange(8, dtype=torch.uint8, device="cuda")) & 1
        return ((c + 16.0 * bit.flatten(-2).float() - 16.0) * d).flatten(-2)
    return ((c - 8.0) * d).flatten(-2)


def _plain_attention(s):
    S, Hkv, D, T, Q, L = s["S"], s["Hkv"], s["D"], s["T"], s["max_q"], s["max_kv"]
    grp = s["Hq"] // Hkv
    j = torch.arange(L, device="cuda")
    slot = s["table"].long()[:, j // T]
    held = (slot >= 0) & (j < s["kv_len"][:, None])
    cell = torch.where(held, slot * T + j % T, 0)
    k = torch.where(held[..., None], _plain_dequant(s["k"][cell], s["type_k"]), 0.0)
    v = torch.where(held[..., None], _plain_dequant(s["v"][cell], s["type_v"]), 0.0)
    k = k.view(S, L, Hkv, D).permute(0, 2, 3, 1).contiguous()
    v = v.view(S, L, Hkv, D).permute(0, 2, 1, 3).contiguous()
    start = s["q_start"].long()
    m = start[1:] - start[:-1]
    i = torch.arange(Q, device="cuda")
    at = (start[:-1, None] + i).clamp(max=s["N"] - 1)
    q = s["q"].float()[at].view(S, Q, Hkv, grp, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, grp * Q, D)
    x = ((q @ k) * (1.0 / math.sqrt(D))).view(S, Hkv, grp, Q, L)
    last = s["kv_len"].long()[:, None] - m[:, None] + i  # the last key a query attends
    seen = held[:, None] & (j <= last[..., None])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(S, Hkv, grp * Q, L) @ v).view(S, Hkv, grp, Q, D) / torch.where(total == 0, 1.0, total)
    o = _plain_walsh(o, s["had_v"]).permute(0, 3, 1, 2, 4).reshape(S, Q, s["Hq"], D)
    t = torch.arange(s["N"], device="cuda")
    r = torch.searchsorted(start[1:].contiguous(), t, right=True)
    s["out"].copy_(o[r, t - start[r]])
    return s["out"]


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


def _own_slots(s):
    kv, ctx = _framework()
    o = s["out"]
    args = kv.SlotMapArgs(n_seq=s["S"], block_tokens=s["T"], n_slots=s["n_slots"], table_stride=s["stride"],
                          max_tokens=s["max_tokens"], n_free=s["free"].numel(), n_new=s["n_new"].data_ptr(),
                          kv_len=s["kv_len"].data_ptr(), pos0=s["pos0"].data_ptr(),
                          free_slots=s["free"].data_ptr(), free_used=s["used"].data_ptr(),
                          table=s["table"].data_ptr(), kv_len_out=o["kv_len"].data_ptr(),
                          q_start=o["q_start"].data_ptr(), positions=o["positions"].data_ptr(),
                          cells=o["cells"].data_ptr(), free_used_out=o["used"].data_ptr(),
                          n_missing=o["missing"].data_ptr())
    return functools.partial(ctx.slot_map, args), {"table": s["table"], **o}


def _own_rows(s):
    kv, ctx = _framework()
    o, e = s["out"], s["q"].element_size()
    N, Hq, D = s["q"].shape
    Hkv = s["k"].shape[1]
    xf = ctx.make_transform(D, s["n_rot"], s["theta"].tolist() if s["n_rot"] else None, s["had"], s["had_v"])
    pool = ctx.make_pool(1, s["n_slots"], s["T"], Hkv * D, Hkv * D, kv.TYPE_F16, kv.TYPE_F16,
                         [o["pool_k"].data_ptr()], [o["pool_v"].data_ptr()], xf)
    type_ = {"f32": kv.TYPE_F32, "f16": kv.TYPE_F16, "bf16": kv.TYPE_BF16}[s["type"]]
    args = kv.QkvArgs(type=type_, out_type=type_, n_tokens=N, n_head=Hq, n_head_kv=Hkv, head_dim=D, eps=EPS,
                      positions=s["positions"].data_ptr(), cells=s["cells"].data_ptr(), q_out=o["q"].data_ptr(),
                      **{n: s[n].data_ptr() for n in "qkv"},
                      **{f"{n}_nb{d}": e * s[n].stride(2 - d) for n in "qkv" for d in (1, 2)},
                      **({"q_weight": s["wq"].data_ptr(), "k_weight": s["wk"].data_ptr()} if s["wq"] is not None
                         else {}),
                      **({n: o[n].data_ptr() for n in ("q_norm", "k_norm")} if "q_norm" in o else {}))
    return functools.partial(ctx.qkv_rows, args, pool), o


def _own_attention(s):
    kv, ctx = _framework()
    types = {"q8_0": kv.TYPE_Q8_0, "q5_0": kv.TYPE_Q5_0, "q4_0": kv.TYPE_Q4_0, "f16": kv.TYPE_F16,
             "bf16": kv.TYPE_BF16}
    E = s["Hkv"] * s["D"]
    xf = ctx.make_transform(s["D"], hadamard_v=s["had_v"])
    pool = ctx.make_pool(1, s["n_slots"], s["T"], E, E, types[s["type_k"]], types[s["type_v"]],
                         [s["k"].data_ptr()], [s["v"].data_ptr()], xf)
    qt = types[s["q_type"]]
    nb1, nb2 = 2 * s["D"], 2 * s["D"] * s["Hq"]
    args = kv.AttnArgs(q=s["q"].data_ptr(), q_type=qt, q_nb1=nb1, q_nb2=nb2, out=s["out"].data_ptr(), out_type=qt,
                       n_tokens=s["N"], n_seq=s["S"], max_q=s["max_q"], max_kv=s["max_kv"], n_head=s["Hq"],
                       n_head_kv=s["Hkv"], head_dim=s["D"], q_start=s["q_start"].data_ptr(),
                       kv_len=s["kv_len"].data_ptr(), table=s["table"].data_ptr(), table_stride=s["stride"], causal=1)
    return functools.partial(ctx.attention, args, pool), s["out"]


def run(state):
    if own:
        if "call" not in state:  # the argument block a program builds once for its buffers
            state["call"] = {"slots": _own_slots, "rows": _own_rows, "attention": _own_attention}[state["kind"]](state)
        call, out = state["call"]
        call()
        return out
    return {"slots": _plain_slots, "rows": _plain_rows, "attention": _plain_attention}[state["kind"]](state)


# -------------------------------------------------------------------- exact
def exact(case, seed):
    """What run() returns, in float64 from the definitions: request by request and head
    by head, sums of squares as dot products, the rotation as a complex product, the
    Walsh-Hadamard transform by butterflies, cached rows decoded one code at a time."""
    if case["kind"] == "slots":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_rows(s) if case["kind"] == "rows" else _exact_attention(s)


def _exact_walsh(x, width):
    if width == 0:
        return x
    y, span = x.reshape(-1, width), 1
    while span < width:
        z = y.view(-1, width // (2 * span), 2, span)
        y = torch.stack([z[:, :, 0] + z[:, :, 1], z[:, :, 0] - z[:, :, 1]], 2).reshape(-1, width)
        span *= 2
    return (y / math.sqrt(width)).view_as(x)


def _exact_rows(s):
    h = s["n_rot"] // 2

    def rows(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / (torch.einsum("thd,thd->th", x, x)[..., None] / x.shape[-1] + EPS).sqrt()
        y = x
        if h:
            angle = torch.outer(s["positions"].float(), s["theta_dev"]).double()
            turn = torch.polar(torch.ones_like(angle), angle)[:, None]
            z = torch.complex(x[..., :h].contiguous(), x[..., h:2 * h].contiguous()) * turn
            y = torch.cat([z.real, z.imag, x[..., 2 * h:]], -1)
        return x, _exact_walsh(y, s["had"])

    qn, q = rows(s["q"], s["wq"])
    kn, k = rows(s["k"], s["wk"])
    out = {"q": q}
    for name, x in (("pool_k", k), ("pool_v", _exact_walsh(s["v"].double(), s["had_v"]))):
        pool = torch.zeros(s["out"][name].shape, dtype=torch.float64, device="cuda")
        kept = s["cells"] >= 0
        pool.index_copy_(0, s["cells"][kept].long(), x.flatten(1)[kept])
        out[name] = pool
    if "q_norm" in s["out"]:
        out.update(q_norm=qn, k_norm=kn)
    return out


def _exact_decode(b, type_):
    g = b.reshape(b.shape[0], -1, GROUP_BYTES[type_])
    if type_ == "f16":
        return g.contiguous().view(torch.float16).double().reshape(b.shape[0], -1)
    x = torch.empty((*g.shape[:2], 32), dtype=torch.float64, device="cuda")
    d = g[..., 0:2].contiguous().view(torch.float16)[..., 0].double()
    for e in range(32):
        if type_ == "q8_0":
            x[..., e] = d * g[..., 2 + e].view(torch.int8).double()
            continue
        code = g[..., GROUP_BYTES[type_] - 16 + e % 16].to(torch.int64)
        code = code % 16 if e < 16 else code // 16
        if type_ == "q5_0":
            code = code + 16 * ((g[..., 2 + e // 8].to(torch.int64) // 2 ** (e % 8)) % 2)
        x[..., e] = d * (code - (8 if type_ == "q4_0" else 16)).double()
    return x.reshape(b.shape[0], -1)


def _exact_attention(s):
    D, grp, T = s["D"], s["Hq"] // s["Hkv"], s["T"]
    out = torch.zeros((s["N"], s["Hq"], D), dtype=torch.float64, device="cuda")
    lens, starts = s["kv_len"].tolist(), s["q_start"].tolist()
    for r in range(s["S"]):
        a, b = starts[r], starts[r + 1]
        at = torch.arange(lens[r], device="cuda")
        slot = s["table"][r].long()[at // T]
        at, slot = at[slot >= 0], slot[slot >= 0]
        k = _exact_decode(s["k"][slot * T + at % T], s["type_k"])
        v = _exact_decode(s["v"][slot * T + at % T], s["type_v"])
        limit = lens[r] - (b - a) + torch.arange(b - a, device="cuda")
        hidden = at[None] > limit[:, None]
        for h in range(s["Hq"]):
            c = slice(h // grp * D, h // grp * D + D)
            x = (s["q"][a:b, h].double() @ k[:, c].T / D ** 0.5).masked_fill_(hidden, -math.inf)
            x = x - torch.logsumexp(x, -1, keepdim=True)
            out[a:b, h] = torch.nan_to_num(x.exp_(), nan=0.0) @ v[:, c]
    return _exact_walsh(out, s["had_v"])
