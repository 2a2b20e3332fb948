"""Batches, float64 references and error bounds of the tests of kvmem_hip_conv_rows
and kvmem_hip_linear_attention.

Bounds, with u = 2^-24 (half a step of fp32) and everything per column of a state:

conv   a sum of W products and a bias errs by (W + 1) u sum |w x|; SiLU has a slope
       below 1.1 and adds |y s(y)| (|y| + 8) 2^-22 (the exponent's argument errs by
       |y| u, exp2, the reciprocal and the products by a step each); a norm divides by
       n = sqrt(sum + eps) and adds |z| (|dy|_2 / n + 2^-20); storing adds half a step.
linear with |k|, |q| the keys' and queries' 2-norms, h the state's bound
           h' = a h + |k| |d|
       (it bounds the state's norm, and the sum of the terms an output is made of), the
       state's error e grows by
           e' = a e max(1, |1 - beta |k|^2|) + c (h' + |k| |beta| (|v| + a |k| h))
       where a token's sums of Dk products and its few other operations are
       c = (Dk + 16) u, and in chunks, whose sums of up to Dk + 64 products have factors
       cut to 22 bits, c = kappa (Dk + 64 + 64) u, kappa the largest absolute row sum of
       a chunk's (1 + A)^-1 (at least 1).  An output errs by
           scale |q| (e' + c h') + half a step,
       and in chunks with a bf16 out, where three factors are cut to 11 bits, by
           scale |q| 3 h' kappa 2^-12 more."""
from __future__ import annotations

import math

import numpy as np
import torch

from conftest import load_pkg

kv = load_pkg()
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE = {"f32": kv.TYPE_F32, "f16": kv.TYPE_F16, "bf16": kv.TYPE_BF16}
U = 2.0 ** -24
CHUNK = 64
FROM = 24  # tokens a request from which a call goes by chunks
FILL = 7.25  # what outputs hold before a call


def half_step(x, type_):
    """Half a step of the type at |x|, its subnormal numbers' spacing at least."""
    fi = torch.finfo(DT[type_])
    return np.abs(x) * fi.eps / 2 + fi.smallest_normal * fi.eps


def ints(values):
    return None if values is None else torch.tensor(values, dtype=torch.int64).to(torch.int32).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


class Requests:
    """Ragged requests: rows of each, tokens that take part, slots of n_slots."""

    def __init__(self, lengths, use=None, slots=None, n_slots=None, tail=0):
        self.lengths = lengths
        self.S = len(lengths)
        self.starts = [0]
        for n in lengths:
            self.starts.append(self.starts[-1] + n)
        self.N = self.starts[-1] + tail
        self.given = use
        self.use = [min(a, b) for a, b in zip(lengths, use)] if use is not None else list(lengths)
        self.n_slots = n_slots or self.S + 2
        self.given_slots = slots
        self.slots = slots if slots is not None else list(range(self.S))
        self.dev = dict(q_start=ints(self.starts), n_use=ints(use), slots=ints(slots))

    def args(self, max_q=None):
        return dict(n_tokens=self.N, n_seq=self.S, max_q=max(self.lengths, default=0) if max_q is None else max_q,
                    n_slots=self.n_slots, **{k: ptr(v) for k, v in self.dev.items()})


def close(got, want, bound, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / bound):.3g} "
                           f"bounds, first at {np.argwhere(bad)[0].tolist()}: {got[bad][0]} for {want[bad][0]}")


# --------------------------------------------------------------- convolution
def conv_reference(x, before, w, bias, silu, norm, norm_dim, eps):
    """Rows x [n, C] behind `before` [W-1, C], float64: (outputs, bounds, new state)."""
    W, n = w.shape[1], x.shape[0]
    all_ = np.concatenate([before, x])
    y = np.zeros_like(x) if bias is None else np.broadcast_to(bias, x.shape).copy()
    m = np.abs(y)
    for j in range(W):
        y += w[:, j] * all_[j:j + n]
        m += np.abs(w[:, j] * all_[j:j + n])
    e = (W + 1) * U * m
    if silu:
        with np.errstate(over="ignore"):
            z = y / (1.0 + np.exp(-y))
        e = 1.1 * e + np.abs(z) * (np.abs(y) + 8) * 2.0 ** -22
        y = z
    if norm:
        h = y[:, :norm].reshape(n, norm // norm_dim, norm_dim)
        r = np.sqrt((h * h).sum(-1, keepdims=True) + eps)
        z = np.divide(h, r, out=np.zeros_like(h), where=r > 0)
        eh = e[:, :norm].reshape(h.shape)
        eh = np.divide(eh + np.abs(z) * np.sqrt((eh * eh).sum(-1, keepdims=True)), r, out=np.zeros_like(h), where=r > 0) \
            + np.abs(z) * 2.0 ** -20
        y = np.concatenate([z.reshape(n, norm), y[:, norm:]], 1)
        e = np.concatenate([eh.reshape(n, norm), e[:, norm:]], 1)
    return y, e, all_[n:]


# ---------------------------------------------------------- linear attention
def kappa(k, g, beta):
    """Largest absolute row sum of (1 + A)^-1 of a chunk's keys [n, Dk]."""
    G = np.cumsum(np.maximum(g, -1e5))
    A = np.tril(beta[:, None] * (k @ k.T) * np.exp(np.minimum(0.0, G[:, None] - G[None])), -1)
    return max(1.0, np.abs(np.linalg.inv(np.eye(len(g)) + A)).sum(1).max())


def linear_reference(q, k, v, g, beta, state, scale, chunked, out_type):
    """One request in float64: q, k [n, Hk, Dk], v [n, H, Dv], g, beta [n, H] or None, state
    [H, Dk, Dv]: (outputs, their bounds, state, its bounds)."""
    n, H, Dv = v.shape
    grp, Dk = H // k.shape[1], k.shape[2]
    kh, qh = np.repeat(k, grp, 1), np.repeat(q, grp, 1)
    g = np.zeros((n, H)) if g is None else g
    S = state.copy()
    hb = np.sqrt((S * S).sum(1))
    e = np.zeros((H, Dv))
    out, bound = np.zeros((n, H, Dv)), np.zeros((n, H, Dv))
    kap = np.ones(H)
    for t in range(n):
        if chunked and t % CHUNK == 0 and beta is not None:
            c = slice(t, min(n, t + CHUNK))
            kap = np.array([kappa(kh[c, h], g[c, h], beta[c, h]) for h in range(H)])
        unit = (kap * (Dk + 128) if chunked else np.full(H, Dk + 16.0))[:, None] * U
        a = np.exp(g[t])[:, None]
        kn = np.sqrt((kh[t] ** 2).sum(-1))[:, None]
        qn = np.sqrt((qh[t] ** 2).sum(-1))[:, None]
        S = a[..., None] * S
        d, more, grow = v[t], 0.0, 1.0
        if beta is not None:
            b = beta[t][:, None]
            d = b * (v[t] - np.einsum("hk,hkv->hv", kh[t], S))
            more = kn * np.abs(b) * (np.abs(v[t]) + a * kn * hb)
            grow = np.maximum(1.0, np.abs(1.0 - b * kn * kn))
        S = S + kh[t][..., None] * d[:, None]
        hb = a * hb + kn * np.abs(d)
        e = a * e * grow + unit * (hb + more)
        out[t] = scale * np.einsum("hk,hkv->hv", qh[t], S)
        bound[t] = scale * qn * (e + unit * hb)
        if chunked and out_type == "bf16":
            bound[t] += scale * qn * 3 * hb * kap[:, None] * 2.0 ** -12
    return out, bound + half_step(out, out_type), S, np.broadcast_to(e[:, None], S.shape) + 1e-30


class Linear:
    """A call's arrays.  Keys and queries are normalized unless `raw`; a head's keys share
    a direction; a token's q, k and v lie side by side."""

    def __init__(self, ctx, rq, Hk, H, Dk, Dv, type_="bf16", out="bf16", delta=True, decay="token", seed=0, scale=0.0,
                 state=True, rate=1.0):
        self.ctx, self.rq, self.dims = ctx, rq, (Hk, H, Dk, Dv)
        self.type, self.out_type, self.delta = type_, out, delta
        self.scale = scale or 1.0 / math.sqrt(Dk)
        gen = torch.Generator().manual_seed(seed)
        N = rq.N

        def unit(x):
            return x / x.norm(dim=-1, keepdim=True)

        rows = torch.empty((N, 2 * Hk * Dk + H * Dv + 16), dtype=DT[type_])
        q, k, v = (rows[:, a:b].view(N, -1, d) for a, b, d in (
            (0, Hk * Dk, Dk), (Hk * Dk, 2 * Hk * Dk, Dk), (2 * Hk * Dk, 2 * Hk * Dk + H * Dv, Dv)))
        q.copy_(unit(torch.randn(q.shape, generator=gen)))
        k.copy_(unit(torch.randn(k.shape, generator=gen) + 0.8 * torch.randn((1, Hk, Dk), generator=gen)))
        v.copy_(torch.randn(v.shape, generator=gen))
        self.rows = rows.cuda()
        self.q, self.k, self.v = (self.rows[:, a:b].view(N, -1, d) for a, b, d in (
            (0, Hk * Dk, Dk), (Hk * Dk, 2 * Hk * Dk, Dk), (2 * Hk * Dk, 2 * Hk * Dk + H * Dv, Dv)))
        self.decay = self.beta = None
        if decay == "token":
            self.decay = (-rate * torch.rand((N, H), generator=gen) ** 3).cuda()
        elif decay == "head":
            self.decay = (-0.1 * rate * torch.rand(H, generator=gen)).cuda()
        if delta:
            self.beta = torch.rand((N, H), generator=gen).cuda()
        self.state = (0.3 * torch.randn((rq.n_slots, H, Dk, Dv), generator=gen)).cuda() if state else None
        self.out = torch.full((N, H, Dv), FILL, dtype=DT[out], device="cuda")
        self.state_out = torch.full((rq.n_slots, H, Dk, Dv), FILL, device="cuda")

    def args(self, max_q=None, **over):
        Hk, H, Dk, Dv = self.dims
        e = self.rows.element_size()
        a = dict(type=TYPE[self.type], out_type=TYPE[self.out_type], n_head_k=Hk, n_head=H, head_dim_k=Dk,
                 head_dim_v=Dv, log_decay=ptr(self.decay), beta=ptr(self.beta),
                 decay_nb=0 if self.decay is None or self.decay.ndim == 1 else 4 * H, beta_nb=4 * H,
                 scale=0.0 if self.scale == 1.0 / math.sqrt(Dk) else self.scale, state=ptr(self.state),
                 state_out=ptr(self.state_out), out=ptr(self.out), **self.rq.args(max_q),
                 **{n: ptr(getattr(self, n)) for n in "qkv"},
                 **{f"{n}_nb{d}": e * getattr(self, n).stride(2 - d) for n in "qkv" for d in (1, 2)})
        return kv.LinearArgs(**{**a, **over})

    def run(self, max_q=None, **over):
        torch.cuda.synchronize()
        self.ctx.linear_attention(self.args(max_q, **over))
        self.ctx.sync()

    def want(self, s, chunked, state=None, use=None):
        """Reference of request s: (outputs, bounds, state, bounds)."""
        rq = self.rq
        rows = slice(rq.starts[s], rq.starts[s] + (rq.use[s] if use is None else use))
        f = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
        g = f(self.decay)
        if g is not None:
            g = np.broadcast_to(g, (rq.N, g.shape[-1]))[rows]
        b = f(self.beta)
        Hk, H, Dk, Dv = self.dims
        if state is None:
            known = self.state is not None and rq.slots[s] < rq.n_slots
            state = f(self.state[rq.slots[s]]) if known else np.zeros((H, Dk, Dv))
        return linear_reference(f(self.q[rows]), f(self.k[rows]), f(self.v[rows]), g, None if b is None else b[rows],
                                state, self.scale, chunked, self.out_type)

    def check(self, chunked=None, out=True, stored=True):
        rq = self.rq
        chunked = max(rq.lengths, default=0) >= FROM if chunked is None else chunked
        got, state = self.out.double().cpu().numpy(), self.state_out.double().cpu().numpy()
        written = np.zeros(rq.N, bool)
        touched = np.zeros(rq.n_slots, bool)
        for s in range(rq.S):
            o, b, S, bs = self.want(s, chunked)
            a, n = rq.starts[s], rq.use[s]
            if out:
                close(got[a:a + n], o, b, f"out of request {s}")
                written[a:a + n] = True
            if stored and rq.slots[s] < rq.n_slots:
                close(state[rq.slots[s]], S, bs, f"state of request {s}")
                touched[rq.slots[s]] = True
        assert (got[~written] == FILL).all(), "rows that take no part were written"
        assert (state[~touched] == FILL).all(), "states that nobody names were written"
