"""Pools, block tables and the float64 reference of the attention tests.

Bound of an output element (vectors over keys j, p the float64 softmax):
  - a cached value is rounded to f16 once it is scaled: 2^-11 |v_j|, at least
    2^-25 absolute;
  - a softmax weight is rounded to f16: 2^-11 p_j; weights are scaled by at
    least 2^4 against the largest before they are rounded, so a small one loses
    at most 2^-25 * 2^-4 of the largest weight of its request;
  - a score errs by delta_j = scale * sum_i |q_i k_ji| * (2^-11 + 2^-11 +
    (D + 8) 2^-24): cached keys and queries rounded to f16, fp32 sums; and by
    2^-22 |x_j| + 2^-22 |max| in the exponent's argument.  Weight and sum both
    move by a factor within e^{+-2 delta}, so p_j by at most expm1(4 delta) p_j
    for delta = max_j;
  - fp32 sums over L keys: (L + 64) 2^-24 of the sum of magnitudes;
  - the output's own rounding, half a step.
hadamard_v spreads the error: each element's bound becomes the mean over its
run times sqrt(width), plus (8 + log2 width) 2^-24 of the run's magnitudes.
lse errs by 2 delta + 2^-20 (1 + |lse|)."""
from __future__ import annotations

import math

import numpy as np
import torch

from conftest import load_pkg

kv = load_pkg()
CACHE = {"q8_0": kv.TYPE_Q8_0, "q5_0": kv.TYPE_Q5_0, "q4_0": kv.TYPE_Q4_0, "f16": kv.TYPE_F16}
OUT = {"f32": (torch.float32, kv.TYPE_F32), "f16": (torch.float16, kv.TYPE_F16), "bf16": (torch.bfloat16, kv.TYPE_BF16)}


def quantize(oracle, type_, x):
    """f32 rows [n, E] -> cached bytes [n, row]."""
    x = np.ascontiguousarray(x, np.float32)
    return x.astype(np.float16).view(np.uint8) if type_ == "f16" else oracle.quantize_rows_f32(CACHE[type_], x)


def decode(oracle, type_, b, E):
    """Cached bytes [n, row] -> float64 rows [n, E]."""
    if type_ == "f16":
        return b.view(np.float16).astype(np.float64)
    return oracle.dequantize_row(CACHE[type_], np.ascontiguousarray(b).reshape(-1), b.shape[0] * E).reshape(
        b.shape[0], E).astype(np.float64)


def walsh(width):
    h = np.ones((1, 1))
    while h.shape[0] < width:
        h = np.block([[h, h], [h, -h]])
    return h


class Case:
    """A pool with the keys of `lens` requests, `m` new queries each, on the GPU."""

    def __init__(self, ctx, oracle, lens, m, Hq, Hkv, D, T, type_k="q4_0", type_v="q4_0", q_type="bf16",
                 out_type="f32", causal=True, holes=0.0, hadamard=0, scale=0.0, seed=0, stride=None, extra_rows=0,
                 k_scale=1.0, v_scale=1.0, q_pad=0, table_fill=kv.NO_SLOT, poison=True, max_kv=None, max_q=None):
        rng = np.random.default_rng([seed, len(lens), Hq, D, T])
        self.ctx, self.oracle, self.lens, self.m = ctx, oracle, list(lens), list(m)
        self.Hq, self.Hkv, self.D, self.T, self.causal, self.hadamard = Hq, Hkv, D, T, causal, hadamard
        self.type_k, self.type_v = type_k, type_v
        S, E = len(lens), Hkv * D
        held = [-(-a // T) for a in lens]
        self.n_slots = sum(held) + 2
        self.stride = stride or max(1, max(held) + 1)
        order = rng.permutation(self.n_slots).astype(np.uint32)
        self.table = np.full((S, self.stride), table_fill, np.uint32)
        at = 0
        n_rows = self.n_slots * T
        self.pool = {}
        live = np.zeros(n_rows, bool)
        for s in range(S):
            for b in range(held[s]):
                self.table[s, b] = order[at]
                live[order[at] * T:order[at] * T + min(T, lens[s] - b * T)] = True
                at += 1
            if holes:
                drop = rng.random(held[s]) < holes
                self.table[s, :held[s]][drop] = rng.choice([kv.NO_SLOT, self.n_slots, self.n_slots + 12345])
        for w, t, sc in (("k", type_k, k_scale), ("v", type_v, v_scale)):
            x = (rng.standard_normal((n_rows, E)) * sc).astype(np.float32)
            x[:, ::37] *= 4.0
            b = quantize(oracle, t, np.clip(x, -65000, 65000))
            if poison:
                b[~live] = 0xFF  # NaN scales where no key lives
            self.pool[w] = b
        N = sum(m)
        self.N, self.rows = N, N + extra_rows
        qdt, self.q_code = OUT[q_type]
        q = torch.from_numpy((rng.standard_normal((max(1, self.rows), Hq, D + q_pad)) * 1.5).astype(np.float32)).to(qdt)
        self.q_host = q[..., :D].double().numpy()
        self.q = q.cuda()[..., :D]
        self.odt, self.o_code = OUT[out_type]
        self.scale = scale or 1.0 / math.sqrt(D)
        self.starts = np.concatenate([[0], np.cumsum(m)]).astype(np.int64)
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.uint32).view(np.int32)).cuda()  # noqa: E731
        self.dev = dict(table=i32(self.table), lens=i32(np.array(lens)), starts=i32(self.starts))
        self.upload()
        self.out = torch.full((max(1, self.rows), Hq, D), 7.25, dtype=self.odt, device="cuda")
        self.lse = torch.full((max(1, self.rows), Hq), 7.25, dtype=torch.float32, device="cuda")
        self.xf = ctx.make_transform(D, hadamard_v=hadamard) if hadamard else None
        self.pool_c = ctx.make_pool(2, self.n_slots, T, E, E, CACHE[type_k], CACHE[type_v],
                                    [0, self.dev["k"].data_ptr()], [0, self.dev["v"].data_ptr()], self.xf)
        self.args = kv.AttnArgs(q=self.q.data_ptr(), q_type=self.q_code, q_nb1=2 * self.q.stride(1),
                                q_nb2=2 * self.q.stride(0), out=self.out.data_ptr(), out_type=self.o_code,
                                lse=self.lse.data_ptr(), n_tokens=self.rows, n_seq=S, max_q=max_q or max(m),
                                max_kv=max(lens) if max_kv is None else max_kv, n_head=Hq, n_head_kv=Hkv, head_dim=D,
                                q_start=self.dev["starts"].data_ptr(), kv_len=self.dev["lens"].data_ptr(),
                                table=self.dev["table"].data_ptr(), table_stride=self.stride, causal=int(causal),
                                scale=scale)

    def upload(self):
        for w in "kv":
            b = torch.from_numpy(self.pool[w])
            if w in self.dev:
                self.dev[w].copy_(b)
            else:
                self.dev[w] = b.cuda()

    def run(self):
        torch.cuda.synchronize()
        self.ctx.attention(self.args, self.pool_c, 1)
        self.ctx.sync()
        return self

    def reference(self, lens=None, m=None, starts=None):
        """(out, bound, lse, lse bound) in float64, [rows, Hq, D]; NaN where nothing is written."""
        lens, m = lens or self.lens, m or self.m
        starts = self.starts if starts is None else starts
        Hq, Hkv, D, T = self.Hq, self.Hkv, self.D, self.T
        out = np.full((self.rows, Hq, D), np.nan)
        bound = np.full_like(out, np.nan)
        lse = np.full((self.rows, Hq), np.nan)
        lb = np.full_like(lse, np.nan)
        room = min(self.args.max_kv, self.stride * T)
        for s in range(len(lens)):
            L = min(lens[s], room)
            j = np.arange(L)
            slot = self.table[s, j // T].astype(np.int64) if L else j
            j, slot = j[slot < self.n_slots], slot[slot < self.n_slots]
            rows = slot * T + j % T
            k = decode(self.oracle, self.type_k, self.pool["k"][rows], Hkv * D).reshape(len(j), Hkv, D)
            v = decode(self.oracle, self.type_v, self.pool["v"][rows], Hkv * D).reshape(len(j), Hkv, D)
            for i in range(min(m[s], self.args.max_q)):
                t = int(starts[s]) + i
                if t >= self.rows:
                    break
                see = j <= lens[s] - m[s] + i if self.causal else j >= 0
                n = int(see.sum())
                if n == 0:
                    out[t], bound[t], lse[t], lb[t] = 0.0, 0.0, -np.inf, 0.0
                    continue
                for h in range(Hq):
                    g = h // (Hq // Hkv)
                    kk, vv, q = k[see, g], v[see, g], self.q_host[t, h]
                    with np.errstate(invalid="ignore", over="ignore"):
                        x = self.scale * (kk @ q)
                        mag = self.scale * (np.abs(kk) @ np.abs(q))
                    top = x.max()
                    p = np.exp(x - top)
                    total = p.sum()
                    p /= total
                    delta = (mag * (2.0 ** -10 + (D + 8) * 2.0 ** -24) + 2.0 ** -22 * (np.abs(x) + abs(top))).max()
                    av = np.abs(vv)
                    o = p @ vv
                    small = 2.0 ** -29 * n / total
                    b = (p @ av) * (math.expm1(min(50.0, 4 * delta)) + 2.0 ** -10 + (n + 64) * 2.0 ** -24) \
                        + small * av.max(0) + 2.0 ** -25
                    w = self.hadamard
                    if w:
                        H = walsh(w) / math.sqrt(w)
                        b = np.repeat(b.reshape(-1, w).sum(1) / math.sqrt(w)
                                      + (8 + math.log2(w)) * 2.0 ** -24 * np.abs(o).reshape(-1, w).sum(1), w)
                        o = (o.reshape(-1, w) @ H).reshape(-1)
                    out[t, h], bound[t, h] = o, b
                    lse[t, h] = top + math.log(total)
                    lb[t, h] = 2 * delta + 2.0 ** -20 * (1 + abs(lse[t, h]))
        return out, bound, lse, lb

    def check(self, **kw):
        out, bound, lse, lb = self.reference(**kw)
        got = self.out.cpu().double().numpy()[:self.rows]
        got_l = self.lse.cpu().double().numpy()[:self.rows]
        half = torch.finfo(self.odt).eps / 2
        blank = np.isnan(out[:, 0, 0]) if self.rows else np.zeros(0, bool)
        assert (got[blank] == 7.25).all() and (got_l[blank] == 7.25).all(), "rows that hold no query were written"
        o, b = out[~blank], bound[~blank]
        g = got[~blank]
        assert np.isfinite(g).all(), "not finite"
        off = np.abs(g - o) - (b + half * (np.abs(o) + b) + 2.0 ** -25)
        assert (off <= 0).all(), f"over the bound by {off.max():.3e} at {np.unravel_index(off.argmax(), off.shape)}"
        gl, wl = got_l[~blank], lse[~blank]
        empty = np.isinf(wl)
        assert np.array_equal(np.isneginf(gl), empty)
        assert (np.abs(gl[~empty] - wl[~empty]) <= lb[~blank][~empty]).all(), "lse"
        # the bound is for the worst signs; rounding errors of many keys average out
        if o.size > 2000 and np.linalg.norm(o) > 0:
            rel = np.linalg.norm(g - o) / np.linalg.norm(o)
            assert rel < max(half, 2.0 ** -9), f"relative error {rel:.2e}"
        return got
