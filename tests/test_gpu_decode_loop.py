"""A batch's calls together, as a program makes them: kvmem_hip_slot_map, then
per layer kvmem_hip_qkv_rows and kvmem_hip_attention -- prompts, single tokens,
drafted tokens and requests that bring nothing, over two layers and one pool;
the same step captured once and replayed as the requests grow; and new tokens
over the window that the reselect engine staged, with blocks it left out.

Each step is checked against float64: the table against the definition, each
cached row against the token's own rotated row (a row that landed in another
token's cell, or at another position, is far off), and the attention's output
against the cached rows and the queries it was given (attention_helpers)."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()

import engine_helpers as eh  # noqa: E402
from attention_helpers import CACHE, Case, decode  # noqa: E402
from test_gpu_qkv_rows import reference as rows_reference  # noqa: E402

EPS = 1e-6
# a code's step against its group's largest magnitude: the most a cached row is off
# (half a step, a whole one where q4_0 and q5_0 saturate); checks add 2^-8 of that magnitude
# for the norm's, RoPE's and rotation's roundings and the scale's
STEP = {"q8_0": 1 / 127, "q5_0": 1 / 16, "q4_0": 1 / 8, "f16": 2.0 ** -10}


def i32(a):
    return torch.from_numpy(np.asarray(a).astype(np.uint32).view(np.int32).copy()).cuda()


class Batch:
    """Requests over one pool, their device state, and the float64 rows of every token they ever had."""

    def __init__(self, ctx, S, Hq, Hkv, D, T, n_slots, stride, max_tokens, types, n_rot, had, layers=2, seed=0,
                 pool=None, table=None, kv_len=None, free=None):
        self.ctx, self.S, self.Hq, self.Hkv, self.D, self.T, self.layers = ctx, S, Hq, Hkv, D, T, layers
        self.n_slots, self.stride, self.max_tokens, self.types, self.n_rot, self.had = (
            n_slots, stride, max_tokens, types, n_rot, had)
        self.rng = np.random.default_rng(seed)
        E = Hkv * D
        self.theta = (np.float32(10000.0) ** (-2.0 * np.arange(max(1, n_rot // 2)) / max(1, n_rot))).astype(np.float32)
        self.xf = ctx.make_transform(D, n_rot, self.theta if n_rot else None, had and D, had)
        if pool is None:
            size = [kv.row_size(CACHE[t], E) for t in types]
            # nothing lives there yet: NaN scales
            self.mem = [[torch.full((n_slots * T, b), 255, dtype=torch.uint8, device="cuda") for b in size]
                        for _ in range(layers)]
            ptrs = [[m[w].data_ptr() for m in self.mem] for w in (0, 1)]
            pool = ctx.make_pool(layers, n_slots, T, E, E, CACHE[types[0]], CACHE[types[1]], *ptrs, self.xf)
        self.pool = pool
        self.len = np.array([0] * S if kv_len is None else kv_len)
        free = self.rng.permutation(n_slots) if free is None else free
        self.d = dict(new=i32(np.zeros(S)), len=i32(self.len), free=i32(free), used=i32([0]),
                      table=i32(np.full((S, stride), kv.NO_SLOT) if table is None else table),
                      len_out=i32(np.zeros(S)), q_start=i32(np.zeros(S + 1)), pos=i32(np.zeros(max_tokens)),
                      cells=i32(np.zeros(max_tokens)), used_out=i32([0]), missing=i32([0]))
        p = {n: t.data_ptr() for n, t in self.d.items()}
        self.map = kv.SlotMapArgs(n_seq=S, block_tokens=T, n_slots=n_slots, table_stride=stride, max_tokens=max_tokens,
                                  n_free=len(free), n_new=p["new"], kv_len=p["len"], free_slots=p["free"],
                                  free_used=p["used"], table=p["table"], kv_len_out=p["len_out"],
                                  q_start=p["q_start"], positions=p["pos"], cells=p["cells"],
                                  free_used_out=p["used_out"], n_missing=p["missing"])
        N = max_tokens
        bf = dict(dtype=torch.bfloat16, device="cuda")
        # the projections' output, one row a token: q heads, then k, then v
        self.proj = [torch.zeros((N, Hq + 2 * Hkv, D), **bf) for _ in range(layers)]
        self.w = [torch.from_numpy((1 + 0.2 * self.rng.standard_normal((2, D))).astype(np.float32)).cuda()
                  for _ in range(layers)]
        self.out = [torch.zeros((N, Hq, D), dtype=torch.float32, device="cuda") for _ in range(layers)]
        self.lse = [torch.zeros((N, Hq), dtype=torch.float32, device="cuda") for _ in range(layers)]
        self.q_seen = [torch.zeros((N, Hq, D), **bf) for _ in range(layers)]
        self.tokens = [[[] for _ in range(S)] for _ in range(layers)]  # float64 (k, v, bounds) by position

    def calls(self, max_q, max_kv, workspace=None):
        """The step's calls, in order; nothing waits for the host."""
        c, d = self.ctx, self.d
        c.slot_map(self.map)
        row, b = 2 * (self.Hq + 2 * self.Hkv) * self.D, 2 * self.D
        for layer in range(self.layers):
            x = self.proj[layer].data_ptr()
            c.qkv_rows(kv.QkvArgs(q=x, k=x + self.Hq * b, v=x + (self.Hq + self.Hkv) * b, type=kv.TYPE_BF16,
                                  out_type=kv.TYPE_BF16, n_tokens=self.max_tokens, n_head=self.Hq,
                                  n_head_kv=self.Hkv, head_dim=self.D, q_nb1=b, q_nb2=row, k_nb1=b, k_nb2=row,
                                  v_nb1=b, v_nb2=row, q_weight=self.w[layer][0].data_ptr(),
                                  k_weight=self.w[layer][1].data_ptr(), eps=EPS, positions=d["pos"].data_ptr(),
                                  cells=d["cells"].data_ptr(), xf=kv.C.pointer(self.xf),
                                  q_out=self.q_seen[layer].data_ptr()), self.pool, layer)
            a = kv.AttnArgs(q=self.q_seen[layer].data_ptr(), q_type=kv.TYPE_BF16, q_nb1=b, q_nb2=b * self.Hq,
                            out=self.out[layer].data_ptr(), out_type=kv.TYPE_F32, lse=self.lse[layer].data_ptr(),
                            n_tokens=self.max_tokens, n_seq=self.S, max_q=max_q, max_kv=max_kv, n_head=self.Hq,
                            n_head_kv=self.Hkv, head_dim=self.D, q_start=d["q_start"].data_ptr(),
                            kv_len=d["len_out"].data_ptr(), table=d["table"].data_ptr(), table_stride=self.stride,
                            causal=1)
            if workspace is not None:
                a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
            c.attention(a, self.pool, layer)
            self.args = a

    def feed(self, new):
        """New projections for `new` tokens of each request."""
        self.new = np.array(new)
        self.d["new"].copy_(i32(new))
        for layer in range(self.layers):
            x = self.rng.standard_normal(tuple(self.proj[layer].shape)).astype(np.float32)
            self.proj[layer].copy_(torch.from_numpy(x).to(torch.bfloat16))
            self.out[layer].fill_(7.25)
            self.lse[layer].fill_(7.25)
        torch.cuda.synchronize()

    def advance(self):
        """The state the next step starts from."""
        self.d["len"].copy_(self.d["len_out"])
        self.d["used"].copy_(self.d["used_out"])
        self.len = self.len + self.new
        torch.cuda.synchronize()

    def cached(self, layer):
        return [m.cpu().numpy() for m in self.mem[layer]]

    def check(self, oracle):
        host = {n: t.cpu().numpy().view(np.uint32) for n, t in self.d.items()}
        after = self.len + self.new
        assert (host["len_out"] == after).all() and host["missing"][0] == 0
        starts = np.concatenate([[0], np.cumsum(self.new)])
        assert (host["q_start"] == starts).all()
        table = host["table"].reshape(self.S, self.stride)
        used = table[table < self.n_slots]
        assert len(set(used.tolist())) == len(used), "a slot twice"
        E = self.Hkv * self.D
        for layer in range(self.layers):
            x = self.proj[layer].float().cpu().numpy()
            w = self.w[layer].cpu().numpy()
            pos = np.concatenate([np.arange(self.len[s], after[s]) for s in range(self.S)]).astype(np.int64)
            N = len(pos)
            h0, h1 = self.Hq, self.Hq + self.Hkv
            k = rows_reference(x[:N, h0:h1], w[1], EPS, pos, self.theta, self.n_rot, self.had and self.D)[2]
            v = rows_reference(x[:N, h1:], None, EPS, pos, self.theta, 0, self.had)[2]
            for s in range(self.S):
                self.tokens[layer][s] += list(zip(k[starts[s]:starts[s + 1]], v[starts[s]:starts[s + 1]]))
            bytes_ = self.cached(layer)
            for s in range(self.S):
                first = int(after[s]) - len(self.tokens[layer][s])
                p = np.arange(first, int(after[s]))
                if not len(p):
                    continue
                cell = table[s, p // self.T].astype(np.int64) * self.T + p % self.T
                for which, t in enumerate(self.types):
                    want = np.stack([r[which] for r in self.tokens[layer][s]]).reshape(len(p), -1, 32)
                    got = decode(oracle, t, bytes_[which][cell], E).reshape(want.shape)
                    most = np.abs(want).max(-1, keepdims=True)
                    assert (np.abs(got - want) <= most * (STEP[t] + 2.0 ** -8) + 1e-6).all(), (layer, s, which)
            c = Case.__new__(Case)
            c.__dict__.update(oracle=oracle, lens=after.tolist(), m=self.new.tolist(), Hq=self.Hq, Hkv=self.Hkv,
                              D=self.D, T=self.T, causal=True, hadamard=self.had, type_k=self.types[0],
                              type_v=self.types[1], n_slots=self.n_slots, stride=self.stride, table=table,
                              pool=dict(zip("kv", bytes_)), rows=self.max_tokens, starts=starts, args=self.args,
                              scale=self.D ** -0.5, q_host=self.q_seen[layer].double().cpu().numpy(),
                              odt=torch.float32, out=self.out[layer], lse=self.lse[layer])
            c.check()


@pytest.mark.parametrize("types,D,Hq,Hkv,T,n_rot,had", [
    (("q4_0", "q4_0"), 256, 24, 4, 128, 64, 64), (("q8_0", "q4_0"), 128, 8, 8, 48, 128, 128),
    (("q5_0", "q5_0"), 64, 16, 2, 16, 64, 0), (("f16", "f16"), 128, 8, 2, 1, 0, 0)])
def test_requests_grow_step_by_step(ctx, oracle, types, D, Hq, Hkv, T, n_rot, had):
    print(f"[decode loop] {types} {D}", flush=True)
    steps = [[37, 0, 130, 1], [1, 5, 1, 1], [1, 1, 0, 1], [0, 0, 0, 0], [3, 60, 1, 2], [1, 1, 1, 1]]
    b = Batch(ctx, 4, Hq, Hkv, D, T, sum(-(-240 // T) for _ in range(4)), -(-240 // T), 200, types, n_rot, had, seed=D)
    for new in steps:
        b.feed(new)
        b.calls(max(max(new), 1), int((b.len + np.array(new)).max()))
        ctx.sync()
        b.check(oracle)
        b.advance()


def test_captured_step_follows_the_requests(ctx, oracle):
    """One graph of a single-token step, replayed while requests grow over block ends; an idle request in between."""
    print("[decode loop] graph", flush=True)
    b = Batch(ctx, 3, 8, 2, 128, 16, 60, 20, 120, ("q4_0", "q4_0"), 64, 64, seed=5)
    b.feed([30, 61, 15])
    b.calls(61, 106)
    ctx.sync()
    b.check(oracle)
    b.advance()
    b.args.max_q, b.args.max_kv = 1, 320
    need = ctx.attention_workspace(b.args, b.pool)
    ws = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    try:
        ctx.set_stream(st.cuda_stream)
        with torch.cuda.graph(g, stream=st):
            b.calls(1, 320, ws)
    finally:
        ctx.set_stream(None)
    for new in ([1, 1, 1], [1, 0, 1], [0, 1, 1], [1, 1, 1], [1, 1, 1], [1, 1, 1]):
        b.feed(new)
        with torch.cuda.stream(st):
            g.replay()
        torch.cuda.synchronize()
        b.check(oracle)
        b.advance()


def test_first_calls_of_a_process_captured(tmp_path):
    """The calls' first launches in a process may be captured ones: a context holds their kernels from its creation."""
    print("[decode loop] first calls", flush=True)
    src = tmp_path / "first.py"
    src.write_text(FIRST)
    root = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, str(src)], cwd=root, capture_output=True, text=True, timeout=100,
                       env={**os.environ, "PYTHONPATH": os.pathsep.join([str(root), str(root.parent)])})
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


FIRST = """
import torch
import conftest
from test_gpu_decode_loop import Batch, kv
ctx = kv.Context(0)
outs = []
for types in (("q4_0", "q8_0"), ("q5_0", "f16"), ("q8_0", "q4_0"), ("f16", "q5_0")):
    b = Batch(ctx, 2, 4, 2, 64, 16, 40, 20, 60, types, 64, 64, layers=1, seed=3)
    b.feed([30, 25])
    st = torch.cuda.Stream()
    ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    ctx.set_stream(st.cuda_stream)
    with torch.cuda.graph(g, stream=st):
        b.calls(30, 64, ws)
    ctx.set_stream(None)
    g.replay()
    torch.cuda.synchronize()
    first = b.out[0].clone()
    b.out[0].fill_(7.25)
    b.calls(30, 64)
    ctx.sync()
    assert torch.equal(b.out[0], first) and bool((first[:55] != 7.25).any())
print("same")
"""


def test_new_tokens_over_the_engines_window(oracle):
    """The window the reselect engine staged, blocks it left out as entries without a slot, continued token by token."""
    print("[decode loop] engine", flush=True)
    L, T, E, D = eh.L, eh.T, eh.E, 64
    cap, nb = 24, 24
    k, v, q = eh.history(cap, seed=61)
    with eh.make_engine(8, 2) as eng:
        eng.set_device_history(k.data_ptr(), v.data_ptr(), cap, nb * T)
        sel = eng.preview(q.data_ptr(), q.shape[1])
        eng.apply(sel)
        ctx = kv.Context.borrow(eng.ctx_handle())
        ctx.sync()
        slots = np.array(eng.block_slots()[:nb])
        assert 0 < (slots >= 0).sum() < nb, "blocks are left out"
        stride, n_slots = nb + 2, eng.n_slots()
        table = np.full((1, stride), kv.NO_SLOT, np.uint32)
        table[0, :nb][slots >= 0] = slots[slots >= 0]
        free = [s for s in range(n_slots) if s not in set(slots.tolist())]
        ptrs = [eng.pool_layer(layer) for layer in range(L)]
        pool = ctx.make_pool(L, n_slots, T, E, E, eng.params.type_k, eng.params.type_v, [p[0] for p in ptrs],
                             [p[1] for p in ptrs])
        b = Batch(ctx, 1, 2 * E // D, E // D, D, T, n_slots, stride, 5, ("q8_0", "q8_0"), 0, 0, layers=L, seed=9,
                  pool=pool, table=table, kv_len=[nb * T], free=free)

        def cached(layer):
            out = []
            for ptr in ptrs[layer]:
                t = torch.empty((n_slots * T, kv.row_size(kv.TYPE_Q8_0, E)), dtype=torch.uint8, device="cuda")
                ctx.d2d_batched([ptr], [t.data_ptr()], [t.numel()])
                ctx.sync()
                out.append(t.cpu().numpy())
            return out

        b.cached = cached
        before = cached(0)
        for new in ([5], [1], [1]):
            b.feed(new)
            b.calls(max(new), nb * T + 8)
            ctx.sync()
            b.check(oracle)
            b.advance()
        held = np.concatenate([np.arange(s * T, (s + 1) * T) for s in slots if s >= 0])
        assert all((a[held] == c[held]).all() for a, c in zip(before, cached(0))), "the staged rows stay"
