"""kvmem_hip_attention with many new tokens a request (more (token, head) rows of
a KV head than the few-query kernel takes: 192 for one request, 64 for many),
against the float64 reference and bounds of attention_helpers: every pair of
cache types, blocks that end inside a step, blocks without a slot, all keys and
causal, query and output types with strides, rotated values, split keys,
infinities and NaN in keys that only the last token attends, queries and values
at f16's ends, rows behind the last request, device lengths past every bound,
repeated, captured and other-stream calls."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
from attention_helpers import Case, quantize  # noqa: E402

TYPES = ["q4_0", "q5_0", "q8_0", "f16"]


def many(ctx, oracle, lens, m, Hq, Hkv, *rest, **kw):
    """A Case whose call must take the many-query kernel."""
    rows = (kw.get("max_q") or max(m)) * (Hq // Hkv)
    assert rows > 192 or (rows > 64 and len(lens) >= 8), "few queries"
    return Case(ctx, oracle, lens, m, Hq, Hkv, *rest, **kw)


def say(*a):
    print("[prompts]", *a, flush=True)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type_k", TYPES)
@pytest.mark.parametrize("type_v", TYPES)
def test_type_pairs(ctx, oracle, type_k, type_v, D):
    say(type_k, type_v, D)
    many(ctx, oracle, [190, 70, 9], [100, 70, 0], 6, 2, D, 64, type_k, type_v, seed=101).run().check()


@pytest.mark.parametrize("T", [1, 7, 48, 100, 512])
@pytest.mark.parametrize("D", [64, 256])
def test_block_sizes(ctx, oracle, T, D):
    say("blocks of", T, D)
    many(ctx, oracle, [177, 130, 259], [70, 3, 33], 4, 1, D, T, "q8_0", "q5_0", seed=102).run().check()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_holes_and_empty_tables(ctx, oracle, D):
    say("holes", D)
    for holes in (0.3, 0.8, 1.0):
        many(ctx, oracle, [300, 129, 64, 500], [60] * 4, 4, 1, D, 16, holes=holes, seed=103).run().check()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_not_causal(ctx, oracle, D):
    say("all keys", D)
    many(ctx, oracle, [300, 5, 0], [70] * 3, 6, 2, D, 32, causal=False, seed=104).run().check()


@pytest.mark.parametrize("q_type", ["f16", "bf16"])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
def test_types_and_strides(ctx, oracle, q_type, out_type):
    say(q_type, out_type)
    many(ctx, oracle, [200, 90], [70, 70], 6, 2, 128, 32, q_type=q_type, out_type=out_type, q_pad=8, seed=105,
         extra_rows=5).run().check()


@pytest.mark.parametrize("D,width", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 256)])
def test_rotated_values(ctx, oracle, D, width):
    say("hadamard", D, width)
    many(ctx, oracle, [200, 3, 0], [70] * 3, 6, 2, D, 32, hadamard=width, seed=106).run().check()
    many(ctx, oracle, [2000], [70], 6, 2, D, 32, hadamard=width, out_type="bf16", seed=107).run().check()


def test_long_cache_is_split(ctx, oracle):
    say("long")
    many(ctx, oracle, [6000, 0, 1, 130, 4097], [34, 34, 1, 34, 34], 6, 1, 128, 128, seed=108, hadamard=64).run().check()
    many(ctx, oracle, [9011], [50], 4, 1, 64, 32, "q8_0", "q4_0", holes=0.2, seed=109).run().check()


def test_tiles_of_256_rows(ctx, oracle):
    """Rows that end at, before and behind a tile of 256; single heads and groups that do not divide it."""
    for m, Hq in ((256, 1), (255, 1), (257, 1), (86, 3), (37, 7)):
        say("rows", m * Hq)
        many(ctx, oracle, [m + 40], [m], Hq, 1, 64, 32, seed=110).run().check()


def test_many_requests(ctx, oracle):
    say("nine requests")
    many(ctx, oracle, [40, 100, 1, 33, 64, 65, 0, 17, 128], [30, 40, 1, 33, 12, 1, 0, 17, 5], 4, 2, 128, 16,
         seed=111).run().check()


def test_large_values_and_queries(ctx, oracle):
    say("ends of f16")
    for t in ("f16", "q8_0"):
        c = many(ctx, oracle, [130, 33], [100, 33], 4, 2, 64, 32, "q8_0", t, seed=112)
        x = np.where(np.random.default_rng(3).random((c.n_slots * 32, 128)) < 0.5, -60000.0, 60000.0)
        c.pool["v"] = quantize(oracle, t, x)
        c.upload()
        c.run().check()
    for f in (2.0 ** 20, 2.0 ** -30):
        c = many(ctx, oracle, [130, 33], [100, 33], 4, 2, 64, 32, "q8_0", "f16", scale=0.125 / f, seed=113)
        c.q.mul_(f)
        c.q_host = c.q_host * f
        c.run().check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type_", ["f16", "q4_0"])
def test_later_keys_do_not_reach_earlier_queries(ctx, oracle, type_, D):
    say("poisoned last key", type_, D)
    c = many(ctx, oracle, [140, 114], [100, 100], 4, 2, D, 32, type_, type_, seed=114)
    clean = c.run().check().copy()
    for bits in (0x7C00, 0x7E00):
        for s in range(2):
            last = c.lens[s] - 1
            row = int(c.table[s, last // 32]) * 32 + last % 32
            for w in "kv":
                c.pool[w][row].view(np.uint16)[0] = bits
        c.upload()
        c.run()
        got = c.out.cpu().double().numpy()
        for s in range(2):
            a, b = int(c.starts[s]), int(c.starts[s + 1])
            assert np.array_equal(got[a:b - 1], clean[a:b - 1])
            assert not np.isfinite(got[b - 1, 0]).all()


def test_bounds_of_a_call(ctx, oracle):
    say("bounds")
    many(ctx, oracle, [300, 90], [100, 60], 4, 1, 64, 32, max_kv=130, seed=115).run().check()
    many(ctx, oracle, [300, 90], [90, 63], 4, 1, 64, 32, max_q=60, seed=116).run().check()
    c = many(ctx, oracle, [300, 90], [60, 60], 4, 1, 64, 32, causal=False, seed=117)
    c.dev["lens"].fill_(-1)
    c.dev["starts"].copy_(torch.tensor([0, 60, 2 ** 31 - 1], dtype=torch.int32))
    c.args.max_kv = 90
    c.run()
    want = c.reference(lens=[90, 90], m=[60, 60])
    assert np.abs(c.out.cpu().double().numpy() - want[0]).max() < 1e-1
    c.dev["starts"].copy_(torch.tensor([130, 7, 0], dtype=torch.int32))  # backwards: no rows
    c.out.fill_(7.25)
    c.run()
    assert (c.out == 7.25).all()


def test_repeats_and_workspaces(ctx, oracle):
    say("repeats")
    c = many(ctx, oracle, [5000, 333], [70, 70], 8, 2, 128, 64, seed=118)
    need = ctx.attention_workspace(c.args, c.pool_c)
    assert need > 0
    a = c.run().out.clone()
    ws = torch.full((need + 64,), 0x7F, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        c.out.fill_(0)
        assert torch.equal(c.run().out, a)
        c.args.workspace, c.args.workspace_bytes = ws.data_ptr(), need
    assert (ws[need:] == 0x7F).all()


def test_captured_calls_by_turns_and_together(ctx, oracle):
    say("graphs")
    cs = [many(ctx, oracle, [3000, 400], [100, 100], 8, 2, 64, 64, seed=119 + i) for i in range(2)]
    eager = [c.run().out.clone() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    graphs, keep = [], []
    try:
        for c, st in zip(cs, streams):
            ws = torch.empty(ctx.attention_workspace(c.args, c.pool_c), dtype=torch.uint8, device="cuda")
            keep.append(ws)
            c.args.workspace, c.args.workspace_bytes = ws.data_ptr(), ws.numel()
            ctx.set_stream(st.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                ctx.attention(c.args, c.pool_c, 1)
            graphs.append(g)
        ctx.set_stream(None)
        for step in range(3):
            for c in cs:
                c.out.fill_(0)
            torch.cuda.synchronize()
            for g, st in zip(graphs, streams):  # both in flight
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for c, e in zip(cs, eager):
                assert torch.equal(c.out, e), step
            for i, c in enumerate(cs):  # shorter requests, other queries
                c.lens = [a - 301 if a > 500 else a - 40 for a in c.lens]
                c.dev["lens"].copy_(torch.tensor(c.lens, dtype=torch.int32))
                c.q.neg_()
                c.q_host = -c.q_host
                c.out.fill_(0)
                c.run()
                eager[i] = c.out.clone()
            cs[0].check()
    finally:
        ctx.set_stream(None)
