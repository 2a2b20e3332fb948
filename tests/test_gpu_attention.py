"""kvmem_hip_attention against a float64 reference over the values the cached
bytes stand for (attention_helpers: bounds counted from the roundings)."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
from attention_helpers import Case, decode, quantize  # noqa: E402

TYPES = ["q4_0", "q5_0", "q8_0", "f16"]
# around every tile and block edge, none, one, and a few hundred keys
LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 700]


def say(*a):
    print("[attention]", *a, flush=True)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type_k", TYPES)
@pytest.mark.parametrize("type_v", TYPES)
def test_single_tokens(ctx, oracle, type_k, type_v, D):
    say("decode", type_k, type_v, D)
    Case(ctx, oracle, LENS, [1] * len(LENS), 12, 2, D, 128, type_k, type_v, seed=1).run().check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("types", [("q4_0", "q4_0"), ("q5_0", "q8_0"), ("q8_0", "q4_0"), ("f16", "f16"), ("f16", "q5_0")])
def test_prompts(ctx, oracle, types, D):
    """Ragged new tokens, from none to more than a tile of rows, some longer than the keys behind them."""
    say("prompts", types, D)
    m = [1, 0, 5, 17, 64, 100, 33]
    lens = [300, 9, 5, 140, 64, 333, 1]  # the last has fewer keys than tokens: its first rows see none
    Case(ctx, oracle, lens, m, 6, 2, D, 64, *types, seed=2).run().check()


@pytest.mark.parametrize("T", [1, 7, 16, 48, 100, 512])
@pytest.mark.parametrize("D", [64, 256])
def test_block_sizes(ctx, oracle, T, D):
    """Blocks that end inside a tile, and tiles that end inside a block."""
    say("blocks of", T, D)
    Case(ctx, oracle, [5, 130, 259, 0], [1, 1, 1, 1], 4, 2, D, T, seed=3).run().check()
    Case(ctx, oracle, [77, 130, 259], [40, 3, 70], 4, 2, D, T, "q8_0", "q5_0", seed=4).run().check()


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (8, 1), (8, 8), (9, 3), (16, 1), (20, 1), (34, 2), (24, 4)])
def test_head_groups(ctx, oracle, Hq, Hkv):
    say("heads", Hq, Hkv)
    Case(ctx, oracle, [1, 70, 200], [1, 1, 1], Hq, Hkv, 128, 32, seed=5).run().check()
    Case(ctx, oracle, [50, 70, 200], [2, 4, 11], Hq, Hkv, 128, 32, seed=6).run().check()
    Case(ctx, oracle, [150], [90], Hq, Hkv, 64, 32, "q8_0", "q8_0", seed=7).run().check()


@pytest.mark.parametrize("m", [1, 2, 3, 40])
def test_holes_and_empty_tables(ctx, oracle, m):
    """Blocks without a slot, slots outside the pool, requests left without any key."""
    say("holes", m)
    for holes in (0.3, 0.8, 1.0):
        Case(ctx, oracle, [300, 129, 64, 1000], [m] * 4, 6, 2, 128, 16, holes=holes, seed=8).run().check()


@pytest.mark.parametrize("m", [1, 6, 70])
def test_not_causal(ctx, oracle, m):
    say("all keys", m)
    Case(ctx, oracle, [300, 5, 0], [m] * 3, 6, 2, 64, 32, causal=False, seed=9).run().check()


@pytest.mark.parametrize("q_type", ["f16", "bf16"])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 50])
def test_types_and_strides(ctx, oracle, q_type, out_type, m):
    say(q_type, out_type, m)
    Case(ctx, oracle, [200, 90], [m, m], 6, 2, 128, 32, q_type=q_type, out_type=out_type, q_pad=8, seed=10).run().check()


@pytest.mark.parametrize("D,width", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 256)])
@pytest.mark.parametrize("m", [1, 30])
def test_rotated_values(ctx, oracle, D, width, m):
    say("hadamard", D, width, m)
    Case(ctx, oracle, [200, 3, 0], [m] * 3, 6, 2, D, 32, hadamard=width, seed=11).run().check()


@pytest.mark.parametrize("m", [1, 20])
def test_long_cache_is_split(ctx, oracle, m):
    """Keys split over workgroups: a long request beside short and empty ones."""
    say("long", m)
    Case(ctx, oracle, [9000, 0, 1, 130, 4097], [m, m, 1, m, m], 6, 1, 128, 128, seed=12, hadamard=64).run().check()
    Case(ctx, oracle, [20011], [m], 4, 2, 64, 32, "q8_0", "q4_0", holes=0.2, seed=13).run().check()


def test_scale_and_large_values(ctx, oracle):
    """An explicit scale; value rows near f16's end; keys whose scores pass 10^4."""
    for m in (1, 20):
        Case(ctx, oracle, [100, 33], [m, m], 4, 2, 64, 32, scale=0.37, seed=14).run().check()
        for t in ("f16", "q8_0"):
            c = Case(ctx, oracle, [100, 33], [m, m], 4, 2, 64, 32, "q8_0", t, v_scale=1.0, seed=15)
            x = np.where(np.random.default_rng(3).random((c.n_slots * 32, 128)) < 0.5, -60000.0, 60000.0)
            c.pool["v"] = quantize(oracle, t, x)
            c.upload()
            c.run().check()
        c = Case(ctx, oracle, [100, 33], [m, m], 4, 2, 64, 32, "f16", "f16", k_scale=3000.0, causal=False, seed=16)
        c.run()
        got = c.out.cpu().double().numpy()
        assert np.isfinite(got).all()
        # one key takes all the weight: its value row comes back
        ref = c.reference()[0]
        assert np.abs(got - ref).max() <= 2.0 ** -10 * np.abs(ref).max()


def test_query_beyond_f16(ctx, oracle):
    """bf16 queries past f16's range (either end) keep their scores."""
    for m in (1, 20):
        for f in (2.0 ** 20, 2.0 ** -30):
            c = Case(ctx, oracle, [100, 33], [m, m], 4, 2, 64, 32, "q8_0", "f16", scale=0.125 / f, seed=17)
            c.q.mul_(f)
            c.q_host = c.q_host * f
            c.run().check()


def test_rows_behind_the_last_request_stay(ctx, oracle):
    for m in (1, 30):
        Case(ctx, oracle, [200, 90], [m, 1], 6, 2, 128, 32, extra_rows=5, seed=18).run().check()


def test_bounds_of_a_call(ctx, oracle):
    """Keys past max_kv or the table, tokens past max_q: never attended, nothing out of range."""
    Case(ctx, oracle, [300, 90], [1, 1], 4, 2, 64, 32, max_kv=130, seed=19).run().check()
    Case(ctx, oracle, [300, 90], [9, 3], 4, 2, 64, 32, max_q=4, seed=20).run().check()
    c = Case(ctx, oracle, [300, 90], [1, 1], 4, 2, 64, 32, seed=21)
    c.args.table_stride = c.stride = 3  # a narrower table: request 1 starts at another entry
    c.table = c.table.reshape(-1)[:6].reshape(2, 3)
    c.run().check()
    # device lengths beyond every bound
    c = Case(ctx, oracle, [300, 90], [2, 2], 4, 2, 64, 32, causal=False, seed=22)
    c.dev["lens"].fill_(-1)
    c.dev["starts"].copy_(torch.tensor([0, 2, 2 ** 31 - 1], dtype=torch.int32))
    c.args.max_kv = 90
    c.run()
    want = c.reference(lens=[90, 90], m=[2, 2])
    assert np.abs(c.out.cpu().double().numpy()[:2] - want[0][:2]).max() < 1e-1
    # starts that run backwards: no rows
    c.dev["starts"].copy_(torch.tensor([3, 1, 0], dtype=torch.int32))
    c.out.fill_(7.25)
    c.run()
    assert (c.out == 7.25).all()


def test_same_slot_twice_and_shared_slots(ctx, oracle):
    """A slot listed twice counts twice; requests may share slots."""
    for m in (1, 20):
        c = Case(ctx, oracle, [160, 160], [m, m], 4, 2, 64, 32, seed=23)
        c.table[0, 1] = c.table[0, 0]
        c.table[1, :4] = c.table[0, :4]
        c.dev["table"].copy_(torch.from_numpy(c.table.view(np.int32)))
        c.run().check()


@pytest.mark.parametrize("m", [2, 8, 40])
@pytest.mark.parametrize("type_", ["f16", "q4_0"])
def test_later_keys_do_not_reach_earlier_queries(ctx, oracle, m, type_):
    """An infinity or NaN in a key or value row reaches only the queries that attend it."""
    say("poisoned last key", m, type_)
    c = Case(ctx, oracle, [100, 64], [m, m], 4, 2, 64, 32, type_, type_, seed=24)
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


def test_queries_without_q_start(ctx, oracle):
    """q_start NULL: one token a request."""
    c = Case(ctx, oracle, LENS, [1] * len(LENS), 6, 2, 128, 32, seed=25, extra_rows=2)
    c.args.q_start = None
    c.args.max_q = 99
    c.run().check()


def test_repeats_bit_for_bit(ctx, oracle):
    for m in (1, 30):
        c = Case(ctx, oracle, [5000, 333], [m, m], 8, 2, 128, 64, seed=26)
        a = c.run().out.clone()
        for _ in range(3):
            c.out.fill_(0)
            assert torch.equal(c.run().out, a)


def test_workspace_and_allocations(ctx, oracle):
    """The caller's workspace gives the context's results; a second call of the same size allocates nothing."""
    for m in (1, 30):
        c = Case(ctx, oracle, [9000, 400], [m, m], 8, 2, 128, 64, seed=27)
        need = ctx.attention_workspace(c.args, c.pool_c)
        assert need > 0
        want = c.run().out.clone()
        before = ctx.scratch_info()["allocations"]
        c.out.fill_(0)
        assert torch.equal(c.run().out, want)
        assert ctx.scratch_info()["allocations"] == before
        ws = torch.full((need + 64,), 0x7F, dtype=torch.uint8, device="cuda")
        c.args.workspace, c.args.workspace_bytes = ws.data_ptr(), need
        c.out.fill_(0)
        assert torch.equal(c.run().out, want)
        assert (ws[need:] == 0x7F).all()


@pytest.mark.parametrize("m", [1, 30])
def test_captured_call(ctx, oracle, m):
    """Two graphs with a workspace each, replayed by turns and together, follow the lengths and queries they find."""
    say("graphs", m)
    cs = [Case(ctx, oracle, [3000, 400], [m, m], 8, 2, 64, 64, seed=28 + i) for i in range(2)]
    eager = [c.run().out.clone() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    graphs, keep = [], []
    try:
        for c, st in zip(cs, streams):
            need = ctx.attention_workspace(c.args, c.pool_c)
            ws = torch.empty(need, dtype=torch.uint8, device="cuda")
            keep.append(ws)
            ctx.set_stream(st.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                with pytest.raises(kv.KvMemError):
                    ctx.attention(c.args, c.pool_c, 1)  # no workspace of its own
                c.args.workspace, c.args.workspace_bytes = ws.data_ptr(), need
                ctx.attention(c.args, c.pool_c, 1)
            graphs.append(g)
        ctx.set_stream(None)
        for step in range(4):
            for c in cs:
                c.out.fill_(0)
            torch.cuda.synchronize()
            for g, st in zip(graphs, streams):  # both in flight
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for c, e in zip(cs, eager):
                assert torch.equal(c.out, e), step
            # shorter requests and other queries for the next replay
            for i, c in enumerate(cs):
                c.lens = [a - 301 if a > 400 else a - 40 for a in c.lens]
                c.dev["lens"].copy_(torch.tensor(c.lens, dtype=torch.int32))
                c.q.neg_()
                c.q_host = -c.q_host
                c.out.fill_(0)
                c.run().check()
                eager[i] = c.out.clone()
    finally:
        ctx.set_stream(None)


def test_other_stream(ctx, oracle):
    """On a caller's stream, behind work queued there."""
    c = Case(ctx, oracle, [300, 90], [1, 1], 4, 2, 64, 32, seed=30)
    want = c.run().out.clone()
    st = torch.cuda.Stream()
    q = c.q.clone()
    c.q.zero_()
    torch.cuda.synchronize()
    ctx.set_stream(st.cuda_stream)
    try:
        with torch.cuda.stream(st):
            x = torch.ones((2048, 2048), device="cuda")
            for _ in range(20):
                x = x @ x * 1e-4
            c.q.copy_(q)
            ctx.attention(c.args, c.pool_c, 1)
        st.synchronize()
    finally:
        ctx.set_stream(None)
    assert torch.equal(c.out, want)


def test_rows_past_4_gib(ctx, oracle):
    """Slots whose byte offsets pass 32 bits."""
    Hkv, D, T = 4, 256, 128
    row = kv.row_size(kv.TYPE_F16, Hkv * D)
    n_slots = (5 << 30) // (row * T)
    big = {w: torch.full((n_slots * T, row), 255, dtype=torch.uint8, device="cuda") for w in "kv"}
    for m in (1, 30):
        c = Case(ctx, oracle, [300], [m], 8, Hkv, D, T, "f16", "f16", seed=31)
        far = [n_slots - 1, 3, n_slots - 5]
        for b, slot in enumerate(far):
            src = int(c.table[0, b]) * T
            for w in "kv":
                big[w][slot * T:slot * T + T].copy_(c.dev[w][src:src + T])
        c.dev["table"][0, :3] = torch.tensor(far, dtype=torch.int32)
        pool = ctx.make_pool(1, n_slots, T, Hkv * D, Hkv * D, kv.TYPE_F16, kv.TYPE_F16, [big["k"].data_ptr()],
                             [big["v"].data_ptr()])
        torch.cuda.synchronize()
        ctx.attention(c.args, pool, 0)
        ctx.sync()
        c.check()


def test_nothing_to_do(ctx, oracle):
    c = Case(ctx, oracle, [30], [1], 4, 2, 64, 32, seed=32)
    for field in ("n_seq", "n_tokens", "max_q"):
        old = getattr(c.args, field)
        setattr(c.args, field, 0)
        c.run()
        assert (c.out == 7.25).all()
        setattr(c.args, field, old)
    c.args.max_kv = 0  # no key fits: every row is empty
    c.run()
    assert (c.out == 0).all() and torch.isneginf(c.lse).all()
    c.args.lse = None
    c.run()
