"""kvmem_hip_slot_map against a plain loop over requests, blocks and tokens:
tables, cells, positions and counts equal word for word -- from one request
with one token to 4096 requests, requests that bring nothing or have nothing,
block sizes that are no power of two, an exhausted free list, tables too
narrow for a request, entries that name no slot, lengths past 32 bits' sum,
and a captured call replayed with other lengths."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
NONE = kv.NO_SLOT
FILL = 0x7b7b7b7b


def expected(n, m, T, W, n_slots, free, used, table, max_tokens, pos0):
    """The definition, one token at a time."""
    table = table.copy()
    S = len(n)
    cells = np.full(max_tokens, -1, np.int64)
    pos = np.zeros(max_tokens, np.int64)
    taken = min(used, len(free))
    missing, t, q_start = 0, 0, [0]
    for s in range(S):
        b0, b1 = -(-n[s] // T), -(-(n[s] + m[s]) // T)
        for b in range(b0, b1):
            if b >= W:
                missing += 1
            elif taken < len(free):
                table[s, b] = free[taken] if free[taken] < n_slots else NONE
                taken += 1
            else:
                table[s, b] = NONE
                missing += 1
        for i in range(min(m[s], max(0, max_tokens - t))):
            p = n[s] + i
            pos[t + i] = (n[s] if pos0 is None else pos0[s]) + i
            slot = table[s, p // T] if p // T < W else NONE
            cells[t + i] = slot * T + p % T if slot < n_slots else -1
        t += m[s]
        q_start.append(t)
    return dict(table=table, kv_len=np.array(n) + np.array(m), q_start=np.array(q_start), positions=pos,
                cells=cells, used=taken, missing=missing)


class Batch:
    def __init__(self, n, m, T, W, n_slots, free, used, table, max_tokens, pos0=None):
        self.args = (n, m, T, W, n_slots, free, used, table, max_tokens, pos0)
        S = len(n)
        u = lambda a: torch.from_numpy(np.asarray(a, np.uint32).view(np.int32).copy()).cuda()  # noqa: E731
        self.t = dict(n=u(n), m=u(m), free=u(free if len(free) else [0]), used=u([used]), table=u(table))
        if pos0 is not None:
            self.t["pos0"] = torch.tensor(pos0, dtype=torch.int32, device="cuda")
        out = lambda k: torch.full((k + 1,), FILL, dtype=torch.int32, device="cuda")  # noqa: E731
        self.o = dict(kv_len=out(S), q_start=out(S + 1), positions=out(max_tokens), cells=out(max_tokens),
                      used=out(1), missing=out(1))
        t, o = self.t, self.o
        self.c = kv.SlotMapArgs(n_seq=S, block_tokens=T, n_slots=n_slots, table_stride=W, max_tokens=max_tokens,
                                n_free=len(free), n_new=t["m"].data_ptr(), kv_len=t["n"].data_ptr(),
                                pos0=t["pos0"].data_ptr() if pos0 is not None else None,
                                free_slots=t["free"].data_ptr(), free_used=t["used"].data_ptr(),
                                table=t["table"].data_ptr(), kv_len_out=o["kv_len"].data_ptr(),
                                q_start=o["q_start"].data_ptr(), positions=o["positions"].data_ptr(),
                                cells=o["cells"].data_ptr(), free_used_out=o["used"].data_ptr(),
                                n_missing=o["missing"].data_ptr())
        torch.cuda.synchronize()

    def check(self, want=None):
        n, m, T, W, n_slots, free, used, table, max_tokens, pos0 = self.args
        want = want or expected(n, m, T, W, n_slots, free, used, table, max_tokens, pos0)
        got = self.t["table"].cpu().numpy().view(np.uint32).reshape(table.shape)
        assert np.array_equal(got, want["table"])
        for name, x in self.o.items():
            g = x.cpu().numpy()
            assert g[-1] == FILL, f"{name}: written past its end"
            w = np.asarray(want[name]).reshape(-1)
            assert np.array_equal(g[:-1].view(np.uint32), (w & 0xffffffff).astype(np.uint32)), name


def random_batch(rng, S, T, most_n, most_m, spare=3, W=None, bad=False, pos=False):
    n = [0 if rng.random() < 0.2 else int(rng.integers(0, most_n + 1)) for _ in range(S)]
    m = [0 if rng.random() < 0.2 else int(rng.integers(0, most_m + 1)) for _ in range(S)]
    need = [-(-(a + b) // T) for a, b in zip(n, m)]
    held = [-(-a // T) for a in n]
    W = W or max(1, max(need) + 1)
    n_slots = sum(need) + max(spare, 0) + 4
    order = rng.permutation(n_slots).astype(np.uint32)
    table = np.full((S, W), 0xabcdef01, np.uint32)  # entries nobody owns stay
    at = 0
    for s in range(S):
        for b in range(min(held[s], W)):
            table[s, b] = order[at]
            at += 1
    used = int(min(3, at))
    free = np.concatenate([order[at - used:at], order[at:max(at, len(order) + min(spare, 0))]])
    if bad:
        free[rng.integers(used, len(free), 2)] = [n_slots, 0xfffffff0]
        for s in range(S):
            if held[s]:
                table[s, 0] = NONE
    pos0 = [int(x) for x in rng.integers(0, 1 << 20, S)] if pos else None
    return Batch(n, m, T, W, n_slots, free, used, table, sum(m) + int(rng.integers(0, 9)), pos0)


@pytest.mark.parametrize("S,T,most_n,most_m", [(1, 128, 0, 1), (1, 1, 5, 3), (2, 128, 127, 2), (3, 16, 16, 16),
                                               (7, 48, 1000, 1), (64, 128, 4000, 1), (65, 32, 300, 77),
                                               (255, 128, 900, 3), (257, 80, 500, 40), (1023, 7, 30, 5),
                                               (4096, 64, 200, 9), (5, 128, 300, 3000)])
def test_matches_the_definition(ctx, S, T, most_n, most_m):
    print(f"[slot_map] S={S} T={T} n<={most_n} m<={most_m}", flush=True)
    rng = np.random.default_rng([S, T, most_n, most_m])
    for pos in (False, True):
        b = random_batch(rng, S, T, most_n, most_m, pos=pos)
        for _ in range(2):  # idempotent
            ctx.slot_map(b.c)
            ctx.sync()
            b.check()


def test_free_list_ends_and_bad_entries(ctx):
    rng = np.random.default_rng(5)
    for spare in (-1, -6, -40):
        b = random_batch(rng, 40, 16, 100, 30, spare=spare)
        ctx.slot_map(b.c)
        ctx.sync()
        b.check()
    b = random_batch(rng, 40, 16, 100, 30, bad=True)
    ctx.slot_map(b.c)
    ctx.sync()
    b.check()
    # no free list at all
    b = Batch([3], [2], 4, 2, 8, [], 0, np.array([[5, 77]], np.uint32), 2)
    ctx.slot_map(b.c)
    ctx.sync()
    b.check()
    assert b.o["cells"][:2].tolist() == [23, -1] and b.o["missing"][0] == 1


def test_table_too_narrow_and_tokens_past_the_end(ctx):
    rng = np.random.default_rng(6)
    b = random_batch(rng, 9, 16, 200, 100, W=5)
    ctx.slot_map(b.c)
    ctx.sync()
    b.check()
    b = Batch([10, 4], [6, 9], 4, 8, 99, list(range(50, 70)), 0, np.arange(16, dtype=np.uint32).reshape(2, 8), 7)
    ctx.slot_map(b.c)
    ctx.sync()
    b.check()
    b = Batch([10, 4], [6, 9], 4, 8, 99, list(range(50, 70)), 0, np.arange(16, dtype=np.uint32).reshape(2, 8), 0)
    ctx.slot_map(b.c)
    ctx.sync()
    b.check()


def test_lengths_past_32_bits_stay_in_range(ctx):
    """Device lengths whose sums pass 32 bits saturate; nothing is written past the arrays."""
    big = 0xfffffff0
    b = Batch([big, 7, big], [100, 3, big], 128, 4, 64, [9, 8], 0, np.full((3, 4), 2, np.uint32), 5)
    ctx.slot_map(b.c)
    ctx.sync()
    want = dict(table=np.full((3, 4), 2, np.uint32), kv_len=[0xffffffff, 10, 0xffffffff],
                q_start=[0, 100, 103, 0xffffffff], positions=[big + i for i in range(5)], cells=[-1] * 5, used=0,
                missing=-(-0xffffffff // 128) - -(-big // 128) + -(-0xffffffff // 128) - -(-big // 128))
    b.check(want)


def test_captured_call_follows_the_lengths(ctx):
    rng = np.random.default_rng(8)
    b = random_batch(rng, 33, 32, 200, 40)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ctx.slot_map(b.c)
        n, m = b.args[0], b.args[1]
        for step in range(4):
            with torch.cuda.stream(stream):
                x = torch.full((64, 64), float(step), device="cuda") @ torch.ones((64, 64), device="cuda")
                graph.replay()
            stream.synchronize()
            assert float(x[0, 0]) == 64.0 * step
            b.check()
            # the next batch: lengths moved on, the same blocks held and free slots taken
            b.args = (b.o["kv_len"][:-1].tolist(), [1] * len(m), *b.args[2:6], int(b.o["used"][0]),
                      b.t["table"].cpu().numpy().view(np.uint32).reshape(b.args[7].shape).copy(), *b.args[8:])
            b.t["n"].copy_(b.o["kv_len"][:-1])
            b.t["m"].fill_(1)
            b.t["used"].copy_(b.o["used"][:1])
            torch.cuda.synchronize()
        assert n != b.args[0]
    finally:
        ctx.set_stream(None)
