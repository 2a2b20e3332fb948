"""kvmem_hip_qkv_rows: per-head norm, RoPE, Walsh-Hadamard rotation and the
quantized rows of new tokens.

Against float64 numpy with bounds counted from the roundings (below), and
bit for bit against the oracle's transform and quantizers where no norm is
applied (the bytes the stage-in writes for the same rows).

Bounds.  e = 2^-24 (half a float32 step).  The sum of D squares errs by at
most (D + 2) e relative, mean, eps, sqrt and the reciprocal add 5 e at most on
a value halved by the root, two products 2 e: y is within g = (D/2 + 10) e of
its value, relative.  cos and sin are within one rounding, two products and a
sum: a rotated element is within (g + 4 e) (|a| + |b|).  Each of the log2(w)
butterfly stages adds e of the sum of magnitudes, the scaling 2 e: within
(g + (8 + log2 w) e) * S, S the sum of magnitudes of the run over sqrt(w).
Stored values add half a step of their type.  A quantized value is within half
a step of d of the row (q4_0, q5_0: one step where the code saturates at the
far end) and within 2^-11 of its code times d (d is stored as f16); a code can
sit on the other side of a tie when the row is off by its bound."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
DT = {"f32": (torch.float32, kv.TYPE_F32), "f16": (torch.float16, kv.TYPE_F16), "bf16": (torch.bfloat16, kv.TYPE_BF16)}
CACHE = {"q8_0": kv.TYPE_Q8_0, "q5_0": kv.TYPE_Q5_0, "q4_0": kv.TYPE_Q4_0, "f16": kv.TYPE_F16}
E32 = 2.0 ** -24


def walsh(width):
    h = np.ones((1, 1))
    while h.shape[0] < width:
        h = np.block([[h, h], [h, -h]])
    return h


def reference(x, w, eps, pos, theta, n_rot, had):
    """(normed, its bound, rotated, its bound) of float64 rows [N, H, D]."""
    x = x.astype(np.float64)
    D = x.shape[-1]
    g = 0.0
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        g = (D / 2 + 10) * E32
    y, yb = x, g * np.abs(x)
    if n_rot:
        h = n_rot // 2
        a = (pos.astype(np.float32)[:, None] * theta[None]).astype(np.float64)[:, None]
        c, s = np.cos(a), np.sin(a)
        x0, x1 = x[..., :h], x[..., h:n_rot]
        y = np.concatenate([x0 * c - x1 * s, x0 * s + x1 * c, x[..., n_rot:]], -1)
        m = (g + 4 * E32) * (np.abs(x0) + np.abs(x1))
        yb = np.concatenate([m, m, yb[..., n_rot:]], -1)
    if had:
        H = walsh(had) / math.sqrt(had)
        run = y.reshape(-1, had)
        S = np.abs(run).sum(-1, keepdims=True) / math.sqrt(had)
        mag = yb.reshape(-1, had).sum(-1, keepdims=True) / math.sqrt(had)
        y = (run @ H).reshape(y.shape)
        yb = np.broadcast_to(mag + (8 + math.log2(had)) * E32 * S, run.shape).reshape(y.shape)
    return x, g * np.abs(x), y, yb


def close(got, want, bound, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half
    got = got.detach().cpu().double().numpy()
    off = np.abs(got - want) - (bound + half * (np.abs(want) + bound) + tiny)
    assert np.isfinite(got).all() and (off <= 0).all(), f"over the bound by {off.max():.3e}"


def rows(rng, N, H, D, dt, pad=0, scale=1.0):
    """A strided device view [N, H, D] (element stride 1) and its values."""
    x = (rng.standard_normal((N, H, D + pad)) * scale).astype(np.float32)
    x[..., ::29] *= 6.0
    t = torch.from_numpy(x).cuda().to(dt)[..., :D]
    return t, t.float().cpu().numpy()


def call(ctx, *, N, Hq, Hkv, D, type_="bf16", out_type=None, n_rot=0, had_k=0, had_v=0, norm=True, cache=None, T=16,
         pad=0, capture=True, seed=0, cells=None, n_slots=None, max_pos=100000, theta=None, scale=1.0):
    rng = np.random.default_rng([seed, N, Hq, Hkv, D])
    dt, tc = DT[type_]
    odt, otc = DT[out_type or type_]
    q, qv = rows(rng, N, Hq, D, dt, pad, scale)
    k, kv_ = rows(rng, N, Hkv, D, dt, pad, scale)
    v, vv = rows(rng, N, Hkv, D, dt, pad, scale)
    wq, wk = ((1 + 0.2 * rng.standard_normal((2, D))).astype(np.float32) if norm else (None, None))
    pos = rng.integers(0, max_pos, N).astype(np.int32)
    theta = (np.float32(10000.0) ** (-2.0 * np.arange(max(1, n_rot // 2)) / max(1, n_rot))).astype(np.float32)
    xf = ctx.make_transform(D, n_rot, theta if n_rot else None, had_k, had_v)
    n_slots = n_slots or -(-N // T) + 2
    if cells is None:
        cells = rng.permutation(n_slots * T)[:N].astype(np.int32)
        if N > 3:
            cells[N // 2] = -1
    dev = dict(pos=torch.from_numpy(pos).cuda(), cells=torch.from_numpy(np.asarray(cells, np.int32)).cuda())
    fill = lambda *s: torch.full(s, float("nan"), dtype=odt, device="cuda")  # noqa: E731
    o = dict(q_out=fill(N, Hq, D), k_out=fill(N, Hkv, D))
    if capture:
        o.update(q_norm=fill(N, Hq, D), k_norm=fill(N, Hkv, D))
    es = q.element_size()
    strides = {f"{n}_nb{d}": es * t.stride(2 - d) for n, t in (("q", q), ("k", k), ("v", v)) for d in (1, 2)}
    weights = {}
    if norm:
        dev["wq"], dev["wk"] = torch.from_numpy(wq).cuda(), torch.from_numpy(wk).cuda()
        weights = dict(q_weight=dev["wq"].data_ptr(), k_weight=dev["wk"].data_ptr())
    pool, pk, pv = None, None, None
    if cache:
        tk, tv = CACHE[cache[0]], CACHE[cache[1]]
        pk = torch.full((n_slots * T, kv.row_size(tk, Hkv * D)), 0xA5, dtype=torch.uint8, device="cuda")
        pv = torch.full((n_slots * T, kv.row_size(tv, Hkv * D)), 0xA5, dtype=torch.uint8, device="cuda")
        pool = ctx.make_pool(2, n_slots, T, Hkv * D, Hkv * D, tk, tv, [0, pk.data_ptr()], [0, pv.data_ptr()], xf)
    args = kv.QkvArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr() if cache else None, type=tc, out_type=otc,
                      n_tokens=N, n_head=Hq, n_head_kv=Hkv, head_dim=D, eps=1e-5, positions=dev["pos"].data_ptr(),
                      cells=dev["cells"].data_ptr() if cache else None, **strides, **weights,
                      **{n: t.data_ptr() for n, t in o.items()})
    if not cache:
        args.xf = kv.C.pointer(xf)
    torch.cuda.synchronize()
    ctx.qkv_rows(args, pool, 1 if cache else 0)
    ctx.sync()
    out = {}
    for name, x, w, h in (("q", qv, wq, had_k), ("k", kv_, wk, had_k), ("v", vv, None, had_v)):
        n, nb, y, yb = reference(x, w, 1e-5, pos, theta, n_rot if name != "v" else 0, h)
        out[name] = (n, nb, y, yb)
        if name != "v":
            close(o[f"{name}_out"], y, yb, odt)
            if capture:
                close(o[f"{name}_norm"], n, nb, odt)
    return dict(out=out, pk=pk, pv=pv, cells=np.asarray(cells), n_slots=n_slots, T=T, raw=(qv, kv_, vv), pos=pos,
                theta=theta)


def check_cache(oracle, r, cache, Hkv, D):
    """Stored rows within their format's step of the float64 rows; other rows untouched."""
    for which, name, pool in (("k", cache[0], r["pk"]), ("v", cache[1], r["pv"])):
        y, yb = (a.reshape(len(r["cells"]), Hkv * D) for a in r["out"][which][2:])
        b = pool.cpu().numpy()
        kept = r["cells"][(r["cells"] >= 0) & (r["cells"] < len(b))]
        assert (np.delete(b, kept, 0) == 0xA5).all(), "a row outside the cells was written"
        for t, c in enumerate(r["cells"]):
            if c < 0 or c >= len(b):
                continue
            if name == "f16":
                got = b[c].view(np.float16).astype(np.float64)
                bound = yb[t] + 2.0 ** -11 * (np.abs(y[t]) + yb[t]) + 2.0 ** -25
            else:
                got = oracle.dequantize_row(CACHE[name], b[c], Hkv * D).astype(np.float64)
                d = np.abs(b[c].reshape(-1, oracle.GROUP_BYTES[CACHE[name]])[:, :2].copy().view(np.float16)
                           .astype(np.float64)).repeat(32)
                top = {"q8_0": 127, "q5_0": 16, "q4_0": 8}[name]
                # half a step, a whole one at the far end of q4_0 / q5_0 (codes reach -top .. top - 1)
                step = np.where((name != "q8_0") & (np.abs(y[t]) > (top - 1) * d), 1.0, 0.5)
                bound = step * d * (1 + 2.0 ** -9) + yb[t] * 2 + 2.0 ** -10 * (np.abs(y[t]) + d)
            off = np.abs(got - y[t]) - bound
            assert (off <= 0).all(), (which, name, t, off.max())


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,n_rot,had", [(64, 64, 64), (64, 0, 0), (128, 128, 128), (128, 48, 64), (256, 64, 256),
                                         (256, 256, 0), (512, 512, 512), (512, 160, 64), (256, 16, 128)])
def test_rows_without_a_pool(ctx, type_, D, n_rot, had):
    print(f"[qkv_rows] {type_} D={D} n_rot={n_rot} had={had}", flush=True)
    for N, Hq, Hkv, out_type in ((1, 24, 4, None), (3, 7, 1, "f32"), (130, 5, 3, "f16")):
        call(ctx, N=N, Hq=Hq, Hkv=Hkv, D=D, type_=type_, out_type=out_type, n_rot=n_rot, had_k=had, seed=D + n_rot)


@pytest.mark.parametrize("cache", [("q4_0", "q4_0"), ("q8_0", "q4_0"), ("q5_0", "q5_0"), ("f16", "f16"), ("q4_0", "f16")])
@pytest.mark.parametrize("Hkv,D,T", [(4, 256, 16), (1, 64, 5), (3, 128, 7), (2, 512, 16)])
def test_rows_into_the_pool(ctx, oracle, cache, Hkv, D, T):
    print(f"[qkv_rows] cache={cache} Hkv={Hkv} D={D} T={T}", flush=True)
    for N in (1, 9, 70):
        r = call(ctx, N=N, Hq=2 * Hkv, Hkv=Hkv, D=D, n_rot=64, had_k=D, had_v=64, cache=cache, T=T, seed=N)
        check_cache(oracle, r, cache, Hkv, D)


@pytest.mark.parametrize("cache", ["q4_0", "q5_0", "q8_0", "f16"])
def test_bytes_are_the_stage_ins(ctx, oracle, cache):
    """Without a norm the cached bytes equal the oracle's transform and quantizers bit for bit."""
    Hkv, D = 4, 256
    for n_rot, had_k, had_v in ((64, 256, 64), (0, 0, 0), (256, 0, 64)):
        r = call(ctx, N=40, Hq=8, Hkv=Hkv, D=D, type_="f16", n_rot=n_rot, had_k=had_k, had_v=had_v, norm=False,
                 cache=(cache, cache), capture=False, seed=n_rot)
        for which, pool, had, rot in ((1, r["pk"], had_k, n_rot), (2, r["pv"], had_v, 0)):
            b = pool.cpu().numpy()
            for t, c in enumerate(r["cells"]):
                if c < 0:
                    continue
                x = oracle.transform_rows(r["raw"][which][t].reshape(1, -1), D, rot, r["theta"] if rot else None,
                                          int(r["pos"][t]), had)
                want = x.astype(np.float16).view(np.uint8) if cache == "f16" else oracle.quantize_rows_f32(CACHE[cache], x)
                assert bool((b[c] == want.reshape(-1)).all()), (which, t)


def test_strided_and_unaligned_views(ctx, oracle):
    for pad in (8, 3, 1):
        r = call(ctx, N=21, Hq=6, Hkv=2, D=128, type_="f16", n_rot=32, pad=pad, cache=("q8_0", "q8_0"), seed=pad)
        check_cache(oracle, r, ("q8_0", "q8_0"), 2, 128)
        call(ctx, N=5, Hq=6, Hkv=2, D=64, type_="f32", n_rot=32, pad=pad, seed=pad)


def test_many_tokens_and_far_positions(ctx, oracle):
    """Several tokens to a workgroup, an odd count, positions up to 2^31 - 1."""
    r = call(ctx, N=4099, Hq=4, Hkv=2, D=128, n_rot=128, had_k=128, had_v=64, cache=("q4_0", "q8_0"), T=128,
             capture=False, max_pos=2 ** 31 - 1)
    check_cache(oracle, r, ("q4_0", "q8_0"), 2, 128)
    call(ctx, N=17001, Hq=2, Hkv=1, D=64, n_rot=64, capture=False)


def test_cells_outside_the_pool_keep_nothing(ctx, oracle):
    cells = np.array([-1, 31, 32, 2 ** 31 - 1, -2 ** 31, 0, 47, 48], np.int32)
    r = call(ctx, N=8, Hq=2, Hkv=2, D=64, cache=("q4_0", "f16"), T=16, n_slots=3, cells=cells)
    check_cache(oracle, r, ("q4_0", "f16"), 2, 64)


def test_zero_rows_and_large_values(ctx):
    """A row of zeros normalises to zeros (eps keeps the root away from 0); f16's largest rows stay finite."""
    N, H, D = 2, 2, 64
    q = torch.zeros((N, H, D), dtype=torch.float16, device="cuda")
    q[1] = 65504.0
    out = torch.full((N, H, D), float("nan"), dtype=torch.float32, device="cuda")
    w = torch.ones(D, device="cuda")
    a = kv.QkvArgs(q=q.data_ptr(), type=kv.TYPE_F16, out_type=kv.TYPE_F32, n_tokens=N, n_head=H, head_dim=D, q_nb1=2 * D,
                   q_nb2=2 * D * H, q_weight=w.data_ptr(), eps=1e-6, q_out=out.data_ptr())
    torch.cuda.synchronize()
    ctx.qkv_rows(a)
    ctx.sync()
    assert (out[0] == 0).all()
    assert torch.allclose(out[1], torch.ones_like(out[1]), rtol=(D / 2 + 10) * E32, atol=0)


def test_only_some_rows(ctx, oracle):
    """k alone, v alone, q alone; n_tokens 0 touches nothing."""
    rng = np.random.default_rng(1)
    N, H, D, T = 5, 2, 64, 8
    x, xv = rows(rng, N, H, D, torch.float16)
    cells = torch.arange(N, dtype=torch.int32, device="cuda")
    pools = [torch.full((T, kv.row_size(kv.TYPE_Q4_0, H * D)), 0xA5, dtype=torch.uint8, device="cuda") for _ in "kv"]
    pool = ctx.make_pool(1, 1, T, H * D, H * D, kv.TYPE_Q4_0, kv.TYPE_Q4_0, [pools[0].data_ptr()], [pools[1].data_ptr()])
    base = dict(type=kv.TYPE_F16, out_type=kv.TYPE_F16, n_head_kv=H, head_dim=D, cells=cells.data_ptr())
    st = dict(nb1=2 * D, nb2=2 * D * H)
    want = oracle.quantize_rows_f16(kv.TYPE_Q4_0, xv.reshape(N, -1).astype(np.float16).view(np.uint16))
    torch.cuda.synchronize()
    for i, n in enumerate("kv"):
        ctx.qkv_rows(kv.QkvArgs(**{n: x.data_ptr()}, n_tokens=0, **{f"{n}_{s}": b for s, b in st.items()}, **base), pool)
        ctx.sync()
        assert (pools[i] == 0xA5).all()
        ctx.qkv_rows(kv.QkvArgs(**{n: x.data_ptr()}, n_tokens=N, **{f"{n}_{s}": b for s, b in st.items()}, **base), pool)
        ctx.sync()
        assert np.array_equal(pools[i].cpu().numpy()[:N], want)
        assert (pools[i].cpu().numpy()[N:] == 0xA5).all()


def test_rows_past_4_gib(ctx, oracle):
    """Cells whose byte offset passes 32 bits."""
    H, D, T = 4, 256, 128
    row = kv.row_size(kv.TYPE_F16, H * D)
    n_slots = (5 << 30) // (row * T)
    pool_t = torch.empty((n_slots * T, row), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(2)
    x, xv = rows(rng, 2, H, D, torch.float16)
    last = n_slots * T - 1
    cells = torch.tensor([last, last - 7], dtype=torch.int32, device="cuda")
    pool = ctx.make_pool(1, n_slots, T, H * D, H * D, kv.TYPE_F16, kv.TYPE_F16, [pool_t.data_ptr()], [pool_t.data_ptr()])
    pool_t[-16:] = 0
    torch.cuda.synchronize()
    ctx.qkv_rows(kv.QkvArgs(k=x.data_ptr(), type=kv.TYPE_F16, out_type=kv.TYPE_F16, n_tokens=2, n_head_kv=H, head_dim=D,
                            k_nb1=2 * D, k_nb2=2 * D * H, cells=cells.data_ptr()), pool)
    ctx.sync()
    got = pool_t[-16:].cpu().numpy().view(np.float16).astype(np.float32)
    assert np.array_equal(got[15], xv[0].reshape(-1)) and np.array_equal(got[8], xv[1].reshape(-1))
    assert (got[[0, 1, 14]] == 0).all()
