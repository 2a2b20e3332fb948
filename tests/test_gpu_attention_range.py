"""kvmem_hip_attention at the ends of the numbers' ranges: bf16 queries up to 2^122
and scales that meet them (the factor that brings their scores back passes fp32,
the scores do not), scores so large that the rounding of a product is more than a
weight's whole range, and quantized keys beyond f16.

Where scores lie far apart one key takes a row's whole weight.  The float64 scores
then have to say so, before the kernel's output is looked at: the best key's lead
is larger than what both scores may err by (mag * (2^-10 + (D + 8) 2^-24), mag the
sum of the magnitudes of a score's terms, as in attention_helpers) and than 40, so
every other weight is below 2^-57 and the row is the best key's value, rounded to
f16 and by the f16 weight that is divided by itself rounded: 2^-10 relative."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
from attention_helpers import Case, decode  # noqa: E402


def times(c, f):
    """Queries times a power of two (exact in bf16)."""
    c.q.mul_(f)
    c.q_host = c.q_host * f
    assert np.isfinite(c.q.double().cpu().numpy()).all()


def check_best_key(c, least=0.7):
    """Rows where one key leads clearly hold its value, and lse its score; they have to be most rows."""
    got = c.run().out.cpu().double().numpy()
    lse = c.lse.cpu().double().numpy()
    clear = total = 0
    for s in range(len(c.lens)):
        j = np.arange(c.lens[s])
        rows = c.table[s, j // c.T].astype(np.int64) * c.T + j % c.T
        k = decode(c.oracle, c.type_k, c.pool["k"][rows], c.Hkv * c.D).reshape(len(j), c.Hkv, c.D)
        v = decode(c.oracle, c.type_v, c.pool["v"][rows], c.Hkv * c.D).reshape(len(j), c.Hkv, c.D)
        for i in range(c.m[s]):
            t = int(c.starts[s]) + i
            n = c.lens[s] - c.m[s] + i + 1 if c.causal else len(j)
            for h in range(c.Hq):
                g = h // (c.Hq // c.Hkv)
                x = c.scale * (k[:n, g] @ c.q_host[t, h])
                err = c.scale * (np.abs(k[:n, g]) @ np.abs(c.q_host[t, h])) * (2.0 ** -10 + (c.D + 8) * 2.0 ** -24)
                best = int(x.argmax())
                lead = x[best] - err[best] - np.delete(x + err, best)
                total += 1
                if n > 1 and lead.min() <= 40 + 2.0 ** -22 * abs(x[best]):
                    continue
                clear += 1
                want = v[best, g]
                assert np.isfinite(got[t, h]).all(), (t, h, "not finite")
                assert (np.abs(got[t, h] - want) <= 2.0 ** -10 * np.abs(want) + 2.0 ** -24).all(), (t, h)
                assert abs(lse[t, h] - x[best]) <= err[best] + 2.0 ** -20 * (1 + abs(x[best])), (t, h, "lse")
    assert clear >= least * total, f"one key leads in {clear} of {total} rows"


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type_k", ["q4_0", "q5_0", "q8_0", "f16"])
@pytest.mark.parametrize("m", [1, 5, 100])
def test_queries_at_bf16s_end(ctx, oracle, m, type_k, D):
    print(f"[range] queries {type_k} {D} {m}", flush=True)
    for f, scale in ((2.0 ** 118, 0.0), (2.0 ** 115, 1.0)):
        c = Case(ctx, oracle, [130, 33], [m, min(m, 33)], 4, 2, D, 32, type_k, "f16", scale=scale, seed=301)
        times(c, f)
        check_best_key(c)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("m", [1, 100])
def test_large_scales_of_small_keys(ctx, oracle, m, D):
    """A large scale takes the factor past fp32 in either kernel; keys of 2^-20 bring the scores back."""
    print(f"[range] scale {D} {m}", flush=True)
    c = Case(ctx, oracle, [130, 33], [m, min(m, 33)], 4, 2, D, 32, "f16", "f16", scale=2.0 ** 17, k_scale=2.0 ** -20, seed=302)
    times(c, 2.0 ** 118)
    check_best_key(c)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("m", [1, 100])
def test_scores_past_24_bits(ctx, oracle, m, D):
    """Scores from 2^24 on: a step of their fp32 is more than the weights' whole range."""
    print(f"[range] scores {D} {m}", flush=True)
    for e in (21, 24, 28, 40, 80):
        c = Case(ctx, oracle, [130, 33], [m, min(m, 33)], 4, 2, D, 32, "f16", "f16", seed=303)
        times(c, 2.0 ** e)
        check_best_key(c)
        # split keys: the parts' maxima lie as far apart
        c = Case(ctx, oracle, [4000], [m], 4, 2, D, 32, "q8_0", "q8_0", seed=304)
        times(c, 2.0 ** e)
        check_best_key(c, 0.5)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("m", [1, 100])
def test_equal_scores_of_any_size(ctx, oracle, m, D):
    """Keys that are all the same: each weighs 1/n whatever the score, the output is the values' mean.  Bound: the
    values' rounding to f16 and the weight's, 2^-10 of the mean magnitude, n + 64 fp32 sums."""
    print(f"[range] equal keys {D} {m}", flush=True)
    for e in (0, 24, 33, 60, 100):
        c = Case(ctx, oracle, [700], [m], 4, 2, D, 32, "q8_0", "f16", causal=False, seed=305)
        c.pool["k"][:] = c.pool["k"][int(c.table[0, 0]) * 32]
        c.upload()
        times(c, 2.0 ** e)
        j = np.arange(700)
        rows = c.table[0, j // 32].astype(np.int64) * 32 + j % 32
        v = decode(oracle, "f16", c.pool["v"][rows], 2 * D).reshape(700, 2, D)[:, [0, 0, 1, 1]]
        got = c.run().out.cpu().double().numpy()
        bound = np.abs(v).mean(0) * (2.0 ** -10 + 764 * 2.0 ** -24) + 2.0 ** -24
        assert np.isfinite(got).all() and (np.abs(got - v.mean(0)) <= bound).all(), e


# largest f16 scale that keeps a code times it below f16's end: 65504 / 128, / 16, / 8
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type_k,above", [("q8_0", [512.0, 4096.0, 65504.0]), ("q5_0", [4100.0, 65504.0]),
                                          ("q4_0", [8192.0, 65504.0])])
@pytest.mark.parametrize("m", [1, 100])
def test_keys_beyond_f16(ctx, oracle, m, type_k, above, D):
    """Quantized keys larger than f16 holds, in some groups of some keys, beside ordinary ones."""
    print(f"[range] keys {type_k} {D} {m}", flush=True)
    rng = np.random.default_rng(D + m)
    gb = {"q8_0": 34, "q5_0": 22, "q4_0": 18}[type_k]
    for scale_of in above:
        for share in (0.01, 0.4, 1.0):
            c = Case(ctx, oracle, [300, 77], [m, min(m, 77)], 6, 2, D, 32, type_k, "f16",
                     scale=2.0 ** -12 / scale_of, seed=306)
            rows = c.pool["k"].reshape(len(c.pool["k"]), -1, gb)
            live = (rows != 0xFF).any(-1).any(-1)
            hit = (rng.random(rows.shape[:2]) < share) & live[:, None]
            d = np.where(rng.random(hit.sum()) < 0.5, -scale_of, scale_of).astype(np.float16)
            rows[..., :2][hit] = d.view(np.uint8).reshape(-1, 2)
            c.upload()
            c.run().check()


def test_keys_beyond_f16_in_split_calls(ctx, oracle):
    """Parts and rotated values, 8-bit scales that stay and change from step to step."""
    for m, had in ((2, 0), (70, 64)):
        c = Case(ctx, oracle, [5000, 800], [m, m], 6, 2, 128, 64, "q8_0", "q8_0", scale=2.0 ** -24, hadamard=had, seed=307)
        rows = c.pool["k"].reshape(len(c.pool["k"]), -1, 34)
        live = np.flatnonzero((rows != 0xFF).any(-1).any(-1))
        for r in live[::97]:
            rows[r, r % rows.shape[1], :2] = np.array([3000.0], np.float16).view(np.uint8)
        c.upload()
        c.run().check()
