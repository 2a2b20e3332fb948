"""kvmem_hip_attention over cached values that are not finite once they are scaled
(infinities, NaN, an 8-bit value beyond f16): the value's dim is not finite in
every row that attends its key, whatever the shape of the call -- all keys, rows
of one token alone in their tile, keys cut by max_kv, split keys, keys in whole
steps and in the last partial one -- and every other element stays within the
float64 reference's bound."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
from attention_helpers import Case  # noqa: E402

BAD = {"inf": 0x7C00, "nan": 0x7E00, "beyond": None}


def poison(c, s, key, bad, dim=5):
    """Makes dim `dim` of KV head 0 of a request's key not finite; the dims that are lost with it."""
    row = int(c.table[s, key // c.T]) * c.T + key % c.T
    if c.type_v == "f16":
        c.pool["v"][row].view(np.uint16)[dim] = BAD[bad]
        return [dim]
    group = c.pool["v"][row]  # the first group of 32 dims
    if bad == "beyond":  # q8_0: 127 * 600 passes f16's range, one code at the others' place does not
        group[:2] = np.array([600.0], np.float16).view(np.uint8)
        group[2:34] = 1
        group[2 + dim] = 127
        return [dim]
    group[:2] = np.array([BAD[bad]], np.uint16).view(np.uint8)
    return list(range(32))


def check(c, s, key, lost):
    """Rows of request s that attend `key` have lost these dims of the heads on KV head 0, and nothing else."""
    with np.errstate(all="ignore"):
        out, bound, _, _ = c.reference()
    got = c.run().out.cpu().double().numpy()
    half = torch.finfo(c.odt).eps / 2
    gone = np.zeros(out.shape, bool)
    for i in range(min(c.m[s], c.args.max_q)):
        if not c.causal or key <= c.lens[s] - c.m[s] + i:
            gone[int(c.starts[s]) + i, :c.Hq // c.Hkv, lost] = True
    assert gone.any()
    assert not np.isfinite(got[gone]).any(), f"{np.isfinite(got[gone]).sum()} of {gone.sum()} elements are finite"
    stay = ~gone & ~np.isnan(bound)
    assert np.isfinite(got[stay]).all()
    off = np.abs(got - out)[stay] - (bound + half * (np.abs(out) + bound) + 2.0 ** -25)[stay]
    assert (off <= 0).all(), f"over the bound by {off.max():.3e}"


def values(type_v):
    return ["inf", "nan"] if type_v == "f16" else ["nan", "beyond"]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type_v", ["f16", "q8_0"])
@pytest.mark.parametrize("m", [1, 70])
def test_all_rows_attend_all_keys(ctx, oracle, type_v, D, m):
    """Not causal: 300 keys end inside a step of the many-query kernel at every head size."""
    print(f"[not finite] all keys {type_v} {D} {m}", flush=True)
    for bad in values(type_v):
        for key in (0, 150, 299):
            c = Case(ctx, oracle, [300, 90], [m, m], 6, 2, D, 32, "q4_0", type_v, causal=False, seed=201)
            lost = poison(c, 0, key, bad)
            c.upload()
            check(c, 0, key, lost)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type_v", ["f16", "q8_0"])
def test_a_tile_of_one_token(ctx, oracle, type_v, D):
    """43 tokens of 6 heads are 258 rows: the last two stand alone in their tile and attend the same keys; so do 200
    heads of one token."""
    print(f"[not finite] one token in a tile {type_v} {D}", flush=True)
    for bad in values(type_v):
        for lens, m, Hq in ((211, 43, 6), (211, 1, 200)):
            for key in (210, 205, 100):
                c = Case(ctx, oracle, [lens], [m], Hq, 1, D, 32, "q4_0", type_v, seed=202)
                lost = poison(c, 0, key, bad)
                c.upload()
                check(c, 0, key, lost)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_keys_cut_by_max_kv(ctx, oracle, D):
    """The bound lies below every row's limit: all rows attend the same keys of a causal call."""
    print(f"[not finite] max_kv {D}", flush=True)
    for m in (2, 70):
        for bad in ("inf", "nan"):
            c = Case(ctx, oracle, [300], [m], 6, 2, D, 32, "q4_0", "f16", max_kv=150, seed=203)
            lost = poison(c, 0, 149, bad)
            c.upload()
            check(c, 0, 149, lost)


@pytest.mark.parametrize("D", [64, 256])
def test_split_keys(ctx, oracle, D):
    """Parts whose keys every row attends, and the last one, whose keys some rows attend."""
    print(f"[not finite] split {D}", flush=True)
    for m in (3, 70):
        for key in (0, 3001, 5000 - m, 4999):
            for type_v, bad in (("f16", "inf"), ("q8_0", "beyond")):
                c = Case(ctx, oracle, [5000], [m], 6, 2, D, 64, "q4_0", type_v, seed=204)
                lost = poison(c, 0, key, bad)
                c.upload()
                check(c, 0, key, lost)
