"""kvmem_hip_qkv_rows' norm over the whole range of float32 and bfloat16 rows: squares
that pass float32's range or fall below it (eps smaller still), and rows on either
side of where that begins, against float64 with test_gpu_qkv_rows' bounds.

Those are relative; products below 2^-126 are multiples of 2^-149 and err by up to
2^-150 whatever their size.  (x r) w is two such products, the first's error times w:
2^-150 (1 + |w|), |w| < 2.  The rotation scales each of its run's 64 elements by 1/8
(64 roundings of 2^-150 beside 64 elements that are off by 3 * 2^-150 / 8) and adds
them, which is exact among multiples of 2^-149: 64 * 2^-150 (1 + 3/8) < 2^-143."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from conftest import load_pkg  # noqa: E402

kv = load_pkg()
from test_gpu_qkv_rows import DT, close, reference  # noqa: E402


def norm(ctx, x, w, eps):
    """The normed rows of a device view [N, H, D], and the rows after a rotation of runs of 64."""
    N, H, D = x.shape
    code = {torch.float32: kv.TYPE_F32, torch.bfloat16: kv.TYPE_BF16}[x.dtype]
    out, turned = (torch.full((N, H, D), float("nan"), device="cuda") for _ in range(2))
    xf = ctx.make_transform(D, hadamard_k=64)
    a = kv.QkvArgs(q=x.data_ptr(), type=code, out_type=kv.TYPE_F32, n_tokens=N, n_head=H, head_dim=D,
                   q_nb1=x.element_size() * D, q_nb2=x.element_size() * D * H, q_weight=w.data_ptr(), eps=eps,
                   xf=kv.C.pointer(xf), q_out=turned.data_ptr(), q_norm=out.data_ptr())
    torch.cuda.synchronize()
    ctx.qkv_rows(a)
    ctx.sync()
    return out, turned


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_rows_of_every_magnitude(ctx, type_, D):
    print(f"[norm range] {type_} {D}", flush=True)
    rng = np.random.default_rng(D)
    # every head of a token at another power of two: neighbours in a wave take different ways
    powers = np.array([0, 120, -110, 59, 61, 64, 100, -38, -42, -46, -70, 1], float)
    x = np.clip(rng.standard_normal((5, len(powers), D)), -4, 4)
    x[..., ::29] *= 6.0
    w = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    x = torch.from_numpy((x * 2.0 ** powers[:, None]).astype(np.float32)).cuda().to(DT[type_][0])
    wd = torch.from_numpy(w).cuda()
    for eps in (0.0, 1e-37, 1e-30, 1e-6, 1e20):
        got, turned = norm(ctx, x, wd, eps)
        n, nb, y, yb = reference(x.float().cpu().numpy(), w, float(np.float32(eps)), None, None, 0, 64)
        assert np.abs(w).max() < 2
        close(got, n, nb + 3 * 2.0 ** -150, torch.float32)
        close(turned, y, yb + 2.0 ** -143, torch.float32)


def test_rows_that_are_not_finite_stay_alone(ctx):
    """An infinity or NaN reaches its own head only; a row of zeros is zeros with an eps."""
    x = torch.ones((2, 8, 64), device="cuda")
    x[0, 1, 3], x[0, 4, 5], x[1, 2] = float("inf"), float("nan"), 0.0
    x[1, 6] = 2.0 ** 100
    w = torch.ones(64, device="cuda")
    got, _ = norm(ctx, x, w, 1e-6)
    assert torch.isnan(got[0, 1, 3]) and (got[0, 1, :3] == 0).all()
    assert torch.isnan(got[0, 4]).all()
    assert (got[1, 2] == 0).all()
    keep = torch.ones((2, 8), dtype=torch.bool)
    keep[0, 1] = keep[0, 4] = keep[1, 2] = False
    assert (got.cpu()[keep] - 1).abs().max() <= 42 * 2.0 ** -24 + 1e-6
