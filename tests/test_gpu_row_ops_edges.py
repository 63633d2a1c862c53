"""Operators on rows of channels on the GPU: values that are not finite through the linear layer, the large tiles with everything that can
stand behind them, equal rows in different places, and the longest grids.

Tolerances as in test_gpu_row_ops: U = 2^-24 is half a step of fp32; a sum of fp32 terms is off by at most (additions one after another) * U *
(sum of the terms' sizes), 128 inside a matrix instruction and the blocks one after another; a result rounded once is off by half a step of
its type; a product with a bf16 result may besides lose what row_ops_ref.cut() counts."""
import pytest
import torch

import row_ops_ref as R
from uncltmo_amd import _hip, row_ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]
INF, NAN = float("inf"), float("nan")


def rnd(*shape, dtype=torch.float32, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (size * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


# ---- what is not finite in the linear layer --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,n,k", [(50, 100, 130), (300, 256, 256), (2100, 2050, 390), (4100, 4096, 1024)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("fmt", ["e5m2", "e4m3"])
def test_linear8_does_not_hide_an_overflow(m, n, k, dtype, fmt):
    """the results that an infinity or a NaN takes part in are NaN, the others those of a zero in its place, bit for bit"""
    x, w, g = rnd(m, k, dtype=dtype), rnd(n, k, seed=1, size=k ** -0.5), rnd(m, n, dtype=dtype, seed=2, size=0.01)

    def step(x, w, g):
        x, w, b = x.clone().requires_grad_(), w.clone().requires_grad_(), torch.zeros(n, device="cuda", requires_grad=True)
        y = row_ops.linear8(x, w, b, fmt)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], g)]
    for value in (INF, -INF, NAN):
        for which in (0, 1, 2):
            src = [x.clone(), w.clone(), g.clone()]
            t = src[which]
            places = [(0, 0), (t.shape[0] // 2, t.shape[1] // 3), (t.shape[0] - 1, t.shape[1] - 1)]
            for i, j in places:
                t[i, j] = 0
            want = step(*src)
            for i, j in places:
                t[i, j] = value
            got = step(*src)
            hit = [torch.zeros_like(v, dtype=torch.bool) for v in want]
            for i, j in places:
                if which == 0:
                    hit[0][i], hit[2][:, j] = True, True               # a row of y, a column of the weight's gradient
                elif which == 1:
                    hit[0][:, i], hit[1][:, j] = True, True            # a column of y, one of x's gradient
                else:
                    hit[1][i], hit[2][j], hit[3][j] = True, True, True  # a row of x's gradient, one of the weight's, one sum
            for name, a, b, h in zip(("y", "gx", "gw", "gb"), got, want, hit):
                assert not torch.isfinite(a[h]).any(), (name, value, which)
                assert torch.equal(a[~h], b[~h]), (name, value, which)
    q = row_ops.quantize8(torch.full((1, 8), INF, device="cuda").index_fill(1, torch.tensor([1], device="cuda"), 2.0))      # quantize8 itself: the largest number
    assert torch.equal(q.values(), torch.full((1, 8), 2.0, device="cuda"))
