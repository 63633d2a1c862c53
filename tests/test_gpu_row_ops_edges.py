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


# ---- the large tiles with everything behind them ---------------------------------------------------------------------------------------
def operand(rows, cols, block, fmt="e4m3", seed=0):
    """a quantised matrix whose bytes behind a row's end are NaN"""
    data, scale = R.quantize(rnd(rows, cols, seed=seed).cpu() * torch.exp2(torch.arange(cols) % 5 - 2.0), block, fmt)
    room = torch.full((rows, -(-cols // 16) * 16 + 16), 0x7F, dtype=torch.uint8, device="cuda")
    room[:, :cols] = data.view(torch.uint8).cuda()
    return row_ops.Quant8(room.view(data.dtype)[:, :cols], scale.cuda(), block)


def reference(a, b, dtype, bias=None, act="none", residual=None):
    """64-bit value of a product and what may be off before the result's rounding; all on the GPU"""
    want, size = R.matmul8(a, b)
    tol = (128 + 8 + -(-a.data.shape[1] // 128)) * R.U * size + (R.cut(a, b) if dtype == torch.bfloat16 else 0.0)
    if bias is not None:
        want = want + bias.double()
        tol = tol + R.U * (want.abs() + bias.double().abs())
    if act == "relu":
        want = want.clamp_min(0)
    elif act == "gelu":
        tol = 1.13 * tol + 16 * R.U * want.abs()                         # the slope is at most 1.13; erf and two products
        want = want * torch.special.ndtr(want)
    if residual is not None:
        want = want + residual.double()
        tol = tol + R.U * want.abs()
    return want, tol


def within(got, want, tol, dtype, what):
    bad = (got.double() - want).abs() > tol + R.HALF[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist())


# M, N and K with sides behind the last tile: 4101 x 3500 goes to 256 x 256 tiles where those are built (bf16 results, b by tiles), 2100 x 2050
# to 128 x 128, 4099 rows leave three behind the last whole tile
LARGE = [(4101, 3500, 1100), (2100, 2050, 384), (4099, 4096, 2048)]


@pytest.mark.parametrize("m,n,k", LARGE)
@pytest.mark.parametrize("block", ["tile", "row"])
@pytest.mark.parametrize("fa", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_large_products_with_bias_activation_and_residual(m, n, k, block, fa, dtype):
    a, b, bias = operand(m, k, "row", fa), operand(n, k, block, seed=1), rnd(n, seed=3)
    res = rnd(m, n, dtype=dtype, seed=4, size=5.0)
    for act in ("gelu", "relu"):
        want, tol = reference(a, b, dtype, bias, act, res)
        out = row_ops.matmul8(a, b, bias=bias, act=act, residual=res, out_dtype=dtype)
        within(out, want, tol, dtype, act)
    wide = torch.full((m, n + 9), 7.0, dtype=dtype, device="cuda")        # rows of a wider buffer at an odd address; what is beside stays
    wide[:, 3:3 + n] = res
    into = wide[:, 3:3 + n]
    row_ops.matmul8(a, b, bias=bias, act=act, residual=into, out_dtype=dtype, out=into)                     # the residual is the result
    assert torch.equal(into, out) and bool((wide[:, :3] == 7).all()) and bool((wide[:, 3 + n:] == 7).all())
    pitched = torch.zeros(m, n + 5, dtype=dtype, device="cuda")[:, :n].copy_(res)
    assert torch.equal(row_ops.matmul8(a, b, bias=bias, act=act, residual=pitched, out_dtype=dtype), out)


@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("m,n,k", [(4099, 4096, 2048), (2100, 4096, 2050)])
def test_large_linear8_with_all_gradients(m, n, k, dtype, wtype):
    x, w, b, g = rnd(m, k, dtype=dtype), rnd(n, k, dtype=wtype, size=k ** -0.5, seed=1), rnd(n, seed=2), rnd(m, n, dtype=dtype, seed=3, size=0.01)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = row_ops.linear8(*leaves)
    gx, gw, gb = torch.autograd.grad(y, leaves, g)

    def q(t, block, fmt, tr=False):
        return row_ops.Quant8(*(v.cuda() for v in R.quantize(t.cpu(), block, fmt, tr)), block)
    for name, got, t, a, o, bias in (("y", y, dtype, q(x, "row", "e4m3"), q(w, "tile", "e4m3"), b), ("gx", gx, dtype, q(g, "row", "e5m2"), q(w, "tile", "e4m3", True), None),
                                     ("gw", gw, wtype, q(g, "row", "e5m2", True), q(x, "row", "e4m3", True), None)):
        want, tol = reference(a, o, t, bias)
        assert got.dtype == t
        within(got, want, tol, t, name)
    bad = (gb.double() - g.double().sum(0)).abs() > 300 * R.U * g.double().abs().sum(0)       # 8 + 16 in a tile, two partial sums a lane, a fold of 32
    assert not bad.any()


# ---- equal rows ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,n,k", [(4099, 4096, 2048), (4099, 2048, 4096), (4160, 4096, 1024), (300, 33000, 1024), (2100, 2050, 384), (28800, 256, 256)])
@pytest.mark.parametrize("block", ["tile", "row"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_equal_rows_give_equal_results_wherever_they_stand(m, n, k, block, dtype):
    """every row of a product is added up the same way: fifty rows over and over"""
    a, b = operand(50, k, "row"), operand(n, k, block, seed=1)
    i = torch.arange(m, device="cuda") % 50
    many = row_ops.Quant8(a.data.view(torch.uint8)[i].view(a.data.dtype), a.scale[i], "row")
    out = row_ops.matmul8(many, b, out_dtype=dtype)
    assert torch.equal(out, out[:50][i])


# ---- the longest grids -----------------------------------------------------------------------------------------------------------------
LONG = 2 ** 27 + 128 + 40                     # columns: a workgroup of 512 threads for each sixteen is more than 2^32 threads


@pytest.mark.parametrize("block", ["tile", "row"])
def test_a_product_of_few_rows_and_over_2_to_the_27_columns(block):
    m, k = 2, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    a = row_ops.Quant8(torch.randint(0, 0x78, (m, k), dtype=torch.uint8, device="cuda", generator=g).view(torch.float8_e4m3fn), torch.ones(m, 1, device="cuda"), "row")
    b = row_ops.Quant8(torch.randint(0, 0x78, (LONG, k), dtype=torch.uint8, device="cuda", generator=g).view(torch.float8_e4m3fn),
                       1 + torch.rand(LONG if block == "row" else (LONG + 127) // 128, 1, device="cuda", generator=g), block)
    bias, res = torch.randn(LONG, device="cuda", generator=g), torch.randn(m, LONG, device="cuda", generator=g)
    out = row_ops.matmul8(a, b, bias=bias, residual=res, out_dtype=torch.float32)
    for first in (0, 2 ** 26 - 256, 2 ** 26, 2 ** 27 - 256, 2 ** 27, 2 ** 27 + 128):             # (whole tiles of 128, so that scales go with them)
        n = slice(first, min(first + 256, LONG))
        part = row_ops.Quant8(b.data[n], b.scale[n if block == "row" else slice(n.start // 128, (n.stop + 127) // 128)], block)
        want, size = R.matmul8(a, part)
        tol = 137 * R.U * (size + bias[n].double().abs() + res[:, n].double().abs())
        assert first % 128 == 0
        within(out[:, n], want + bias[n].double() + res[:, n].double(), tol, torch.float32, first)


def test_a_weights_gradient_of_over_2_to_the_27_channels():
    """rows of ones of both signs: their mean square is exactly 1"""
    x = torch.ones(2, LONG, dtype=torch.bfloat16, device="cuda")
    x[:, ::3] = -1
    gy = rnd(2, LONG, dtype=torch.bfloat16)
    w = torch.ones(LONG, device="cuda", requires_grad=True)
    y = row_ops.rms_norm(x, w, 1e-6)
    assert bool((y == x).all())                                              # 1 - 5e-7 rounds to 1
    gw, = torch.autograd.grad(y, [w], gy)
    want = (gy.float() * x.float()).sum(0)                                   # exact but for one rounding
    assert bool(((gw - want).abs() <= 1e-6 * gy.float().abs().sum(0)).all())


# ---- rows whose squares leave fp32 -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("cols", [5, 13, 32, 64, 300, 1000, 3000, 8200, 20001])
def test_norm_of_large_values(cols, dtype):
    """tolerances as for other rows (test_gpu_row_ops): scaling by a power of two rounds nothing"""
    x, gy, w = rnd(12, cols, dtype=dtype), rnd(12, cols, dtype=dtype, seed=1), 1 + 0.1 * rnd(cols, seed=2)
    size = torch.tensor([1.0, 2.0 ** 62, 2.0 ** 64, 2.0 ** 66, 1.0, 2.0 ** 90, 2.0 ** 120, 1.0, 2.0 ** 64, 2.0 ** -20, 2.0 ** 118, 2.0 ** 70], device="cuda")
    x = (x.float() * size[:, None]).to(dtype)
    x[4, 1] = INF
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = row_ops.rms_norm(xs, ws, 1e-6)
    gx, gw = torch.autograd.grad(y, [xs, ws], gy)
    ok = torch.arange(12, device="cuda") != 4
    others = torch.arange(cols, device="cuda") != 1                         # (1 / rms of the row with an infinity is 0)
    want, _ = R.norm(x[ok], w, 1e-6)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert bool(((y[ok].double() - want).abs() <= (R.HALF[dtype] + 96 * R.U) * want.abs() + tiny).all())
    assert bool(torch.isnan(y[4, 1])) and bool((y[4, others] == 0).all())
    want, size, want_w, size_w = R.norm_backward(gy[ok], None, x[ok], w, 1e-6)
    assert bool(((gw.double() - want_w).abs() <= 160 * R.U * size_w)[others].all()) and bool(torch.isnan(gw[1]))
    assert bool(((gx[ok].double() - want).abs() <= R.HALF[dtype] * want.abs() + 128 * R.U * size + 2 * tiny).all())
    q, _ = row_ops.rms_norm_quant8(x, w)
    q1, _ = row_ops.rms_norm_quant8((x.float() * torch.where(x.float().abs().amax(1) > 2.0 ** 40, 2.0 ** -60, 1.0)[:, None]).to(dtype), w)
    assert bool(((q.values()[ok] - q1.values()[ok]).abs() <= 2.0 ** -3 * q1.values()[ok].abs() + 2.0 ** -8 * q1.scale.amax()).all())
