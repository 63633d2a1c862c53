"""Operators on rows of channels on the GPU against their restatements (row_ops_ref): flags, dropped sums and 8-bit operands bit for bit,
everything else against 64 bits.

Tolerances, as counted before the first run.  U = 2^-24 is half a step of fp32.  A result rounded once to its type is off by half a step of
it, relative.  A sum of fp32 terms is off by at most (additions one after another) * U * (sum of the terms' sizes): a row is added up by at
least 64 threads with shuffles behind them, at most 64 terms a thread and 8 levels; a product of 128-blocks adds 128 terms inside a matrix
instruction and the blocks one after another; a weight's gradient adds at most 64 rows a slot, 4 folds and 32 + 5 partial rows.  A product
with a bf16 result may besides lose what row_ops_ref.cut() counts."""
import pytest
import torch

import row_ops_ref as R
from uncltmo_amd import _hip, row_ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]
EPS = 1e-6
LOW = {t: torch.finfo(t).tiny * torch.finfo(t).eps for t in DTYPES}       # the smallest number's step


def rnd(*shape, dtype=torch.float32, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (size * torch.randn(*shape, generator=g)).to(dtype)


def within(got, want, tol, what=""):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError("%s: %d of %d outside; first at %s: got %.9g want %.9g tolerance %.3g"
                             % (what, int(bad.sum()), bad.numel(), i, got[i], want[i], tol[i]))


def wide(x, pitch_more, front):
    """the same rows inside a wider buffer: another pitch, another alignment"""
    rows, cols = x.shape
    buf = torch.full((rows * (cols + pitch_more) + front,), float("nan"), dtype=x.dtype, device="cuda")
    v = buf[front:].view(rows, cols + pitch_more)[:, :cols]
    v.copy_(x)
    return v


# ---- dropout -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols,span", [(1, 1, 1), (3, 7, 1), (5, 8, 1), (70, 9, 4), (144, 256, 1), (600, 32, 150), (33, 100, 33), (2, 2051, 1), (9, 4096, 1)])
def test_dropout_bit_for_bit(dtype, rows, cols, span):
    x, r = rnd(rows, cols, dtype=dtype), rnd(rows, cols, dtype=dtype, seed=1)
    for p, seed, offset, res in ((0.1, 3, 0, None), (0.5, 2 ** 63 + 12345, 2 ** 40 + 7, r), (0.0, 1, 2, r), (1.0, 1, 2, r), (1.0, 5, 0, None), (1e-6, 4, 4, None)):
        got = row_ops.dropout(x.cuda(), p, seed, offset, residual=None if res is None else res.cuda(), span=span)
        assert torch.equal(got.cpu(), R.dropout(x, res, p, seed, offset, span)), (p, seed)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dropout_views_and_axes(dtype):
    x, r = rnd(37, 40, dtype=dtype), rnd(37, 40, dtype=dtype, seed=2)
    want = R.dropout(x, r, 0.3, 11, 5)
    for more, front in ((3, 1), (8, 0), (1, 3)):
        assert torch.equal(row_ops.dropout(wide(x, more, front), 0.3, 11, 5, residual=wide(r, more + 2, front)).cpu(), want)
    m = rnd(2, 40, 5, 6, dtype=dtype).cuda().contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)      # the generator's maps
    got = row_ops.dropout(m, 0.4, 9, span=30)
    assert got.shape == m.shape and torch.equal(got.cpu().reshape(60, 40), R.dropout(m.cpu().reshape(60, 40), None, 0.4, 9, 0, 30))
    t = rnd(40, 37, dtype=dtype).cuda().t()                                                                        # columns apart: copied
    assert torch.equal(row_ops.dropout(t, 0.4, 9).cpu(), R.dropout(t.cpu(), None, 0.4, 9, 0))
    e = rnd(1, 40, dtype=dtype).cuda().expand(5, 40)
    assert torch.equal(row_ops.dropout(e, 0.4, 9).cpu(), R.dropout(e.cpu().contiguous(), None, 0.4, 9, 0))
    for shape in ((0, 8), (4, 0), (2, 0, 8)):
        assert row_ops.dropout(torch.empty(shape, dtype=dtype, device="cuda"), 0.5, 1).shape == shape
    assert torch.equal(row_ops.dropout(x[0].cuda(), 0.3, 11, 5).cpu(), R.dropout(x[:1], None, 0.3, 11, 5)[0])


def test_dropout_clears_what_is_not_finite():
    x = torch.full((64, 64), float("inf"))
    x[::2] = float("nan")
    keep, _ = R.flags(64, 64, 0.5, 3, 0)
    got = row_ops.dropout(x.cuda(), 0.5, 3).cpu()
    assert (got[~keep] == 0).all() and not torch.isfinite(got[keep]).any()


def test_dropout_gradient_and_seed_tensor():
    x, r, g = (rnd(50, 33, seed=s) for s in (1, 2, 3))
    xg, rg = x.cuda().requires_grad_(), r.cuda().requires_grad_()
    seed = torch.tensor([77, 2 ** 35], dtype=torch.int64, device="cuda")
    y = row_ops.dropout(xg, 0.25, seed, offset=4, residual=rg, span=5)
    assert torch.equal(y.detach().cpu(), R.dropout(x, r, 0.25, 77, 2 ** 35 + 4, 5))
    y.backward(g.cuda())
    assert torch.equal(xg.grad.cpu(), R.dropout(g, None, 0.25, 77, 2 ** 35 + 4, 5)) and torch.equal(rg.grad.cpu(), g)
    y = row_ops.dropout(xg, 0.25, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    neg = torch.tensor([-3, -1], dtype=torch.int64, device="cuda")                    # two's complement, as the counter takes it
    assert torch.equal(row_ops.dropout(x.cuda(), 0.25, neg).cpu(), R.dropout(x, None, 0.25, -3, -1))
    assert torch.equal(row_ops.dropout(x.cuda(), 0.25, -3, -1).cpu(), R.dropout(x, None, 0.25, -3, -1))


def test_rows_behind_the_last_and_far_offsets():
    """rows more than 2^31 elements apart; bytes between and behind them stay as they are"""
    pitch, cols = (1 << 30) + 8, 48
    buf = torch.zeros(2 * pitch + cols + 64, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, cols), (pitch, 1))
    src = rnd(3, cols, dtype=torch.bfloat16)
    x.copy_(src)
    assert torch.equal(row_ops.dropout(x, 0.3, 5).cpu(), R.dropout(src, None, 0.3, 5, 0))
    y, h = row_ops.add_rms_norm(x, x, None, EPS)
    assert torch.equal(h.cpu(), (2 * src.float()).to(torch.bfloat16))
    q = row_ops.quantize8(x)
    assert torch.equal(q.data.cpu().view(torch.uint8), R.quantize(src, "row", "e4m3")[0].view(torch.uint8))
    d = _hip.RmsnormDesc()
    d.dtype, d.rows, d.cols, d.eps, d.span = _hip.BF16, 3, cols, EPS, 1
    d.x, d.ldx, d.y, d.ldy = x.data_ptr(), pitch, x.data_ptr(), pitch                  # in place
    _hip.check(_hip.lib().uncl_rmsnorm(d, _hip.stream_ptr()), "uncl_rmsnorm")
    want, _ = R.norm(src, None, EPS)
    within(x, want, (2.0 ** -8 + 96 * R.U) * want.abs())
    x.zero_()
    assert int(buf.count_nonzero()) == 0


# ---- residual addition and RMS norm ----------------------------------------------------------------------------------------------------
WIDTHS = [1, 5, 8, 13, 32, 64, 100, 256, 320, 520, 1000, 2048, 2056, 4096, 8200, 16384, 16392, 20001]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_forward_backward(dtype, cols):
    rows = 300 if cols < 600 else (67 if cols < 5000 else 5)
    x, r = rnd(rows, cols, dtype=dtype, size=3.0), rnd(rows, cols, dtype=dtype, seed=1)
    gy, gh = rnd(rows, cols, dtype=dtype, seed=2), rnd(rows, cols, dtype=dtype, seed=3)
    w = 1 + 0.3 * rnd(cols, seed=4)
    x[rows // 2] = 0                                                                     # a row of zeros
    r[rows // 2] = 0
    p = 0.2
    xs, rs, ws = x.cuda().requires_grad_(), r.cuda().requires_grad_(), w.cuda().requires_grad_()
    y, h = row_ops.add_rms_norm(xs, rs, ws, EPS, p=p, seed=9, offset=2)
    want_h = R.dropout(x, r, p, 9, 2)
    assert torch.equal(h.detach().cpu(), want_h)
    want_y, _ = R.norm(want_h, w, EPS)
    half = R.HALF[dtype]
    within(y, want_y, (half + 96 * R.U) * want_y.abs() + LOW[dtype], "y")
    gx, gr, gw = torch.autograd.grad([y, h], [xs, rs, ws], [gy.cuda(), gh.cuda()])
    want, size, want_w, size_w = R.norm_backward(gy, gh, want_h, w, EPS)
    tiny = LOW[dtype]
    within(gr, want, half * want.abs() + 128 * R.U * size + tiny, "g_res")
    keep, factor = R.flags(rows, cols, p, 9, 2)
    within(gx, want * keep * factor, (half * want.abs() + 130 * R.U * size) * keep * factor + tiny, "g_x")
    within(gw, want_w, 160 * R.U * size_w, "g_w")
    # one gradient only, no weight, nothing dropped: the same numbers for both summands
    xs, rs = x.cuda().requires_grad_(), r.cuda().requires_grad_()
    y, h = row_ops.add_rms_norm(xs, rs, None, EPS)
    h0 = (x.float() + r.float()).to(dtype)
    gx, gr = torch.autograd.grad(y, [xs, rs], gy.cuda())
    want, size, _, _ = R.norm_backward(gy, None, h0, None, EPS)
    within(gr, want, half * want.abs() + 128 * R.U * size + tiny, "g_res alone")
    assert torch.equal(gx, gr)
    gx, gr = torch.autograd.grad(row_ops.add_rms_norm(xs, rs, None, EPS)[1], [xs, rs], gh.cuda())
    assert torch.equal(gx.cpu(), gh) and torch.equal(gr.cpu(), gh)


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (2, 256), (4608, 256), (50000, 32), (3000, 520), (2500, 2056)])
def test_norm_of_many_rows_and_the_weights_gradient(rows, cols):
    x, gy, w = rnd(rows, cols, dtype=torch.bfloat16), rnd(rows, cols, dtype=torch.bfloat16, seed=1), 1 + 0.1 * rnd(cols, seed=2)
    xs, ws = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = row_ops.rms_norm(xs, ws, EPS)
    want_y, _ = R.norm(x, w, EPS)
    within(y, want_y, (2.0 ** -8 + 96 * R.U) * want_y.abs() + 1e-37, "y")
    gx, gw = torch.autograd.grad(y, [xs, ws], gy.cuda())
    want, size, want_w, size_w = R.norm_backward(gy, None, x, w, EPS)
    within(gx, want, 2.0 ** -8 * want.abs() + 128 * R.U * size + 1e-37, "g_x")
    within(gw, want_w, 160 * R.U * size_w, "g_w")
    y2 = row_ops.rms_norm(xs, ws, EPS)
    again = torch.autograd.grad(y2, [xs, ws], gy.cuda())
    assert torch.equal(y, y2) and torch.equal(gx, again[0]) and torch.equal(gw, again[1])      # fixed order: the same bits


def test_norm_gradient_against_differences():
    """directional derivative of a weighted sum of y and h: fp32 kernels, central differences of the 64-bit form; step 1e-5, whose own
    error is 1e-10 of the third derivative's size"""
    x, r, w, gy, gh = (rnd(20, 72, seed=s) for s in range(5))
    w = w[0]
    dx, dr, dw = rnd(20, 72, seed=7).double(), rnd(20, 72, seed=8).double(), rnd(72, seed=9).double()
    keep, factor = R.flags(20, 72, 0.2, 3, 0)

    def f(t):
        h = (r.double() + t * dr) + (x.double() + t * dx) * keep * factor
        y, _ = R.norm(h, w.double() + t * dw, EPS)
        return ((y * gy).sum() + (h * gh).sum()).item()
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    xs, rs, ws = (t.cuda().requires_grad_() for t in (x, r, w))
    y, h = row_ops.add_rms_norm(xs, rs, ws, EPS, p=0.2, seed=3)
    gx, gr, gw = torch.autograd.grad([y, h], [xs, rs, ws], [gy.cuda(), gh.cuda()])
    terms = [(gx.double().cpu() * dx), (gr.double().cpu() * dr), (gw.double().cpu() * dw)]
    got, size = sum(t.sum().item() for t in terms), sum(t.abs().sum().item() for t in terms)
    assert abs(got - want) < 1e-5 * size


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_norm_views_empty_and_one_dimension(dtype):
    x, r, w = rnd(37, 100, dtype=dtype), rnd(37, 100, dtype=dtype, seed=1), 1 + 0.1 * rnd(100, seed=2)
    ref = row_ops.add_rms_norm(x.cuda(), r.cuda(), w.cuda(), EPS)
    for more, front in ((3, 1), (8, 0), (1, 3)):
        got = row_ops.add_rms_norm(wide(x, more, front), wide(r, more + 2, front), w.cuda(), EPS)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    strided_w = torch.stack([w, w], 1).cuda()[:, 0]
    assert torch.equal(row_ops.rms_norm(ref[1], strided_w, EPS), ref[0])
    assert torch.equal(row_ops.rms_norm(ref[1][3], w.cuda(), EPS), ref[0][3])
    m = rnd(2, 32, 5, 6, dtype=dtype).cuda().contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    assert torch.equal(row_ops.rms_norm(m), row_ops.rms_norm(m.reshape(60, 32)).view(2, 5, 6, 32))
    for shape in ((0, 8), (2, 0, 8), (4, 0)):
        e = torch.empty(shape, dtype=dtype, device="cuda", requires_grad=True)
        ws = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y, h = row_ops.add_rms_norm(e, e, ws, EPS, p=0.1)
        assert y.shape == h.shape == torch.Size(shape)
        gx, gw = torch.autograd.grad(y, [e, ws], torch.empty_like(y))
        assert gx.shape == torch.Size(shape) and int(gw.count_nonzero()) == 0


@pytest.mark.parametrize("cols", [64, 16400])
def test_norm_of_a_row_with_nan_leaves_the_others(cols):
    x = rnd(9, cols)
    x[4, 7] = float("nan")
    y = row_ops.rms_norm(x.cuda()).cpu()
    assert torch.isnan(y[4]).all() and torch.isfinite(y[[0, 1, 2, 3, 5, 6, 7, 8]]).all()
    xs, g = x.cuda().requires_grad_(), rnd(9, cols, seed=1).cuda()
    _, h = row_ops.add_rms_norm(xs, torch.zeros_like(xs), None, EPS)                   # a gradient of the sum alone passes as it is
    assert torch.equal(torch.autograd.grad(h, [xs], g)[0], g)


def test_gradients_that_are_one_number_everywhere():
    """a sum's gradient is one element seen from everywhere: rows without a pitch"""
    x, w = rnd(40, 72).cuda().requires_grad_(), rnd(24, 72, seed=1).cuda().requires_grad_()
    ones = torch.ones(40, 72, device="cuda")
    for f, leaves in ((lambda: row_ops.dropout(x, 0.3, 1), [x]), (lambda: row_ops.rms_norm(x), [x]), (lambda: row_ops.linear8(x, w), [x, w])):
        got = torch.autograd.grad(f().sum(), leaves)
        want = torch.autograd.grad(f(), leaves, torch.ones_like(f()))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    y, h = row_ops.add_rms_norm(x, ones, None, EPS)
    got, = torch.autograd.grad(y.sum() + 2 * h.sum(), [x])
    y, h = row_ops.add_rms_norm(x, ones, None, EPS)
    assert torch.equal(got, torch.autograd.grad([y, h], [x], [ones, 2 * ones])[0])


# ---- 8-bit operands --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (128, 128), (130, 257), (5, 40), (300, 64), (1, 4096), (257, 1000)])
def test_quantize_bit_for_bit(dtype, fmt, rows, cols):
    x = rnd(rows, cols, dtype=dtype) * torch.exp2(torch.randint(-6, 6, (rows, cols), generator=torch.Generator().manual_seed(1)).float()).to(dtype)
    x[:, cols // 2] = 0
    x[rows // 2] *= 0                                                                    # whole blocks of zeros
    for block in ("row", "tile"):
        for transpose in (False, True):
            for src in (x.cuda(), wide(x, 5, 3)):
                q = row_ops.quantize8(src, block, transpose, fmt)
                data, scale = R.quantize(x, block, fmt, transpose)
                assert torch.equal(q.scale.cpu(), scale), (block, transpose)
                assert torch.equal(q.data.cpu().view(torch.uint8), data.view(torch.uint8)), (block, transpose)
                assert q.data.stride(0) % 16 == 0 and q.block == block
    assert torch.equal(row_ops.quantize8(x.cuda().view(1, rows, cols), fmt=fmt).data.view(torch.uint8),
                       row_ops.quantize8(x.cuda(), fmt=fmt).data.view(torch.uint8))


def test_quantize_of_values_that_are_not_finite():
    x = rnd(130, 140)
    x[0, 0], x[1, 1], x[2, 2], x[129, 139], x[5] = float("inf"), -float("inf"), float("nan"), float("nan"), float("inf")
    x[7] = 1e-38
    x[8, :128] = 3e38
    for block in ("row", "tile"):
        for transpose in (False, True):
            q = row_ops.quantize8(x.cuda(), block, transpose)
            data, scale = R.quantize(x, block, "e4m3", transpose)
            assert torch.equal(q.scale.cpu(), scale) and torch.isfinite(scale).all()
            nan = torch.isnan(data.float())
            assert torch.equal(torch.isnan(q.data.cpu().float()), nan) and int(nan.sum()) == 2
            assert torch.equal(q.data.cpu().float()[~nan], data.float()[~nan])
    for shape in ((0, 8), (4, 0)):
        e = torch.empty(shape, device="cuda")
        assert row_ops.quantize8(e).data.shape == shape and row_ops.quantize8(e, "tile", True).data.shape == shape[::-1]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [1, 8, 32, 100, 128, 130, 256, 520, 2056, 16392])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_norm_into_8_bits(dtype, cols, fmt):
    """the norm's result is off by 96 U before it is rounded; the scale by that and one rounding, and a value moves by half a step of the
    8-bit format (2^-4 / 2^-3 of itself, or half of the smallest number's step, 2^-10 / 2^-17 scales)"""
    rows = 70 if cols < 3000 else 3
    x, r, w = rnd(rows, cols, dtype=dtype), rnd(rows, cols, dtype=dtype, seed=1), 1 + 0.1 * rnd(cols, seed=2)
    x[1] = 0
    r[1] = 0
    q, h = row_ops.rms_norm_quant8(x.cuda(), w.cuda(), residual=r.cuda(), fmt=fmt)
    want_h = (x.float() + r.float()).to(dtype)
    assert torch.equal(h.cpu(), want_h)
    y, _ = R.norm(want_h, w, EPS)
    scale = torch.stack([b.abs().amax(1) for b in y.split(128, 1)], 1).clamp_min(2.0 ** -100) / R.TOP[fmt]
    within(q.scale, scale, 100 * R.U * scale, "scale")
    half, low = (2.0 ** -4, 2.0 ** -10) if fmt == "e4m3" else (2.0 ** -3, 2.0 ** -17)
    got = R.values(q.data.cpu(), q.scale.cpu(), "row")
    within(got, y, (1 + 200 * R.U) * torch.maximum(half * y.abs(), low * scale.repeat_interleave(128, 1)[:, :cols]) + 200 * R.U * y.abs(), "values")
    q2, h2 = row_ops.rms_norm_quant8(h, w.cuda(), fmt=fmt)
    assert h2 is h and torch.equal(q2.data.view(torch.uint8), q.data.view(torch.uint8)) and torch.equal(q2.scale, q.scale)


# ---- product -----------------------------------------------------------------------------------------------------------------------------
def operand(rows, cols, block, fmt="e4m3", seed=0):
    """a quantised matrix whose bytes behind a row's end are NaN"""
    data, scale = R.quantize(rnd(rows, cols, seed=seed) * torch.exp2(torch.arange(cols) % 5 - 2.0), block, fmt)
    room = torch.full((rows, -(-cols // 16) * 16 + 16), 0x7F, dtype=torch.uint8, device="cuda")
    room[:, :cols] = data.view(torch.uint8).cuda()
    return (data, scale, block), row_ops.Quant8(room.view(data.dtype)[:, :cols], scale.cuda(), block)


def check_product(m, n, k, block="tile", fa="e4m3", act="none", dtype=torch.float32, bias=True, residual=False):
    ra, a = operand(m, k, "row", fa)
    rb, b = operand(n, k, block, seed=1)
    want, size = R.matmul8(ra, rb)
    bv = rnd(n, seed=3) if bias else None
    rv = rnd(m, n, dtype=dtype, seed=4) if residual else None
    tol = (128 + 8 + -(-k // 128)) * R.U * size + (R.cut(ra, rb) if dtype == torch.bfloat16 else 0.0)
    if bias:
        want, tol = want + bv.double(), tol + R.U * (want.abs() + bv.double().abs())
    if act == "relu":
        want = want.clamp_min(0)
    elif act in ("lrelu", "sigmoid", "tanh", "msig"):             # slopes up to 1; an exponential and a division
        want = {"lrelu": lambda v: torch.where(v > 0, v, 0.2 * v), "sigmoid": torch.sigmoid, "tanh": torch.tanh, "msig": lambda v: torch.sigmoid(3 * v)}[act](want)
        tol = tol + 64 * R.U
    elif act == "gelu":
        tol = 1.13 * tol + 16 * R.U * want.abs()                 # the slope is at most 1.13; erf and two products
        want = want * torch.special.ndtr(want)
    if residual:
        want = want + rv.double()
        tol = tol + R.U * want.abs()
    out = row_ops.matmul8(a, b, bias=None if bv is None else bv.cuda(), act=act, residual=None if rv is None else rv.cuda(), out_dtype=dtype)
    within(out, want, tol + R.HALF[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0.0), "product %s" % ((m, n, k, block, fa, act, dtype),))
    return a, b, out


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 127), (100, 300), (128, 1192), (257, 129), (300, 2065)])
def test_product_sizes(m, n, k):
    check_product(m, n, k)


@pytest.mark.parametrize("m", [3, 40, 200])
@pytest.mark.parametrize("block", ["tile", "row"])
@pytest.mark.parametrize("fa", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_product_formats(m, block, fa, dtype):
    check_product(m, 200, 400, block, fa, dtype=dtype)
    check_product(m * 9, 1100, 70, block, fa, dtype=dtype)


@pytest.mark.parametrize("act", ["lrelu", "sigmoid", "tanh", "msig"])
@pytest.mark.parametrize("m,k", [(5, 128), (200, 100), (70, 1100)])
def test_product_rarer_activations(act, m, k):
    check_product(m, 130, k, act=act, residual=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n", [(5, 37), (70, 260), (1000, 300)])
def test_product_outputs(dtype, m, n):
    for act in ("none", "relu", "gelu"):
        for residual in (False, True):
            check_product(m, n, 256, act=act, dtype=dtype, bias=residual or act != "none", residual=residual)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(2100, 2050, 384), (28800, 256, 256), (4101, 3500, 1100), (300, 33000, 1024), (4099, 4096, 2048), (4099, 2048, 4096)])
def test_product_of_many_tiles(m, n, k, dtype):
    """the large shapes against a 64-bit product on the GPU of what the operands stand for"""
    _, a = operand(m, k, "row")
    _, b = operand(n, k, "tile", seed=1)
    want, size = R.matmul8(a, b)
    out = row_ops.matmul8(a, b, out_dtype=dtype)
    tol = (128 + 8 + -(-k // 128)) * R.U * size + (R.cut(a, b) if dtype == torch.bfloat16 else 0.0)
    bad = (out.double() - want).abs() > tol + R.HALF[dtype] * (want.abs() + tol) + 2.0 ** -25
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())
    assert torch.equal(out, row_ops.matmul8(a, b, out_dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(65, 65, 1024), (256, 200, 4608), (129, 1000, 2100), (70, 16, 30000)])
def test_product_of_few_tiles_and_long_sums(m, n, k, dtype):
    """workgroups share a tile's K; without scratch memory one takes all of it"""
    check_product(m, n, k, act="gelu", dtype=dtype, residual=True)
    a, b, out = check_product(m, n, k, "row", "e5m2", dtype=dtype)
    assert _hip.lib().uncl_matmul8_workspace_bytes(m, n, k) > 0
    one = torch.empty_like(out)
    d = _hip.Matmul8Desc()
    d.M, d.N, d.K, d.a_fmt, d.b_fmt = m, n, k, _hip.E5M2, _hip.E4M3
    d.a, d.lda, d.a_scale, d.a_scale_row, d.a_scale_block = a.data.data_ptr(), a.data.stride(0), a.scale.data_ptr(), a.scale.stride(0), a.scale.stride(1)
    bs = b.scale.t().contiguous()
    d.b, d.ldb, d.b_scale, d.b_scale_row, d.b_scale_block = b.data.data_ptr(), b.data.stride(0), bs.data_ptr(), 1, n
    bias = rnd(n, seed=3).cuda()
    d.bias, d.out, d.ldo, d.out_dtype = bias.data_ptr(), one.data_ptr(), n, _hip.dtype_code(dtype)
    _hip.check(_hip.lib().uncl_matmul8(d, None, _hip.stream_ptr()), "uncl_matmul8")
    want, size = R.matmul8((a.data, a.scale, "row"), (b.data, b.scale, "row"))
    want = (want + bias).cpu()
    tol = (128 + 10 + -(-k // 128)) * R.U * (size.cpu() + bias.abs().double().cpu()) + (R.cut((a.data, a.scale, "row"), (b.data, b.scale, "row")).cpu() if dtype == torch.bfloat16 else 0.0)
    within(one, want, tol + R.HALF[dtype] * (want.abs() + tol) + 2.0 ** -25, "one workgroup a tile")


def test_product_layouts():
    m, n, k = 70, 90, 200
    a, b, want = check_product(m, n, k, bias=False)
    odd = torch.zeros(m, k + 3, dtype=torch.uint8, device="cuda")                       # an odd pitch: copied to 16-byte borders
    odd[:, :k] = a.data.view(torch.uint8)
    a2 = row_ops.Quant8(odd.view(torch.float8_e4m3fn)[:, :k], a.scale, "row")
    assert torch.equal(row_ops.matmul8(a2, b, out_dtype=torch.float32), want)
    a3 = row_ops.Quant8(a.data, a.scale.t().contiguous().t(), "row")                    # scales block by block
    b3 = row_ops.Quant8(b.data.contiguous(), torch.stack([b.scale, b.scale], 2)[..., 1], "tile")
    assert torch.equal(row_ops.matmul8(a3, b3, out_dtype=torch.float32), want)
    buf = torch.full((m, n + 7), 5.0, device="cuda")                                    # rows of a wider buffer; what is beside stays
    got = row_ops.matmul8(a, b, out_dtype=torch.float32, out=buf[:, 3:3 + n])
    assert torch.equal(got, want) and (buf[:, :3] == 5).all() and (buf[:, 3 + n:] == 5).all() and got.data_ptr() == buf[:, 3:].data_ptr()
    acc = torch.ones(m, n, device="cuda")
    row_ops.matmul8(a, b, out_dtype=torch.float32, residual=acc, out=acc)               # in place: added to
    assert torch.equal(acc, want + 1)
    r = rnd(n, m).cuda().t()                                                            # a residual with columns apart
    assert torch.equal(row_ops.matmul8(a, b, out_dtype=torch.float32, residual=r), want + r)
    run = torch.arange((m + 1) * n, device="cuda", dtype=torch.float32).view(m + 1, n) % 64    # a residual one row above the result
    above = run[:-1].clone()
    row_ops.matmul8(a, b, out_dtype=torch.float32, residual=run[:-1], out=run[1:])
    assert torch.equal(run[1:], want + above)
    e = row_ops.matmul8(row_ops.Quant8(a.data[:0], a.scale[:0], "row"), b)
    assert e.shape == (0, n)


@pytest.mark.parametrize("m,k", [(3, 128), (100, 256), (70, 4096)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_product_activations_of_what_is_not_finite(m, k, dtype):
    _, a = operand(m, k, "row")
    _, b = operand(5, k, "tile")
    inf, nan = float("inf"), float("nan")
    bias = torch.tensor([inf, -inf, nan, -1e30, 1e30 if dtype != torch.float16 else 6e4], device="cuda")
    for act, want in (("none", [inf, -inf, nan]), ("relu", [inf, 0.0, nan]), ("lrelu", [inf, -inf, nan]), ("gelu", [inf, 0.0, nan]),
                      ("sigmoid", [1.0, 0.0, nan]), ("tanh", [1.0, -1.0, nan]), ("msig", [1.0, 0.0, nan])):
        out = row_ops.matmul8(a, b, bias=bias, act=act, out_dtype=dtype).float()
        assert torch.equal(out[:, :3].nan_to_num(7.0, 8.0, -8.0), torch.tensor(want, device="cuda").nan_to_num(7.0, 8.0, -8.0).expand(m, 3)), act
        if act in ("relu", "gelu"):
            assert (out[:, 3] == 0).all() and torch.isfinite(out[:, 4]).all()


def test_product_refusals():
    _, a = operand(8, 64, "row")
    _, b = operand(8, 64, "tile")
    _, c = operand(8, 65, "tile")
    f = torch.zeros(8, device="cuda")
    for call, kind in ((lambda: row_ops.matmul8(b, b), ValueError), (lambda: row_ops.matmul8(a, c), ValueError), (lambda: row_ops.matmul8(a, b, act="swish"), ValueError),
                       (lambda: row_ops.matmul8(a, b, out_dtype=torch.int32), TypeError), (lambda: row_ops.matmul8(a, b, bias=f.half()), TypeError),
                       (lambda: row_ops.matmul8(a, b, bias=f[:7]), ValueError), (lambda: row_ops.matmul8(a, b, residual=torch.zeros(8, 8, device="cuda")), TypeError),
                       (lambda: row_ops.matmul8(a, row_ops.Quant8(b.data, b.scale[:, :0], "tile")), ValueError),
                       (lambda: row_ops.matmul8(a, row_ops.Quant8(b.data.float(), b.scale, "tile")), TypeError),
                       (lambda: row_ops.matmul8(a, row_ops.quantize8(torch.zeros(8, 64, device="cuda"), "tile", fmt="e5m2")), TypeError),
                       (lambda: row_ops.matmul8(a, b, bias=f.requires_grad_()), RuntimeError),
                       (lambda: row_ops.matmul8(a, b, out=torch.zeros(8, 8, dtype=torch.bfloat16, device="cuda").t()[:, ::2]), ValueError),
                       (lambda: row_ops.quantize8(torch.zeros(4, 4, device="cuda"), "column"), ValueError),
                       (lambda: row_ops.quantize8(torch.zeros(4, 4, device="cuda"), fmt="e3m4"), ValueError),
                       (lambda: row_ops.quantize8(torch.zeros(4, 4, device="cuda", dtype=torch.float64)), TypeError),
                       (lambda: row_ops.quantize8(torch.zeros(4, 4, device="cuda", requires_grad=True)), RuntimeError),
                       (lambda: row_ops.dropout(torch.zeros(4, 4, device="cuda"), 1.5, 1), ValueError),
                       (lambda: row_ops.dropout(torch.zeros(4, 4, device="cuda"), 0.5, 1, span=0), ValueError),
                       (lambda: row_ops.dropout(torch.zeros(4, 4, device="cuda"), 0.5, 1, span=2 ** 64 + 1), ValueError),
                       (lambda: row_ops.dropout(torch.zeros(4, 4, device="cuda"), 0.5, 1.5), TypeError),
                       (lambda: row_ops.dropout(torch.zeros(4, 4, device="cuda"), 0.5, torch.zeros(2, dtype=torch.int64)), _hip.HipError),
                       (lambda: row_ops.dropout(torch.zeros((), device="cuda"), 0.5, 1), ValueError),
                       (lambda: row_ops.add_rms_norm(torch.zeros(4, 4, device="cuda"), torch.zeros(4, 5, device="cuda")), ValueError),
                       (lambda: row_ops.add_rms_norm(torch.zeros(4, 4, device="cuda"), torch.zeros(4, 4, device="cuda").half()), TypeError),
                       (lambda: row_ops.rms_norm(torch.zeros(4, 4, device="cuda"), torch.ones(5, device="cuda")), ValueError),
                       (lambda: row_ops.rms_norm(torch.zeros(4, 4, device="cuda"), eps=0.0), ValueError),
                       (lambda: row_ops.linear8(torch.zeros(4, 4, device="cuda"), torch.zeros(5, 3, device="cuda")), ValueError),
                       (lambda: row_ops.linear8(torch.zeros(1, 1, device="cuda").expand(2 ** 22 + 1, 1), torch.zeros(1, 1, device="cuda")), ValueError),
                       (lambda: row_ops.linear8(torch.zeros(4, 4, device="cuda"), torch.zeros(5, 4, device="cuda"), grad_fmt="fp8"), ValueError)):
        with pytest.raises(kind):
            call()


# ---- the linear layer of a training step -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (50, 100, 130), (300, 256, 256), (129, 33, 520)])
@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_linear8(m, n, k, dtype, wtype):
    x, w, b, g = rnd(m, k, dtype=dtype), rnd(n, k, dtype=wtype, size=k ** -0.5, seed=1), rnd(n, seed=2), rnd(m, n, dtype=dtype, seed=3, size=0.01)
    xs, ws, bs = (t.cuda().requires_grad_() for t in (x, w, b))
    y = row_ops.linear8(xs, ws, bs)
    gx, gw, gb = torch.autograd.grad(y, [xs, ws, bs], g.cuda())
    Q = lambda t, block, fmt, tr=False: (*R.quantize(t, block, fmt, tr), block)  # noqa: E731
    for got, ops, length, t, add in (
            (y, (Q(x, "row", "e4m3"), Q(w, "tile", "e4m3")), k, dtype, b.double()),
            (gx, (Q(g, "row", "e5m2"), Q(w, "tile", "e4m3", True)), n, dtype, 0.0),
            (gw, (Q(g, "row", "e5m2", True), Q(x, "row", "e4m3", True)), m, wtype, 0.0)):
        want, size = R.matmul8(*ops)
        tol = (128 + 9 + -(-length // 128)) * R.U * size + R.U * (want + add).abs() + (R.cut(*ops) if t == torch.bfloat16 else 0.0)
        assert got.dtype == t
        within(got, want + add, tol + R.HALF[t] * ((want + add).abs() + tol), "linear8")
    within(gb, g.double().sum(0), 300 * R.U * g.double().abs().sum(0), "bias")
    y3 = row_ops.linear8(xs.detach().view(1, m, k), ws, None)
    assert y3.shape == (1, m, n)
    only, = torch.autograd.grad(y3, [ws], g.cuda().view(1, m, n))
    assert torch.equal(only, gw)


def test_linear8_without_rows():
    x, w, b = torch.empty(0, 32, device="cuda", requires_grad=True), rnd(16, 32).cuda().requires_grad_(), rnd(16).cuda().requires_grad_()
    y = row_ops.linear8(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty(0, 16, device="cuda"))
    assert y.shape == (0, 16) and gx.shape == (0, 32) and int(gw.count_nonzero()) == 0 and int(gb.count_nonzero()) == 0


@pytest.mark.parametrize("which", ["x", "w", "b", "xb", "wb"])
def test_linear8_only_the_gradients_asked_for(which):
    x, w, b, g = rnd(200, 130, dtype=torch.bfloat16).cuda(), rnd(72, 130, seed=1).cuda(), rnd(72, seed=2).cuda(), rnd(200, 72, dtype=torch.bfloat16, seed=3).cuda()
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = dict(zip("xwb", torch.autograd.grad(row_ops.linear8(*full), full, g)))
    some = {n: t.clone().requires_grad_(n in which) for n, t in zip("xwb", (x, w, b))}
    got = torch.autograd.grad(row_ops.linear8(some["x"], some["w"], some["b"]), [some[n] for n in which], g)
    assert all(torch.equal(v, want[n]) for n, v in zip(which, got))
    with torch.no_grad():
        assert torch.equal(row_ops.linear8(*full), row_ops.linear8(x, w, b))


def test_linear8_of_views_and_changed_operands():
    """rows of wider buffers; x and weight changed after the forward pass: the gradients are those of the values it saw"""
    x, w, g = rnd(150, 100, dtype=torch.bfloat16), rnd(60, 100, seed=1), rnd(150, 60, dtype=torch.bfloat16, seed=2)
    xs, ws = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    want = torch.autograd.grad(row_ops.linear8(xs, ws), [xs, ws], g.cuda())
    xv, wv = wide(x, 5, 3).requires_grad_(), wide(w, 3, 1).requires_grad_()
    y = row_ops.linear8(xv, wv)
    with torch.no_grad():
        xv.zero_()
        wv.zero_()
    got = torch.autograd.grad(y, [xv, wv], wide(g, 7, 1))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- together --------------------------------------------------------------------------------------------------------------------------
def mlp(x, stream, w, seed, offset, p=0.1):
    """a channel MLP behind a dropped branch, as a training step runs it"""
    y, h = row_ops.add_rms_norm(x, stream, w["n"], EPS, p=p, seed=seed, offset=offset)
    z = torch.nn.functional.gelu(row_ops.linear8(y, w["w1"], w["b1"]))
    return row_ops.dropout(row_ops.linear8(z, w["w2"], w["b2"]), p, seed, offset + 1, residual=h)


def weights(c, m):
    return {"n": 1 + 0.1 * rnd(c, seed=1), "w1": rnd(m, c, size=c ** -0.5, seed=2), "b1": 0.1 * rnd(m, seed=3), "w2": rnd(c, m, size=m ** -0.5, seed=4),
            "b2": 0.1 * rnd(c, seed=5)}


def test_mlp_serving_against_64_bits():
    """norm into 8 bits, product with GELU, quantise, product with residual: against 64 bits on the operands that the steps hand over"""
    c, hid, rows = 256, 384, 144
    w = weights(c, hid)
    x, s = rnd(rows, c, dtype=torch.bfloat16), rnd(rows, c, dtype=torch.bfloat16, seed=9)
    wd = {k: v.cuda() for k, v in w.items()}
    q1, q2 = row_ops.quantize8(wd["w1"], "tile"), row_ops.quantize8(wd["w2"], "tile")
    with torch.no_grad():
        a, h = row_ops.rms_norm_quant8(x.cuda(), wd["n"], residual=s.cuda())
        z = row_ops.matmul8(a, q1, bias=wd["b1"], act="gelu")
        az = row_ops.quantize8(z)
        out = row_ops.matmul8(az, q2, bias=wd["b2"], residual=h)
    cpu = lambda q: (q.data.cpu(), q.scale.cpu(), q.block)  # noqa: E731
    want, size = R.matmul8(cpu(a), cpu(q1))
    want = want + w["b1"].double()
    tol = 1.13 * (140 * R.U * (size + w["b1"].abs().double()) + R.cut(cpu(a), cpu(q1))) + 16 * R.U * want.abs()
    want = want * torch.special.ndtr(want)
    within(z, want, tol + 2.0 ** -8 * (want.abs() + tol), "first product")
    want, size = R.matmul8(cpu(az), cpu(q2))
    want = want + w["b2"].double() + h.double().cpu()
    tol = 140 * R.U * (size + h.double().cpu().abs() + 1) + R.cut(cpu(az), cpu(q2))
    within(out, want, tol + 2.0 ** -8 * (want.abs() + tol), "second product")
    # and the whole against the same layer without any 8-bit rounding: an operand is off by at most 2^-4 of itself, at random, so that a sum of
    # hundreds of products is off by a few hundredths of its own size
    y, _ = R.norm(h.cpu(), w["n"], EPS)
    full = torch.nn.functional.gelu(y @ w["w1"].double().t() + w["b1"].double()) @ w["w2"].double().t() + w["b2"].double()
    got = out.double().cpu() - h.double().cpu()
    assert ((got - full).norm() / full.norm()).item() < 2.0 ** -4


def test_mlp_training_in_a_captured_graph():
    """forward and backward captured once: replays with the seed tensor moved on equal eager passes at the same seeds, bit for bit"""
    c, hid, rows = 256, 512, 288
    w = {k: v.cuda().requires_grad_() for k, v in weights(c, hid).items()}
    x = rnd(rows, c, dtype=torch.bfloat16).cuda().requires_grad_()
    s = rnd(rows, c, dtype=torch.bfloat16, seed=9).cuda().requires_grad_()
    g = rnd(rows, c, dtype=torch.bfloat16, seed=10).cuda()
    leaves = [x, s, *w.values()]

    def step(seed):
        out = mlp(x, s, w, seed, 3)
        return [out, *torch.autograd.grad(out, leaves, g)]
    eager = []
    for k in range(3):
        eager.append([t.detach().clone() for t in step(torch.tensor([5, 100 * k], dtype=torch.int64, device="cuda"))])
    seed = torch.tensor([5, 0], dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(seed)
    for k in (0, 1, 2, 1):
        seed.copy_(torch.tensor([5, 100 * k], dtype=torch.int64))
        with torch.no_grad():
            row_ops.rms_norm(x)                                  # the program's own work between replays
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, eager[k]):
            assert torch.equal(a.detach(), b)
    assert not torch.equal(eager[0][0], eager[1][0])


def test_other_streams_and_repeated_calls():
    x, w = rnd(5000, 256, dtype=torch.bfloat16).cuda(), (1 + 0.1 * rnd(256)).cuda()
    wq = row_ops.quantize8(rnd(512, 256).cuda(), "tile")
    q, _ = row_ops.rms_norm_quant8(x, w)
    want = row_ops.matmul8(q, wq)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for k in range(6):
        with torch.cuda.stream(streams[k % 3]):
            q, _ = row_ops.rms_norm_quant8(x, w)
            outs.append(row_ops.matmul8(q, wq))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device():
    x = rnd(40, 64).cuda(1).requires_grad_()
    y, h = row_ops.add_rms_norm(x, x.detach(), None, EPS, p=0.2, seed=1)
    gx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    x0 = x.detach().cuda(0).requires_grad_()
    y0, h0 = row_ops.add_rms_norm(x0, x0.detach(), None, EPS, p=0.2, seed=1)
    assert torch.equal(y.cuda(0), y0) and torch.equal(gx.cuda(0), torch.autograd.grad(y0, [x0], torch.ones_like(y0))[0])
