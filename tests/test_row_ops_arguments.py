"""What the Python entry points of the operators on rows of channels (uncltmo_amd.row_ops) decide before a launch, without a GPU: the device
check and the launch are replaced, so that sizes can be those of tensors that no memory holds."""
import pytest
import torch

from uncltmo_amd import row_ops

E4M3 = torch.float8_e4m3fn


@pytest.fixture
def calls(monkeypatch):
    """entry points called, in place of launches"""
    seen = []
    monkeypatch.setattr(row_ops, "_need", lambda t, what, dtypes, shape=None, dev=None: t)
    monkeypatch.setattr(row_ops, "_call", lambda dev, what, fn, *args: seen.append(what))
    return seen


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def q8(rows, cols, block, pitch=None):
    """a matrix in 8 bits without memory"""
    pitch = pitch or (cols + 15) & ~15
    data = meta(rows, pitch, dtype=E4M3)[:, :cols]
    return row_ops.Quant8(data, meta(rows if block == "row" else (rows + 127) // 128, (cols + 127) // 128, dtype=torch.float32), block)


# sizes that a 32-bit field would keep the low bits of, and the first ones over the limits
WIDE = [(2 ** 32,), (2 ** 32 + 8,), (3, 2 ** 32 + 8), (2 ** 30 + 1,), (1, 2, 2 ** 31)]


@pytest.mark.parametrize("shape", WIDE + [(2 ** 32 + 1, 4), (2 ** 17, 2 ** 16, 1)], ids=str)
def test_rows_and_channels_over_the_limits_are_refused(calls, shape):
    x = meta(*shape)
    for call in (lambda: row_ops.dropout(x, 0.5, 1), lambda: row_ops.rms_norm(x), lambda: row_ops.add_rms_norm(x, x, p=0.1),
                 lambda: row_ops.rms_norm_quant8(x), lambda: row_ops.quantize8(x), lambda: row_ops.quantize8(x, "tile"),
                 lambda: row_ops.quantize8(x, transpose=True), lambda: row_ops.linear8(x, meta(8, shape[-1]))):
        with pytest.raises(ValueError):
            call()
    assert not calls


def test_rows_and_channels_at_the_limits_are_taken(calls):
    for x in (meta(2 ** 30), meta(2 ** 32, 1)):
        row_ops.dropout(x, 0.5, 1)
        row_ops.rms_norm(x)
        row_ops.quantize8(x)
    assert calls == ["uncl_dropout", "uncl_rmsnorm", "uncl_quant8"] * 2


@pytest.mark.parametrize("m,n,k", [(2 ** 32 + 5, 8, 16), (2 ** 32, 8, 16), (8, 2 ** 32 + 8, 16), (2 ** 30 + 1, 8, 16), (8, 2 ** 30 + 1, 16), (8, 8, 2 ** 32 + 128),
                                   (8, 8, 2 ** 22 + 1)])
def test_products_over_the_limits_are_refused(calls, m, n, k):
    with pytest.raises(ValueError):
        row_ops.matmul8(q8(m, k, "row"), q8(n, k, "tile"))
    assert not calls


def test_forward_mode_derivatives_are_refused(calls):
    """a dual tensor needs no requires_grad; its tangent must not get lost"""
    x, other, w = torch.ones(4, 16), torch.zeros(4, 16), torch.ones(16)
    quants = row_ops.Quant8(x.to(E4M3), torch.ones(4, 1), "row"), row_ops.Quant8(x.to(E4M3), torch.ones(1, 1), "tile")
    with torch.autograd.forward_ad.dual_level():
        d, dw = (torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w))
        for call in (lambda: row_ops.dropout(d, 0.5, 1), lambda: row_ops.dropout(x, 0.5, 1, residual=d), lambda: row_ops.rms_norm(d), lambda: row_ops.rms_norm(x, dw),
                     lambda: row_ops.add_rms_norm(x, d), lambda: row_ops.rms_norm_quant8(d), lambda: row_ops.quantize8(d), lambda: row_ops.linear8(d, other),
                     lambda: row_ops.linear8(x, d), lambda: row_ops.matmul8(*quants, residual=torch.autograd.forward_ad.make_dual(other[:, :4], other[:, :4]))):
            for mode in (torch.enable_grad, torch.no_grad):              # (no_grad leaves forward mode on)
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        assert not calls
        row_ops.dropout(x, 0.5, 1)                                       # no tangent: an ordinary call
    assert calls == ["uncl_dropout"]


def test_product_into_a_given_tensor_is_a_change_that_autograd_sees(calls):
    """written as torch's own in-place operations are: a backward pass that saved the tensor raises instead of reading the new numbers"""
    a, b = row_ops.Quant8(torch.ones(4, 16).to(E4M3), torch.ones(4, 1), "row"), row_ops.Quant8(torch.ones(16, 16).to(E4M3), torch.ones(1, 1), "tile")
    x = torch.ones(4, 16, requires_grad=True)
    h = x * 2
    y = h * h                                                            # saves h
    with torch.no_grad():
        row_ops.matmul8(a, b, residual=h.detach(), out_dtype=torch.float32, out=h.detach())
    assert calls == ["uncl_matmul8"] and h._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        t = torch.zeros(4, 16)
        assert row_ops.matmul8(a, b, out_dtype=torch.float32, out=t) is t
    empty = row_ops.Quant8(a.data[:0], a.scale[:0], "row")
    row_ops.matmul8(empty, b, out_dtype=torch.float32, out=torch.zeros(0, 16))
    assert len(calls) == 2


def test_quantised_tiles_have_a_limit_of_rows(calls):
    most = 65535 * 128
    for kw in (dict(block="tile"), dict(transpose=True), dict(block="tile", transpose=True)):
        row_ops.quantize8(meta(most, 8), **kw)
        with pytest.raises(ValueError, match="8388480"):
            row_ops.quantize8(meta(most + 1, 8), **kw)
    row_ops.quantize8(meta(most + 1, 8))
    assert calls == ["uncl_quant8"] * 4


def test_layouts_that_the_product_does_not_read_are_copied(calls, monkeypatch):
    """one row whose stride is any number, and rows far apart: taken like every other layout, within the entry's limits"""
    sent = []
    monkeypatch.setattr(row_ops, "_call", lambda dev, what, fn, desc, *args: sent.append({k: getattr(desc._obj, k) for k in ("M", "lda", "ldb", "a_scale_row", "b_scale_row")}))
    b = q8(8, 256, "tile")
    far = meta(2 ** 21 * 2, 2, dtype=torch.float32).as_strided((1, 2), (2 ** 21, 1))
    row_ops.matmul8(row_ops.Quant8(q8(1, 256, "row").data, far, "row"), b)                       # scales of one row
    row_ops.matmul8(q8(1, 256, "row"), row_ops.Quant8(b.data, far, "tile"))
    row_ops.matmul8(q8(3, 256, "row", 2 ** 22 + 16), b)                                          # rows of a and of b
    row_ops.matmul8(q8(3, 256, "row"), q8(8, 256, "tile", 2 ** 22 + 16))
    assert len(sent) == 4
    for d in sent:
        assert d["lda"] <= 2 ** 22 and d["ldb"] <= 2 ** 22 and 0 <= d["a_scale_row"] <= 2 ** 20 and 0 <= d["b_scale_row"] <= 2 ** 20, d


def test_scales_that_want_a_gradient_are_refused(calls):
    a, b = row_ops.Quant8(torch.ones(4, 16).to(E4M3), torch.ones(4, 1), "row"), row_ops.Quant8(torch.ones(16, 16).to(E4M3), torch.ones(1, 1), "tile")
    for qa, qb in ((a._replace(scale=torch.ones(4, 1, requires_grad=True)), b), (a, b._replace(scale=torch.ones(1, 1, requires_grad=True)))):
        with pytest.raises(RuntimeError, match="no gradient"):
            row_ops.matmul8(qa, qb)
        with torch.no_grad():
            row_ops.matmul8(qa, qb)
    assert calls == ["uncl_matmul8"] * 2
