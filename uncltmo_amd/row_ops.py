"""Operators on rows of channels: dropout from a counter, the residual addition with an RMS norm behind it, and the matrix product of 8-bit
operands (csrc/row_ops.hip, csrc/quant8.hip, csrc/matmul8.hip).

A row is one pixel or graph node: the LAST axis of a tensor holds its channels.  An (N, C, H, W) map of the generator, which lies channel-last
in memory, goes in as `x.permute(0, 2, 3, 1)` -- a view.  Leading axes may have any strides that make one row pitch (slices of a wider
buffer among them); other layouts are copied first.  Tensors are fp32, bf16 or fp16 on an MI355X; there is no CPU path.

    training   y, h = add_rms_norm(branch, stream, weight, p=0.1, seed=seed, offset=layer)     # h: the new residual stream
               z = linear8(y, w1, b1)                                                          # 8-bit products, forward and gradients
    serving    q, h = rms_norm_quant8(branch, weight, residual=stream)
               z = matmul8(q, w1_q8, bias=b1, act="gelu")                                      # w1_q8 = quantize8(w1, "tile"), once
"""
import ctypes as C
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _hip

BLOCK = 128
_TILED_ROWS = 65535 * BLOCK               # one workgroup a tile of 128 x 128, tiles of rows along the grid's second axis
_FMT = {"e4m3": _hip.E4M3, "e5m2": _hip.E5M2}
_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_F8_TYPES = (torch.float8_e4m3fn, torch.float8_e5m2)
_F8_CODE = {torch.float8_e4m3fn: _hip.E4M3, torch.float8_e5m2: _hip.E5M2}
_ACT = {"none": _hip.ACT_NONE, "relu": _hip.ACT_RELU, "lrelu": _hip.ACT_LRELU, "gelu": _hip.ACT_GELU, "sigmoid": _hip.ACT_SIGMOID,
        "tanh": _hip.ACT_TANH, "msig": _hip.ACT_MSIG}
_CODE = {torch.float32: _hip.F32, torch.bfloat16: _hip.BF16, torch.float16: _hip.F16}
_DTYPES = tuple(_CODE)
_U64 = (1 << 64) - 1
# the handle alone of torch.cuda.current_stream(device): the Stream object around it takes 2 us of a call's 10 to make
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(dev, what, fn, *args):
    """One entry point of the library on the tensors' device and that device's current stream."""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, _stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev.index))
    if rc:
        _hip.check(rc, what)


def _need(t, what, dtypes, shape=None, dev=None):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and (shape is None or t.shape == shape) and (dev is None or t.device == dev):
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError("uncltmo_amd: %s must be a tensor, got %s" % (what, type(t).__name__))
    if not t.is_cuda:
        raise _hip.HipError("%s is on %s; the HIP path needs it on the MI355X" % (what, t.device))
    if t.dtype not in dtypes:
        raise TypeError("uncltmo_amd: %s must be %s, got %s" % (what, " / ".join(str(d).replace("torch.", "") for d in dtypes), t.dtype))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("uncltmo_amd: %s must have shape %s, got %s" % (what, tuple(shape), tuple(t.shape)))
    raise ValueError("uncltmo_amd: %s is on %s, the other tensors on %s" % (what, t.device, dev))


def _pitch(t):
    """Distance between neighbouring rows in elements, or None if the rows of `t` are not evenly spaced."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return None
    pitch = run = None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if pitch is None:
            pitch, run = stride, stride * size
        elif stride != run:
            return None
        else:
            run *= size
    pitch = t.shape[-1] if pitch is None else pitch
    return pitch if pitch >= t.shape[-1] else None


def _rows(t):
    """(tensor whose rows have one pitch, pitch)"""
    if t.is_contiguous():
        return t, t.shape[-1]
    p = _pitch(t)
    if p is None:
        t = t.contiguous()
        p = t.shape[-1]
    return t, p


def _extent(x):
    """(rows, channels), within what the entry points take: they hold channels in 32 bits, and ctypes would cut a larger number off unasked"""
    if x.dim() == 0:
        raise ValueError("uncltmo_amd: a tensor of rows needs an axis of channels")
    s = x.shape
    rows, cols = s[0] if len(s) == 2 else s[:-1].numel(), s[-1]
    if rows > 1 << 32 or cols > 1 << 30:
        raise ValueError("uncltmo_amd: up to 2^32 rows of up to 2^30 channels, got %d of %d" % (rows, cols))
    return rows, cols


def _seed_args(p, seed, offset, span, dev):
    """checked (p, span, seed tensor or None, seed, offset)"""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("uncltmo_amd: the dropout probability must be in [0, 1], got %r" % p)
    if not isinstance(span, int) or not 1 <= span < 1 << 63:
        raise ValueError("uncltmo_amd: span (rows that share their flags) must be a positive integer of 64 bits, got %r" % (span,))
    if not isinstance(offset, int):
        raise TypeError("uncltmo_amd: offset must be an integer, got %s" % type(offset).__name__)
    if isinstance(seed, torch.Tensor):
        _need(seed, "seed", (torch.int64,), (2,), dev)
        if not seed.is_contiguous():
            raise ValueError("uncltmo_amd: a seed tensor must be contiguous")
        return p, span, seed, 0, offset & _U64
    if not isinstance(seed, int):
        raise TypeError("uncltmo_amd: seed must be an integer or a device tensor of two int64 (seed, offset), got %s" % type(seed).__name__)
    return p, span, None, seed & _U64, offset & _U64


def _dropout(x, res, drop):
    rows, cols = _extent(x)
    x, ldx = _rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ldr = 0
    if res is not None:
        res, ldr = _rows(res)
    p, span, dev_seed, seed, offset = drop
    _call(x.device, "uncl_dropout", _hip.lib().uncl_dropout, x.data_ptr(), ldx, None if res is None else res.data_ptr(), ldr, y.data_ptr(), cols,
          _CODE[x.dtype], rows, cols, p, span, None if dev_seed is None else dev_seed.data_ptr(), seed, offset)
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, drop):
        ctx.drop = drop[:2] + (None,) + drop[3:]
        ctx.on_device = drop[2] is not None
        if ctx.on_device:
            ctx.save_for_backward(drop[2])       # autograd refuses a backward pass whose seed was changed in between
        return _dropout(x.detach(), None if res is None else res.detach(), drop)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        need = ctx.needs_input_grad
        drop = ctx.drop[:2] + (ctx.saved_tensors[0],) + ctx.drop[3:] if ctx.on_device else ctx.drop
        return _dropout(g, None, drop) if need[0] else None, g if need[1] else None, None


def dropout(x, p, seed, offset=0, residual=None, span=1):
    """residual + keep * x / (1 - p): the flags come from a counter (Philox4x32-10 of `seed`, `offset` and the element's place), no mask is
    stored, and the backward pass makes the same flags again.

    seed: an integer, or an int64 device tensor (seed, offset) that every launch reads -- the form for a captured graph, whose program
    changes it in place between replays.  offset: a number of its own for each call that shares a seed (layer, step); added to the seed
    tensor's.  span: so many consecutive rows share their flags; H * W for an (N, H, W, C) map drops whole channels of a sample, 1 single
    elements.  p is held in 16 bits (rounded to a multiple of 2^-16, the factor with it).  Dropped elements are 0 whatever x holds.  Every
    call drops: leave it out where nothing shall be dropped."""
    _need(x, "x", _DTYPES)
    if residual is not None:
        _need(residual, "residual", (x.dtype,), x.shape, x.device)
    drop = _seed_args(p, seed, offset, span, x.device)
    if not _wants_grad(x, residual):
        return _dropout(x, residual, drop)
    return _DropoutFn.apply(x, residual, drop)


def _norm_desc(x, res, w, eps, drop):
    d = _hip.RmsnormDesc()
    rows, cols = _extent(x)
    d.dtype, d.rows, d.cols, d.eps = _CODE[x.dtype], rows, cols, eps
    x, d.ldx = _rows(x)
    d.x = x.data_ptr()
    if res is not None:
        res, d.ldr = _rows(res)
        d.res = res.data_ptr()
    if w is not None:
        d.weight = w.data_ptr()
    d.span = 1
    if drop is not None:
        d.p, d.span, dev_seed, d.seed, d.offset = drop
        if dev_seed is not None:
            d.seed_dev = dev_seed.data_ptr()
    return d, x, res


def _norm(x, res, w, eps, drop, need_grad):
    """(y, h or None where nothing is added or dropped, 1 / rms or None)"""
    w = None if w is None else w.contiguous()
    d, xr, rr = _norm_desc(x, res, w, eps, drop)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    d.y, d.ldy = y.data_ptr(), d.cols
    h = rstd = None
    if res is not None or drop is not None:
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        d.h, d.ldh = h.data_ptr(), d.cols
    if need_grad:
        rstd = torch.empty(d.rows, dtype=torch.float32, device=x.device)
        d.rstd = rstd.data_ptr()
    _call(x.device, "uncl_rmsnorm", _hip.lib().uncl_rmsnorm, C.byref(d))
    return y, h, rstd


class _NormFn(torch.autograd.Function):
    """(x, residual, weight) -> (y, h); h is None where nothing is added or dropped"""

    @staticmethod
    def forward(ctx, x, res, w, eps, drop):
        ctx.set_materialize_grads(False)
        y, h, rstd = _norm(x, res, w, eps, drop, True)
        ctx.save_for_backward(x if h is None else h, rstd, w, None if drop is None else drop[2])
        # the backward pass runs on autograd's own thread, where Python is slow: what is known now is filled in now
        d = ctx.desc = _hip.RmsnormBwdDesc()
        d.rows, d.cols = _extent(x)
        d.dtype, d.span = _CODE[x.dtype], 1
        ctx.drop = drop is not None
        if drop is not None:
            d.p, d.span, _, d.seed, d.offset = drop
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gh):
        h, rstd, w, dev_seed = ctx.saved_tensors
        if gy is None and gh is None:
            return (None,) * 5
        need, dev, d, lib = ctx.needs_input_grad, h.device, _hip.RmsnormBwdDesc(), _hip.lib()
        C.memmove(C.byref(d), C.byref(ctx.desc), C.sizeof(d))
        if gy is not None:
            gy, d.ldgy = _rows(gy)
            d.gy = gy.data_ptr()
        if gh is not None:
            gh, d.ldgh = _rows(gh)
            d.gh = gh.data_ptr()
        h, d.ldh = _rows(h)
        d.h, d.rstd = h.data_ptr(), rstd.data_ptr()
        if w is not None:
            w = w.contiguous()
            d.weight = w.data_ptr()
        g_res = g_x = g_w = ws = None
        if need[1] or not ctx.drop:
            g_res = torch.empty(h.shape, dtype=h.dtype, device=dev)
            d.g_res, d.ldgr = g_res.data_ptr(), d.cols
        if not ctx.drop:
            g_x = g_res if need[0] else None
        elif need[0]:
            g_x = torch.empty(h.shape, dtype=h.dtype, device=dev)
            d.g_x, d.ldgx = g_x.data_ptr(), d.cols
            if dev_seed is not None:
                d.seed_dev = dev_seed.data_ptr()
        if need[2]:
            g_w = torch.empty(w.shape, dtype=torch.float32, device=dev)
            d.g_w = g_w.data_ptr()
            ws = torch.empty(lib.uncl_rmsnorm_backward_workspace_bytes(d.rows, d.cols), dtype=torch.uint8, device=dev)
        _call(dev, "uncl_rmsnorm_backward", lib.uncl_rmsnorm_backward, C.byref(d), None if ws is None else ws.data_ptr())
        return g_x, g_res if need[1] else None, g_w, None, None


def _norm_checks(x, residual, weight, eps):
    _need(x, "x", _DTYPES)
    _extent(x)
    if residual is not None:
        _need(residual, "residual", (x.dtype,), x.shape, x.device)
    if weight is not None:
        _need(weight, "weight", (torch.float32,), x.shape[-1:], x.device)
    eps = float(eps)
    if not eps > 0.0:
        raise ValueError("uncltmo_amd: eps must be positive (a row of zeros has no root mean square), got %r" % eps)
    return eps


def _wants_grad(a, b=None, c=None):
    """whether the call belongs on autograd's tape.  A dual tensor needs no requires_grad (and torch.no_grad() does not stop it): its tangent would
    get lost without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (a, b, c)):
        raise NotImplementedError("uncltmo_amd: the operators on rows of channels have no forward-mode derivatives")
    return torch.is_grad_enabled() and ((a is not None and a.requires_grad) or (b is not None and b.requires_grad) or (c is not None and c.requires_grad))


def rms_norm(x, weight=None, eps=1e-6):
    """x / sqrt(mean over the channels of x^2 + eps) * weight; weight: fp32, one number a channel.  ("Pixel norm" on a channel-last map.)"""
    eps = _norm_checks(x, None, weight, eps)
    return (_NormFn.apply(x, None, weight, eps, None) if _wants_grad(x, weight) else _norm(x, None, weight, eps, None, False))[0]


def add_rms_norm(x, residual, weight=None, eps=1e-6, p=0.0, seed=0, offset=0, span=1):
    """(y, h): h = residual + dropout(x, p, ...), the residual stream behind a branch, in the tensors' type, and y = rms_norm(h, weight, eps),
    in one pass over memory.  p = 0 drops nothing; seed / offset / span as in dropout().  Gradients flow through both results."""
    if residual is None:
        raise TypeError("uncltmo_amd: add_rms_norm needs a residual; rms_norm is the form without one")
    eps = _norm_checks(x, residual, weight, eps)
    drop = _seed_args(p, seed, offset, span, x.device)
    drop = drop if drop[0] > 0.0 else None
    if _wants_grad(x, residual, weight):
        return _NormFn.apply(x, residual, weight, eps, drop)
    return _norm(x, residual, weight, eps, drop, False)[:2]


class Quant8(NamedTuple):
    """A matrix in 8 bits.  data: (rows, cols) float8_e4m3fn or float8_e5m2; scale: fp32, (rows, ceil(cols / 128)) for block = "row" (one for
    128 neighbours of a row), (ceil(rows / 128), ceil(cols / 128)) for block = "tile"."""
    data: torch.Tensor
    scale: torch.Tensor
    block: str

    def values(self):
        """the fp32 matrix that the 8-bit numbers and their scales stand for"""
        r, c = self.data.shape
        s = self.scale.repeat_interleave(BLOCK, 1)[:, :c]
        return self.data.float() * (s if self.block == "row" else s.repeat_interleave(BLOCK, 0)[:r])


def _fmt(fmt):
    if fmt not in _FMT:
        raise ValueError("uncltmo_amd: the 8-bit format must be 'e4m3' or 'e5m2', got %r" % (fmt,))
    return _FMT[fmt]


def _no_grad(what, *ts):
    if _wants_grad(*ts):
        raise RuntimeError("uncltmo_amd: %s has no gradient; call it under torch.no_grad() or on detached tensors" % what)


def _empty8(rows, cols, fmt, block, dev):
    """rows on lines of memory (16-byte borders if they are shorter than one); row scales lie block by block, as the product reads them"""
    pitch, kb = (cols + 127) & ~127 if cols >= BLOCK else (cols + 15) & ~15, (cols + 127) // BLOCK
    data = torch.empty(rows, pitch, dtype=_F8[fmt], device=dev)
    if pitch != cols:
        data = data[:, :cols]
    scale = (torch.empty_strided((rows, kb), (1, rows), dtype=torch.float32, device=dev) if block == "row"
             else torch.empty((rows + 127) // BLOCK, kb, dtype=torch.float32, device=dev))
    return Quant8(data, scale, block)


def rms_norm_quant8(x, weight=None, residual=None, eps=1e-6, fmt="e4m3"):
    """(Quant8, h): add_rms_norm / rms_norm with y in 8 bits, one scale for 128 channels of a row, ready for matmul8; h = x + residual in
    their type (x itself without a residual).  The rows of all leading axes, in order.  No gradient."""
    eps = _norm_checks(x, residual, weight, eps)
    code = _fmt(fmt)
    _no_grad("rms_norm_quant8", x, weight, residual)
    rows, cols = _extent(x)
    weight = None if weight is None else weight.contiguous()
    d, xr, rr = _norm_desc(x, residual, weight, eps, None)
    q = _empty8(rows, cols, fmt, "row", x.device)
    h = x
    if residual is not None:
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        d.h, d.ldh = h.data_ptr(), cols
    d.y, d.ldy, d.y_fmt = q.data.data_ptr(), max(cols, q.data.stride(0)), code
    d.y_scale, d.scale_row, d.scale_block = q.scale.data_ptr(), q.scale.stride(0), q.scale.stride(1)
    _call(x.device, "uncl_rmsnorm", _hip.lib().uncl_rmsnorm, C.byref(d))
    return q, h


def quantize8(x, block="row", transpose=False, fmt="e4m3"):
    """x (rows, cols) -- leading axes of a larger tensor are its rows -- in 8 bits, block by block: scale = max(amax, 2^-100) / largest number
    of the format, data = x / scale rounded to the nearest, ties to even.  block "row": 1 x 128 (activations, gradients); "tile": 128 x 128
    (weights).  transpose: the result is (cols, rows), its blocks along x's rows.  Infinities become the largest number, NaN stays NaN;
    neither counts for the block's scale.  By tiles or transposed: up to 65535 x 128 rows."""
    _need(x, "x", _DTYPES)
    code = _fmt(fmt)
    if block not in ("row", "tile"):
        raise ValueError("uncltmo_amd: block must be 'row' or 'tile', got %r" % (block,))
    _no_grad("quantize8", x)
    rows, cols = _extent(x)
    if rows > _TILED_ROWS and (block == "tile" or transpose):
        raise ValueError("uncltmo_amd: quantize8 by tiles or transposed takes up to %d rows, got %d" % (_TILED_ROWS, rows))
    x, ldx = _rows(x)
    q = _empty8(cols if transpose else rows, rows if transpose else cols, fmt, block, x.device)
    _call(x.device, "uncl_quant8", _hip.lib().uncl_quant8, x.data_ptr(), _CODE[x.dtype], rows, cols, ldx, q.data.data_ptr(), q.data.stride(0), code,
          q.scale.data_ptr(), q.scale.stride(0), q.scale.stride(1), int(block == "tile"), int(bool(transpose)))
    return q


def _operand(t):
    """8-bit rows as the product reads them: on 16-byte borders, at most 2^22 bytes apart, readable up to the next one behind a row's end; (tensor,
    pitch)"""
    (rows, cols), (pitch, step) = t.shape, t.stride()
    room = (cols + 15) & ~15
    if (step == 1 or cols == 1) and pitch >= cols and pitch % 16 == 0 and pitch <= 1 << 22 and t.data_ptr() % 16 == 0 and (
            pitch >= room and t.storage_offset() + (rows - 1) * pitch + room <= t.untyped_storage().nbytes()):
        return t, pitch
    out = torch.zeros(rows, room, dtype=torch.uint8, device=t.device)
    out[:, :cols] = t.view(torch.uint8) if t.is_contiguous() else t.contiguous().view(torch.uint8)
    return out.view(t.dtype)[:, :cols], room


def _scale(t, most=1 << 20):
    """block scales with rows as near as the product wants them, within 32-bit offsets or neighbours; (tensor, its two strides)"""
    if t.shape[0] == 1:                                      # (whatever a single row's stride says)
        return t, (1, t.stride(1))
    if not (1 if most == 1 else 0) <= t.stride(0) <= most:
        t = t.t().contiguous().t()
    return t, t.stride()


def _quant_checks(q, what, blocks, dtypes):
    if not isinstance(q, Quant8):
        raise TypeError("uncltmo_amd: %s must be a Quant8 (see quantize8), got %s" % (what, type(q).__name__))
    if q.block not in blocks:
        raise ValueError("uncltmo_amd: %s must have blocks by %s, got %r" % (what, " or ".join(blocks), q.block))
    data = _need(q.data, what + ".data", dtypes)
    if data.dim() != 2:
        raise ValueError("uncltmo_amd: %s.data must be a matrix, got shape %s" % (what, tuple(data.shape)))
    r, c = data.shape
    _need(q.scale, what + ".scale", (torch.float32,), (r if q.block == "row" else (r + 127) // BLOCK, (c + 127) // BLOCK), data.device)
    return data


def matmul8(a, b, bias=None, act="none", residual=None, out_dtype=torch.bfloat16, out=None):
    """act(a b^T + bias) + residual of 8-bit operands a (M, K; e4m3 or e5m2, blocks by row) and b (N, K; e4m3, blocks by tile or by row): (M, N)
    in out_dtype, sums in fp32.
    bias: fp32 (N); act: none / relu / lrelu / gelu / sigmoid / tanh / msig; residual: (M, N) in out_dtype.  out: a tensor of that shape and
    type to write (the residual itself among them).  No gradient: linear8 is the form for training."""
    ad = _quant_checks(a, "a", ("row",), _F8_TYPES)
    bd = _quant_checks(b, "b", ("tile", "row"), (torch.float8_e4m3fn,))
    dev = ad.device
    (m, k), (n, kb) = ad.shape, bd.shape
    if k != kb or bd.device != dev:
        raise ValueError("uncltmo_amd: a is (M, K) = %s on %s, b (N, K) = %s on %s" % ((m, k), dev, (n, kb), bd.device))
    if k == 0:
        raise ValueError("uncltmo_amd: matmul8 needs a common axis of at least one element")
    if max(m, n) > 1 << 30 or k > 1 << 22:
        raise ValueError("uncltmo_amd: matmul8 takes up to 2^30 rows and results and a common axis of up to 2^22, got %d, %d and %d" % (m, n, k))
    if act not in _ACT:
        raise ValueError("uncltmo_amd: unknown activation %r" % (act,))
    if out_dtype not in _CODE:
        raise TypeError("uncltmo_amd: out_dtype must be float32, bfloat16 or float16, got %s" % out_dtype)
    d = _hip.Matmul8Desc()
    if bias is not None:
        bias = _need(bias, "bias", (torch.float32,), (n,), dev).contiguous()
        d.bias = bias.data_ptr()
    if residual is not None:
        _need(residual, "residual", (out_dtype,), (m, n), dev)
    _no_grad("matmul8", bias, residual, out)
    _no_grad("matmul8", a.scale, b.scale)
    given = out is not None
    if not given:
        out, ldo = torch.empty(m, n, dtype=out_dtype, device=dev), n
    else:
        _need(out, "out", (out_dtype,), (m, n), dev)
        ldo = _pitch(out)
        if ldo is None:
            raise ValueError("uncltmo_amd: out must have rows of neighbouring elements, got strides %s" % (out.stride(),))
    if m == 0 or n == 0:
        return out
    if residual is not None:
        residual, d.ldr = _rows(residual)
        if residual.data_ptr() != out.data_ptr() or d.ldr != ldo:        # rows of the one that are other rows of the other would be read too late
            if residual.untyped_storage().data_ptr() == out.untyped_storage().data_ptr():
                residual, d.ldr = residual.clone(memory_format=torch.contiguous_format), n
        d.res = residual.data_ptr()
    tile = b.block == "tile"
    (ad, lda), (bd, ldb), (sa, sas), (sb, sbs) = _operand(ad), _operand(bd), _scale(a.scale), _scale(b.scale, 1 << 20 if tile else 1)
    d.M, d.N, d.K, d.a_fmt, d.b_fmt, d.b_tile = m, n, k, _F8_CODE[ad.dtype], _hip.E4M3, tile
    d.a, d.lda, d.a_scale, (d.a_scale_row, d.a_scale_block) = ad.data_ptr(), lda, sa.data_ptr(), sas
    d.b, d.ldb, d.b_scale, (d.b_scale_row, d.b_scale_block) = bd.data_ptr(), ldb, sb.data_ptr(), sbs
    d.act, d.out_dtype, d.out, d.ldo = _ACT[act], _CODE[out_dtype], out.data_ptr(), ldo
    lib = _hip.lib()
    size = lib.uncl_matmul8_workspace_bytes(m, n, k) if m > 64 else 0
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _call(dev, "uncl_matmul8", lib.uncl_matmul8, C.byref(d), None if ws is None else ws.data_ptr())
    if given:                                                # autograd's saved copy of it, if there is one, is no longer what was saved
        torch.autograd.graph.increment_version(out)
    return out


def _linear8(x, w, bias, grad_fmt, for_x, for_w):
    """(y, what the backward pass needs: the descriptor's sizes and a buffer)"""
    lib, dev = _hip.lib(), x.device
    d = _hip.Linear8Desc()
    d.M, d.K = _extent(x)
    d.N = w.shape[0]
    d.dtype, d.w_dtype, d.grad_fmt, d.for_x, d.for_w = _CODE[x.dtype], _CODE[w.dtype], _FMT[grad_fmt], for_x, for_w
    y = torch.empty((*x.shape[:-1], d.N), dtype=x.dtype, device=dev)
    if d.M == 0:
        return y, d, None
    x, d.ldx = _rows(x)
    w, d.ldw = _rows(w)
    d.x, d.w, d.y, d.ldy = x.data_ptr(), w.data_ptr(), y.data_ptr(), d.N
    if bias is not None:
        bias = bias.contiguous()
        d.bias = bias.data_ptr()
    saved = torch.empty(lib.uncl_linear8_saved_bytes(d.M, d.N, d.K, for_x, for_w), dtype=torch.uint8, device=dev) if for_x or for_w else None
    ws = torch.empty(lib.uncl_linear8_workspace_bytes(d.M, d.N, d.K, 0), dtype=torch.uint8, device=dev)
    _call(dev, "uncl_linear8_forward", lib.uncl_linear8_forward, C.byref(d), None if saved is None else saved.data_ptr(), ws.data_ptr())
    return y, d, saved


class _Linear8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, grad_fmt):
        need = ctx.needs_input_grad
        y, ctx.desc, saved = _linear8(x, w, bias, grad_fmt, int(need[0]), int(need[1]))
        ctx.save_for_backward(saved)
        ctx.shapes = x.shape, w.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (saved,), need, lib, dev = ctx.saved_tensors, ctx.needs_input_grad, _hip.lib(), g.device
        shape, wtype = ctx.shapes
        f = ctx.desc
        gx = torch.empty(shape, dtype=g.dtype, device=dev) if need[0] else None
        gw = torch.empty(f.N, f.K, dtype=wtype, device=dev) if need[1] else None
        gb = torch.empty(f.N, dtype=torch.float32, device=dev) if need[2] else None
        if f.M == 0:
            return gx, None if gw is None else gw.zero_(), None if gb is None else gb.zero_(), None
        d = _hip.Linear8Desc()
        d.M, d.N, d.K, d.dtype, d.w_dtype, d.grad_fmt, d.for_x, d.for_w = f.M, f.N, f.K, f.dtype, f.w_dtype, f.grad_fmt, f.for_x, f.for_w
        g, d.ldgy = _rows(g)
        d.gy = g.data_ptr()
        if gx is not None:
            d.gx, d.ldgx = gx.data_ptr(), f.K
        if gw is not None:
            d.gw, d.ldgw = gw.data_ptr(), f.K
        if gb is not None:
            d.gb = gb.data_ptr()
        ws = torch.empty(lib.uncl_linear8_workspace_bytes(f.M, f.N, f.K, 1), dtype=torch.uint8, device=dev)
        _call(dev, "uncl_linear8_backward", lib.uncl_linear8_backward, C.byref(d), None if saved is None else saved.data_ptr(), ws.data_ptr())
        return gx, gw, gb, None


def linear8(x, weight, bias=None, grad_fmt="e5m2"):
    """x weight^T + bias with all three products of a training step in 8 bits: x and weight are quantised to e4m3 (rows / tiles of 128), the
    gradient of the output to grad_fmt by rows -- along its columns for x's gradient, along its rows, like x, for weight's.  weight (N, K)
    fp32, bf16 or fp16; bias fp32 (N).  The result and x's gradient have x's type, weight's gradient weight's (summed in fp32).  The rounding
    of the operands is not differentiated (straight through).  What the backward pass needs of x and weight is kept in 8 bits.  An infinity in
    x, weight or the gradient counts as NaN and makes NaN of every result it takes part in (a loss scale sees the step that overflowed); the
    bias' gradient is the plain sum.  Up to 2^22 rows, channels and results (each is a common axis of one of the products)."""
    _need(x, "x", _DTYPES)
    rows, k = _extent(x)
    _need(weight, "weight", _DTYPES, None, x.device)
    if weight.dim() != 2 or weight.shape[1] != k or k == 0 or weight.shape[0] == 0:
        raise ValueError("uncltmo_amd: weight must be (N, %d) with N > 0 and channels to sum over, got %s" % (k, tuple(weight.shape)))
    if max(rows, k, weight.shape[0]) > 1 << 22:
        raise ValueError("uncltmo_amd: linear8 takes up to 2^22 rows, channels and results, got %d, %d and %d" % (rows, k, weight.shape[0]))
    if bias is not None:
        _need(bias, "bias", (torch.float32,), (weight.shape[0],), x.device)
    _fmt(grad_fmt)
    if not _wants_grad(x, weight, bias):
        return _linear8(x, weight, bias, grad_fmt, 0, 0)[0]
    return _Linear8Fn.apply(x, weight, bias, grad_fmt)
