"""Cases, plain forms and 64-bit values of the operators on rows of channels (uncltmo_amd.row_ops): dropout from a counter, the residual
addition with the RMS norm behind it (and its 8-bit output), the matrix product of 8-bit operands with a scale for each block of 128, and
the linear layer of a training step built from three such products.

A row is one pixel or graph node of a channel-last tensor.  The generator's bottleneck has 144 nodes of 256 channels a sample (200 tiles of a
2160 x 3840 frame set = 28800 rows, 32 training frames = 4608), its last decoder stage maps of 252 x 252 pixels with 32 channels."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP = {"e4m3": 448.0, "e5m2": 57344.0}
AMAX_MIN = 2.0 ** -100
BLOCK = 128
EPS = 1e-6


# --------------------------------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------------------------------
def _dropout(rows, cols, dtype, p, train, residual, span=1):
    return {"op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "p": p, "train": train, "residual": residual, "span": span}


def _norm(rows, cols, dtype, p, train):
    return {"op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "p": p, "train": train}


def _norm8(rows, cols, dtype):
    return {"op": "norm8", "rows": rows, "cols": cols, "dtype": dtype}


def _matmul8(m, n, k, act, residual, dtype):
    return {"op": "matmul8", "m": m, "n": n, "k": k, "act": act, "residual": residual, "dtype": dtype}


def _linear8(m, n, k):
    return {"op": "linear8", "m": m, "n": n, "k": k}


def listed():
    return [
        # one sample's bottleneck nodes: the smallest call of a training step
        dict(name="dropout_nodes", **_dropout(144, 256, "bf16", 0.05, False, True)),
        # a training batch's last decoder stage, whole channels dropped, forward and gradient
        dict(name="dropout_maps_train", **_dropout(16 * 252 * 252, 32, "bf16", 0.1, True, False, 252 * 252)),
        # one token of a wide channel product
        dict(name="norm_token", **_norm(1, 4096, "bf16", 0.0, False)),
        # the bottleneck of 32 training frames, its branch dropped
        dict(name="norm_nodes_train", **_norm(4608, 256, "bf16", 0.05, True)),
        # pixel norm behind a decoder convolution of 8 training frames
        dict(name="norm_pixels_train", **_norm(8 * 252 * 252, 32, "bf16", 0.0, True)),
        # 200 tiles' nodes on their way into an 8-bit product
        dict(name="norm8_tiles", **_norm8(28800, 256, "fp16")),
        # one token: the weight is all there is to read
        dict(name="matmul8_token", **_matmul8(1, 4096, 4096, "none", True, "bf16")),
        # a ragged batch of rows and a weight with odd sides
        dict(name="matmul8_ragged", **_matmul8(1037, 1000, 1192, "relu", False, "fp16")),
        # first product of the bottleneck's channel MLP over 200 tiles
        dict(name="matmul8_tiles", **_matmul8(28800, 1024, 256, "gelu", False, "bf16")),
        # the largest: a long batch of rows through a wide square weight
        dict(name="matmul8_wide", **_matmul8(8192, 4096, 4096, "none", True, "bf16")),
        # the channel MLP of 32 training frames: output and both gradients
        dict(name="linear8_nodes", **_linear8(4608, 1024, 256)),
        # a wide layer of a training step with an odd number of rows
        dict(name="linear8_wide", **_linear8(4099, 4096, 2048)),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "norm", "norm8", "matmul8", "matmul8", "linear8"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op == "matmul8":
        n, k = _log(rng, 16, 8192), _log(rng, 16, 8192)
        m = _log(rng, 1, max(1, min(32768, 8192 * 4096 * 4096 // (n * k))))
        return _matmul8(m, n, k, rng.choice(["none", "relu", "gelu"]), rng.random() < 0.5, dtype)
    if op == "linear8":
        n, k = _log(rng, 64, 4096), _log(rng, 64, 4096)
        return _linear8(_log(rng, 16, max(16, min(8192, 4099 * 4096 * 2048 // (n * k)))), n, k)
    if op == "dropout":
        cols = _log(rng, 8, 2048)
        rows = _log(rng, 1, min(1 << 19, 30_000_000 // cols))
        return _dropout(rows, cols, dtype, rng.choice([0.05, 0.1, 0.5]), rng.random() < 0.5, rng.random() < 0.5,
                        1 if rng.random() < 0.6 else _log(rng, 2, max(2, rows // 2)))
    cols = _log(rng, 16, 8192)
    rows = _log(rng, 1, min(1 << 19, 16_000_000 // cols))
    if op == "norm8":
        return _norm8(rows, cols, dtype)
    return _norm(rows, cols, dtype, rng.choice([0.0, 0.05, 0.1]), rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------------------------
def _rows_of(gen, rows, cols, dtype, size=1.0):
    """activations: normal rows whose channels have sizes of their own, a few of them ten times the others'"""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    size_c = 0.5 + torch.rand(cols, generator=gen, device="cuda")
    size_c = torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.01, 10 * size_c, size_c)
    return x.mul_(size * size_c).to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": dict(case), "seed": 0x5851F42D4C957F2D ^ seed, "offset": 7 + seed % 1000}
    op = case["op"]
    if op in ("dropout", "norm", "norm8"):
        rows, cols, dtype = case["rows"], case["cols"], case["dtype"]
        s["x"] = _rows_of(gen, rows, cols, dtype)
        if op != "dropout" or case["residual"]:
            s["residual"] = _rows_of(gen, rows, cols, dtype, 2.0)
        if op != "dropout":
            s["weight"] = 1 + 0.2 * torch.randn(cols, generator=gen, device="cuda")
        if case.get("train"):
            s["gy"] = _rows_of(gen, rows, cols, dtype, 0.1)
            if op == "norm":
                s["gh"] = _rows_of(gen, rows, cols, dtype, 0.1)
        if case.get("train"):
            for name in ("x", "residual", "weight"):
                if name in s:
                    s[name].requires_grad_(True)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    if op == "matmul8":
        s["a"], s["a_scale"] = _pitched(*_q8_rows(_rows_of(gen, m, k, "fp32"), "e4m3"))
        s["b"], s["b_scale"] = _pitched(*_q8_tiles(torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k), "e4m3"))
        s["bias"] = 0.1 * torch.randn(n, generator=gen, device="cuda")
        s["residual"] = _rows_of(gen, m, n, case["dtype"]) if case["residual"] else None
        return s
    s["x"] = _rows_of(gen, m, k, "bf16").requires_grad_(True)
    s["weight"] = (torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)).requires_grad_(True)
    s["bias"] = (0.1 * torch.randn(n, generator=gen, device="cuda")).requires_grad_(True)
    s["gy"] = _rows_of(gen, m, n, "bf16", 0.01)
    return s


def _pitched(q, scale):
    """8-bit rows start on 16-byte borders, as the quantisers lay them out; row scales lie block by block"""
    rows, cols = q.shape
    room = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=q.device)
    room[:, :cols] = q.view(torch.uint8)
    if scale.shape[0] == rows:
        scale = scale.t().contiguous().t()
    return room.view(q.dtype)[:, :cols], scale


# --------------------------------------------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------------------------------------------
def _flags(p, seed, offset, rows, cols, span):
    """1 where an element is kept: 16-bit words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3),
    eight a counter, against round(p 2^16)"""
    limit = int(round(p * 65536))
    groups = -(-cols // 8)
    i = torch.arange(-(-rows // span) * groups, dtype=torch.int64, device="cuda")
    low = 0xFFFFFFFF
    c = [i & low, i >> 32, torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        # a product of 32 by 32 bits wraps in int64, and its halves come out all the same
        x, y = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((y >> 32) & low) ^ c[1] ^ k0, y & low, ((x >> 32) & low) ^ c[3] ^ k1, x & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], dim=1)
    keep = (words >= limit).view(-1, groups * 8)[:, :cols]
    return (keep.repeat_interleave(span, dim=0)[:rows] if span > 1 else keep), (65536.0 / (65536 - limit) if limit < 65536 else 0.0)


def _drop(x, flags):
    keep, size = flags
    return torch.where(keep, x.float() * torch.tensor(size, dtype=torch.float32, device=x.device), 0.0)


def _plain_dropout(s):
    c, x = s["case"], s["x"].detach()
    flags = _flags(c["p"], s["seed"], s["offset"], c["rows"], c["cols"], c["span"])
    y = _drop(x, flags)
    if "residual" in s:
        y = y + s["residual"].detach().float()
    out = [y.to(x.dtype)]
    if c["train"]:
        out.append(_drop(s["gy"], flags).to(x.dtype))
        if "residual" in s:
            out.append(s["gy"])
    return out


def _plain_norm(s):
    c, x, w = s["case"], s["x"].detach(), s["weight"].detach()
    flags = _flags(c["p"], s["seed"], s["offset"], c["rows"], c["cols"], 1) if c["p"] else None
    h = ((x.float() if flags is None else _drop(x, flags)) + s["residual"].detach().float()).to(x.dtype)
    hf = h.float()
    r = torch.rsqrt(hf.square().mean(1, keepdim=True) + EPS)
    n = hf * r
    out = [(n * w).to(x.dtype), h]
    if c["train"]:
        g = s["gy"].float()
        gw = g * w
        gh = s["gh"].float() + r * (gw - n * (gw * n).mean(1, keepdim=True))
        out += [(gh if flags is None else _drop(gh, flags)).to(x.dtype), gh.to(x.dtype), (g * n).sum(0)]
    return out


def _scales(amax, fmt):
    scale = amax.clamp_min(AMAX_MIN) * torch.tensor(1.0 / TOP[fmt], dtype=torch.float32, device=amax.device)
    return scale, torch.reciprocal(scale)


def _blocks(x, rows_too):
    """x with its columns (and rows) filled up with zeros to whole blocks of 128, the blocks in axes of their own"""
    r, c = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -c % BLOCK, 0, -r % BLOCK if rows_too else 0))
    return x.view(-1, BLOCK if rows_too else 1, x.shape[1] // BLOCK, BLOCK)


def _q8(x, fmt, rows_too):
    r, c = x.shape
    b = _blocks(x, rows_too)
    scale, inverse = _scales(b.abs().amax(dim=(1, 3)), fmt)
    q = (b * inverse[:, None, :, None]).clamp(-TOP[fmt], TOP[fmt]).reshape(-1, b.shape[2] * BLOCK)[:r, :c]
    return q.to(F8[fmt]), scale


def _q8_rows(x, fmt):
    return _q8(x, fmt, False)


def _q8_tiles(x, fmt):
    return _q8(x, fmt, True)


def _values(q, scale):
    """the values that 8-bit numbers and their blocks' scales stand for"""
    r, c = q.shape
    b = _blocks(q.float(), scale.shape[0] != r)
    return (b * scale[:, None, :, None]).reshape(-1, b.shape[2] * BLOCK)[:r, :c]


def _product(a, b):
    """a b^T of quantised operands, block after block of the common axis"""
    return _values(*a) @ _values(*b).t()


def _plain_matmul8(s):
    c = s["case"]
    y = _product((s["a"], s["a_scale"]), (s["b"], s["b_scale"])) + s["bias"]
    if c["act"] == "relu":
        y = y.clamp_min(0)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[c["dtype"]])


def _plain_linear8(s):
    x, w, g = s["x"].detach(), s["weight"].detach(), s["gy"]
    y = _product(_q8_rows(x, "e4m3"), _q8_tiles(w, "e4m3")) + s["bias"].detach()
    gx = _product(_q8_rows(g, "e5m2"), _q8_tiles(w.t(), "e4m3"))
    gw = _product(_q8_rows(g.t(), "e5m2"), _q8_rows(x.t(), "e4m3"))
    return [y.to(x.dtype), gx.to(x.dtype), gw, g.float().sum(0)]


def run(state):
    if own:
        return _own(state)
    return {"dropout": _plain_dropout, "norm": _plain_norm, "norm8": _plain_norm8, "matmul8": _plain_matmul8,
            "linear8": _plain_linear8}[state["case"]["op"]](state)


def _plain_norm8(s):
    x = s["x"]
    h = (x.float() + s["residual"].float()).to(x.dtype)
    hf = h.float()
    y = hf * torch.rsqrt(hf.square().mean(1, keepdim=True) + EPS) * s["weight"]
    q, scale = _q8_rows(y, "e4m3")
    return [q, scale, h]


def _own(s):
    from uncltmo_amd import row_ops
    c = s["case"]
    op = c["op"]
    if op == "dropout":
        x, r = s["x"], s.get("residual")
        if c["span"] > 1:
            y = row_ops.dropout(x, c["p"], s["seed"], s["offset"], residual=r, span=c["span"])
        else:
            y = row_ops.dropout(x, c["p"], s["seed"], s["offset"], residual=r)
        if not c["train"]:
            return [y]
        return [y, *torch.autograd.grad(y, [x] if r is None else [x, r], s["gy"])]
    if op == "norm":
        y, h = row_ops.add_rms_norm(s["x"], s["residual"], s["weight"], EPS, p=c["p"], seed=s["seed"], offset=s["offset"])
        if not c["train"]:
            return [y, h]
        return [y, h, *torch.autograd.grad([y, h], [s["x"], s["residual"], s["weight"]], [s["gy"], s["gh"]])]
    if op == "norm8":
        q, h = row_ops.rms_norm_quant8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return [q.data, q.scale, h]
    if op == "matmul8":
        return row_ops.matmul8(row_ops.Quant8(s["a"], s["a_scale"], "row"), row_ops.Quant8(s["b"], s["b_scale"], "tile"), bias=s["bias"],
                               act=c["act"], residual=s["residual"], out_dtype=DTYPES[c["dtype"]])
    y = row_ops.linear8(s["x"], s["weight"], s["bias"])
    return [y, *torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["gy"])]


# --------------------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op in ("dropout", "norm", "norm8"):
        n, e = case["rows"] * case["cols"], 2 if case["dtype"] != "fp32" else 4
        if op == "norm8":
            return {"bytes": n * (3 * e + 1) + 4 * case["rows"] * -(-case["cols"] // BLOCK) + 4 * case["cols"], "flops": 8 * n}
        if op == "dropout":
            back = 2 if case["train"] else 0
            return {"bytes": n * e * (2 + case["residual"] + back), "flops": 2 * n}
        # forward x, residual -> h, y; backward gy, gh, h -> gradients of x (dropped branch) and of the residual
        back = (5 if case["p"] else 4) if case["train"] else 0
        return {"bytes": n * e * (4 + back) + 8 * case["cols"], "flops": (6 + (12 if case["train"] else 0)) * n}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "matmul8":
        e = 2 if case["dtype"] != "fp32" else 4
        kb = -(-k // BLOCK)
        return {"bytes": m * k + n * k + 4 * m * kb + 4 * -(-n // BLOCK) * kb + m * n * e * (1 + case["residual"]) + 4 * n, "flops": 2 * m * n * k}
    # x, weight, gy in; y, two gradients out
    return {"bytes": 2 * m * k * 2 + 2 * m * n * 2 + 2 * n * k * 4 + 8 * n, "flops": 6 * m * n * k}


# --------------------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------------------------------------------
def _exact_keep(case, s, span):
    """the flags by numpy's unsigned 64-bit integers"""
    rows, cols = case["rows"], case["cols"]
    t, per = int(round(case["p"] * 65536)), (cols + 7) // 8
    i = np.arange(((rows + span - 1) // span) * per, dtype=np.uint64)
    lo, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    a, b = i & lo, i >> s32
    c, d = np.full_like(i, s["offset"]) & lo, np.full_like(i, s["offset"]) >> s32
    key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32 % 2 ** 32]
    for _ in range(10):
        u, v = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (v >> s32) ^ b ^ np.uint64(key[0]), v & lo, (u >> s32) ^ d ^ np.uint64(key[1]), u & lo
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack([a, b, c, d], 1).astype("<u4").view("<u2").reshape(-1, per * 8)
    keep = torch.from_numpy(words >= t).cuda() if t < 65536 else torch.zeros(words.shape, dtype=torch.bool, device="cuda")
    return keep[:, :cols][torch.arange(rows, device="cuda") // span], 65536 / (65536 - t) if t < 65536 else 0.0


def _round8(v, fmt):
    """to the nearest number of the 8-bit format, ties to even, in 64 bits"""
    bits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    e = (torch.frexp(v.abs()).exponent.double() - 1).clamp_min(low)
    step = torch.exp2(e - bits)
    return ((v / step).round() * step).clamp(-TOP[fmt], TOP[fmt])


def _exact_q8(x, fmt, rows):
    """64-bit 8-bit values and scales of blocks of 128 columns and `rows` rows; the scale, its inverse and their product with x are held in 32
    bits by definition"""
    r, c = x.shape
    f32 = lambda t: t.to(torch.float32).double()  # noqa: E731
    full = torch.zeros(-(-r // rows) * rows, -(-c // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:r, :c] = x.double()
    parts = full.unflatten(0, (-1, rows)).unflatten(2, (-1, BLOCK))
    amax = parts.abs().amax(dim=(1, 3)).clamp_min(AMAX_MIN)
    scale = f32(amax * float(np.float32(1 / TOP[fmt])))
    q = _round8(f32(parts * f32(1 / scale)[:, None, :, None]), fmt)
    return q.flatten(2, 3).flatten(0, 1)[:r, :c], scale


def _exact_values(q, scale, rows):
    full = scale.double().repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    return q.double() * full


def _exact_linear(x, w, g, bias):
    va = lambda t, fmt, rows: _exact_values(*_exact_q8(t, fmt, rows), rows)  # noqa: E731
    y = va(x, "e4m3", 1) @ va(w, "e4m3", BLOCK).t() + bias.double()
    gx = va(g, "e5m2", 1) @ va(w.t(), "e4m3", BLOCK).t()
    gw = va(g.t(), "e5m2", 1) @ va(x.t(), "e4m3", 1).t()
    return [y, gx, gw, g.double().sum(0)]


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    op = case["op"]
    if op == "dropout":
        keep, size = _exact_keep(case, s, case["span"])
        y = s["x"].double().mul_(size).mul_(keep)
        out = [y.add_(s["residual"].double()) if case["residual"] else y]
        if case["train"]:
            out.append(s["gy"].double().mul_(size).mul_(keep))
            if case["residual"]:
                out.append(s["gy"].double())
        return out
    if op in ("norm", "norm8"):
        x, w = s["x"].double(), s["weight"].double()
        keep, size = _exact_keep(case, s, 1) if case.get("p") else (None, 1.0)
        if keep is not None:
            x = x * size * keep
        h = (x + s["residual"].double()).to(s["x"].dtype).double()          # the sum is held in the tensors' type by definition
        rms = (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt()
        u = h / rms
        if op == "norm8":
            q, scale = _exact_q8(u * w, "e4m3", 1)
            return [q, scale, h]
        out = [u * w, h]
        if case["train"]:
            g = s["gy"].double()
            v = g * w
            gh = (v - u * (v * u).sum(1, keepdim=True) / h.shape[1]) / rms + s["gh"].double()
            out += [gh if keep is None else gh * size * keep, gh, (g * u).sum(0)]
        return out
    if op == "matmul8":
        y = _exact_values(s["a"], s["a_scale"], 1) @ _exact_values(s["b"], s["b_scale"], BLOCK).t() + s["bias"].double()
        if case["act"] == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        return y if s["residual"] is None else y + s["residual"].double()
    return _exact_linear(s["x"], s["weight"], s["gy"], s["bias"])
