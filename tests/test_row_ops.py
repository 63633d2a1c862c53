"""Operators on rows of channels (uncltmo_amd.row_ops), what needs no GPU: the counter's published test vectors, the layouts of the C
structs, the refusals of the C entries (before any launch) and of the Python functions."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import row_ops_ref as R
from uncltmo_amd import _hip, row_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_counter_against_published_vectors():
    """known answers of Philox4x32-10 (counter, key -> four words)"""
    for c, k, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                       ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                       ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                        (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in R.philox(np.array([c], dtype=np.uint64), k)[0]) == want


def test_flags_share_rows_and_keep_the_expectation():
    keep, factor = R.flags(600, 37, 0.1, 5, 2 ** 40, span=3)
    assert torch.equal(keep[0], keep[2]) and not torch.equal(keep[2], keep[3])
    keep, factor = R.flags(4000, 100, 0.1, 5, 9)
    n, q = keep.numel(), 1 / factor
    assert abs(keep.float().mean().item() - q) < 5 * (q * (1 - q) / n) ** 0.5          # five standard deviations of a mean of n flags
    assert abs(q - 0.9) < 2.0 ** -17


def test_struct_layouts_match_the_c_side():
    exe = os.path.join(ROOT, "build", "row_ops_sizes")
    os.makedirs(os.path.dirname(exe), exist_ok=True)
    with open(exe + ".c", "w") as f:
        f.write('#include <stdio.h>\n#include <stddef.h>\n#include "uncltmo_hip.h"\nint main(){printf("%zu %zu %zu %zu %zu %zu %zu %zu\\n", '
                "sizeof(uncl_rmsnorm_desc), sizeof(uncl_rmsnorm_bwd_desc), sizeof(uncl_matmul8_desc), sizeof(uncl_linear8_desc), "
                "offsetof(uncl_rmsnorm_desc, offset), offsetof(uncl_rmsnorm_bwd_desc, offset), offsetof(uncl_matmul8_desc, ldo), "
                "offsetof(uncl_linear8_desc, gb));return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), exe + ".c", "-o", exe])
    got = [int(v) for v in subprocess.check_output([exe]).split()]
    ds = (_hip.RmsnormDesc, _hip.RmsnormBwdDesc, _hip.Matmul8Desc, _hip.Linear8Desc)
    assert got == [C.sizeof(d) for d in ds] + [ds[0].offset.offset, ds[1].offset.offset, ds[2].ldo.offset, ds[3].gb.offset]


def test_entries_refuse_bad_arguments_before_any_launch():
    lib, bad = _hip.lib(), -1
    buf = (C.c_float * 64)()
    p = (C.addressof(buf) + 15) & ~15

    def drop(x=p, ldx=8, res=None, ldr=0, y=p, ldy=8, dt=_hip.F32, rows=2, cols=8, prob=0.5, span=1):
        return lib.uncl_dropout(x, ldx, res, ldr, y, ldy, dt, rows, cols, prob, span, None, 1, 2, None)
    for kw in (dict(x=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(res=p, ldr=7), dict(dt=3), dict(rows=-1), dict(cols=-1), dict(prob=-0.1),
               dict(prob=1.5), dict(prob=float("nan")), dict(span=0), dict(rows=2 ** 32 + 1), dict(cols=2 ** 30 + 1, ldx=2 ** 31, ldy=2 ** 31)):
        assert drop(**kw) == bad, kw
    assert drop(rows=0, x=None) == 0 and drop(cols=0, y=None) == 0

    def make(cls, base, **kw):
        d = cls()
        for k, v in {**base, **kw}.items():
            setattr(d, k, v)
        return C.byref(d)
    base = dict(dtype=_hip.F32, rows=2, cols=8, eps=1e-6, x=p, ldx=8, y=p, ldy=8, span=1)
    for kw in (dict(x=None), dict(y=None), dict(eps=0.0), dict(eps=float("nan")), dict(eps=-1.0), dict(ldx=7), dict(ldy=7), dict(res=p, ldr=7), dict(h=p, ldh=7),
               dict(dtype=9), dict(rows=-1), dict(rows=2 ** 32 + 1), dict(cols=2 ** 30 + 1, ldx=2 ** 31, ldy=2 ** 31), dict(y_fmt=3), dict(y_fmt=_hip.E4M3), dict(p=2.0), dict(span=0)):
        assert lib.uncl_rmsnorm(make(_hip.RmsnormDesc, base, **kw), None) == bad, kw
    assert lib.uncl_rmsnorm(None, None) == bad and lib.uncl_rmsnorm(make(_hip.RmsnormDesc, base, rows=0, x=None), None) == 0
    base = dict(dtype=_hip.F32, rows=2, cols=8, h=p, ldh=8, rstd=p, gy=p, ldgy=8, g_res=p, ldgr=8, span=1)
    for kw in (dict(h=None), dict(rstd=None), dict(ldh=7), dict(ldgy=7), dict(gh=p, ldgh=7), dict(ldgr=7), dict(g_x=p, ldgx=7), dict(g_w=p), dict(span=0),
               dict(p=-1.0), dict(dtype=7), dict(rows=-3), dict(rows=2 ** 33), dict(cols=2 ** 30 + 1, ldh=2 ** 31, ldgy=2 ** 31, ldgr=2 ** 31)):
        assert lib.uncl_rmsnorm_backward(make(_hip.RmsnormBwdDesc, base, **kw), None, None) == bad, kw
    assert lib.uncl_rmsnorm_backward(None, None, None) == bad and lib.uncl_rmsnorm_backward_workspace_bytes(0, 8) == 0
    assert lib.uncl_rmsnorm_backward_workspace_bytes(10 ** 7, 40) <= 1024 * 40 * 4

    def quant(x=p, dt=_hip.F32, rows=2, cols=8, ldx=8, q=p, ldq=16, fmt=_hip.E4M3, scale=p, tile=0, tr=0):
        return lib.uncl_quant8(x, dt, rows, cols, ldx, q, ldq, fmt, scale, 1, 1, tile, tr, None)
    for kw in (dict(x=None), dict(q=None), dict(scale=None), dict(dt=4), dict(fmt=0), dict(fmt=3), dict(ldx=7), dict(ldq=7), dict(rows=-1), dict(rows=2 ** 33), dict(cols=2 ** 30 + 1, ldx=2 ** 31, ldq=2 ** 31), dict(tr=1, rows=20),
               dict(tile=1, rows=65535 * 128 + 1), dict(tr=1, rows=65535 * 128 + 1, ldq=2 ** 31)):
        assert quant(**kw) == bad, kw
    assert quant(rows=0, x=None) == 0
    base = dict(M=2, N=2, K=8, a_fmt=1, b_fmt=1, b_tile=1, a=p, lda=16, a_scale=p, b=p, ldb=16, b_scale=p, out=p, ldo=2, out_dtype=_hip.F32)
    for kw in (dict(a=None), dict(b=None), dict(a_scale=None), dict(b_scale=None), dict(out=None), dict(a_fmt=0), dict(b_fmt=3), dict(b_fmt=2), dict(lda=2 ** 22 + 16), dict(a_scale_row=2 ** 20 + 1), dict(b_scale_row=-1), dict(b_tile=0, b_scale_row=2), dict(lda=8), dict(lda=24), dict(ldb=20),
               dict(K=17), dict(K=0), dict(a=p + 8), dict(b=p + 4), dict(ldo=1), dict(res=p, ldr=1), dict(act=9), dict(act=-1), dict(out_dtype=5), dict(M=-1),
               dict(M=2 ** 30 + 1), dict(M=2 ** 30, N=2 ** 30, ldo=2 ** 30)):
        assert lib.uncl_matmul8(make(_hip.Matmul8Desc, base, **kw), None, None) == bad, kw
    assert lib.uncl_matmul8(make(_hip.Matmul8Desc, base, M=0, a=None), None, None) == 0 and lib.uncl_matmul8(None, None, None) == bad
    assert lib.uncl_matmul8_workspace_bytes(28800, 1024, 256) == 0 and lib.uncl_matmul8_workspace_bytes(256, 64, 4608) > 0 and lib.uncl_matmul8_workspace_bytes(0, 4, 4) == 0
    base = dict(M=2, N=8, K=8, dtype=_hip.BF16, w_dtype=_hip.F32, grad_fmt=2, for_x=1, for_w=1, x=p, ldx=8, w=p, ldw=8, y=p, ldy=8, gy=p, ldgy=8, gx=p, ldgx=8, gw=p, ldgw=8)
    both = (dict(M=-1), dict(N=0), dict(K=0), dict(M=2 ** 22 + 1), dict(N=2 ** 22 + 1), dict(dtype=3), dict(w_dtype=-1), dict(grad_fmt=0), dict(grad_fmt=3))
    for kw in both + (dict(x=None), dict(w=None), dict(y=None), dict(ldx=7), dict(ldw=7), dict(ldy=7)):
        assert lib.uncl_linear8_forward(make(_hip.Linear8Desc, base, **kw), p, p, None) == bad, kw
    for kw in both + (dict(gy=None), dict(ldgy=7), dict(ldgx=7), dict(ldgw=7), dict(for_x=0), dict(for_w=0)):
        assert lib.uncl_linear8_backward(make(_hip.Linear8Desc, base, **kw), p, p, None) == bad, kw
    d = make(_hip.Linear8Desc, base)
    assert lib.uncl_linear8_forward(d, None, p, None) == bad and lib.uncl_linear8_forward(d, p, None, None) == bad and lib.uncl_linear8_forward(None, p, p, None) == bad
    assert lib.uncl_linear8_backward(d, None, p, None) == bad and lib.uncl_linear8_backward(d, p, None, None) == bad and lib.uncl_linear8_backward(None, p, p, None) == bad
    empty = make(_hip.Linear8Desc, base, M=0, x=None)
    assert lib.uncl_linear8_forward(empty, None, None, None) == 0 and lib.uncl_linear8_backward(empty, None, None, None) == 0
    assert lib.uncl_linear8_saved_bytes(100, 8, 8, 0, 0) == 0 and lib.uncl_linear8_saved_bytes(0, 8, 8, 1, 1) == 0


def test_host_tensors_and_wrong_kinds_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: row_ops.dropout(x, 0.5, 1), lambda: row_ops.rms_norm(x), lambda: row_ops.add_rms_norm(x, x),
                 lambda: row_ops.rms_norm_quant8(x), lambda: row_ops.quantize8(x), lambda: row_ops.linear8(x, x),
                 lambda: row_ops.matmul8(row_ops.Quant8(x.to(torch.float8_e4m3fn), torch.ones(4, 1), "row"),
                                         row_ops.Quant8(x.to(torch.float8_e4m3fn), torch.ones(1, 1), "tile"))):
        with pytest.raises(_hip.HipError):
            call()
    with pytest.raises(TypeError):
        row_ops.dropout([1.0], 0.5, 1)
    with pytest.raises(TypeError):
        row_ops.matmul8(x, x)
    with pytest.raises(TypeError):
        row_ops.add_rms_norm(x, None)


def test_row_pitch_of_views():
    x = torch.zeros(6, 5, 32)
    assert row_ops._pitch(x) == 32 and row_ops._pitch(x[..., 8:24]) == 32 and row_ops._pitch(x[:, 2]) == 160
    assert row_ops._pitch(x[:, :3]) is None and row_ops._pitch(x.transpose(0, 1)) is None and row_ops._pitch(x[..., ::2]) is None
    assert row_ops._pitch(torch.zeros(1, 32).expand(6, 32)) is None                    # rows that are one place in memory: copied
    assert row_ops._pitch(torch.zeros(7)) == 7 and row_ops._pitch(x[:1, :1]) == 32
    n = torch.zeros(2, 32, 6, 6).contiguous(memory_format=torch.channels_last)
    assert row_ops._pitch(n.permute(0, 2, 3, 1)) == 32
