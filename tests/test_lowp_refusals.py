"""CPU checks of the C entry points' refusals: every bad argument answers
JB_ERR_INVALID with a message before any device call."""
import math

import pytest

from jammi_b200 import _lib as L

P = 4096  # stands for a device pointer: a refused call never reads it


def refused(fn, *args):
    st = fn(*args)
    msg = L.lib().jb_last_error().decode()
    assert st == L.ERR_INVALID, (st, msg)
    assert msg
    return msg


def rms(**kw):
    a = dict(x=P, r=None, gamma=P, sum=None, y=P, q=None, scale=None, dtype=L.DT_BF16, rows=4, cols=8, eps=1e-6) | kw
    return refused(L.lib().jb_op_rmsnorm, a["x"], a["r"], a["gamma"], a["sum"], a["y"], a["q"], a["scale"], a["dtype"],
                   a["rows"], a["cols"], a["eps"], None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=2 ** 31 - 1), dict(cols=0), dict(cols=-3), dict(dtype=L.DT_S8), dict(dtype=9), dict(y=None),
                                dict(q=P, scale=P), dict(y=None, q=P), dict(y=None, scale=P), dict(scale=P),
                                dict(sum=P), dict(eps=-1.0), dict(eps=math.nan), dict(x=None), dict(gamma=None)])
def test_rmsnorm_refuses(kw):
    assert "rmsnorm" in rms(**kw)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=2 ** 31 - 1), dict(cols=0), dict(dtype=L.DT_S32), dict(q=None), dict(scale=None),
                                dict(y=None)])
def test_dequantize_rows_refuses(kw):
    a = dict(q=P, scale=P, y=P, dtype=L.DT_F32, rows=2, cols=8) | kw
    refused(L.lib().jb_op_dequantize_rows, a["q"], a["scale"], a["y"], a["dtype"], a["rows"], a["cols"], None)


@pytest.mark.parametrize("fn", ["jb_op_quantize_mxfp4", "jb_op_dequantize_mxfp4"])
@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=2 ** 31 - 1), dict(cols=2 ** 31 - 32), dict(cols=0), dict(cols=48), dict(cols=-32), dict(dtype=L.DT_S8), dict(x=None),
                                dict(q=None), dict(scale=None), dict(x=P + 8), dict(q=P + 4), dict(scale=P + 2)])
def test_mxfp4_rows_refuse(fn, kw):
    a = dict(x=P, dtype=L.DT_BF16, q=P, scale=P, rows=4, cols=64) | kw
    args = [a["x"], a["dtype"], a["q"], a["scale"]] if "_quantize" in fn else [a["q"], a["scale"], a["x"], a["dtype"]]
    assert fn in refused(getattr(L.lib(), fn), *args, a["rows"], a["cols"], None)


@pytest.mark.parametrize("kw", [dict(M=-1), dict(M=2 ** 31 - 1), dict(N=2 ** 31 - 8), dict(K=2 ** 31 - 32), dict(N=0), dict(N=12), dict(K=0), dict(K=48), dict(c_dtype=L.DT_S32),
                                dict(epi=-1), dict(epi=4), dict(epi=L.EPI_RESIDUAL), dict(res=P), dict(aq=None),
                                dict(ws=None), dict(c=None), dict(aq=P + 8), dict(c=P + 2), dict(asc=P + 1),
                                dict(epi=L.EPI_RESIDUAL, res=P + 4)])
def test_linear_mxfp4_refuses(kw):
    a = dict(aq=P, asc=P, wq=P, ws=P, bias=None, res=None, c=P, c_dtype=L.DT_BF16, M=4, N=16, K=64, epi=L.EPI_NONE) | kw
    refused(L.lib().jb_op_linear_mxfp4, a["aq"], a["asc"], a["wq"], a["ws"], a["bias"], a["res"], a["c"], a["c_dtype"],
            a["M"], a["N"], a["K"], a["epi"], None)


def test_mxfp4_scale_bytes():
    f = L.lib().jb_mxfp4_scale_bytes
    assert [f(1, 32), f(128, 128), f(129, 128), f(128, 160), f(0, 64), f(-1, 64)] == [512, 512, 1024, 1024, 0, 0]
    assert f(2 ** 31 - 1, 4096) == 2 ** 24 * 32 * 512


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(batch=2 ** 31 - 1), dict(rows=2 ** 31 - 1), dict(heads=0), dict(kv=0), dict(kv=3), dict(d=24), dict(d=256), dict(d=0),
                                dict(max_len=-1), dict(rows=-1), dict(left=-1), dict(right=-5), dict(sinks=-1),
                                dict(dtype=L.DT_S8), dict(qkv=None), dict(cu=None), dict(ctx=None), dict(qkv=P + 2),
                                dict(ctx=P + 8), dict(heads=2 ** 22, kv=2 ** 21)])
def test_attention_window_refuses(kw):
    a = dict(qkv=P, cu=P, ctx=P, dtype=L.DT_BF16, batch=2, heads=4, kv=2, d=64, max_len=16, rows=32, left=4, right=4,
             sinks=0) | kw
    refused(L.lib().jb_op_attention_window, a["qkv"], a["cu"], a["ctx"], a["dtype"], a["batch"], a["heads"], a["kv"],
            a["d"], a["max_len"], a["rows"], a["left"], a["right"], a["sinks"], None)


@pytest.mark.parametrize("cols", [2 ** 30 + 1, 2 ** 31 - 256, 2 ** 31 - 1])
def test_columns_that_32_bit_steps_would_pass_are_refused(cols):
    """A row's last step past its end must not wrap to a negative column."""
    for kw in (dict(), dict(y=None, q=P, scale=P), dict(dtype=L.DT_F32), dict(r=P, sum=P)):
        assert "cols" in rms(cols=cols, **kw)
    for dtype in (L.DT_F32, L.DT_BF16, L.DT_F16):
        assert "cols" in refused(L.lib().jb_op_dequantize_rows, P, P, P, dtype, 1, cols, None)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_buffers_between_elements_are_refused(off):
    """A load of half an element would fault on the device."""
    lib = L.lib()
    for dtype in (L.DT_F32, L.DT_BF16, L.DT_F16):
        wide = off % (4 if dtype == L.DT_F32 else 2)
        for kw in ([dict(x=P + off), dict(r=P + off), dict(r=P, sum=P + off), dict(y=P + off)] if wide else []):
            assert "aligned" in rms(dtype=dtype, **kw)
        for kw in (dict(gamma=P + off), dict(y=None, q=P, scale=P + off)):
            assert "aligned" in rms(dtype=dtype, **kw)
        if wide:
            assert "aligned" in refused(lib.jb_op_dequantize_rows, P, P, P + off, dtype, 2, 8, None)
        assert "aligned" in refused(lib.jb_op_dequantize_rows, P, P + off, P, dtype, 2, 8, None)
    assert "bias" in refused(lib.jb_op_linear_mxfp4, P, P, P, P, P + off, None, P, L.DT_BF16, 4, 16, 64, L.EPI_NONE, None)
    assert "cu_seqlens" in refused(lib.jb_op_attention_window, P, P + off, P, L.DT_BF16, 2, 4, 2, 64, 16, 32, 4, 4, 0, None)
