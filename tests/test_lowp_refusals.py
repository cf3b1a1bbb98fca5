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


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(cols=0), dict(cols=-3), dict(dtype=L.DT_S8), dict(dtype=9), dict(y=None),
                                dict(q=P, scale=P), dict(y=None, q=P), dict(y=None, scale=P), dict(scale=P),
                                dict(sum=P), dict(eps=-1.0), dict(eps=math.nan), dict(x=None), dict(gamma=None)])
def test_rmsnorm_refuses(kw):
    assert "rmsnorm" in rms(**kw)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(cols=0), dict(dtype=L.DT_S32), dict(q=None), dict(scale=None),
                                dict(y=None)])
def test_dequantize_rows_refuses(kw):
    a = dict(q=P, scale=P, y=P, dtype=L.DT_F32, rows=2, cols=8) | kw
    refused(L.lib().jb_op_dequantize_rows, a["q"], a["scale"], a["y"], a["dtype"], a["rows"], a["cols"], None)
