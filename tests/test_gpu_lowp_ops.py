"""GPU parity of the RMS norm, the MXFP4 format and windowed attention
against plain float64 implementations, through the public entry points.

A rounding is off by at most half a step: u = ``torch.finfo(t).eps / 2`` of
the value (bf16 2^-8, f16 2^-11, f32 2^-24); the tolerances count those.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def _ops():
    from jammi_b200 import ops
    return ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ── RMS norm ────────────────────────────────────────────────────────────────

def rms_ref(x, gamma, r):
    s = x.double() + (r.double() if r is not None else 0)
    return s, s / torch.sqrt(s.square().mean(1, keepdim=True) + EPS) * gamma.double()


def rms_f32_error(cols):
    """Relative error of y = s * rstd * gamma before its last rounding, in f32
    roundings u = 2^-24: s (1); the sum of squares, every term positive, in
    at most cols + 8 additions on any path, halved by the square root (its
    terms carry 2 of s and 1 of the square); the division, the addition of
    eps, the root and the reciprocal (4); two products (2)."""
    return (1 + ((cols + 8) + 3) / 2 + 4 + 2) * 2.0 ** -24


def sum_depth(cols):
    """Additions on the longest path of the kernels' sums: a thread's own
    elements, then a tree.  A thread holds at most 64 (wide rows) or
    ceil(cols / 256) elements in two partial sums."""
    return max(64, -(-cols // 256)) + 16


RMS_SHAPES = [(1, 1), (1, 8), (3, 7), (12, 768), (5, 33), (257, 384), (1000, 1024), (9, 1032), (130, 1536), (33, 2056),
              (17, 4096), (5, 4100), (3, 16384), (2, 16392), (2, 20001)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("rows,cols", RMS_SHAPES)
def test_rmsnorm(dev, rows, cols, res, dt):
    t, g = DTYPES[dt], _gen(rows * 31 + cols + res)
    x = (torch.randn((rows, cols), generator=g, device=dev) * 3).to(t)
    r = torch.randn((rows, cols), generator=g, device=dev).to(t) if res else None
    gamma = 1 + 0.2 * torch.randn((cols,), generator=g, device=dev)
    got = _ops().rmsnorm(x, gamma, EPS, residual=r)
    y, h = got if res else (got, None)
    s, ref = rms_ref(x, gamma, r)
    u = torch.finfo(t).eps / 2
    rel = rms_f32_error(sum_depth(cols)) + u
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    assert y.dtype == t
    assert ((y.double() - ref).abs() <= rel * ref.abs() * (1 + u) + tiny).all()
    if res:
        # one rounding of the exact sum's f32 value
        assert ((h.double() - s).abs() <= (u + 2.0 ** -24) * s.abs() * (1 + u) + tiny).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("rows,cols", RMS_SHAPES)
def test_rmsnorm_quantize(dev, rows, cols, res, dt):
    t, g = DTYPES[dt], _gen(rows * 37 + cols + res)
    x = (torch.randn((rows, cols), generator=g, device=dev) * 3).to(t)
    r = torch.randn((rows, cols), generator=g, device=dev).to(t) if res else None
    gamma = 1 + 0.2 * torch.randn((cols,), generator=g, device=dev)
    q, scale, *h = _ops().rmsnorm_quantize(x, gamma, EPS, residual=r)
    s, ref = rms_ref(x, gamma, r)
    amax = ref.abs().amax(1)
    rel = rms_f32_error(sum_depth(cols))
    # the scale: y's error and one division
    assert ((scale.double() - amax / 127).abs() <= (rel + 2.0 ** -23) * amax / 127).all()
    # the code: y / scale is at most 127, off by the errors of y, of the
    # largest y, of 127 / a and of the product, and rint moves it by a half
    off = (q.double() - ref * (127 / amax)[:, None]).abs()
    assert off.max() <= 0.5 + 127 * (2 * rel + 2.0 ** -22), off.max()
    assert (q.abs().amax(1) == 127).all()
    if res:
        u = torch.finfo(t).eps / 2
        assert ((h[0].double() - s).abs() <= (u + 2.0 ** -24) * s.abs() * (1 + u) + 1e-7).all()


@pytest.mark.parametrize("cols", [768, 4096, 771])
def test_rmsnorm_quantize_special_rows(dev, cols):
    x = torch.randn((7, cols), generator=_gen(1), device=dev)
    x[0] = 0
    x[1, 5] = math.nan
    x[2, cols - 1] = math.inf
    x[3] *= 1e-30  # mean(s^2) underflows: eps alone
    x[4] = 0
    x[4, 3] = 1e-41  # the row's only value, subnormal
    x[5, 0] = -math.inf
    gamma = torch.ones(cols, device=dev)
    q, scale = _ops().rmsnorm_quantize(x, gamma, EPS)
    assert scale[0] == 0 and (q[0] == 0).all()
    for r in (1, 2, 5):
        assert scale[r].isnan() and (q[r] == 0).all()
    assert q[3].abs().max() == 127 and q[4, 3] == 127 and (q[4].abs().sum() == 127)
    _, ref = rms_ref(x, gamma, None)
    off = (q[3].double() - ref[3] * 127 / ref[3].abs().max()).abs().max()
    assert off <= 0.5 + 127 * (2 * rms_f32_error(sum_depth(cols)) + 2.0 ** -22)
    y = _ops().dequantize_rows(q, scale, torch.float32)
    assert (y[0] == 0).all() and y[1].isnan().all()


@pytest.mark.parametrize("cols", [768, 2048, 770])
def test_rmsnorm_in_place(dev, cols):
    """sum may replace x or the residual, y may replace the other."""
    from jammi_b200 import _lib as L
    g = _gen(3)
    x = torch.randn((50, cols), generator=g, device=dev).bfloat16()
    r = torch.randn((50, cols), generator=g, device=dev).bfloat16()
    gamma = torch.rand((cols,), generator=g, device=dev)
    y, h = _ops().rmsnorm(x, gamma, EPS, residual=r)
    for a, b in ((x.clone(), r.clone()), (r.clone(), x.clone())):
        L.check(L.lib().jb_op_rmsnorm(a.data_ptr(), b.data_ptr(), gamma.data_ptr(), a.data_ptr(), b.data_ptr(), None,
                                      None, L.DT_BF16, 50, cols, EPS, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(a, h) and torch.equal(b, y)


def test_rmsnorm_unaligned_views(dev):
    """A base address that is not a multiple of 16 bytes gives the same rows."""
    g = _gen(4)
    flat = torch.randn((11 * 768 + 1,), generator=g, device=dev).half()
    gamma = torch.rand((769,), generator=g, device=dev)
    x = flat[1:].view(11, 768)
    want_q, want_s = _ops().rmsnorm_quantize(x.clone(), gamma[1:].clone(), EPS)
    q, s = _ops().rmsnorm_quantize(x, gamma[1:], EPS)
    # the two kernels sum in different orders
    assert ((s - want_s).abs() <= want_s * 2 * rms_f32_error(sum_depth(768))).all()
    assert (q.int() - want_q.int()).abs().max() <= 1


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (64, 768), (1001, 1000), (7, 4096), (0, 8)])
def test_dequantize_rows(dev, rows, cols, dt):
    g = _gen(rows + cols)
    q = torch.randint(-127, 128, (rows, cols), generator=g, device=dev, dtype=torch.int8)
    scale = torch.rand((rows,), generator=g, device=dev)
    y = _ops().dequantize_rows(q, scale, DTYPES[dt])
    assert torch.equal(y, (q.float() * scale[:, None]).to(DTYPES[dt]))


def test_rmsnorm_empty_and_refusals(dev):
    ops = _ops()
    gamma = torch.ones(8, device=dev)
    assert ops.rmsnorm(torch.empty((0, 8), device=dev), gamma, EPS).shape == (0, 8)
    q, s = ops.rmsnorm_quantize(torch.empty((0, 8), device=dev), gamma, EPS)
    assert q.shape == (0, 8) and s.shape == (0,)
    x = torch.ones((4, 8), device=dev)
    for bad in (dict(x=x.t()), dict(x=x[:, ::2]), dict(x=x.double()), dict(x=x.cpu()), dict(gamma=gamma[:7]),
                dict(gamma=gamma.half()), dict(gamma=gamma.cpu()), dict(residual=x[:3]), dict(residual=x.half()),
                dict(x=x[0])):
        a = dict(x=x, gamma=gamma, residual=None) | bad
        with pytest.raises(ValueError):
            ops.rmsnorm(a["x"], a["gamma"], EPS, residual=a["residual"])
        with pytest.raises(ValueError):
            ops.rmsnorm_quantize(a["x"], a["gamma"], EPS, residual=a["residual"])
