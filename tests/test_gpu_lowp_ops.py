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
              (17, 4096), (5, 4100), (3, 16384), (2, 16392), (2, 20001), (700, 16400), (3, 32768), (2, 32776), (1300, 201), (30, 1501), (5, 4095), (3, 256), (3, 1023), (7, 2049), (70, 225), (33, 226), (40, 993), (40, 994), (9, 2017), (9, 2018), (11, 4065), (11, 4066)]


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


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("cols", [8, 200, 201, 768, 771, 1024, 1536, 4096, 4100, 16384, 20001, 32768, 40000])
def test_rmsnorm_of_rows_whose_squares_leave_f32(dev, cols, res, dt):
    """Magnitudes whose squares overflow, underflow or lose bits, with eps of the same size or 0;
    ordinary rows between them keep their values."""
    t, g, ops = DTYPES[dt], _gen(cols + res), _ops()
    size = torch.tensor([1.0, 1e25, 1.0, 3e37, 1e18, 2e19, 1e-25, 1.0, 1e-38, 1e-19, 1e-22], device=dev)
    x = torch.randn((size.numel(), cols), generator=g, device=dev).clamp(-4, 4)
    x[:, 0] = 1.0  # no row is 0 throughout
    x = (x * size[:, None]).to(t)
    r = (torch.randn((size.numel(), cols), generator=g, device=dev).clamp(-4, 4) * size[:, None]).to(t) if res else None
    gamma = 1 + 0.2 * torch.rand((cols,), generator=g, device=dev)
    u, rel = torch.finfo(t).eps / 2, rms_f32_error(sum_depth(cols))
    s = x.double() + (r.double() if res else 0)
    assert s.abs().max() < 3.4e38
    for eps in (0.0, 1e-6, 1e-37, 1e-43):
        ref = s / torch.sqrt(s.square().mean(1, keepdim=True) + torch.tensor(eps).double().item()) * gamma.double()
        y = ops.rmsnorm(x, gamma, eps, residual=r)
        y = (y[0] if res else y).double()
        # a result below f32's normal range is off by units of its last place
        off = ((y - ref).abs() - (rel + u) * ref.abs() * (1 + u) - 2.0 ** -130).amax(1)
        assert (off <= 0).all(), (eps, off)
        q, scale = ops.rmsnorm_quantize(x, gamma, eps, residual=r)[:2]
        amax = ref.abs().amax(1)
        assert ((scale.double() - amax / 127).abs() <= (rel + 2.0 ** -23) * amax / 127 + 2.0 ** -148).all(), eps
        big = amax > 1e-30  # (scale itself keeps its bits)
        code = (q.double() - ref * (127 / amax)[:, None])[big].abs()
        assert code.max() <= 0.5 + 127 * (2 * rel + 2.0 ** -22), (eps, code.max())


def test_rmsnorm_of_zeros_without_eps(dev):
    """0 / 0: NaN, as the formula has it; with a NaN or an infinity in the row too."""
    for cols in (64, 771, 4096, 5001):
        x = torch.zeros((4, cols), device=dev)
        x[1, 3], x[2, 3], x[3, 3] = math.nan, math.inf, 2.0
        gamma = torch.ones(cols, device=dev)
        y = _ops().rmsnorm(x, gamma, 0.0)
        assert y[0].isnan().all() and y[1].isnan().all()
        assert y[2, 3].isnan() and (y[2, :3] == 0).all() and (y[2, 4:] == 0).all()
        assert y[3].isfinite().all()
        q, scale = _ops().rmsnorm_quantize(x, gamma, 0.0)
        assert scale[:3].isnan().all() and (q[:3] == 0).all() and q[3, 3] == 127


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


# ── MXFP4 ───────────────────────────────────────────────────────────────────

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def mx_ref(x):
    """(values, codes, scale bytes) of x's MXFP4 form in float64, block by block of 32."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    powers = torch.tensor([2.0 ** p for p in range(-149, 128)], dtype=torch.float64, device=x.device)
    floor = torch.searchsorted(powers, top, right=True) - 1 - 149
    e = torch.where(top > 0, floor - 2, torch.full_like(floor, -127)).clamp(-127, 127)
    bad = ~torch.isfinite(b).all(-1)
    z = b.abs() * torch.exp2(-e.double())[..., None]
    gap = (z[..., None] - torch.tensor(E2M1, dtype=torch.float64, device=x.device)).abs()
    near = gap.amin(-1, keepdim=True)
    even = torch.tensor([i % 2 == 0 for i in range(8)], device=x.device)
    hit = gap == near
    code = torch.where((hit & even).any(-1), (hit & even).int().argmax(-1), hit.int().argmax(-1))
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    v = torch.tensor(E2M1, dtype=torch.float64, device=x.device)[code] * torch.exp2(e.double())[..., None]
    v = torch.where(bad[..., None], torch.full_like(v, math.nan), torch.where(torch.signbit(b), -v, v))
    neg = torch.signbit(b) & ~bad[..., None]
    byte = torch.where(bad, torch.full_like(e, 255), e + 127)
    return v.reshape(x.shape), (code + 8 * neg).reshape(x.shape), byte


def scale_bytes(scale, rows, cols):
    """The scale tiles as [rows, cols / 32], and what pads them."""
    rt, ct, _ = scale.shape
    full = scale.reshape(rt, ct, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, ct * 4).long()
    pad = full.clone()
    pad[:rows, :cols // 32] = 0
    return full[:rows, :cols // 32], pad


MX_SHAPES = [(1, 32), (1, 64), (12, 768), (127, 96), (128, 256), (129, 288), (300, 1024), (1000, 160), (40, 4096)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,cols", MX_SHAPES)
def test_quantize_mxfp4(dev, rows, cols, dt):
    g = _gen(rows + cols)
    x = torch.randn((rows, cols), generator=g, device=dev)
    x *= torch.exp2(torch.randint(-12, 12, (rows, cols // 32, 1), generator=g, device=dev).float()).expand(
        -1, -1, 32).reshape(rows, cols)
    x = x.to(DTYPES[dt])
    q, scale = _ops().quantize_mxfp4(x)
    v, code, byte = mx_ref(x)
    got = torch.stack((q & 15, q >> 4), -1).reshape(rows, cols)
    assert torch.equal(got.long(), code.long())
    sb, pad = scale_bytes(scale, rows, cols)
    assert torch.equal(sb, byte.long()) and not pad.any()
    for t in DTYPES.values():
        assert torch.equal(_ops().dequantize_mxfp4(q, scale, t), v.to(t))


def test_quantize_mxfp4_borders(dev):
    """Every border between two codes, its neighbours, saturation, tiny and huge blocks, zeros,
    and blocks that are not finite."""
    x = torch.zeros((12, 64), device=dev)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device=dev)
    x[0, 0], x[0, 1:9], x[0, 9:17] = 7.75, mids, -mids  # scale 2^0; 7.75 saturates at 6
    x[1, 0], x[1, 1:9] = 4.0, torch.nextafter(mids, torch.tensor(9.0, device=dev)).clamp(max=6.0)
    x[2, 0], x[2, 1:9] = -4.0, torch.nextafter(mids, torch.tensor(0.0, device=dev))
    x[3] = 2.0 ** -126
    x[4, 3] = 1e-41
    x[5, 40] = torch.finfo(torch.float32).max
    x[5, 41] = -1e-30
    x[6, 2] = math.nan
    x[7, 63] = -math.inf
    x[8, 31], x[8, 32] = -0.0, 2.0 ** 127
    x[9] = -6.0
    x[10, ::2] = 3.0
    q, scale = _ops().quantize_mxfp4(x)
    v, code, byte = mx_ref(x)
    got = torch.stack((q & 15, q >> 4), -1).reshape(12, 64)
    assert torch.equal(got.long(), code.long())
    assert torch.equal(scale_bytes(scale, 12, 64)[0], byte.long())
    y = _ops().dequantize_mxfp4(q, scale, torch.float32)
    assert torch.equal(torch.nan_to_num(y, nan=-1.0), torch.nan_to_num(v.float(), nan=-1.0))
    assert y[6, :32].isnan().all() and not y[6, 32:].isnan().any()


def gelu64(z):
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


LIN_SHAPES = [(1, 8, 32), (12, 2304, 768), (3, 72, 64), (127, 200, 96), (129, 264, 160), (64, 1024, 4096), (300, 1536, 384),
              (2000, 1160, 288), (5000, 768, 768), (4100, 1000, 1056), (2850, 1000, 1056)]


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("M,N,K", LIN_SHAPES)
def test_linear_mxfp4_places(dev, M, N, K, out):
    """One non-zero activation per row: every output is one weight exactly, which
    shows each code and each scale byte in its place."""
    ops, g = _ops(), _gen(M + N + K)
    x = torch.zeros((M, K), device=dev)
    at = torch.randint(0, K, (M,), generator=g, device=dev)
    at[0], at[-1] = 0, K - 1
    x[torch.arange(M, device=dev), at] = torch.exp2(torch.randint(-8, 8, (M,), generator=g, device=dev).float())
    w = torch.randn((N, K), generator=g, device=dev)
    w *= torch.exp2(torch.randint(-6, 6, (N, K // 32), generator=g, device=dev).float()).repeat_interleave(32, 1)
    aq, wq = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    c = ops.linear_mxfp4(*aq, *wq, out_dtype=DTYPES[out])
    ops.sync()
    # |x| <= 128 and |w| <= 2^10: inside f16; a power of two times an e2m1 value: no rounding in any type
    want = x[torch.arange(M, device=dev), at][:, None].double() * mx_ref(w)[0][:, at].T
    assert torch.equal(c.double(), want.to(DTYPES[out]).double())


def linear_check(c, a, w, bias, res, epi, K):
    """Float64 of the quantised operands.  The accumulator: the products of a
    block are exact, and each of the K / 16 partial sums is off by at most two
    units of 2^-24 of the terms' magnitudes (truncated alignment counted);
    then bias, activation (1e-6 max(1, |z|)), residual and the output's own
    rounding u."""
    z = a @ w.T
    mag = a.abs() @ w.abs().T
    if bias is not None:
        z = z + bias.double()
        mag = mag + bias.double().abs()
    off = (K / 16 * 2 + 4) * 2.0 ** -24 * mag
    if epi == "gelu":
        z, off = gelu64(z), 1.13 * off + 1e-6 * z.abs().clamp(min=1)
    elif epi == "quick_gelu":
        z, off = z * torch.sigmoid(1.702 * z), 1.1 * off + 1e-6 * z.abs().clamp(min=1)
    elif epi == "residual":
        z = z + res.double()
        off = off + 2.0 ** -23 * res.double().abs()
    u = torch.finfo(c.dtype).eps / 2
    tiny = torch.finfo(c.dtype).smallest_normal * torch.finfo(c.dtype).eps
    err = (c.double() - z).abs()
    ok = err <= off * (1 + u) + u * z.abs() + tiny
    assert ok.all(), (err / (off + u * z.abs() + tiny)).max()


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("epi", ["none", "gelu", "quick_gelu", "residual"])
@pytest.mark.parametrize("M,N,K", LIN_SHAPES)
def test_linear_mxfp4(dev, M, N, K, epi, out):
    from jammi_b200 import _lib as L
    ops, g, t = _ops(), _gen(M * 3 + N + K), DTYPES[out]
    a = torch.randn((M, K), generator=g, device=dev)
    w = torch.randn((N, K), generator=g, device=dev) / math.sqrt(K)
    bias = torch.randn((N,), generator=g, device=dev) if epi != "quick_gelu" else None
    res = torch.randn((M, N), generator=g, device=dev).to(t) if epi == "residual" else None
    aq, wq = ops.quantize_mxfp4(a), ops.quantize_mxfp4(w)
    codes = {"none": L.EPI_NONE, "gelu": L.EPI_GELU, "quick_gelu": L.EPI_QUICK_GELU, "residual": L.EPI_RESIDUAL}
    c = ops.linear_mxfp4(*aq, *wq, bias=bias, residual=res, epilogue=codes[epi], out_dtype=t)
    ops.sync()
    linear_check(c, mx_ref(a)[0], mx_ref(w)[0], bias, res, epi, K)


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("epi", ["none", "gelu", "residual"])
@pytest.mark.parametrize("M,N,K", [(20001, 1544, 288), (9000, 4096, 64), (40000, 392, 672)])
def test_linear_mxfp4_accumulators_handed_back(dev, M, N, K, epi, out):
    """Six and more tiles per CTA or pair of CTAs: each of the two accumulators is written again behind
    the reads of both CTAs' epilogues, with one set of bits at every run."""
    from jammi_b200 import _lib as L
    ops, g, t = _ops(), _gen(M + N + K), DTYPES[out]
    a = torch.randn((M, K), generator=g, device=dev)
    w = torch.randn((N, K), generator=g, device=dev) / math.sqrt(K)
    bias = torch.randn((N,), generator=g, device=dev)
    res = torch.randn((M, N), generator=g, device=dev).to(t) if epi == "residual" else None
    aq, wq = ops.quantize_mxfp4(a), ops.quantize_mxfp4(w)
    codes = {"none": L.EPI_NONE, "gelu": L.EPI_GELU, "residual": L.EPI_RESIDUAL}
    runs = [ops.linear_mxfp4(*aq, *wq, bias=bias, residual=res, epilogue=codes[epi], out_dtype=t) for _ in range(6)]
    ops.sync()
    assert all(torch.equal(r, runs[0]) for r in runs)
    aw, ww = ops.dequantize_mxfp4(*aq, torch.float32).double(), ops.dequantize_mxfp4(*wq, torch.float32).double()
    for lo in range(0, M, 4000):
        linear_check(runs[0][lo:lo + 4000], aw[lo:lo + 4000], ww, bias, None if res is None else res[lo:lo + 4000], epi, K)


@pytest.mark.parametrize("epi", ["gelu", "quick_gelu"])
def test_linear_mxfp4_activations_over_their_range(dev, epi):
    """Weights of zero: the bias is what the activation gets.  Its error is the 1e-6 max(1, |z|) that
    the framework's other linears keep to."""
    from jammi_b200 import _lib as L
    z = torch.cat([torch.linspace(-20, 20, 8192), torch.tensor([0.0, -0.0, 1e30, -1e30, 3e38, -3e38, 1e-30, -1e-30]),
                   torch.tensor([math.inf, -math.inf, math.nan, 40.0, -40.0, 90.0, -90.0, 1e4])]).to(dev)
    aq = _ops().quantize_mxfp4(torch.ones((2, 32), device=dev))
    wq = _ops().quantize_mxfp4(torch.zeros((z.numel(), 32), device=dev))
    c = _ops().linear_mxfp4(*aq, *wq, bias=z, epilogue=L.EPI_GELU if epi == "gelu" else L.EPI_QUICK_GELU,
                            out_dtype=torch.float32)
    _ops().sync()
    assert torch.equal(torch.nan_to_num(c[0], nan=-7.0), torch.nan_to_num(c[1], nan=-7.0))
    z, y = z.double(), c[0].double()
    assert y[z.isnan()].isnan().all() and (y[z == math.inf] == math.inf).all()
    fin = z.isfinite()
    want = (gelu64(z) if epi == "gelu" else z * torch.sigmoid(1.702 * z))[fin]
    assert ((y[fin] - want).abs() <= 1e-6 * z[fin].abs().clamp(min=1)).all()


@pytest.mark.parametrize("out", DTYPES)
def test_linear_mxfp4_gelu_error_where_it_is_stated(dev, out):
    """|error| <= 3e-7 before the output's own rounding on |x| <= 8, and 2^-9 of the value down to
    x = -6.15 (where it is 1e-9)."""
    from jammi_b200 import _lib as L
    z = torch.linspace(-8, 8, 64000).to(dev)
    aq = _ops().quantize_mxfp4(torch.ones((1, 32), device=dev))
    wq = _ops().quantize_mxfp4(torch.zeros((z.numel(), 32), device=dev))
    c = _ops().linear_mxfp4(*aq, *wq, bias=z, epilogue=L.EPI_GELU, out_dtype=DTYPES[out])[0]
    _ops().sync()
    u = torch.finfo(c.dtype).eps / 2 if out != "f32" else 0  # f32's own is in the 3e-7
    tiny = torch.finfo(c.dtype).smallest_normal * torch.finfo(c.dtype).eps
    want = z.double() * torch.special.ndtr(z.double())
    err = (c.double() - want).abs()
    assert (err <= 3e-7 * (1 + u) + u * want.abs() + tiny).all(), err.max()
    near = (z >= -6.15) & (z <= 0)
    assert (err <= ((2.0 ** -9 * (1 + u) + u) * want.abs() + tiny))[near].all()


def test_linear_mxfp4_residual_in_place_and_nan_rows(dev):
    from jammi_b200 import _lib as L
    ops, g = _ops(), _gen(8)
    M, N, K = 333, 328, 128
    a, w = torch.randn((M, K), generator=g, device=dev), torch.randn((N, K), generator=g, device=dev)
    a[7, 40] = math.nan
    w[9, 100] = math.inf
    aq, wq = ops.quantize_mxfp4(a), ops.quantize_mxfp4(w)
    res = torch.randn((M, N), generator=g, device=dev).bfloat16()
    want = ops.linear_mxfp4(*aq, *wq, residual=res, epilogue=L.EPI_RESIDUAL)
    L.check(L.lib().jb_op_linear_mxfp4(aq[0].data_ptr(), aq[1].data_ptr(), wq[0].data_ptr(), wq[1].data_ptr(), None,
                                       res.data_ptr(), res.data_ptr(), L.DT_BF16, M, N, K, L.EPI_RESIDUAL,
                                       torch.cuda.current_stream().cuda_stream))
    ops.sync()
    assert torch.equal(torch.nan_to_num(res.float(), nan=1e9), torch.nan_to_num(want.float(), nan=1e9))
    nan = want.isnan()
    assert nan[7].all() and nan[:, 9].all() and nan.sum() == M + N - 1


def test_mxfp4_refusals(dev):
    ops = _ops()
    x = torch.ones((4, 64), device=dev)
    for bad in (x[:, :48].contiguous(), x.t(), x.double(), x.cpu(), x[0], x[:, :0]):
        with pytest.raises(ValueError):
            ops.quantize_mxfp4(bad)
    q, s = ops.quantize_mxfp4(x)
    w, ws = ops.quantize_mxfp4(torch.ones((16, 64), device=dev))
    odd, odds = ops.quantize_mxfp4(torch.ones((15, 64), device=dev))
    short, shorts = ops.quantize_mxfp4(torch.ones((16, 32), device=dev))
    from jammi_b200 import _lib as L
    from jammi_b200._lib import JbError
    for args, kw in (((q, s, short, shorts), {}), ((q, s[0], w, ws), {}), ((q.cpu(), s, w, ws), {}),
                     ((q, s, w, ws), dict(bias=torch.ones(15, device=dev))),
                     ((q, s, w, ws), dict(bias=torch.ones(16, device=dev).half())),
                     ((q, s, w, ws), dict(residual=torch.ones((4, 16), device=dev), epilogue=L.EPI_RESIDUAL)),
                     ((q, s, w, ws), dict(out_dtype=torch.int32)), ((q.int(), s, w, ws), {})):
        with pytest.raises(ValueError):
            ops.linear_mxfp4(*args, **kw)
    for args, kw in (((q, s, odd, odds), {}), ((q, s, w, ws), dict(epilogue=L.EPI_RESIDUAL)), ((q, s, w, ws), dict(epilogue=7)),
                     ((q, s, w, ws), dict(residual=torch.ones((4, 16), device=dev).bfloat16()))):
        with pytest.raises(JbError) as e:
            ops.linear_mxfp4(*args, **kw)
        assert e.value.status == L.ERR_INVALID
    with pytest.raises(ValueError):
        ops.dequantize_mxfp4(q, s, torch.int8)
    none = ops.quantize_mxfp4(torch.empty((0, 64), device=dev))
    assert none[0].shape == (0, 32) and none[1].shape == (0, 1, 512)
    assert ops.dequantize_mxfp4(*none).shape == (0, 64)
    assert ops.linear_mxfp4(*none, w, ws).shape == (0, 16)


# ── windowed attention ──────────────────────────────────────────────────────

def window_ref(qkv, lens, h, hk, left, right, sinks, hide=None):
    """Float64, row by row; also sum_j p_j |v_j| / sum_j p_j and max |q k| / sqrt(d) for the error bound.
    ``hide`` [tokens]: keys with p = 0."""
    d = qkv.shape[1] // (h + 2 * hk)
    x = qkv.double()
    out, mag = torch.zeros((qkv.shape[0], h * d), dtype=torch.float64, device=qkv.device), None
    mag, top, at = out.clone(), 0.0, 0
    for n in lens:
        if n:
            q, k, v = x[at:at + n].split([h * d, hk * d, hk * d], 1)
            q = q.reshape(n, h, d).transpose(0, 1)
            k = k.reshape(n, hk, d).transpose(0, 1).repeat_interleave(h // hk, 0)
            v = v.reshape(n, hk, d).transpose(0, 1).repeat_interleave(h // hk, 0)
            i, j = torch.arange(n, device=x.device)[:, None], torch.arange(n, device=x.device)[None]
            seen = (j <= i + right) & ((j >= i - left) | (j < sinks))
            if hide is not None:
                seen = seen & ~hide[at:at + n]
            s = (q @ k.transpose(1, 2) / math.sqrt(d)).masked_fill(~seen, -math.inf)
            top = max(top, (q.abs() @ k.abs().transpose(1, 2)).max().item() / math.sqrt(d))
            p = torch.softmax(s, -1)
            out[at:at + n] = (p @ v).transpose(0, 1).reshape(n, h * d)
            mag[at:at + n] = (p @ v.abs()).transpose(0, 1).reshape(n, h * d)
        at += n
    return out, mag, top


def window_check(got, qkv, lens, h, hk, left, right, sinks, tensor_cores, first=0, hide=None):
    """An output is sum p v / sum p.  Scores: d products and sums in f32, off by (d + 4) 2^-24 of
    sum |q k| / sqrt(d) =: top, so p is off by that share (and 2^-21 for the exponential and its
    argument's rounding at |argument| <= 2 top log2 e).  On tensor cores each p is also rounded to
    the rows' 16-bit type (u), against an unrounded sum.  The sums over up to n keys in f32 add
    n 2^-24.  All of it is a share of sum p |v| / sum p; the store rounds once."""
    ref, mag, top = window_ref(qkv, lens, h, hk, left, right, sinks, hide)
    d = qkv.shape[1] // (h + 2 * hk)
    u = torch.finfo(qkv.dtype).eps / 2
    share = 2 * ((d + 8) * 2.0 ** -24 * top + 2.0 ** -21) + max(lens, default=0) * 2.0 ** -23 + (u if tensor_cores else 0)
    T = sum(lens)
    err = (got.double() - ref)[:T].abs()
    assert got.dtype == qkv.dtype and got.shape == ref.shape
    bound = share * mag[:T] + u * (ref[:T].abs() + share * mag[:T]) + torch.finfo(qkv.dtype).smallest_normal * 2 * u
    assert (err <= bound)[first:].all(), (err / bound)[first:].max().item()


WINDOWS = [(64, 64, 0), (64, 64, 1), (0, 0, 0), (0, 0, 3), (128, 0, 0), (255, 0, 4), (17, 200, 5), (300, 5, 130),
           (2 ** 31 - 1, 2 ** 31 - 1, 0), (2 ** 31 - 1, 0, 2 ** 31 - 1), (1, 1, 700)]
LENS = [[1], [12], [0, 5, 0, 0, 129, 64, 1, 127, 128, 0], [300, 1, 257, 512, 40], [1000]]


def run_window(dev, lens, h, hk, d, t, left, right, sinks, seed, extra=3, scale=1.0):
    g = _gen(seed)
    T = sum(lens)
    qkv = (torch.randn((T + extra, (h + 2 * hk) * d), generator=g, device=dev) * scale).to(t)
    qkv[T:] = math.nan  # rows behind the last sequence
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    got = _ops().attention_window(qkv, cu, h, max(lens), left, right, sinks=sinks, kv_heads=hk)
    _ops().sync()
    return qkv, got


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
def test_attention_window_64(dev, lens, left, right, sinks, dt):
    t = DTYPES[dt]
    qkv, got = run_window(dev, lens, 3, 3, 64, t, left, right, sinks, sum(lens) + left % 1000 + sinks % 1000)
    window_check(got, qkv, lens, 3, 3, left, right, sinks, t != torch.float32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(4, 2, 64), (6, 1, 64), (2, 2, 128), (4, 1, 128), (3, 3, 32), (4, 2, 32), (4, 2, 16), (5, 5, 8)])
@pytest.mark.parametrize("left,right,sinks", [(64, 64, 1), (100, 0, 4), (2 ** 31 - 1, 2 ** 31 - 1, 0)])
def test_attention_window_heads(dev, h, hk, d, left, right, sinks, dt):
    t, lens = DTYPES[dt], [200, 3, 0, 129, 391]
    qkv, got = run_window(dev, lens, h, hk, d, t, left, right, sinks, h * 100 + d)
    window_check(got, qkv, lens, h, hk, left, right, sinks, t != torch.float32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(12, 12, 64), (6, 3, 64), (8, 4, 128), (12, 12, 32)])
@pytest.mark.parametrize("left,right,sinks", [(64, 64, 1), (64, 64, 0), (300, 20, 4)])
@pytest.mark.parametrize("batch,lo,hi", [(256, 32, 256), (40, 0, 700), (2100, 1, 20)])
def test_attention_window_many_rows(dev, batch, lo, hi, left, right, sinks, h, hk, d, dt):
    """More query blocks than any GPU has slots for: every slot works through several, of mixed
    sizes; 2100 rows pass the kernel's table of row offsets."""
    t = DTYPES[dt]
    lens = torch.randint(lo, hi + 1, (batch,), generator=torch.Generator().manual_seed(batch)).tolist()
    qkv, got = run_window(dev, lens, h, hk, d, t, left, right, sinks, batch + left + d)
    window_check(got, qkv, lens, h, hk, left, right, sinks, t != torch.float32)


@pytest.mark.parametrize("batch", [1, 31, 33, 767, 768, 769, 1536, 1537, 2048, 2049])
@pytest.mark.parametrize("longest", [1, 30, 200])
def test_attention_window_batches_around_the_offset_scan(dev, batch, longest):
    """Row offsets are scanned 768 at a time, up to 2048 rows."""
    lens = torch.randint(0, longest + 1, (batch,), generator=torch.Generator().manual_seed(batch + longest)).tolist()
    lens[-1] = longest
    qkv, got = run_window(dev, lens, 2, 1, 64, torch.bfloat16, 20, 20, 2, batch)
    window_check(got, qkv, lens, 2, 1, 20, 20, 2, True)


@pytest.mark.parametrize("batch,longest", [(2049, 3), (4095, 9), (4097, 0), (30000, 5), (300000, 1), (6145, 200), (2000000, 3)])
@pytest.mark.parametrize("left,right,sinks", [(2, 1, 1), (10 ** 9, 10 ** 9, 0)])
def test_attention_window_batches_of_any_size(dev, batch, longest, left, right, sinks):
    """More rows than the table of offsets, a max_len that says nothing, empty rows among them and
    one long one: the work follows the tokens, not batch * max_len."""
    lens = torch.randint(0, longest + 1, (batch,), generator=torch.Generator().manual_seed(batch))
    lens[batch // 2], lens[0], lens[-1] = 1000, 0, 0
    T, d, t = int(lens.sum()), 64, torch.bfloat16
    qkv = torch.randn((T + 2, 3 * d), generator=_gen(batch), device=dev).to(t)
    cu = torch.zeros(batch + 1, dtype=torch.int32)
    cu[1:] = lens.cumsum(0)
    got = _ops().attention_window(qkv, cu.to(dev), 1, 2 ** 31 - 1, left, right, sinks=sinks)
    _ops().sync()
    kept = lens[lens > 0]
    some = torch.randperm(kept.numel(), generator=torch.Generator().manual_seed(1))[:400]
    at = torch.cat([torch.zeros(1, dtype=torch.long), kept.cumsum(0)])
    picks = sorted(set(some.tolist()) | {0, kept.numel() - 1, int(kept.argmax())})
    index = torch.cat([torch.arange(at[i], at[i + 1]) for i in picks]).to(dev)
    window_check(got[index], qkv[index], [int(kept[i]) for i in picks], 1, 1, left, right, sinks, True)
    if longest == 1:  # rows of one token give their value
        one = torch.repeat_interleave(kept == 1, kept).to(dev)
        assert torch.equal(got[:T][one], qkv[:T][one][:, 2 * d:])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_attention_window_long_rows_and_large_scores(dev, dt):
    t, lens = DTYPES[dt], [5000, 17, 2049]
    qkv, got = run_window(dev, lens, 2, 2, 64, t, 64, 64, 2, 5, scale=3.0)
    window_check(got, qkv, lens, 2, 2, 64, 64, 2, t != torch.float32)


def test_attention_window_unbounded_is_full_attention(dev):
    """The framework's own full and causal attention are the window's limits."""
    ops, lens = _ops(), [130, 64, 1, 300]
    qkv, got = run_window(dev, lens, 4, 4, 64, torch.float32, 10 ** 6, 10 ** 6, 0, 11, extra=0)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    # both f32: scores differ by the order of 64 products
    assert (ops.attention(qkv, cu, 4, 300) - got).abs().max() <= 2e-5
    _, causal = run_window(dev, lens, 4, 4, 64, torch.float32, 10 ** 6, 0, 0, 11, extra=0)
    assert (ops.attention(qkv, cu, 4, 300, causal=True) - causal).abs().max() <= 2e-5


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attention_window_leaves_other_rows(dev, dt):
    """ctx rows behind the last sequence keep their bytes; NaN in keys that the window hides does
    not reach the output."""
    from jammi_b200 import _lib as L
    t, g = DTYPES[dt], _gen(2)
    n, h, d = 400, 2, 64
    qkv = torch.randn((n + 70, 3 * h * d), generator=g, device=dev).to(t)
    clean = qkv.clone()
    qkv[:, h * d:][n:] = math.inf
    qkv[5:100, h * d:] = math.nan  # hidden from queries >= 200 by a window of 64
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    ctx = torch.full((n + 70, h * d), 7.0, device=dev, dtype=t)
    L.check(L.lib().jb_op_attention_window(qkv.data_ptr(), cu.data_ptr(), ctx.data_ptr(), L.DT_BF16 if dt == "bf16" else
                                           L.DT_F32, 1, h, h, d, n, n + 70, 64, 64, 2,
                                           torch.cuda.current_stream().cuda_stream))
    _ops().sync()
    assert (ctx[n:] == 7.0).all()
    # the hidden keys may be anything: the float64 reference of the clean rows
    # is the value for queries 200 and up.  Rows that share a block of queries
    # with NaN keys are computed again with unrounded p, the others with p
    # rounded to 16 bits: two values, each inside the bound, which counts that
    # rounding once (so bits cannot be compared)
    clean[n:] = 0
    full = torch.where(torch.arange(n + 70, device=dev)[:, None] < n, ctx, torch.zeros_like(ctx))
    window_check(full, clean, [n], h, h, 64, 64, 2, dt == "bf16", first=200)
    assert ctx[5:100].isnan().all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("left,right", [(64, 64), (300, 20)])
@pytest.mark.parametrize("gap", [60, 100, 123, 125, 127, 129, 200, 2000, -100, -2000])
@pytest.mark.parametrize("at,of", [(0, 2), (1, 2), (16, 32), (5, 32), (48, 500), (200, 500)])
def test_attention_window_scores_far_apart(dev, gap, at, of, left, right, dt):
    """A query's scores with some of the keys that it sees, or that its neighbours see, lie ``gap``
    powers of two above the others."""
    t, n, d, g = DTYPES[dt], 500, 64, _gen(gap)
    qkv = torch.zeros((n, 3 * d), device=dev)
    qkv[:, 0] = 8.0
    qkv[at::of, d] = gap * math.log(2)  # 8 k / sqrt(64) log2(e) = gap
    qkv[:, 2 * d:] = torch.randn((n, d), generator=g, device=dev)
    qkv = qkv.to(t)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = _ops().attention_window(qkv, cu, 1, n, left, right)
    _ops().sync()
    window_check(got, qkv, [n], 1, 1, left, right, 0, t != torch.float32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("left,right,sinks", [(64, 64, 0), (300, 20, 3), (10 ** 6, 10 ** 6, 0)])
@pytest.mark.parametrize("gap", [10, 14, 18, 22])
def test_attention_window_columns_of_small_weights(dev, gap, left, right, sinks, d, dt):
    """Some keys outweigh the others by 2^gap, and half of the columns are 0 in their values: what is
    left there are the small weights, whose bits P has to keep."""
    t, n, g = DTYPES[dt], 700, _gen(gap + d)
    qkv = torch.zeros((n, 3 * d), device=dev)
    qkv[:, 0] = math.sqrt(d)
    qkv[:, 1:4] = torch.randn((n, 3), generator=g, device=dev)
    qkv[:, d + 1:d + 4] = torch.randn((n, 3), generator=g, device=dev)
    heavy = torch.arange(n, device=dev) % 50 == 20
    qkv[heavy, d] = gap * math.log(2)  # sqrt(d) k / sqrt(d) log2(e) = gap
    qkv[:, 2 * d:] = torch.randn((n, d), generator=g, device=dev) * 500
    qkv[heavy, 2 * d:2 * d + d // 2] = 0
    qkv = qkv.to(t)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = _ops().attention_window(qkv, cu, 1, n, left, right, sinks=sinks)
    _ops().sync()
    window_check(got, qkv, [n], 1, 1, left, right, sinks, t != torch.float32)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("left,right", [(3, 0), (100, 0), (2, 2)])
@pytest.mark.parametrize("gap", [20, 40, 70, 95, 110])
@pytest.mark.parametrize("small", [-20, -40, -75, -100])
def test_attention_window_small_values_beside_hidden_scores(dev, small, gap, left, right, dt):
    """Keys that some of the queries do not see score ``gap`` powers of two above the others, and the
    values are around 2^small (half of the columns; the others around 1): products of weights relative
    to such a score and the values leave f32's range, the outputs do not."""
    t, n, d, g = DTYPES[dt], 500, 64, _gen(gap - small)
    qkv = torch.zeros((n, 3 * d), device=dev)
    qkv[:, 0] = 8.0
    qkv[:, 1:4] = torch.randn((n, 3), generator=g, device=dev)
    qkv[:, d + 1:d + 4] = torch.randn((n, 3), generator=g, device=dev)
    qkv[16::32, d] = gap * math.log(2)  # 8 k / sqrt(64) log2(e) = gap
    qkv[:, 2 * d:] = torch.randn((n, d), generator=g, device=dev)
    qkv[:, 2 * d:2 * d + 32] *= 2.0 ** small
    qkv = qkv.to(t)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = _ops().attention_window(qkv, cu, 1, n, left, right)
    _ops().sync()
    window_check(got, qkv, [n], 1, 1, left, right, 0, t != torch.float32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("left,right,sinks", [(64, 64, 0), (300, 300, 0), (300, 20, 3)])
def test_attention_window_scores_of_minus_infinity(dev, left, right, sinks, d, dt):
    """Keys at minus infinity, a query's own and whole leading blocks among them, weigh nothing."""
    t, n, g = DTYPES[dt], 700, _gen(d + left)
    qkv = torch.randn((n, 3 * d), generator=g, device=dev)
    hide = torch.arange(n, device=dev) % 2 == 1
    if left == 300 and not sinks:
        hide[:200] = True
    root = math.sqrt(d)
    qkv[:, 0] = root / 2
    qkv[:, d] = torch.where(hide, -math.inf, -28.0)  # visible keys: scores near -14
    qkv = qkv.to(t)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = _ops().attention_window(qkv, cu, 1, n, left, right, sinks=sinks)
    _ops().sync()
    clean = qkv.clone()
    clean[hide, d] = -28.0
    window_check(got, clean, [n], 1, 1, left, right, sinks, t != torch.float32, hide=hide)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("left,right,sinks", [(64, 64, 1), (300, 20, 3), (10 ** 6, 0, 0)])
def test_attention_window_infinite_value(dev, left, right, sinks, dt):
    """An infinite value reaches the queries that see it, in its column, and nothing else."""
    t, n, d, key, g = DTYPES[dt], 900, 64, 400, _gen(left)
    qkv = torch.randn((n, 3 * d), generator=g, device=dev).to(t)
    clean = qkv.clone()
    qkv[key, 2 * d + 5] = math.inf
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = _ops().attention_window(qkv, cu, 1, n, left, right, sinks=sinks)
    _ops().sync()
    i = torch.arange(n, device=dev)
    sees = (key <= i + right) & (key >= i - left)
    assert (got[sees, 5] == math.inf).all()
    got[sees, 5] = window_ref(clean, [n], 1, 1, left, right, sinks)[0].to(t)[sees, 5]
    window_check(got, clean, [n], 1, 1, left, right, sinks, t != torch.float32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("h,hk,d", [(4, 2, 64), (2, 2, 32), (2, 1, 128)])
@pytest.mark.parametrize("left,right,sinks", [(10 ** 6, 0, 0), (64, 64, 2), (300, 0, 5), (0, 10 ** 6, 0)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_attention_window_channel_that_is_not_finite(dev, bad, left, right, sinks, h, hk, d, dt):
    """A channel of V that is not finite in some of the tokens: the queries that see one of them have it
    in that column alone, the others (in blocks that hold such a token, too) keep every column."""
    t, g, lens = DTYPES[dt], _gen(d + left % 97), [2600, 5, 333]
    n = sum(lens)
    qkv = torch.randn((n, (h + 2 * hk) * d), generator=g, device=dev).to(t)
    clean = qkv.clone()
    tokens = torch.tensor([900, 1500, 2599, 2602, 2605 + 200], device=dev)
    col = (h + hk) * d + 7  # of the first key / value head
    qkv[tokens, col] = bad
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    got = _ops().attention_window(qkv, cu, h, max(lens), left, right, sinks=sinks, kv_heads=hk)
    _ops().sync()
    ref = window_ref(clean, lens, h, hk, left, right, sinks)[0].to(t)
    start = torch.repeat_interleave(cu[:-1].long(), cu.diff().long())
    end = torch.repeat_interleave(cu[1:].long(), cu.diff().long())
    i = torch.arange(n, device=dev)[:, None]
    sees = ((tokens >= start[:, None]) & (tokens < end[:, None]) & (tokens <= i + right) &
            ((tokens >= i - left) | (tokens - start[:, None] < sinks))).any(1)
    assert sees.any() and not sees.all()
    for head in range(h // hk):  # the query heads of that key / value head
        c = got[:, head * d + 7]
        assert (c[sees].isnan() if math.isnan(bad) else c[sees] == bad).all()
        c[sees] = ref[sees, head * d + 7]
    window_check(got, clean, lens, h, hk, left, right, sinks, t != torch.float32)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_attention_window_long_causal_row_with_an_infinite_channel(dev, dt):
    """Every query block has hidden values that are not finite, every query tens of thousands of visible
    keys: nothing waits for the columns that are computed again."""
    t, n, d = DTYPES[dt], 60000, 64
    qkv = torch.randn((n, 3 * d), generator=_gen(6), device=dev).to(t)
    clean = qkv.clone()
    qkv[:, 2 * d + 9] = math.inf
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = _ops().attention_window(qkv, cu, 1, n, n, 0)
    _ops().sync()
    assert (got[:, 9] == math.inf).all()
    got[:, 9] = 0
    assert got.isfinite().all()
    rows = torch.tensor([0, 1, 127, 128, 5000, 31999, n - 129, n - 2, n - 1], device=dev)
    u = torch.finfo(t).eps / 2
    x = clean.double()
    for r in rows.tolist():
        s = x[:r + 1, d:2 * d] @ x[r, :d] / math.sqrt(d)
        p = torch.softmax(s, 0)
        top = (x[:r + 1, d:2 * d].abs() @ x[r, :d].abs()).max().item() / math.sqrt(d)
        want, mag = p @ x[:r + 1, 2 * d:], p @ x[:r + 1, 2 * d:].abs()
        share = 2 * ((d + 8) * 2.0 ** -24 * top + 2.0 ** -21) + (r + 1) * 2.0 ** -23 + u  # as window_check
        err = (got[r].double() - want).abs()
        err[9] = 0
        assert (err <= share * mag + u * (want.abs() + share * mag)).all(), (r, err.max())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("cu", [[0, 300, 300, 900], [0, 5, -7, 20, 2 ** 31 - 1], [600, 20, -(2 ** 31), 40, 900]])
def test_attention_window_offsets_that_do_not_fit(dev, cu, dt):
    """Rows longer than max_len are cut; offsets that go back, are negative or lie behind the
    buffer make rows of what is inside it."""
    t, n, d, longest = DTYPES[dt], 800, 64, 250
    qkv = torch.randn((n, 3 * d), generator=_gen(len(cu)), device=dev).to(t)
    ctx = torch.full((n, d), 7.0, device=dev, dtype=t)
    from jammi_b200 import _lib as L
    offsets = torch.tensor(cu, dtype=torch.int32, device=dev)
    L.check(L.lib().jb_op_attention_window(qkv.data_ptr(), offsets.data_ptr(), ctx.data_ptr(), {"f32": L.DT_F32, "bf16": L.DT_BF16,
                                           "f16": L.DT_F16}[dt], len(cu) - 1, 1, 1, d, longest, n, 64, 64, 1,
                                           torch.cuda.current_stream().cuda_stream))
    _ops().sync()
    rows = [(a, min(b, n, a + longest)) for a, b in zip(cu, cu[1:]) if a >= 0]
    written = torch.zeros(n, dtype=torch.bool, device=dev)
    for a, b in rows:
        if b > a:
            written[a:b] = True
            window_check(ctx[a:b], qkv[a:b], [b - a], 1, 1, 64, 64, 1, t != torch.float32)
    assert (ctx[~written] == 7.0).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_attention_window_values_of_nan_alone(dev, dt):
    """No query waits long for a long row without one finite value."""
    n, d = 40000, 64
    qkv = torch.randn((n, 3 * d), generator=_gen(1), device=dev).to(DTYPES[dt])
    qkv[:, 2 * d:] = math.nan
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    got = _ops().attention_window(qkv, cu, 1, n, n, n)
    _ops().sync()
    assert got.isnan().all()


def test_attention_window_refusals(dev):
    from jammi_b200 import _lib as L
    from jammi_b200._lib import JbError
    ops = _ops()
    qkv, cu = torch.ones((10, 3 * 64), device=dev), torch.tensor([0, 10], dtype=torch.int32, device=dev)
    for a in ((qkv.t(), cu, 1), (qkv.cpu(), cu, 1), (qkv, cu.cpu(), 1), (qkv, cu.long(), 1), (qkv, cu, 5), (qkv, cu, 0),
              (qkv.double(), cu, 1), (qkv[0], cu, 1), (qkv, cu[:0], 1), (qkv, cu.reshape(1, 2), 1)):
        with pytest.raises(ValueError):
            ops.attention_window(*a, 10, 4, 4)
    with pytest.raises(ValueError):
        ops.attention_window(qkv, cu, 2, 10, 4, 4, kv_heads=3)
    for kw in (dict(left=-1), dict(right=-1), dict(sinks=-2), dict(max_len=-1)):
        a = dict(max_len=10, left=4, right=4, sinks=0) | kw
        with pytest.raises(JbError) as e:
            ops.attention_window(qkv, cu, 1, a["max_len"], a["left"], a["right"], sinks=a["sinks"])
        assert e.value.status == L.ERR_INVALID
    with pytest.raises(JbError):
        ops.attention_window(torch.ones((4, 3 * 24), device=dev), cu, 1, 4, 1, 1)  # head_dim 24
    assert ops.attention_window(qkv[:0], cu[:1], 1, 0, 4, 4).shape == (0, 64)


def test_sizes_beyond_32_bits_are_refused(dev):
    """What ctypes would cut to its low 32 bits."""
    ops = _ops()
    qkv, cu = torch.ones((10, 3 * 64), device=dev), torch.tensor([0, 10], dtype=torch.int32, device=dev)
    for i in range(4):
        for beyond in (2 ** 31, 2 ** 32, 2 ** 40 + 3, -2 ** 32):
            a = [10, 4, 4, 0]
            a[i] = beyond
            with pytest.raises(ValueError):
                ops.attention_window(qkv, cu, 1, *a[:3], sinks=a[3])
    long = torch.empty((2 ** 31 + 8, 1), dtype=torch.int8, device=dev)
    one = torch.ones((1,), device=dev)
    with pytest.raises(ValueError):
        ops.rmsnorm(long.bfloat16(), one, EPS)
    with pytest.raises(ValueError):
        ops.dequantize_rows(long, one)
    q, s = ops.quantize_mxfp4(torch.ones((4, 64), device=dev))
    w, ws = ops.quantize_mxfp4(torch.ones((16, 64), device=dev))
    with pytest.raises(ValueError):
        ops.linear_mxfp4(q, s, w, ws, epilogue=2 ** 32)
    assert ops.attention_window(qkv, cu, 1, 10, 2 ** 31 - 1, 2 ** 31 - 1, sinks=2 ** 31 - 1).isfinite().all()


# ── together ────────────────────────────────────────────────────────────────

class Layer:
    """A pre-norm encoder layer at low precision: x + r -> RMS norm -> int8 rows -> int8 QKV linear ->
    windowed attention -> MXFP4 output linear added to the sum -> RMS norm -> MXFP4 FFN with GELU."""

    H, HEADS, F = 256, 4, 1024

    def __init__(self, seed):
        ops, g = _ops(), _gen(seed)
        H, F = self.H, self.F
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.g1, self.g2 = 1 + 0.1 * rand(H), 1 + 0.1 * rand(H)
        self.qkv = ops.quantize_rows(rand(3 * H, H) / math.sqrt(H))
        self.out = ops.quantize_mxfp4(rand(H, H) / math.sqrt(H))
        self.up = ops.quantize_mxfp4(rand(F, H) / math.sqrt(H))
        self.down = ops.quantize_mxfp4(rand(H, F) / math.sqrt(F))
        self.b_up, self.b_down = 0.1 * rand(F), 0.1 * rand(H)

    def __call__(self, x, r, cu, longest):
        from jammi_b200 import _lib as L
        ops = _ops()
        q, s, h = ops.rmsnorm_quantize(x, self.g1, EPS, residual=r)
        qkv = ops.linear_s8(q, s, *self.qkv, out_dtype=torch.bfloat16)
        ctx = ops.attention_window(qkv, cu, self.HEADS, longest, 64, 64, sinks=1)
        a = ops.linear_mxfp4(*ops.quantize_mxfp4(ctx), *self.out, residual=h, epilogue=L.EPI_RESIDUAL)
        y = ops.rmsnorm(a, self.g2, EPS)
        up = ops.linear_mxfp4(*ops.quantize_mxfp4(y), *self.up, bias=self.b_up, epilogue=L.EPI_GELU)
        z = ops.linear_mxfp4(*ops.quantize_mxfp4(up), *self.down, bias=self.b_down, residual=a, epilogue=L.EPI_RESIDUAL)
        return dict(h=h, q=q, s=s, qkv=qkv, ctx=ctx, a=a, y=y, up=up, z=z)


def layer_inputs(lens, seed):
    g = _gen(seed)
    T = sum(lens)
    x = torch.randn((T, Layer.H), generator=g, device="cuda").bfloat16()
    r = torch.randn((T, Layer.H), generator=g, device="cuda").bfloat16()
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    return x, r, cu


LAYER_LENS = [70, 1, 300, 0, 12, 256]


def test_layer_each_stage_on_what_it_got(dev):
    """The whole run, every stage held to float64 of its own operator on the tensors that reached it."""
    layer, (x, r, cu) = Layer(1), layer_inputs(LAYER_LENS, 2)
    t = layer(x, r, cu, max(LAYER_LENS))
    _ops().sync()
    s, ref = rms_ref(x, layer.g1, r)
    amax, rel = ref.abs().amax(1), rms_f32_error(sum_depth(Layer.H))
    assert ((t["q"].double() - ref * (127 / amax)[:, None]).abs() <= 0.5 + 127 * (2 * rel + 2.0 ** -22)).all()
    acc = t["q"].double() @ layer.qkv[0].double().T * t["s"].double()[:, None] * layer.qkv[1].double()
    assert ((t["qkv"].double() - acc).abs() <= (2.0 ** -8 + 2.0 ** -22) * acc.abs()).all()
    window_check(t["ctx"], t["qkv"], LAYER_LENS, Layer.HEADS, Layer.HEADS, 64, 64, 1, True)
    value = lambda m: _ops().dequantize_mxfp4(*m, torch.float32).double()  # noqa: E731
    linear_check(t["a"], mx_ref(t["ctx"])[0], value(layer.out), None, t["h"], "residual", Layer.H)
    linear_check(t["up"], mx_ref(t["y"])[0], value(layer.up), layer.b_up, None, "gelu", Layer.H)
    linear_check(t["z"], mx_ref(t["up"])[0], value(layer.down), layer.b_down, t["a"], "residual", Layer.F)


def test_layer_captured_replayed_and_on_two_streams(dev):
    """Two captured runs replayed at once on two streams, on new inputs copied into theirs, give the
    eager runs' bits: nothing is kept from one call for the next, and nothing is shared."""
    layer, lens = Layer(3), LAYER_LENS
    runs = []
    for k in range(2):
        static = layer_inputs(lens, 10 + k)
        layer(*static, max(lens))  # warm-up: attributes, the error flag
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = layer(*static, max(lens))
        runs.append((static, stream, graph, out))
    for turn in range(3):
        fresh = [layer_inputs(lens, 100 + 10 * turn + k) for k in range(2)]
        want = [layer(*f, max(lens)) for f in fresh]
        torch.cuda.synchronize()
        for (static, stream, graph, out), f in zip(runs, fresh):
            with torch.cuda.stream(stream):
                for a, b in zip(static, f):
                    a.copy_(b)
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), w in zip(runs, want):
            for k in w:
                assert torch.equal(out[k], w[k]), k
    _ops().sync()
    del runs


def test_ops_run_on_the_current_stream(dev):
    """A call waits for the work before it on its own stream only."""
    ops = _ops()
    x = torch.zeros((4096, 1024), device=dev).bfloat16()
    gamma = torch.ones(1024, device=dev)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            x.add_(1.0)
        q, s = ops.rmsnorm_quantize(x, gamma, EPS)
        m = ops.quantize_mxfp4(x)
        y = ops.dequantize_mxfp4(*m, torch.float32)
    side.synchronize()
    assert (q == 127).all() and (y == 16.0).all()  # 20 / 4 = 5 ties to the even code 6: 4 * 4


def test_window_two_calls_at_once_on_two_streams(dev):
    ops = _ops()
    lens = torch.randint(32, 257, (200,), generator=torch.Generator().manual_seed(1)).tolist()
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    qs = [torch.randn((sum(lens), 3 * 12 * 64), generator=_gen(k), device=dev).bfloat16() for k in range(2)]
    want = [ops.attention_window(q, cu, 12, 256, 64, 64, sinks=1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for _ in range(5):
        for st, q in zip(streams, qs):
            with torch.cuda.stream(st):
                got.append(ops.attention_window(q, cu, 12, 256, 64, 64, sinks=1))
    torch.cuda.synchronize()
    ops.sync()
    assert all(torch.equal(g, want[k % 2]) for k, g in enumerate(got))


def test_kernels_of_every_kind_at_once_on_four_streams(dev):
    """Kernels that take an SM's tensor memory, alone and by pairs of SMs, beside each other and beside the
    framework's own linear: each gives the bits that it gives alone."""
    ops, g = _ops(), _gen(21)
    lens = torch.randint(1, 400, (300,), generator=torch.Generator().manual_seed(2)).tolist()
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    T = sum(lens)
    wide, narrow = (torch.randn((T, 3 * 4 * d), generator=g, device=dev).bfloat16() for d in (128, 32))
    a, w = ops.quantize_mxfp4(torch.randn((20001, 288), generator=g, device=dev)), ops.quantize_mxfp4(
        torch.randn((1544, 288), generator=g, device=dev))
    few, deep = ops.quantize_mxfp4(torch.randn((50, 4096), generator=g, device=dev)), ops.quantize_mxfp4(
        torch.randn((1024, 4096), generator=g, device=dev))
    x, m = torch.randn((4000, 768), generator=g, device=dev).bfloat16(), torch.randn((768, 768), generator=g, device=dev).bfloat16()
    calls = [[lambda: ops.attention_window(wide, cu, 4, 400, 64, 64, sinks=1), lambda: ops.linear_mxfp4(*a, *w)],
             [lambda: ops.linear_mxfp4(*a, *w), lambda: ops.attention_window(narrow, cu, 4, 400, 300, 0)],
             [lambda: ops.linear(x, m), lambda: ops.linear_mxfp4(*few, *deep)],
             [lambda: ops.attention_window(narrow, cu, 4, 400, 20, 20), lambda: ops.rmsnorm(x, torch.ones(768, device=dev), EPS)]]
    want = [[f() for f in stream] for stream in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], []
    for _ in range(12):
        for st, fs, ws in zip(streams, calls, want):
            with torch.cuda.stream(st):
                got += [(f(), w) for f, w in zip(fs, ws)]
    torch.cuda.synchronize()
    ops.sync()
    for have, one in got:
        assert torch.equal(have[:T] if have.shape[0] == T else have, one)
