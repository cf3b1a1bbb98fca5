"""Single-op entry points over torch CUDA tensors (device pointers only).

Each function calls one C-ABI op of libjammi_b200.so on the current torch
stream.  They exist for op-level parity tests and for callers that compose
their own forward; the encoder forward itself runs entirely inside the
library (``jb_encode_text`` / ``jb_encode_image``).
"""
from __future__ import annotations

import torch

from . import _lib as L
from ._lib import check, lib

_DT = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16, torch.int8: L.DT_S8,
       torch.int32: L.DT_S32}


def _s(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _p(t):
    return 0 if t is None else t.data_ptr()


def _contig(*ts):
    for t in ts:
        if t is not None and not t.is_contiguous():
            raise ValueError("tensors must be contiguous")


def sync(device=None):
    """``jb_op_sync``: synchronise the current stream and raise on a device-side timeout."""
    check(lib().jb_op_sync(torch.cuda.current_stream(device).cuda_stream))


def linear(a: torch.Tensor, w: torch.Tensor, bias=None, residual=None, epilogue: int = L.EPI_NONE,
           out_dtype=None) -> torch.Tensor:
    """``epi(a @ w.T + bias)``; a [M, K], w [N, K] both f32 or both bf16."""
    _contig(a, w, bias, residual)
    M, K = a.shape
    N = w.shape[0]
    out_dtype = out_dtype or a.dtype
    c = torch.empty((M, N), dtype=out_dtype, device=a.device)
    check(lib().jb_op_linear(_p(a), _DT[a.dtype], _p(w), _DT[w.dtype], _p(bias), _p(residual),
                             _p(c), _DT[out_dtype], M, N, K, epilogue, _s(a)))
    return c


def linear_s8(aq: torch.Tensor, a_scale, wq: torch.Tensor, w_scale, bias=None, residual=None,
              epilogue: int = L.EPI_NONE, out_dtype=torch.int32) -> torch.Tensor:
    """int8 linear: s32 accumulators (out_dtype int32) or dequantised output."""
    _contig(aq, a_scale, wq, w_scale, bias, residual)
    M, K = aq.shape
    N = wq.shape[0]
    c = torch.empty((M, N), dtype=out_dtype, device=aq.device)
    check(lib().jb_op_linear_s8(_p(aq), _p(a_scale), _p(wq), _p(w_scale), _p(bias), _p(residual),
                                _p(c), _DT[out_dtype], M, N, K, epilogue, _s(aq)))
    return c


def quantize_rows(x: torch.Tensor, activation: int = L.EPI_NONE):
    """Per-row int8 of x, or of activation(x) rounded to x's dtype
    (activation EPI_GELU): returns (q int8 [R, C], scale f32 [R])."""
    _contig(x)
    R, C = x.shape
    q = torch.empty((R, C), dtype=torch.int8, device=x.device)
    s = torch.empty((R,), dtype=torch.float32, device=x.device)
    if activation == L.EPI_NONE:
        check(lib().jb_op_quantize_rows(_p(x), _DT[x.dtype], _p(q), _p(s), R, C, _s(x)))
    else:
        check(lib().jb_op_quantize_rows_act(_p(x), _DT[x.dtype], int(activation), _p(q), _p(s), R, C,
                                            _s(x)))
    return q, s


def layernorm(x: torch.Tensor, gamma, beta, eps: float, residual=None) -> torch.Tensor:
    _contig(x, gamma, beta, residual)
    R, C = x.shape
    y = torch.empty_like(x)
    check(lib().jb_op_layernorm(_p(x), _p(residual), _p(gamma), _p(beta), _p(y), _DT[x.dtype], R, C,
                                float(eps), _s(x)))
    return y


def _refuse(name, t, shape, dtypes, index):
    """The ValueError that says what ``_check`` found wrong."""
    if t is None:
        raise ValueError(f"{name} is missing")
    if not t.is_cuda or (index is not None and t.get_device() != index):
        where = "a CUDA device" if index is None else f"cuda:{index}"
        raise ValueError(f"{name} must be on {where}, not on {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    raise ValueError(f"{name}: {t.dtype} is not one of {', '.join(map(str, dtypes))}")


def _check(name, t, shape, dtypes, index=None):
    """Raises ValueError unless ``t`` is a contiguous CUDA tensor of ``shape`` (None: any) and one
    of ``dtypes``, on device ``index`` (None: any)."""
    if (t is None or t.dtype not in dtypes or not t.is_contiguous() or not t.is_cuda or
            (shape is not None and t.shape != shape) or (index is not None and t.get_device() != index)):
        _refuse(name, t, shape, dtypes, index)


_INT_MAX = 2 ** 31 - 1  # ctypes would pass what lies beyond it by its low 32 bits


def _too_large():
    raise ValueError("sizes must be below 2^31")


_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_F32 = (torch.float32,)

# The current stream's handle without building a Stream object (3 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_entry = {}


def _call(name, index, *args):
    """One library call on device ``index`` and its current torch stream."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(lib(), name)
    if _current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status)


def _rms_args(x, gamma, residual):
    """The device index and the shape of a valid call."""
    _check("x", x, None, _FLOATS)
    shape, index = x.shape, x.get_device()
    if len(shape) != 2:
        raise ValueError("x must be [rows, cols]")
    if shape[0] > _INT_MAX or shape[1] > _INT_MAX:
        _too_large()
    _check("gamma", gamma, shape[1:], _F32, index)
    if residual is not None:
        _check("residual", residual, shape, (x.dtype,), index)
    return index, shape


def rmsnorm(x: torch.Tensor, gamma: torch.Tensor, eps: float, residual=None):
    """RMS norm of ``x`` [R, C] (+ ``residual``): ``s * rsqrt(mean(s^2) + eps) * gamma`` with
    ``s = x + residual`` in f32.  Returns y, or (y, s rounded to x's dtype) when a residual is
    given.  x f32, bf16 or f16; gamma f32 [C]; C up to 2^30; eps >= 0 (a row of zeros with eps 0
    is NaN)."""
    index, (R, C) = _rms_args(x, gamma, residual)
    y = torch.empty_like(x)
    h = None if residual is None else torch.empty_like(x)
    if R:
        _call("jb_op_rmsnorm", index, x.data_ptr(), _p(residual), gamma.data_ptr(), _p(h), y.data_ptr(),
              None, None, _DT[x.dtype], R, C, eps)
    return y if h is None else (y, h)


def rmsnorm_quantize(x: torch.Tensor, gamma: torch.Tensor, eps: float, residual=None):
    """``rmsnorm`` with its output as per-row int8: (q int8 [R, C], scale f32 [R]) -- the
    activations of ``linear_s8`` -- and the rounded sum as a third value when a residual is given.
    The unrounded f32 norm is quantised; a row that is not finite has scale NaN and q 0."""
    index, (R, C) = _rms_args(x, gamma, residual)
    q = x.new_empty((R, C), dtype=torch.int8)
    scale = x.new_empty((R,), dtype=torch.float32)
    h = None if residual is None else torch.empty_like(x)
    if R:
        _call("jb_op_rmsnorm", index, x.data_ptr(), _p(residual), gamma.data_ptr(), _p(h), None,
              q.data_ptr(), scale.data_ptr(), _DT[x.dtype], R, C, eps)
    return (q, scale) if h is None else (q, scale, h)


def dequantize_rows(q: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values that int8 rows stand for: ``q[r, c] * scale[r]`` in ``dtype`` (f32, bf16, f16)."""
    _check("q", q, None, (torch.int8,))
    if q.dim() != 2:
        raise ValueError("q must be [rows, cols]")
    if max(q.shape) > _INT_MAX:
        _too_large()
    _check("scale", scale, q.shape[:1], _F32, q.get_device())
    if dtype not in _FLOATS:
        raise ValueError(f"{dtype} is not one of {', '.join(map(str, _FLOATS))}")
    y = q.new_empty(q.shape, dtype=dtype)
    if q.shape[0]:
        _call("jb_op_dequantize_rows", q.get_device(), q.data_ptr(), scale.data_ptr(), y.data_ptr(), _DT[dtype],
              q.shape[0], q.shape[1])
    return y


_U8 = (torch.uint8,)


def quantize_mxfp4(x: torch.Tensor):
    """MXFP4 form of ``x`` [R, C] (f32, bf16 or f16; C a multiple of 32): codes uint8 [R, C / 2],
    the even column in the low half, and scale bytes uint8 [ceil(R / 128), ceil(C / 128), 512] in
    the order ``linear_mxfp4`` reads (``jb_op_quantize_mxfp4``)."""
    _check("x", x, None, _FLOATS)
    shape = x.shape
    if len(shape) != 2 or shape[1] % 32 or not shape[1]:
        raise ValueError("x must be [rows, cols] with cols a multiple of 32")
    R, C = shape
    if R > _INT_MAX or C > _INT_MAX:
        _too_large()
    q = x.new_empty((R, C // 2), dtype=torch.uint8)
    scale = q.new_empty(((R + 127) // 128, (C + 127) // 128, 512))
    if R:
        _call("jb_op_quantize_mxfp4", x.get_device(), x.data_ptr(), _DT[x.dtype], q.data_ptr(), scale.data_ptr(), R, C)
    return q, scale


def _check_mxfp4(name, q, scale, index=None):
    """Raises ValueError unless q and scale are MXFP4 rows on device ``index`` (None: any); their
    device, rows and columns."""
    _check(name, q, None, _U8, index)
    shape, index = q.shape, q.get_device()
    if len(shape) != 2 or shape[1] % 16 or not shape[1]:
        raise ValueError(f"{name} must be [rows, cols / 2] with cols a multiple of 32")
    R, C = shape[0], 2 * shape[1]
    if R > _INT_MAX or C > _INT_MAX:
        _too_large()
    tiles = ((R + 127) // 128, (C + 127) // 128, 512)
    if (scale is None or scale.shape != tiles or scale.dtype is not torch.uint8 or not scale.is_contiguous() or
            scale.get_device() != index):
        _refuse(name + "'s scale", scale, tiles, _U8, index)
    return index, R, C


def dequantize_mxfp4(q: torch.Tensor, scale: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The values [R, C] that ``quantize_mxfp4``'s codes and scales stand for, in ``dtype``."""
    index, R, C = _check_mxfp4("q", q, scale)
    if dtype not in _FLOATS:
        raise ValueError(f"{dtype} is not one of {', '.join(map(str, _FLOATS))}")
    y = q.new_empty((R, C), dtype=dtype)
    if R:
        _call("jb_op_dequantize_mxfp4", index, q.data_ptr(), scale.data_ptr(), y.data_ptr(), _DT[dtype], R, C)
    return y


def linear_mxfp4(aq: torch.Tensor, a_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, bias=None,
                 residual=None, epilogue: int = L.EPI_NONE, out_dtype=torch.bfloat16) -> torch.Tensor:
    """``epi(a @ w.T + bias)`` [M, N] of MXFP4 activations [M, K] and weights [N, K], both as
    ``quantize_mxfp4`` returns them; N a multiple of 8, ``out_dtype`` f32, bf16 or f16 (the
    residual's too), bias f32 [N]."""
    index, M, K = _check_mxfp4("aq", aq, a_scale)
    _, N, columns = _check_mxfp4("wq", wq, w_scale, index)
    if columns != K:
        raise ValueError("aq and wq must have the same number of columns")
    if out_dtype not in _FLOATS:
        raise ValueError(f"{out_dtype} is not one of {', '.join(map(str, _FLOATS))}")
    if bias is not None:
        _check("bias", bias, (N,), _F32, index)
    if residual is not None:
        _check("residual", residual, (M, N), (out_dtype,), index)
    if epilogue > _INT_MAX or epilogue < -_INT_MAX:
        _too_large()
    c = aq.new_empty((M, N), dtype=out_dtype)
    if M:
        _call("jb_op_linear_mxfp4", index, aq.data_ptr(), a_scale.data_ptr(), wq.data_ptr(), w_scale.data_ptr(),
              _p(bias), _p(residual), c.data_ptr(), _DT[out_dtype], M, N, K, epilogue)
    return c


def attention(qkv: torch.Tensor, cu_seqlens: torch.Tensor, heads: int, max_len: int,
              causal: bool = False, tma: bool = False) -> torch.Tensor:
    """qkv [T, 3*heads*d] packed rows, cu_seqlens int32 [B+1] -> ctx [T, heads*d]
    (``causal``: query i sees keys j <= i of its row; ``tma``: pass the row
    count, which selects the model forwards' TMA / tcgen05 kernels)."""
    _contig(qkv, cu_seqlens)
    T, three_h = qkv.shape
    H = three_h // 3
    ctx = torch.empty((T, H), dtype=qkv.dtype, device=qkv.device)
    if tma:
        check(lib().jb_op_attention_rows(_p(qkv), _p(cu_seqlens), _p(ctx), _DT[qkv.dtype],
                                         cu_seqlens.numel() - 1, heads, H // heads, max_len, T,
                                         1 if causal else 0, _s(qkv)))
        return ctx
    fn = lib().jb_op_attention_causal if causal else lib().jb_op_attention
    check(fn(_p(qkv), _p(cu_seqlens), _p(ctx), _DT[qkv.dtype], cu_seqlens.numel() - 1, heads,
             H // heads, max_len, _s(qkv)))
    return ctx


def attention_window(qkv: torch.Tensor, cu_seqlens: torch.Tensor, heads: int, max_len: int, left: int, right: int,
                     sinks: int = 0, kv_heads=None) -> torch.Tensor:
    """Windowed attention over packed rows: qkv [T, (heads + 2 * kv_heads) * d] (Q|K|V), cu_seqlens
    int32 [B+1] -> ctx [T, heads*d].  Query i of a row sees key j iff ``j <= i + right and
    (j >= i - left or j < sinks)``; ``kv_heads`` None means ``heads``; d 8, 16, 32, 64 or 128.
    ``max_len`` bounds the rows' lengths: of a longer row the first ``max_len`` tokens are a row.
    What no row holds, behind ``cu_seqlens[-1]`` for instance, is left unwritten."""
    kv_heads = heads if kv_heads is None else kv_heads
    _check("qkv", qkv, None, _FLOATS)
    _check("cu_seqlens", cu_seqlens, None, (torch.int32,), qkv.get_device())
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError("heads must be a positive multiple of kv_heads")
    shape, offsets = qkv.shape, cu_seqlens.shape
    if len(shape) != 2 or not shape[1] or shape[1] % (heads + 2 * kv_heads):
        raise ValueError("qkv must be [tokens, (heads + 2 * kv_heads) * head_dim]")
    if len(offsets) != 1 or not offsets[0]:
        raise ValueError("cu_seqlens must be [batch + 1]")
    T, d = shape[0], shape[1] // (heads + 2 * kv_heads)
    if (max(T, d, offsets[0], max_len, left, right, sinks) > _INT_MAX or
            min(max_len, left, right, sinks) < -_INT_MAX):
        _too_large()
    ctx = qkv.new_empty((T, heads * d))
    _call("jb_op_attention_window", qkv.get_device(), qkv.data_ptr(), cu_seqlens.data_ptr(), ctx.data_ptr(),
          _DT[qkv.dtype], offsets[0] - 1, heads, kv_heads, d, max_len, T, left, right, sinks)
    return ctx


def pool_normalize(hidden: torch.Tensor, cu_seqlens: torch.Tensor, pooling: int = L.POOL_MEAN):
    _contig(hidden, cu_seqlens)
    T, H = hidden.shape
    B = cu_seqlens.numel() - 1
    out = torch.empty((B, H), dtype=torch.float32, device=hidden.device)
    check(lib().jb_op_pool_normalize(_p(hidden), _DT[hidden.dtype], _p(cu_seqlens), _p(out), B, H,
                                     pooling, _s(hidden)))
    return out


def preprocess_rgb8(images, target: int, mean, std, device="cuda") -> torch.Tensor:
    """RGB8 ``[h, w, 3]`` arrays -> f32 [B, 3, target, target] on the device
    (``jb_op_preprocess_rgb8``: white square pad, Catmull-Rom resize, normalise)."""
    from .encoders import pack_rgb8
    buf, offs, ws, hs = pack_rgb8(images)
    dev = torch.device(device)
    d_buf = torch.from_numpy(buf).to(dev)
    d_off = torch.from_numpy(offs).to(dev)
    d_w = torch.from_numpy(ws).to(dev)
    d_h = torch.from_numpy(hs).to(dev)
    m = torch.tensor(list(mean), dtype=torch.float32)
    s = torch.tensor(list(std), dtype=torch.float32)
    out = torch.empty((len(images), 3, target, target), dtype=torch.float32, device=dev)
    max_side = int(max(max(int(a), int(b)) for a, b in zip(ws, hs))) if len(images) else 1
    check(lib().jb_op_preprocess_rgb8(_p(d_buf), _p(d_off), _p(d_w), _p(d_h), len(images), max_side,
                                      target, m.data_ptr(), s.data_ptr(), _p(out), _s(out)))
    return out


def set_attention_tcgen05(on: bool):
    """``jb_set_attention_tcgen05``: every bf16 head-dim-64 row on the tcgen05
    attention kernel (process-wide; on by default), or off: the mma.sync kernel."""
    lib().jb_set_attention_tcgen05(1 if on else 0)


def wait_flag(flag: torch.Tensor, expect: int, limit_ms: int):
    """``jb_op_wait_flag``: a bounded device-side wait until flag[0] == expect;
    on expiry the next ``sync`` raises JbError (JB_ERR_TIMEOUT)."""
    if flag.dtype != torch.int32 or flag.numel() < 1:
        raise ValueError("flag must be an int32 tensor")
    check(lib().jb_op_wait_flag(_p(flag), int(expect), int(limit_ms), _s(flag)))


THRESHOLD_KINDS = {"mean": 0, "median": 1}


def fit_binary_threshold(vectors: torch.Tensor, kind: str = "median") -> torch.Tensor:
    """Per-dimension threshold tau of a Binary sidecar over the first
    min(rows, 100000) rows of f32 ``vectors`` [rows, dim] ("mean" or "median")."""
    _contig(vectors)
    rows, dim = vectors.shape
    tau = torch.empty(dim, dtype=torch.float32, device=vectors.device)
    check(lib().jb_op_fit_binary_threshold(_p(vectors), rows, dim, THRESHOLD_KINDS[kind], _p(tau), _s(vectors)))
    return tau


def pack_threshold_bits(vectors: torch.Tensor, tau: torch.Tensor) -> torch.Tensor:
    """uint8 [rows, ceil(dim / 8)]: bit i = vectors[:, i] > tau[i], LSB-first."""
    _contig(vectors, tau)
    rows, dim = vectors.shape
    out = torch.empty((rows, (dim + 7) // 8), dtype=torch.uint8, device=vectors.device)
    check(lib().jb_op_pack_threshold_bits(_p(vectors), rows, dim, _p(tau), _p(out), _s(vectors)))
    return out


def exact_search(corpus: torch.Tensor, queries: torch.Tensor, k: int, tie_rank=None):
    """Exact cosine search: (idx int64 [q, min(k, n)], dist f32 [q, min(k, n)])
    in ascending (distance, tie rank) order; ``tie_rank`` int32/uint32 [n]
    (distinct) or None for row order.  Synchronises to surface input errors."""
    _contig(corpus, queries, tie_rank)
    n, dim = corpus.shape
    nq = queries.shape[0]
    scratch = torch.empty((nq, n), dtype=torch.float32, device=corpus.device)
    idx = torch.empty((nq, k), dtype=torch.int64, device=corpus.device)
    dist = torch.empty((nq, k), dtype=torch.float32, device=corpus.device)
    check(lib().jb_op_exact_search(_p(corpus), n, dim, _p(tie_rank), _p(queries), nq, k, _p(scratch),
                                   _p(idx), _p(dist), _s(corpus)))
    sync(corpus.device)
    kk = min(k, n)
    return idx[:, :kk], dist[:, :kk]
