"""Projections in 8-bit floats with a scale for each block of 128, and what feeds them.

The functions take torch tensors as device memory (include/mlxr_fp8.h has the C entries):

- ``rms_norm`` norms rows of the residual stream, adds the residual on the way, and can leave its result
  in 8 bits;
- ``quantize_fp8`` rounds rows to 8 bits, ``quantize_fp8_weight`` weights;
- ``fp8_matmul`` multiplies rows with weights.

``Fp8Rows`` are rows [M, K] with their scales [M, ceil(K / 128)], ``Fp8Weight`` is a projection [N, K] with scales
[ceil(N / 128), ceil(K / 128)]; an element stands for itself times its scale.  ``Linear`` takes both.
"""
import collections
import ctypes

from . import paged, qgemm
from .paged import E4M3, _code, _on, _stream
from .qgemm import QGemmError

BLOCK = 128
_I64, _P, _I = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int

Fp8Rows = collections.namedtuple("Fp8Rows", "data scales")
Fp8Rows.__doc__ = """Rows in 8 bits: data [M, K] float8_e4m3fn, scales [M, ceil(K / 128)] float32, both contiguous."""

_SIGS = {
    "mlxr_rms_norm": (_I, [_I, _I, _P, _I, _I64, _P, _I64, _P, _I, ctypes.c_float, _P, _P, _I, _P, _P]),
    "mlxr_quantize_fp8": (_I, [_I, _I, _P, _I, _I64, _P, _P, _P]),
    "mlxr_quantize_fp8_weight": (_I, [_I, _I, _P, _I, _P, _P, _P]),
    "mlxr_fp8_matmul_workspace_size": (_I, [_I, _I, _I, _I, ctypes.POINTER(ctypes.c_size_t)]),
    "mlxr_fp8_matmul": (_I, [_I, _I, _I, _P, _P, _P, _P, _P, _I, _P, _I, _P, ctypes.c_size_t, _P]),
    "mlxr_fp8_linear_workspace_size": (_I, [_I, _I, _I, _I, ctypes.POINTER(ctypes.c_size_t)]),
    "mlxr_fp8_linear": (_I, [_I, _I, _I, _P, _I, _I64, _P, _P, _P, _I, _P, _I, _P, ctypes.c_size_t, _P]),
    "mlxr_fp8_test_force": (_I, [_I, _I]),
}
_bound = None


def _lib():
    global _bound
    if _bound is None:
        l = paged._lib()
        for name, (res, args) in _SIGS.items():
            f = getattr(l, name)
            f.restype, f.argtypes = res, args
        _bound = l
    return _bound


def _rows(x, index, what, stream):
    """x [..., K] as rows: (x or what takes its place, rows, K, row stride in elements); copied only where no stride says it."""
    shape = x.shape
    if not shape or x.get_device() != index or index < 0:
        raise QGemmError(-3, f"{what} must be [..., K] on a GPU")
    k = shape[-1]
    if k == 0:
        raise QGemmError(-3, f"{what}: rows must not be empty")
    if x.is_contiguous():
        return x, x.numel() // k, k, k
    x = x.reshape(-1, k) if stream is None else _on(stream, x.reshape, -1, k)
    st = x.stride()
    if (st[1] != 1 and k > 1) or st[0] < 0:
        x = _on(stream, x.clone, memory_format=paged._torch.contiguous_format)
        st = x.stride()
    return x, x.shape[0], k, st[0]


def _out8(m, k, like, stream):
    torch = paged._torch
    return Fp8Rows(_on(stream, torch.empty, (m, k), dtype=torch.float8_e4m3fn, device=like.device),
                   _on(stream, torch.empty, (m, -(-k // BLOCK)), dtype=torch.float32, device=like.device))


def rms_norm(x, weight=None, eps=1e-5, residual=None, quantize=False, out_dtype=None, stream=None):
    """s / sqrt(mean(s^2) + eps) * weight over the last dimension of s = x (+ residual), in fp32 (mlxr_rms_norm).

    x and ``residual``: one shape and dtype (float32, float16, bfloat16); ``weight`` [K] of any of them.  Returns the
    normed tensor in x's dtype (or ``out_dtype``), with ``quantize`` as ``Fp8Rows`` of [rows, K]; with a residual
    also the sum s in x's dtype: (normed, sum)."""
    lib = _bound or _lib()
    torch, codes, index, shape, xt = paged._torch, paged._x_codes, x.get_device(), x.shape, x.dtype
    x2, m, k, xs = _rows(x, index, "rms_norm: x", stream)
    dt = codes.get(xt)
    if dt is None:
        _code(codes, xt, "x")
    r2 = total = pr = pt = pw = None
    rs = wt = 0
    if residual is not None:
        if residual.shape != shape or residual.dtype is not xt:
            raise QGemmError(-3, "rms_norm: the residual must have x's shape and dtype and be on its GPU")
        r2, _, _, rs = _rows(residual, index, "rms_norm: the residual", stream)
        total = torch.empty_like(x, memory_format=torch.contiguous_format) if stream is None else \
            _on(stream, torch.empty, shape, dtype=xt, device=x.device)
        pr, pt = r2.data_ptr(), total.data_ptr()
    if weight is not None:
        if weight.shape != (k,) or weight.get_device() != index or not weight.is_contiguous():
            raise QGemmError(-3, f"rms_norm: weight must be a contiguous [{k}] tensor on GPU {index}")
        pw, wt = weight.data_ptr(), _code(codes, weight.dtype, "weight")
    ps = None
    if quantize:
        if out_dtype is not None:
            raise QGemmError(-1, "rms_norm: quantize and out_dtype exclude each other")
        out = _out8(m, k, x, stream)
        po, ot, ps = out.data.data_ptr(), E4M3, out.scales.data_ptr()
    else:
        if stream is None:
            out = torch.empty_like(x, dtype=out_dtype, memory_format=torch.contiguous_format)
        else:
            out = _on(stream, torch.empty, shape, dtype=out_dtype or xt, device=x.device)
        po, ot = out.data_ptr(), dt if out_dtype is None else _code(codes, out_dtype, "out")
    rc = lib.mlxr_rms_norm(m, k, x2.data_ptr(), dt, xs, pr, rs, pw, wt, eps, pt, po, ot, ps, _stream(stream, index))
    if rc:
        qgemm._check(rc)
    return out if total is None else (out, total)


def quantize_fp8(x, stream=None):
    """Rows x [..., K] in 8 bits, with a scale max|x| / 448 for each 128 elements (mlxr_quantize_fp8): ``Fp8Rows`` of
    [rows, K]."""
    lib, index = _bound or _lib(), x.get_device()
    dt = _code(paged._x_codes, x.dtype, "x")
    x2, m, k, xs = _rows(x, index, "quantize_fp8: x", stream)
    out = _out8(m, k, x, stream)
    rc = lib.mlxr_quantize_fp8(m, k, x2.data_ptr(), dt, xs, out[0].data_ptr(), out[1].data_ptr(), _stream(stream, index))
    if rc:
        qgemm._check(rc)
    return out


class Fp8Weight:
    """A projection in 8 bits: ``data`` [N, K] float8_e4m3fn, ``scales`` [ceil(N / 128), ceil(K / 128)] float32 (what
    block-scaled checkpoints hold), contiguous on one GPU; K a multiple of 16."""

    __slots__ = ("data", "scales", "N", "K")

    def __init__(self, data, scales):
        _lib()
        torch, shape = paged._torch, data.shape
        if len(shape) != 2 or shape[1] % 16 or shape[0] == 0 or shape[1] == 0:
            raise QGemmError(-3, "Fp8Weight: data must be [N, K], K a multiple of 16")
        if data.dtype is not torch.float8_e4m3fn or not data.is_contiguous() or data.get_device() < 0 or data.data_ptr() % 16:
            raise QGemmError(-1, "Fp8Weight: data must be contiguous float8_e4m3fn on a GPU, at a multiple of 16 bytes")
        want = (-(-shape[0] // BLOCK), -(-shape[1] // BLOCK))
        if scales.dtype is not torch.float32 or scales.shape != want or not scales.is_contiguous() or \
                scales.get_device() != data.get_device():
            raise QGemmError(-3, f"Fp8Weight: scales must be contiguous float32 {list(want)} on data's GPU")
        self.data, self.scales = data, scales
        self.N, self.K = shape


def quantize_fp8_weight(w, stream=None):
    """Weights w [N, K] in 8 bits with a scale max|w| / 448 for each 128 x 128 (mlxr_quantize_fp8_weight)."""
    lib = _lib()
    if w.dim() != 2 or w.get_device() < 0 or w.shape[1] % 16 or w.numel() == 0:
        raise QGemmError(-3, "quantize_fp8_weight: w must be [N, K] on a GPU, K a multiple of 16")
    torch, (n, k) = paged._torch, w.shape
    dt = _code(paged._x_codes, w.dtype, "w")
    w = w if w.is_contiguous() else _on(stream, w.contiguous)
    data = _on(stream, torch.empty, (n, k), dtype=torch.float8_e4m3fn, device=w.device)
    scales = _on(stream, torch.empty, (-(-n // BLOCK), -(-k // BLOCK)), dtype=torch.float32, device=w.device)
    qgemm._check(lib.mlxr_quantize_fp8_weight(n, k, w.data_ptr(), dt, data.data_ptr(), scales.data_ptr(),
                                              _stream(stream, w.get_device())))
    return Fp8Weight(data, scales)


def fp8_matmul(x, w, bias=None, out=None, out_dtype=None, stream=None):
    """x W^T (+ bias) with W an ``Fp8Weight`` [N, K] (mlxr_fp8_matmul, mlxr_fp8_linear).

    x: ``Fp8Rows`` [M, K], or [..., K] in float16, bfloat16 or float32, which is rounded by ``quantize_fp8`` first.  Returns
    [M, N] ([..., N]) in x's dtype (of ``Fp8Rows`` bfloat16), ``out_dtype``, or in ``out``."""
    lib, torch = _bound or _lib(), paged._torch
    if not isinstance(w, Fp8Weight):
        raise QGemmError(-1, "fp8_matmul: w must be an Fp8Weight")
    n, k, wd = w.N, w.K, w.data
    index = wd.get_device()
    rows = isinstance(x, Fp8Rows)
    if rows:
        data, scales = x
        lead, dtype = data.shape[:-1], torch.bfloat16
        if data.dim() != 2 or data.shape[1] != k:
            raise QGemmError(-3, f"Input shape must be [M, {k}]")
        m = data.shape[0]
        if data.dtype is not torch.float8_e4m3fn or scales.dtype is not torch.float32 or data.get_device() != index or \
                scales.get_device() != index or scales.shape != (m, -(-k // BLOCK)) or not data.is_contiguous() or \
                not scales.is_contiguous():
            raise QGemmError(-1, f"fp8_matmul: rows must be contiguous float8_e4m3fn [M, {k}] with float32 scales "
                                 f"[M, {-(-k // BLOCK)}] on GPU {index}")
        if data.data_ptr() % 16:
            data = _on(stream, data.clone)
    else:
        shape, dtype = x.shape, x.dtype
        if not shape or shape[-1] != k:
            raise QGemmError(-3, f"Input shape must be [..., {k}]")
        if x.get_device() != index:
            raise QGemmError(-1, "fp8_matmul: x must be on the weight's GPU")
        lead, xt = shape[:-1], _code(paged._x_codes, dtype, "x")
        data, m, _, stride = _rows(x, index, "fp8_matmul: x", stream)
    pb, bt = None, 0
    if bias is not None:
        if bias.shape != (n,) or bias.get_device() != index or not bias.is_contiguous():
            raise QGemmError(-3, "Bias shape must be [N]")
        pb, bt = bias.data_ptr(), _code(paged._x_codes, bias.dtype, "bias")
    if out is None:
        out = _on(stream, torch.empty, (*lead, n), dtype=out_dtype or dtype, device=wd.device)
    elif out.shape != (*lead, n) or not out.is_contiguous() or out.get_device() != index or out.data_ptr() % 16:
        raise QGemmError(-1, f"out must be a contiguous {[*lead, n]} tensor on GPU {index}, at a multiple of 16 bytes")
    yt = _code(paged._x_codes, out.dtype, "out")
    size = ctypes.c_size_t()
    rc = (lib.mlxr_fp8_matmul_workspace_size if rows else lib.mlxr_fp8_linear_workspace_size)(m, n, k, yt, ctypes.byref(size))
    if rc:
        qgemm._check(rc)
    nb = size.value
    ws = _on(stream, torch.empty, nb, dtype=torch.uint8, device=wd.device) if nb else None
    rest = (wd.data_ptr(), w.scales.data_ptr(), pb, bt, out.data_ptr(), yt, ws.data_ptr() if nb else None, nb,
            _stream(stream, index))
    if rows:
        rc = lib.mlxr_fp8_matmul(m, n, k, data.data_ptr(), scales.data_ptr(), *rest)
    else:
        rc = lib.mlxr_fp8_linear(m, n, k, data.data_ptr(), xt, stride, *rest)
    if rc:
        qgemm._check(rc)
    return out
