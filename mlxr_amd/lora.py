"""Low-rank adapters of many requests beside shared (quantized) projections.

``lora_apply`` adds each token's own adapter to the outputs of projections that read the same
input (include/mlxr_lora.h): ``out[t] = y[t] + scale * (x[t] A^T) B^T`` with the A, B and scale of
adapter ``ids[t]``.  ``LoraBank`` keeps a projection's adapters in the layout that it takes.
"""
import ctypes
import struct

from . import paged, qgemm
from .paged import _code, _on, _stream, _vector
from .qgemm import QGemmError

MAX_ADAPTERS, MAX_RANK = 4096, 128
_P, _I = ctypes.c_void_p, ctypes.c_int


class Item(ctypes.Structure):
    """mlxr_lora_item."""
    _fields_ = [("a_dev", _P), ("b_dev", _P), ("y_dev", _P), ("out_dev", _P), ("N", _I), ("y_dtype", _I)]


_pack_item = struct.Struct("@4P2i").pack  # the same as bytes

_SIGS = {
    "mlxr_lora_workspace_size": (_I, [_I, _P] + [_I] * 4 + [ctypes.POINTER(ctypes.c_size_t)]),
    "mlxr_lora_apply": (_I, [_I, _P] + [_I] * 4 + [_P, _I, ctypes.c_int64, _P, _P, _P, _P, ctypes.c_size_t, _P]),
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


def lora_apply(x, ids, a, b, y, scales=None, ranks=None, outs=None, stream=None):
    """For each projection i that reads x [tokens, K]: y[i] + scale * (x A^T) B^T with the adapter
    ``ids`` [tokens] (int32; outside [0, adapters): none) of each token (mlxr_lora_apply).

    a[i] [adapters, rank, K] and b[i] [adapters, N_i, rank] have x's dtype (float16 / bfloat16), one
    rank (a multiple of 8, up to 128) for all; ``ranks`` [adapters] (int32) says how much of it each
    adapter uses.  ``scales`` [adapters] float32.  outs[i] may be y[i].  Returns the outputs."""
    lib, index, n, torch = _lib(), x.get_device(), len(a), paged._torch
    if x.dim() != 2 or index < 0:
        raise QGemmError(-3, "Input shape must be [tokens, K] on a GPU")
    tokens, K = x.shape
    if len(b) != n or len(y) != n or (outs is not None and len(outs) != n):
        raise QGemmError(-1, "one A, one B, one y (and one output) per projection")
    pi = _vector(ids, tokens, "ids", index)
    if n == 0:
        return []
    if a[0].dim() != 3:
        raise QGemmError(-3, "a[0] must be [adapters, rank, K]")
    adapters, rank, _ = shape = a[0].shape
    ps = None if scales is None else _vector(scales, adapters, "scales", index, paged._float32)
    pr = None if ranks is None else _vector(ranks, adapters, "ranks", index)
    xt = x.dtype
    dt = _code(paged._x_codes, xt, "x")
    xs = x.stride()
    if xs[1] != 1 or xs[0] % 8 or xs[0] < 0 or x.data_ptr() % 16:
        x = _on(stream, x.clone, memory_format=torch.contiguous_format)
        xs = x.stride()
        if xs[0] % 8:
            raise QGemmError(-3, "lora: K must be a multiple of 8")
    given = outs is not None
    if not given:
        make = torch.empty_like
        outs = [make(t) for t in y] if stream is None else [_on(stream, make, t) for t in y]
    items = b""
    codes = paged._x_codes
    for i in range(n):
        A, B, t, o = a[i], b[i], y[i], outs[i]
        bs, ts = B.shape, t.shape
        if A.shape != shape or shape[2] != K:
            raise QGemmError(-3, f"a[{i}] must be [{adapters}, {rank}, {K}]")
        if len(bs) != 3 or bs[0] != adapters or bs[2] != rank:
            raise QGemmError(-3, f"b[{i}] must be [{adapters}, N, {rank}]")
        N = bs[1]
        if A.dtype is not xt or B.dtype is not xt or A.get_device() != index or B.get_device() != index or \
                not A.is_contiguous() or not B.is_contiguous():
            raise QGemmError(-1, f"a[{i}] and b[{i}] must be contiguous, of x's dtype and device")
        if len(ts) != 2 or ts[0] != tokens or ts[1] != N or t.get_device() != index or not t.is_contiguous() or \
                given and (o.shape != ts or o.dtype is not t.dtype or o.get_device() != index or not o.is_contiguous()):
            raise QGemmError(-1, f"y[{i}] and its output must be contiguous [{tokens}, {N}] tensors of one dtype on GPU {index}")
        items += _pack_item(A.data_ptr(), B.data_ptr(), t.data_ptr(), o.data_ptr(), N, _code(codes, t.dtype, "y"))
    nb = ctypes.c_size_t()
    qgemm._check(lib.mlxr_lora_workspace_size(n, items, tokens, K, adapters, rank, ctypes.byref(nb)))
    nb = nb.value
    ws = _on(stream, torch.empty, nb, dtype=torch.uint8, device=x.device) if nb else None
    qgemm._check(lib.mlxr_lora_apply(n, items, tokens, K, adapters, rank, x.data_ptr(), dt, xs[0], pi, ps, pr,
                                     ws.data_ptr() if nb else None, nb, _stream(stream, index)))
    return outs


class LoraBank:
    """The adapters of one projection [N, K]: A [adapters, rank, K], B [adapters, N, rank], a scale and a
    rank for each, filled by ``load``."""

    def __init__(self, adapters, rank, N, K, dtype=None, device="cuda"):
        torch = qgemm._torch()
        if not 0 < adapters <= MAX_ADAPTERS or not 0 < rank <= MAX_RANK or N <= 0 or K <= 0 or K % 8:
            raise QGemmError(-1, f"LoraBank: up to {MAX_ADAPTERS} adapters of rank up to {MAX_RANK}, K a multiple of 8")
        dtype = dtype or torch.bfloat16
        room = -(-rank // 8) * 8
        self.N, self.K, self.rank = N, K, rank
        self.a = torch.zeros((adapters, room, K), dtype=dtype, device=device)
        self.b = torch.zeros((adapters, N, room), dtype=dtype, device=device)
        self.scales = torch.zeros(adapters, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(adapters, dtype=torch.int32, device=device)

    def load(self, i, a, b, scale=1.0):
        """Adapter i: a [r, K], b [N, r] with r up to the bank's rank, and its scale."""
        r = a.shape[0]
        if a.dim() != 2 or b.dim() != 2 or r > self.rank or a.shape[1] != self.K or tuple(b.shape) != (self.N, r):
            raise QGemmError(-3, f"LoraBank: an adapter is [r, {self.K}] and [{self.N}, r], r up to {self.rank}")
        self.a[i, :r].copy_(a)
        self.b[i, :, :r].copy_(b)
        self.scales[i] = scale
        self.ranks[i] = r
        return self

    def apply(self, x, ids, y, out=None, stream=None):
        """y + the tokens' adapters (out may be y)."""
        return lora_apply(x, ids, [self.a], [self.b], [y], self.scales, self.ranks, None if out is None else [out], stream)[0]
