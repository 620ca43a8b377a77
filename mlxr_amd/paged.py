"""Paged key-value cache: page tables and slots on the device, writes of new tokens, decode attention.

The functions take torch tensors as device memory (include/mlxr_paged.h has the C entries):

- ``page_resize`` brings the requests of a batch to new lengths: pages go back to the pool, pages
  are taken from it, and the slots of the new tokens are listed;
- ``paged_append`` writes keys and values into those slots;
- ``paged_attention`` attends with one new token per request over its cached tokens.

``PagedKVCache`` holds the stores of several layers with the pool and the tables they share.
A store is ``[num_pages, kv_heads, page_size, head_dim]`` in any memory order whose last
dimension is contiguous (a ``[pages, page_size, heads, dim]`` tensor is passed as
``t.permute(0, 2, 1, 3)``), float16, bfloat16 or float8_e4m3fn with a float32 scale per kv head.
"""
import collections
import ctypes
import struct

from . import qgemm
from .qgemm import BF16, F16, F32, QGemmError

E4M3 = 3
MAX_ROWS = 4096

_I64, _P, _I = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int


class Cache(ctypes.Structure):
    """mlxr_paged_cache (the strides' arrays as their elements)."""
    _fields_ = [("k_dev", _P), ("v_dev", _P), ("k_scale_dev", _P), ("v_scale_dev", _P),
                ("k0", _I64), ("k1", _I64), ("k2", _I64), ("v0", _I64), ("v1", _I64), ("v2", _I64),
                ("dtype", _I), ("num_pages", _I), ("page_size", _I), ("kv_heads", _I), ("head_dim", _I)]


# the same structure as bytes, which a call takes for its address: a third of the time of a Structure
_pack_cache = struct.Struct("@4P6q5i4x").pack

_SIGS = {
    "mlxr_page_resize": (_I, [_I] * 3 + [_P, _I64, _I] + [_P] * 9 + [_I, _P, _P]),
    "mlxr_paged_append": (_I, [_P, _I, _P, _I64, _I64, _P, _I64, _I64, _I, _P, _P]),
    "mlxr_paged_attention_workspace_size": (_I, [_P, _I, _I, _I, ctypes.POINTER(ctypes.c_size_t)]),
    "mlxr_paged_attention": (_I, [_P, _I, _I, _P, _I, _I64, _I64, _P, _I64, _I, _P, ctypes.c_float, _I, _P, _I, _P, _P,
                                  ctypes.c_size_t, _P]),
}

_bound = None
_torch = None
_x_codes, _cache_codes = {}, {}


def _lib():
    """The library with this module's entries declared."""
    global _bound, _torch
    if _bound is None:
        l = qgemm.lib()
        for name, (res, args) in _SIGS.items():
            f = getattr(l, name)
            f.restype, f.argtypes = res, args
        import torch
        _torch = torch
        _x_codes.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
        _cache_codes.update({torch.float16: F16, torch.bfloat16: BF16, torch.float8_e4m3fn: E4M3})
        _bound = l
    return _bound


def _code(codes, dtype, what):
    c = codes.get(dtype)
    if c is None:
        raise QGemmError(-1, f"{what} has an unsupported dtype {dtype}")
    return c


def _stream(stream, index):
    """Handle of the torch stream a call runs on: the given one, or the device's current one."""
    return _torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream


def _on(stream, make, *args, **kw):
    """A tensor that belongs to the call's stream."""
    if stream is None:
        return make(*args, **kw)
    with _torch.cuda.stream(stream):
        return make(*args, **kw)


def _i32(t, what, device, dims=1):
    if t.dtype != _torch.int32 or t.dim() != dims or t.device != device or (t.stride()[-1] != 1 and t.shape[-1] > 1):
        raise QGemmError(-1, f"{what} must be a{' contiguous' if dims == 1 else ''} {dims}-dimensional int32 tensor on {device}")
    return t.data_ptr()


def _per_head(t, heads, what, device):
    if t.dtype != _torch.float32 or t.shape != (heads,) or not t.is_contiguous() or t.device != device:
        raise QGemmError(-1, f"{what} must be a contiguous float32 [{heads}] tensor on {device}")
    return t.data_ptr()


def _cache(k, v, k_scale, v_scale):
    """mlxr_paged_cache of two stores, its dtype code and the stores' shape."""
    shape, ks, vs, d = k.shape, k.stride(), v.stride(), k.device
    if len(shape) != 4 or v.shape != shape:
        raise QGemmError(-3, "key and value stores must be [num_pages, kv_heads, page_size, head_dim] of one shape")
    if v.dtype != k.dtype or v.device != d or not k.is_cuda:
        raise QGemmError(-1, "key and value stores must have one dtype and be on one GPU")
    if ks[3] != 1 or vs[3] != 1:
        raise QGemmError(-3, "the last dimension of a store must be contiguous")
    pages, heads, page, dim = shape
    if pages == 1 or heads == 1 or page == 1:  # strides of single places mean nothing
        ks, vs = ([s if n > 1 else 0 for s, n in zip(t, shape)] for t in (ks, vs))
    code = _code(_cache_codes, k.dtype, "the cache")
    return _pack_cache(k.data_ptr(), v.data_ptr(), _per_head(k_scale, heads, "k_scale", d) if k_scale is not None else 0,
                       _per_head(v_scale, heads, "v_scale", d) if v_scale is not None else 0, ks[0], ks[1], ks[2], vs[0], vs[1],
                       vs[2], code, pages, page, heads, dim), code, shape


def _rows16(t, stream):
    """t [n, heads, dim] with rows that start at multiples of 16 bytes: t itself, or a copy."""
    s, size = t.stride(), t.element_size()
    if (s[2] == 1 or t.shape[2] == 1) and s[0] * size % 16 == 0 and s[1] * size % 16 == 0 and s[0] >= 0 and t.data_ptr() % 16 == 0:
        return t
    return _on(stream, t.clone, memory_format=_torch.contiguous_format)


Resized = collections.namedtuple("Resized", "lens free_count starts slots positions refused")
Resized.__doc__ = """What ``page_resize`` gives: the rows' lengths [rows], free pages left [1], first new token of
each row [rows + 1], slots and positions of the new tokens [tokens] (-1 past them), rows refused [1]."""


def page_resize(table, lens, want, free, free_count, page_size, tokens, stream=None):
    """Brings the rows of ``table`` [rows, width] from ``lens`` to ``want`` tokens (mlxr_page_resize).

    ``free`` [num_pages] is the pool's stack of free pages, its first ``free_count`` [1] entries; both
    it and the table are changed in place.  ``tokens``: places for the new tokens' slots.  All
    tensors int32.  Returns ``Resized``; nothing is copied to the host."""
    lib, d = _lib(), table.device
    pt, pl, pw = _i32(table, "table", d, 2), _i32(lens, "lens", d), _i32(want, "want", d)
    pf, pc = _i32(free, "free", d), _i32(free_count, "free_count", d)
    rows, width = table.shape
    if not table.is_cuda or lens.shape != (rows,) or want.shape != (rows,) or free_count.shape != (1,):
        raise QGemmError(-3, "page_resize: lens and want must be [rows], free_count [1], on the table's GPU")
    if not 0 <= tokens < 1 << 31 or not 0 < page_size < 1 << 31:
        raise QGemmError(-1, "page_resize: tokens must not be negative and page_size must be positive")
    buf = _on(stream, _torch.empty, 2 * (rows + tokens) + 3, dtype=_torch.int32, device=d)
    p0 = buf.data_ptr()
    p1 = p0 + 4 * rows
    p2 = p1 + 4
    p3 = p2 + 4 * (rows + 1)
    p4 = p3 + 4 * tokens
    qgemm._check(lib.mlxr_page_resize(rows, page_size, free.shape[0], pt, table.stride()[0], width, pl, pw, pf, pc, p0, p1, p2,
                                      p3, p4, tokens, p4 + 4 * tokens, _stream(stream, d.index)))
    return Resized._make(buf.split((rows, 1, rows + 1, tokens, tokens, 1)))


def paged_append(k, v, k_store, v_store, slots, k_scale=None, v_scale=None, stream=None):
    """Writes keys and values [tokens, kv_heads, head_dim] into the slots [tokens] (int32; tokens whose
    slot is -1 are left out) of the stores, divided by their head's scale (mlxr_paged_append)."""
    lib = _lib()
    c, _, (_, heads, _, dim) = _cache(k_store, v_store, k_scale, v_scale)
    d, shape = k_store.device, k.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape:
        raise QGemmError(-3, "keys and values must be [tokens, kv_heads, head_dim]")
    if k.device != d or v.device != d or v.dtype != k.dtype:
        raise QGemmError(-1, "keys and values must have one dtype and be on the cache's GPU")
    n, ps = shape[0], _i32(slots, "slots", d)
    if slots.shape != (n,):
        raise QGemmError(-3, "slots must be [tokens]")
    dt = _code(_x_codes, k.dtype, "keys")
    k, v = _rows16(k, stream), _rows16(v, stream)
    ks, vs = k.stride(), v.stride()
    qgemm._check(lib.mlxr_paged_append(c, n, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], dt, ps,
                                       _stream(stream, d.index)))


def paged_attention(q, k_store, v_store, table, lens, scale=None, window=0, k_scale=None, v_scale=None, out=None,
                    out_dtype=None, return_lse=False, stream=None):
    """Attention of one new token per row, q [rows, heads, head_dim], over the row's cached tokens
    (mlxr_paged_attention): ``lens`` [rows] counts them, the new one included, ``table`` [rows, width]
    names their pages; how the work is split goes by what the table could hold, so pass ``table[:, :n]``
    where no row needs more than n pages.  ``scale`` defaults to head_dim ** -0.5; ``window`` keeps the last tokens only
    (0: all).  Rows of length 0 give zeros.  Returns out [rows, heads, head_dim] (q's dtype or
    ``out_dtype``), with ``return_lse`` also the log of the softmax's sum, float32 [rows, heads]."""
    lib = _lib()
    c, _, (_, _, _, dim) = _cache(k_store, v_store, k_scale, v_scale)
    d, shape = k_store.device, q.shape
    if len(shape) != 3 or shape[2] != dim:
        raise QGemmError(-3, "queries must be [rows, heads, head_dim]")
    if q.device != d:
        raise QGemmError(-1, "queries must be on the cache's GPU")
    rows, heads, _ = shape
    pt, pl = _i32(table, "table", d, 2), _i32(lens, "lens", d)
    width = table.shape[1]
    if table.shape[0] != rows or lens.shape[0] != rows:
        raise QGemmError(-3, "table and lens must have one row per query")
    if not 0 <= window < 1 << 31:
        raise QGemmError(-1, "paged_attention: window must not be negative")
    dt = _code(_x_codes, q.dtype, "queries")
    if out is None:
        out = _on(stream, _torch.empty, shape, dtype=out_dtype or q.dtype, device=d)
    elif out.shape != shape or not out.is_contiguous() or out.device != d:
        raise QGemmError(-1, f"out must be a contiguous [{rows}, {heads}, {dim}] tensor on {d}")
    odt = _code(_x_codes, out.dtype, "out")
    q = _rows16(q, stream)
    lse = _on(stream, _torch.empty, (rows, heads), dtype=_torch.float32, device=d) if return_lse else None
    nb = ctypes.c_size_t()
    qgemm._check(lib.mlxr_paged_attention_workspace_size(c, rows, heads, width, ctypes.byref(nb)))
    nb = nb.value
    ws = _on(stream, _torch.empty, nb, dtype=_torch.uint8, device=d) if nb else None
    qs = q.stride()
    qgemm._check(lib.mlxr_paged_attention(c, rows, heads, q.data_ptr(), dt, qs[0], qs[1], pt, table.stride()[0], width, pl,
                                          dim ** -0.5 if scale is None else scale, window, out.data_ptr(), odt,
                                          lse.data_ptr() if return_lse else None, ws.data_ptr() if nb else None, nb, _stream(stream, d.index)))
    return (out, lse) if return_lse else out


class PagedKVCache:
    """Key and value stores of ``layers`` layers over one pool of pages, and the requests' page tables.

    Row r of the tables is a request; ``resize`` brings the requests to new lengths (0 frees a
    row), ``append`` and ``attend`` work on one layer with the slots and tables that it left."""

    def __init__(self, layers, num_pages, page_size, kv_heads, head_dim, rows, max_tokens, dtype=None, device="cuda",
                 k_scale=None, v_scale=None):
        torch = qgemm._torch()
        if min(layers, num_pages, page_size, kv_heads, head_dim, rows, max_tokens) <= 0:
            raise QGemmError(-1, "PagedKVCache: sizes must be positive")
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        dtype = dtype or torch.bfloat16
        self.page_size, self.k_scale, self.v_scale = page_size, k_scale, v_scale
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        i32 = {"dtype": torch.int32, "device": device}
        self.table = torch.full((rows, -(-max_tokens // page_size)), -1, **i32)
        self.lens = torch.zeros(rows, **i32)
        self.free = torch.arange(num_pages, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)

    def resize(self, want, tokens, stream=None):
        """Requests to ``want`` [rows] tokens; returns ``Resized`` (slots of up to ``tokens`` new tokens)."""
        r = page_resize(self.table, self.lens, want, self.free, self.free_count, self.page_size, tokens, stream=stream)
        self.lens, self.free_count = r.lens, r.free_count
        return r

    def append(self, layer, k, v, slots, stream=None):
        paged_append(k, v, self.k[layer], self.v[layer], slots, self.k_scale, self.v_scale, stream=stream)

    def attend(self, layer, q, **options):
        return paged_attention(q, self.k[layer], self.v[layer], self.table, self.lens, k_scale=self.k_scale,
                               v_scale=self.v_scale, **options)
