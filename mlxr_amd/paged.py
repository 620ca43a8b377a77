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
_torch = _int32 = _float32 = None
_x_codes, _cache_codes = {}, {}


def _lib():
    """The library with this module's entries declared."""
    global _bound, _torch, _int32, _float32
    if _bound is None:
        l = qgemm.lib()
        for name, (res, args) in _SIGS.items():
            f = getattr(l, name)
            f.restype, f.argtypes = res, args
        import torch
        _torch, _int32, _float32 = torch, torch.int32, torch.float32
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


def _vector(t, n, what, index, dtype=None):
    """Address of a contiguous [n] tensor of int32 (or dtype) on GPU `index`."""
    dtype = dtype or _int32
    if t.dtype is not dtype or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
        raise QGemmError(-1 if t.dtype is not dtype or t.get_device() != index or t.dim() != 1 else -3,
                         f"{what} must be a contiguous {str(dtype)[6:]} [{n}] tensor on GPU {index}")
    return t.data_ptr()


def _table(t, index):
    """Address of a page table [rows, width] on GPU `index`."""
    if t.dtype is not _int32 or t.dim() != 2 or t.get_device() != index or (t.stride()[1] != 1 and t.shape[1] > 1):
        raise QGemmError(-1, f"table must be a 2-dimensional int32 tensor with contiguous rows on GPU {index}")
    return t.data_ptr()


def _cache(k, v, k_scale, v_scale):
    """mlxr_paged_cache of two stores, their heads, head_dim and GPU."""
    shape, ks, vs, index = k.shape, k.stride(), v.stride(), k.get_device()
    if len(shape) != 4 or v.shape != shape:
        raise QGemmError(-3, "key and value stores must be [num_pages, kv_heads, page_size, head_dim] of one shape")
    if v.dtype is not k.dtype or v.get_device() != index or index < 0:
        raise QGemmError(-1, "key and value stores must have one dtype and be on one GPU")
    if ks[3] != 1 or vs[3] != 1:
        raise QGemmError(-3, "the last dimension of a store must be contiguous")
    pages, heads, page, dim = shape
    if pages == 1 or heads == 1 or page == 1:  # strides of single places mean nothing
        ks, vs = ([s if n > 1 else 0 for s, n in zip(t, shape)] for t in (ks, vs))
    code = _code(_cache_codes, k.dtype, "the cache")
    return _pack_cache(k.data_ptr(), v.data_ptr(),
                       0 if k_scale is None else _vector(k_scale, heads, "k_scale", index, _float32),
                       0 if v_scale is None else _vector(v_scale, heads, "v_scale", index, _float32), ks[0], ks[1], ks[2], vs[0],
                       vs[1], vs[2], code, pages, page, heads, dim), heads, dim, index


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
    it and the table are changed in place.  ``tokens``: places for the new tokens' slots.  Where the pool has too few
    pages for a row, it and all later rows that need any are refused.  All tensors int32.  Returns ``Resized``; nothing is copied to the host."""
    lib, index, shape = _lib(), table.get_device(), table.shape
    if index < 0:
        raise QGemmError(-1, "page_resize: table must be on a GPU")
    pt = _table(table, index)
    rows, width = shape
    pl, pw = _vector(lens, rows, "lens", index), _vector(want, rows, "want", index)
    pages = free.shape[0]
    pf, pc = _vector(free, pages, "free", index), _vector(free_count, 1, "free_count", index)
    if not 0 <= tokens < 1 << 31 or not 0 < page_size < 1 << 31:
        raise QGemmError(-1, "page_resize: tokens must not be negative and page_size must be positive")
    buf = _on(stream, _torch.empty, 2 * (rows + tokens) + 3, dtype=_int32, device=table.device)
    p0 = buf.data_ptr()
    p1 = p0 + 4 * rows
    p2 = p1 + 4
    p3 = p2 + 4 * (rows + 1)
    p4 = p3 + 4 * tokens
    qgemm._check(lib.mlxr_page_resize(rows, page_size, pages, pt, table.stride()[0], width, pl, pw, pf, pc, p0, p1, p2,
                                      p3, p4, tokens, p4 + 4 * tokens, _stream(stream, index)))
    return Resized._make(buf.unsafe_split_with_sizes((rows, 1, rows + 1, tokens, tokens, 1)))


def paged_append(k, v, k_store, v_store, slots, k_scale=None, v_scale=None, stream=None):
    """Writes keys and values [tokens, kv_heads, head_dim] into the slots [tokens] (int32; tokens whose
    slot is -1 are left out) of the stores, divided by their head's scale (mlxr_paged_append)."""
    lib = _lib()
    c, heads, dim, index = _cache(k_store, v_store, k_scale, v_scale)
    shape = k.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape:
        raise QGemmError(-3, "keys and values must be [tokens, kv_heads, head_dim]")
    if k.get_device() != index or v.get_device() != index or v.dtype is not k.dtype:
        raise QGemmError(-1, "keys and values must have one dtype and be on the cache's GPU")
    n = shape[0]
    ps = _vector(slots, n, "slots", index)
    dt = _code(_x_codes, k.dtype, "keys")
    k, v = _rows16(k, stream), _rows16(v, stream)
    ks, vs = k.stride(), v.stride()
    qgemm._check(lib.mlxr_paged_append(c, n, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], dt, ps,
                                       _stream(stream, index)))


def paged_attention(q, k_store, v_store, table, lens, scale=None, window=0, k_scale=None, v_scale=None, out=None,
                    out_dtype=None, return_lse=False, stream=None):
    """Attention of one new token per row, q [rows, heads, head_dim], over the row's cached tokens
    (mlxr_paged_attention): ``lens`` [rows] counts them, the new one included, ``table`` [rows, width]
    names their pages; how the work is split goes by what the table could hold, so pass ``table[:, :n]``
    where no row needs more than n pages.  ``scale`` defaults to head_dim ** -0.5; ``window`` keeps the last tokens only
    (0: all).  Rows of length 0 give zeros.  Returns out [rows, heads, head_dim] (q's dtype or
    ``out_dtype``), with ``return_lse`` also the log of the softmax's sum, float32 [rows, heads]."""
    lib = _lib()
    c, _, dim, index = _cache(k_store, v_store, k_scale, v_scale)
    shape = q.shape
    if len(shape) != 3 or shape[2] != dim:
        raise QGemmError(-3, "queries must be [rows, heads, head_dim]")
    if q.get_device() != index:
        raise QGemmError(-1, "queries must be on the cache's GPU")
    rows, heads, _ = shape
    pt, (table_rows, width) = _table(table, index), table.shape
    if table_rows != rows:
        raise QGemmError(-3, "table must have one row per query")
    pl = _vector(lens, rows, "lens", index)
    if not 0 <= window < 1 << 31:
        raise QGemmError(-1, "paged_attention: window must not be negative")
    dt = _code(_x_codes, q.dtype, "queries")
    if out is None:
        if out_dtype is None and q.is_contiguous():
            out = _on(stream, _torch.empty_like, q)
        else:
            out = _on(stream, _torch.empty, shape, dtype=out_dtype or q.dtype, device=q.device)
    elif out.shape != shape or not out.is_contiguous() or out.get_device() != index:
        raise QGemmError(-1, f"out must be a contiguous [{rows}, {heads}, {dim}] tensor on GPU {index}")
    odt = _code(_x_codes, out.dtype, "out")
    q = _rows16(q, stream)
    lse = _on(stream, _torch.empty, (rows, heads), dtype=_float32, device=q.device) if return_lse else None
    nb = ctypes.c_size_t()
    qgemm._check(lib.mlxr_paged_attention_workspace_size(c, rows, heads, width, ctypes.byref(nb)))
    nb = nb.value
    ws = _on(stream, _torch.empty, nb, dtype=_torch.uint8, device=q.device) if nb else None
    qs = q.stride()
    qgemm._check(lib.mlxr_paged_attention(c, rows, heads, q.data_ptr(), dt, qs[0], qs[1], pt, table.stride()[0], width, pl,
                                          dim ** -0.5 if scale is None else scale, window, out.data_ptr(), odt,
                                          lse.data_ptr() if return_lse else None, ws.data_ptr() if nb else None, nb,
                                          _stream(stream, index)))
    return (out, lse) if return_lse else out


class PagedKVCache:
    """Key and value stores of ``layers`` layers over one pool of pages, and the requests' page tables.

    Row r of the tables is a request; ``resize`` brings the requests to new lengths (0 frees a
    row), ``append`` and ``attend`` work on one layer with the slots and tables that it left.  All state
    (``table``, ``lens``, ``free``, ``free_count``) stays in the same memory, so that a captured step goes on
    from where the last one left it."""

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
        """Requests to ``want`` [rows] tokens; returns ``Resized`` (slots of up to ``tokens`` new tokens).  Rows that
        need pages are served in their order until the pool has too few for one; it and all later ones that need any are
        refused: they keep their lengths and have no new token (``starts`` of the next row is theirs)."""
        r = page_resize(self.table, self.lens, want, self.free, self.free_count, self.page_size, tokens, stream=stream)
        _on(stream, _torch._foreach_copy_, [self.lens, self.free_count], [r.lens, r.free_count])  # one launch
        return r

    def append(self, layer, k, v, slots, stream=None):
        paged_append(k, v, self.k[layer], self.v[layer], slots, self.k_scale, self.v_scale, stream=stream)

    def attend(self, layer, q, longest=None, **options):
        """paged_attention over the rows of a layer.  ``longest``: no row holds more tokens (None: not known), which
        the split of the work goes by; tokens past it would be left out."""
        table = self.table if longest is None else self.table[:, :max(1, -(-longest // self.page_size))]
        return paged_attention(q, self.k[layer], self.v[layer], table, self.lens, k_scale=self.k_scale,
                               v_scale=self.v_scale, **options)
