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

from . import qgemm
from .qgemm import QGemmError

E4M3 = 3
MAX_ROWS = 4096

_I64, _P, _I = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int


class Cache(ctypes.Structure):
    """mlxr_paged_cache (the strides' arrays as their elements)."""
    _fields_ = [("k_dev", _P), ("v_dev", _P), ("k_scale_dev", _P), ("v_scale_dev", _P),
                ("k0", _I64), ("k1", _I64), ("k2", _I64), ("v0", _I64), ("v1", _I64), ("v2", _I64),
                ("dtype", _I), ("num_pages", _I), ("page_size", _I), ("kv_heads", _I), ("head_dim", _I)]


_SIGS = {
    "mlxr_page_resize": (_I, [_I] * 3 + [_P, _I64, _I] + [_P] * 9 + [_I, _P, _P]),
    "mlxr_paged_append": (_I, [_P, _I, _P, _I64, _I64, _P, _I64, _I64, _I, _P, _P]),
    "mlxr_paged_attention_workspace_size": (_I, [_P, _I, _I, ctypes.POINTER(ctypes.c_size_t)]),
    "mlxr_paged_attention": (_I, [_P, _I, _I, _P, _I, _I64, _I64, _P, _I64, _I, _P, ctypes.c_float, _I, _P, _I, _P, _P,
                                  ctypes.c_size_t, _P]),
}

_bound = None


def _lib():
    global _bound
    if _bound is None:
        l = qgemm.lib()
        for name, (res, args) in _SIGS.items():
            f = getattr(l, name)
            f.restype, f.argtypes = res, args
        _bound = l
    return _bound


_codes = {}


def _code(dtype, what, cache=False):
    if not _codes:
        torch = qgemm._torch()
        _codes.update({torch.float32: qgemm.F32, torch.float16: qgemm.F16, torch.bfloat16: qgemm.BF16,
                       torch.float8_e4m3fn: E4M3})
    c = _codes.get(dtype)
    if c is None or (c == qgemm.F32 if cache else c == E4M3):
        raise QGemmError(-1, f"{what} has an unsupported dtype {dtype}")
    return c


def _on(stream, device):
    """The torch stream a call runs on, its handle, and the context that makes new tensors belong to it."""
    torch = qgemm._torch()
    if stream is None:
        return torch.cuda.current_stream(device).cuda_stream, None
    return stream.cuda_stream, torch.cuda.stream(stream)


def _empty(ctx, shape, dtype, device):
    torch = qgemm._torch()
    if ctx is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with ctx:
        return torch.empty(shape, dtype=dtype, device=device)


def _i32(t, what, device, dims=1):
    torch = qgemm._torch()
    if t.dtype != torch.int32 or t.dim() != dims or t.device != device or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise QGemmError(-1, f"{what} must be a{' contiguous' if dims == 1 else ''} {dims}-dimensional int32 tensor on {device}")
    return t


def _scale(t, heads, what, device):
    if t is None:
        return None
    if t.dtype != qgemm._torch().float32 or tuple(t.shape) != (heads,) or not t.is_contiguous() or t.device != device:
        raise QGemmError(-1, f"{what} must be a contiguous float32 [{heads}] tensor on {device}")
    return t.data_ptr()


def _cache(k, v, k_scale, v_scale):
    if k.dim() != 4 or v.shape != k.shape:
        raise QGemmError(-3, "key and value stores must be [num_pages, kv_heads, page_size, head_dim] of one shape")
    if v.dtype != k.dtype or v.device != k.device or k.device.type != "cuda":
        raise QGemmError(-1, "key and value stores must have one dtype and be on one GPU")
    pages, heads, page, dim = k.shape
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise QGemmError(-3, "the last dimension of a store must be contiguous")
    d = k.device
    return Cache(k.data_ptr(), v.data_ptr(), _scale(k_scale, heads, "k_scale", d), _scale(v_scale, heads, "v_scale", d),
                 ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], _code(k.dtype, "the cache", True), pages, page, heads, dim)


def _rows16(t):
    """t [n, heads, dim] with rows that start at multiples of 16 bytes: t itself, or a copy."""
    s, unit = t.stride(), 16 // t.element_size()
    if s[2] == 1 and s[0] % unit == 0 and s[1] % unit == 0 and s[0] >= 0 and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


Resized = collections.namedtuple("Resized", "lens free_count starts slots positions refused")
Resized.__doc__ = """What ``page_resize`` gives: the rows' lengths [rows], free pages left [1], first new token of
each row [rows + 1], slots and positions of the new tokens [tokens] (-1 past them), rows refused [1]."""


def page_resize(table, lens, want, free, free_count, page_size, tokens, stream=None):
    """Brings the rows of ``table`` [rows, width] from ``lens`` to ``want`` tokens (mlxr_page_resize).

    ``free`` [num_pages] is the pool's stack of free pages, its first ``free_count`` [1] entries; both
    it and the table are changed in place.  ``tokens``: places for the new tokens' slots.  All
    tensors int32.  Returns ``Resized``; nothing is copied to the host."""
    torch = qgemm._torch()
    d = table.device
    _i32(table, "table", d, 2)
    for t, what in ((lens, "lens"), (want, "want"), (free, "free"), (free_count, "free_count")):
        _i32(t, what, d)
    rows, width = table.shape
    if d.type != "cuda" or lens.shape[0] != rows or want.shape[0] != rows or free_count.shape[0] != 1:
        raise QGemmError(-3, "page_resize: lens and want must be [rows], free_count [1], on the table's GPU")
    if tokens < 0:
        raise QGemmError(-1, "page_resize: tokens must not be negative")
    ptr, ctx = _on(stream, d)
    # one allocation, each part at a multiple of 16 bytes
    parts = [rows, 1, rows + 1, tokens, tokens, 1]
    at = [0]
    for n in parts:
        at.append(at[-1] + (n + 3) // 4 * 4)
    buf = _empty(ctx, at[-1], torch.int32, d)
    base = buf.data_ptr()
    p = [base + 4 * x for x in at]
    qgemm._check(_lib().mlxr_page_resize(rows, int(page_size), free.shape[0], table.data_ptr(), table.stride(0), width,
                                              lens.data_ptr(), want.data_ptr(), free.data_ptr(), free_count.data_ptr(),
                                              p[0], p[1], p[2], p[3], p[4], tokens, p[5], ptr))
    return Resized(*[buf[x:x + n] for x, n in zip(at, parts)])


def paged_append(k, v, k_store, v_store, slots, k_scale=None, v_scale=None, stream=None):
    """Writes keys and values [tokens, kv_heads, head_dim] into the slots [tokens] (int32; tokens whose
    slot is -1 are left out) of the stores, divided by their head's scale (mlxr_paged_append)."""
    c = _cache(k_store, v_store, k_scale, v_scale)
    d = k_store.device
    if k.dim() != 3 or k.shape[1] != c.kv_heads or k.shape[2] != c.head_dim or v.shape != k.shape:
        raise QGemmError(-3, "keys and values must be [tokens, kv_heads, head_dim]")
    if k.device != d or v.device != d or v.dtype != k.dtype:
        raise QGemmError(-1, "keys and values must have one dtype and be on the cache's GPU")
    _i32(slots, "slots", d)
    n = k.shape[0]
    if slots.shape[0] != n:
        raise QGemmError(-3, "slots must be [tokens]")
    dt = _code(k.dtype, "keys")
    ptr, ctx = _on(stream, d)
    if ctx is None:
        k, v = _rows16(k), _rows16(v)
    else:
        with ctx:
            k, v = _rows16(k), _rows16(v)
    ks, vs = k.stride(), v.stride()
    qgemm._check(_lib().mlxr_paged_append(ctypes.byref(c), n, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], dt,
                                               slots.data_ptr(), ptr))


def paged_attention(q, k_store, v_store, table, lens, scale=None, window=0, k_scale=None, v_scale=None, out=None,
                    out_dtype=None, return_lse=False, stream=None):
    """Attention of one new token per row, q [rows, heads, head_dim], over the row's cached tokens
    (mlxr_paged_attention): ``lens`` [rows] counts them, the new one included, ``table`` [rows, width]
    names their pages.  ``scale`` defaults to head_dim ** -0.5; ``window`` keeps the last tokens only
    (0: all).  Rows of length 0 give zeros.  Returns out [rows, heads, head_dim] (q's dtype or
    ``out_dtype``), with ``return_lse`` also the log of the softmax's sum, float32 [rows, heads]."""
    torch = qgemm._torch()
    c = _cache(k_store, v_store, k_scale, v_scale)
    d = k_store.device
    if q.dim() != 3 or q.shape[2] != c.head_dim:
        raise QGemmError(-3, "queries must be [rows, heads, head_dim]")
    if q.device != d:
        raise QGemmError(-1, "queries must be on the cache's GPU")
    rows, heads, dim = q.shape
    _i32(table, "table", d, 2)
    _i32(lens, "lens", d)
    if table.shape[0] != rows or lens.shape[0] != rows:
        raise QGemmError(-3, "table and lens must have one row per query")
    dt = _code(q.dtype, "queries")
    ptr, ctx = _on(stream, d)
    if out is None:
        out = _empty(ctx, (rows, heads, dim), out_dtype or q.dtype, d)
    elif tuple(out.shape) != (rows, heads, dim) or not out.is_contiguous() or out.device != d:
        raise QGemmError(-1, f"out must be a contiguous [{rows}, {heads}, {dim}] tensor on {d}")
    odt = _code(out.dtype, "out")
    if ctx is None:
        q = _rows16(q)
    else:
        with ctx:
            q = _rows16(q)
    lse = _empty(ctx, (rows, heads), torch.float32, d) if return_lse else None
    lib, cp = _lib(), ctypes.byref(c)
    n = ctypes.c_size_t()
    qgemm._check(lib.mlxr_paged_attention_workspace_size(cp, rows, heads, ctypes.byref(n)))
    ws = _empty(ctx, n.value, torch.uint8, d)
    qs = q.stride()
    qgemm._check(lib.mlxr_paged_attention(cp, rows, heads, q.data_ptr(), dt, qs[0], qs[1], table.data_ptr(), table.stride(0),
                                          table.shape[1], lens.data_ptr(), dim ** -0.5 if scale is None else float(scale),
                                          int(window), out.data_ptr(), odt, lse.data_ptr() if lse is not None else None,
                                          ws.data_ptr(), n.value, ptr))
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
