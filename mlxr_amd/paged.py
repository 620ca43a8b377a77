"""Paged key-value cache: page tables and slots on the device, writes of new tokens, decode attention.

The functions take torch tensors as device memory (include/mlxr_paged.h has the C entries):

- ``page_resize`` brings the requests of a batch to new lengths: pages go back to the pool, pages
  are taken from it, and the slots of the new tokens are listed;
- ``paged_append`` writes keys and values into those slots;
- ``paged_attention`` attends with one new token per request over its cached tokens;
- ``paged_tree_attention`` attends with many drafted tokens per request, a tree (``tree_mask``) or a chain of them;
- ``paged_accept``, ``paged_copy`` and ``paged_fork`` move tokens within the cache, in all layers at once.

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
MAX_WORDS = 64  # of a tree's mask

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
    "mlxr_paged_tree_attention_workspace_size": (_I, [_P] + [_I] * 6 + [ctypes.POINTER(ctypes.c_size_t)]),
    "mlxr_paged_tree_attention": (_I, [_P] + [_I] * 3 + [_P, _I, _I64, _I64, _P, _I64, _I, _P, _P, _P, _I, ctypes.c_float, _P, _I,
                                                         _P, _P, ctypes.c_size_t, _P]),
    "mlxr_tree_mask": (_I, [_I, _I, _P, _P, _P, _I, _P, _P, _P]),
    "mlxr_paged_accept": (_I, [_P, _I, _I64, _I64, _I, _P, _I64, _I, _P, _P, _P, _I64, _I, _P, _P, _P]),
    "mlxr_paged_copy": (_I, [_P, _I, _I64, _I64, _I, _P, _P, _P]),
    "mlxr_paged_fork": (_I, [_P, _I, _I64, _I64, _I, _P, _I64, _I, _P, _P, _P, _P, _I, _P]),
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


def tree_mask(parents, starts, words, positions=None, stream=None):
    """Masks of drafted trees for ``paged_tree_attention`` (mlxr_tree_mask): ``parents`` [tokens] (int32) is the index of each
    node's parent among its row's nodes (before its own; -1: a root), ``starts`` [rows + 1] the rows' first nodes.  Returns the
    mask [tokens, words] (int64) and the nodes' positions [tokens] in the text: with ``positions`` (page_resize's) those
    of the roots' plus their depth, else the depth."""
    lib, index = _lib(), parents.get_device()
    if index < 0 or parents.dim() != 1 or starts.dim() != 1 or starts.shape[0] < 1:
        raise QGemmError(-3, "tree_mask: parents [tokens] and starts [rows + 1] must be on a GPU")
    n, rows = parents.shape[0], starts.shape[0] - 1
    pp, ps = _vector(parents, n, "parents", index), _vector(starts, rows + 1, "starts", index)
    px = None if positions is None else _vector(positions, n, "positions", index)
    mask = _on(stream, _torch.empty, (n, words if 0 < words <= MAX_WORDS else 1), dtype=_torch.int64, device=parents.device)
    out = _on(stream, _torch.empty, n, dtype=_int32, device=parents.device)
    qgemm._check(lib.mlxr_tree_mask(rows, n, ps, pp, px, words, mask.data_ptr(), out.data_ptr(), _stream(stream, index)))
    return mask, out


def paged_tree_attention(q, k_store, v_store, table, lens, starts, mask=None, scale=None, k_scale=None, v_scale=None, out=None,
                         out_dtype=None, return_lse=False, stream=None):
    """Attention of drafted tokens, q [tokens, heads, head_dim], over their rows' cached tokens (mlxr_paged_tree_attention).

    Row r's queries are starts[r] .. starts[r + 1] - 1 (``starts`` [rows + 1] as page_resize gives them; later queries are
    padding), its nodes the last as many of its ``lens`` [rows] cached tokens.  A node sees the tokens before them and
    the nodes whose bits its ``mask`` [tokens, words] (int64; bit j % 64 of word j / 64) has; without a mask itself
    and the nodes before it.  Returns out [tokens, heads, head_dim] (q's dtype or ``out_dtype``; zeros for padding and for
    nodes that see nothing), with ``return_lse`` also the log of the softmax's sum, float32 [tokens, heads]."""
    lib = _lib()
    c, _, dim, index = _cache(k_store, v_store, k_scale, v_scale)
    shape = q.shape
    if len(shape) != 3 or shape[2] != dim:
        raise QGemmError(-3, "queries must be [tokens, heads, head_dim]")
    if q.get_device() != index:
        raise QGemmError(-1, "queries must be on the cache's GPU")
    tokens, heads, _ = shape
    pt, (rows, width) = _table(table, index), table.shape
    pl, ps = _vector(lens, rows, "lens", index), _vector(starts, rows + 1, "starts", index)
    pm, words = None, 0
    if mask is not None:
        if mask.dim() != 2 or mask.shape[0] != tokens:
            raise QGemmError(-3, "mask must be [tokens, words]")
        if mask.dtype is not _torch.int64 or mask.get_device() != index or not mask.is_contiguous():
            raise QGemmError(-1, f"mask must be a contiguous int64 tensor on GPU {index}")
        pm, words = mask.data_ptr(), mask.shape[1]
    dt = _code(_x_codes, q.dtype, "queries")
    if out is None:
        out = _on(stream, _torch.empty_like, q, dtype=out_dtype, memory_format=_torch.contiguous_format)
    elif out.shape != shape or not out.is_contiguous() or out.get_device() != index:
        raise QGemmError(-1, f"out must be a contiguous [{tokens}, {heads}, {dim}] tensor on GPU {index}")
    odt = _code(_x_codes, out.dtype, "out")
    q = _rows16(q, stream)
    lse = _on(stream, _torch.empty, (tokens, heads), dtype=_float32, device=q.device) if return_lse else None
    nb = ctypes.c_size_t()
    qgemm._check(lib.mlxr_paged_tree_attention_workspace_size(c, rows, tokens, heads, width, dt, odt, ctypes.byref(nb)))
    nb = nb.value
    ws = _on(stream, _torch.empty, nb, dtype=_torch.uint8, device=q.device) if nb else None
    qs = q.stride()
    qgemm._check(lib.mlxr_paged_tree_attention(c, rows, tokens, heads, q.data_ptr(), dt, qs[0], qs[1], pt, table.stride()[0], width,
                                               pl, ps, pm, words, dim ** -0.5 if scale is None else scale, out.data_ptr(), odt,
                                               lse.data_ptr() if return_lse else None, ws.data_ptr() if nb else None, nb,
                                               _stream(stream, index)))
    return (out, lse) if return_lse else out


def _layers(k, v):
    """mlxr_paged_cache of the first of a model's layers' stores [layers, pages, heads, page, dim] (or of one layer's), the
    layers, their strides and the GPU."""
    shape, ks, vs, index = k.shape, k.stride(), v.stride(), k.get_device()
    if len(shape) == 4:
        shape, ks, vs = (1, *shape), (0, *ks), (0, *vs)
    if len(shape) != 5 or v.shape != k.shape or shape[0] == 0:
        raise QGemmError(-3, "key and value stores must be [layers, num_pages, kv_heads, page_size, head_dim] of one shape")
    if v.dtype is not k.dtype or v.get_device() != index or index < 0:
        raise QGemmError(-1, "key and value stores must have one dtype and be on one GPU")
    layers, pages, heads, page, dim = shape
    if (ks[4] != 1 or vs[4] != 1) and dim > 1:
        raise QGemmError(-3, "the last dimension of a store must be contiguous")
    if pages == 1 or heads == 1 or page == 1:  # strides of single places mean nothing
        ks, vs = ([s if n > 1 else 0 for s, n in zip(t, shape)] for t in (ks, vs))
    code = _code(_cache_codes, k.dtype, "the cache")
    return _pack_cache(k.data_ptr(), v.data_ptr(), 0, 0, ks[1], ks[2], ks[3], vs[1], vs[2], vs[3], code, pages, page, heads,
                       dim), layers, ks[0], vs[0], index


def paged_accept(k_store, v_store, table, lens, starts, path, counts, stream=None):
    """Keeps the accepted path of each row's drafted tokens (mlxr_paged_accept): the last starts[r + 1] - starts[r] of its
    ``lens`` [rows] tokens are the nodes of a tree; nodes ``path`` [rows, depth] (ascending), the first ``counts`` [rows] of
    them, move together behind the row's other tokens in every layer of the stores [layers, num_pages, kv_heads, page_size,
    head_dim].  All int32.  Returns the new lengths [rows]; ``page_resize`` to them gives the other nodes' pages back."""
    lib = _lib()
    c, layers, kl, vl, index = _layers(k_store, v_store)
    pt, (rows, width) = _table(table, index), table.shape
    pl, ps, pc = _vector(lens, rows, "lens", index), _vector(starts, rows + 1, "starts", index), _vector(counts, rows, "counts", index)
    if path.dim() != 2 or path.shape[0] != rows:
        raise QGemmError(-3, "path must have one row per request")
    if path.dtype is not _int32 or path.get_device() != index or (path.shape[1] > 1 and path.stride()[1] != 1):
        raise QGemmError(-1, f"path must be an int32 tensor with contiguous rows on GPU {index}")
    out = _on(stream, _torch.empty, rows, dtype=_int32, device=table.device)
    qgemm._check(lib.mlxr_paged_accept(c, layers, kl, vl, rows, pt, table.stride()[0], width, pl, ps, path.data_ptr(),
                                       path.stride()[0], path.shape[1], pc, out.data_ptr(), _stream(stream, index)))
    return out


def paged_copy(k_store, v_store, src, dst, stream=None):
    """Copies the tokens in slots ``src`` to slots ``dst`` [tokens] (int32; -1: left out), bit for bit, in every layer of the
    stores (mlxr_paged_copy).  No slot may be twice in dst, or in both."""
    lib = _lib()
    c, layers, kl, vl, index = _layers(k_store, v_store)
    n = src.shape[0] if src.dim() else 0
    qgemm._check(lib.mlxr_paged_copy(c, layers, kl, vl, n, _vector(src, n, "src", index), _vector(dst, n, "dst", index),
                                     _stream(stream, index)))


def paged_fork(k_store, v_store, table, sources, grown, stream=None):
    """Fills the new tokens of a ``page_resize`` (``grown``) with those at the same positions of rows ``sources`` [rows]
    (int32; -1: not filled), in every layer (mlxr_paged_fork)."""
    lib = _lib()
    c, layers, kl, vl, index = _layers(k_store, v_store)
    pt, (rows, width) = _table(table, index), table.shape
    n = grown.slots.shape[0]
    qgemm._check(lib.mlxr_paged_fork(c, layers, kl, vl, rows, pt, table.stride()[0], width, _vector(sources, rows, "sources", index),
                                     _vector(grown.starts, rows + 1, "starts", index), _vector(grown.slots, n, "slots", index),
                                     _vector(grown.positions, n, "positions", index), n, _stream(stream, index)))


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
        # zeros: tokens that are counted before they are written (more than `resize` lists) attend to nothing of other owners of the memory
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
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

    def attend_tree(self, layer, q, starts, mask=None, longest=None, **options):
        """paged_tree_attention of a layer's drafted tokens, which are the last of their rows (``starts`` as the ``resize`` that made
        room for them gave).  ``longest``: as for ``attend``."""
        table = self.table if longest is None else self.table[:, :max(1, -(-longest // self.page_size))]
        return paged_tree_attention(q, self.k[layer], self.v[layer], table, self.lens, starts, mask, k_scale=self.k_scale,
                                    v_scale=self.v_scale, **options)

    def accept(self, grown, path, counts, stream=None):
        """After a pass over drafted tokens (``grown``: what the ``resize`` that made room for them gave): each row keeps
        the nodes of its accepted path, which become its last tokens, and gives back the pages of the others
        (paged_accept, page_resize).  Returns ``Resized``."""
        lens = paged_accept(self.k, self.v, self.table, self.lens, grown.starts, path, counts, stream=stream)
        return self.resize(lens, 0, stream=stream)

    def fork(self, sources, tokens, stream=None):
        """Rows whose ``sources`` [rows] (int32) names another row become copies of it; rows with -1 (or anything that is no row) stay.  ``tokens``: at
        least as many as are copied in all.  A row that becomes a copy must be empty (resize it to 0 before).  Returns
        ``Resized``; rows for which the pool had no pages are refused as by ``resize``."""
        rows = self.lens.shape[0]
        _vector(sources, rows, "sources", self.lens.get_device())

        def wanted():
            at = sources.clamp(0, rows - 1)
            return _torch.where(at == sources, self.lens[at.long()], self.lens)
        grown = self.resize(_on(stream, wanted), tokens, stream=stream)
        paged_fork(self.k, self.v, self.table, sources, grown, stream=stream)
        return grown
