"""Attention of drafted tokens over a paged cache, and masks of trees, against plain float64 forms."""
import ctypes
import math
import random

import pytest

import mlxr_amd as mx
from mlxr_amd import paged

P = ctypes.c_void_p


def _cache(**kw):
    c = dict(k_dev=64, v_dev=128, k_scale_dev=None, v_scale_dev=None, k0=2048 * 8, k1=2048, k2=128, v0=2048 * 8, v1=2048,
             v2=128, dtype=mx.BF16, num_pages=10, page_size=16, kv_heads=8, head_dim=128)
    c.update(kw)
    return paged.Cache(**c)


# ------------------------------------------------------------------------------ refusals (no GPU)

def test_refusals():
    L, n = paged._lib(), ctypes.c_size_t()

    def call(c=None, rows=2, tokens=6, heads=32, q=64, qdt=mx.BF16, qt=4096, qh=128, table=64, width=4, lens=64, starts=64, mask=64,
             words=1, out=64, odt=mx.BF16, ws=64, nb=1 << 40):
        return L.mlxr_paged_tree_attention(ctypes.byref(c or _cache()), rows, tokens, heads, P(q), qdt, qt, qh, P(table), width, width,
                                           P(lens), P(starts), P(mask), words, 0.1, P(out), odt, None, P(ws), nb, None)
    assert call(rows=-1) == -1 and call(tokens=-1) == -1 and call(heads=0) == -1 and call(width=0) == -1 and call(tokens=0) == 0
    assert call(rows=0) == -1 and call(rows=4097) == -3 and call(heads=33) == -3 and call(tokens=1 << 22) == -3
    assert call(width=1 << 27) == -3 and call(c=_cache(head_dim=12)) == -3
    assert call(qdt=mx.F32) == -1 and call(qdt=mx.F16) == -1 and call(odt=3) == -1
    assert call(words=0) == -3 and call(words=65) == -3
    for name in ("q", "table", "lens", "starts", "out"):
        assert call(**{name: 0}) == -1, name
    assert call(q=72) == -3 and call(out=72) == -3 and call(qt=4095) == -3 and call(qh=4) == -3 and call(ws=72) == -3
    assert call(width=100, ws=0) == -1 and call(width=100, nb=16) == -1

    def size(rows=2, tokens=6, heads=32, width=4, qdt=mx.BF16, odt=mx.BF16):
        return L.mlxr_paged_tree_attention_workspace_size(ctypes.byref(_cache()), rows, tokens, heads, width, qdt, odt, ctypes.byref(n))
    assert size() == 0 and n.value == 0 and size(width=400) == 0 and n.value > 0 and size(tokens=0) == 0 and n.value == 0
    assert size(qdt=mx.F16) == -1 and size(odt=3) == -1 and size(width=0) == -1
    assert L.mlxr_paged_tree_attention_workspace_size(ctypes.byref(_cache()), 1, 1, 8, 4, mx.BF16, mx.BF16, None) == -1

    def mask(rows=2, tokens=6, starts=64, parents=64, words=1, out=64):
        return L.mlxr_tree_mask(rows, tokens, P(starts), P(parents), None, words, P(out), None, None)
    assert mask(rows=-1) == -1 and mask(tokens=-1) == -1 and mask(words=0) == -1 and mask(words=65) == -3 and mask(rows=4097) == -3
    assert mask(tokens=0) == 0 and mask(starts=0) == -1 and mask(parents=0) == -1 and mask(out=0) == -1


def test_launches_too_large_are_refused():
    """Sizes whose launch would have 2^32 threads or more, and the largest below."""
    L, n = paged._lib(), ctypes.c_size_t()

    def size(rows, tokens, heads, kv, dim=128, width=4):
        c = _cache(kv_heads=kv, head_dim=dim)
        return L.mlxr_paged_tree_attention_workspace_size(ctypes.byref(c), rows, tokens, heads, width, mx.BF16, mx.BF16, ctypes.byref(n))
    assert size(4096, 4096, 1024, 1024) == 0 and size(1024, 4, 4096, 4096) == 0
    assert size(4096, 4096, 4096, 4096) == -3 and size(4096, 1, 1025, 1025) == -3 and size(1025, 4, 4096, 4096) == -3
    assert "kv heads" in L.mlxr_qgemm_last_error().decode()
    assert size(1, 1 << 23, 8, 8) == 0 and size(1, 1 << 23, 8, 8, dim=136) == -3 and size(1, (1 << 23) - 1, 8, 8, dim=256) == 0
    c = _cache(kv_heads=4096)
    assert L.mlxr_paged_tree_attention(ctypes.byref(c), 4096, 1, 4096, P(64), mx.BF16, 4096 * 128, 128, P(64), 4, 4, P(64), P(64), P(64), 1, 0.1,
                                       P(64), mx.BF16, None, P(64), 1 << 40, None) == -3


def test_workspace_holds_what_can_be_written():
    """Two partial sums (columns x head_dim, and two floats a column) for each workgroup that a CU holds, of 256 CUs, and the rows' tiles."""
    L, n = paged._lib(), ctypes.c_size_t()
    for dim, tokens, columns, resident in ((128, 513, 256, 1), (128, 100, 128, 2), (128, 4, 64, 2), (64, 4, 64, 4), (64, 513, 128, 2), (256, 4, 64, 2)):
        c = _cache(head_dim=dim, kv_heads=8)
        assert L.mlxr_paged_tree_attention_workspace_size(ctypes.byref(c), 4 if tokens == 100 else 1, tokens, 32, 3000, mx.BF16, mx.BF16, ctypes.byref(n)) == 0
        assert 0 < n.value <= 256 * resident * 2 * columns * (dim + 2) * 4 + 64, (dim, tokens, n.value)


def test_wrapper_refusals():
    import torch
    k, t = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 3), dtype=torch.int32)
    one = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(mx.QGemmError, match="on one GPU"):
        mx.paged_tree_attention(torch.zeros((2, 8, 64), dtype=torch.bfloat16), k, k, t, one, one)
    with pytest.raises(mx.QGemmError, match="on a GPU"):
        mx.tree_mask(one, one, 1)


# ------------------------------------------------------------------------------ the kernels

def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f8": torch.float8_e4m3fn}[name]


def _i32(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _words(rows_of_bits, words):
    """[tokens, words] int64 of Python integers of bits."""
    import torch
    got = []
    for b in rows_of_bits:
        w = [b >> 64 * i & (1 << 64) - 1 for i in range(words)]
        got.append([v - (1 << 64) if v >> 63 else v for v in w])
    return torch.tensor(got, dtype=torch.int64, device="cuda").view(len(rows_of_bits), words)


def _tree(n, rng):
    """Parents and bits of a random tree."""
    parents = [rng.randrange(-1, i) if i else -1 for i in range(n)]
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return parents, bits


class Batch:
    """Rows with a context and drafts each, their cache and queries."""

    def __init__(self, context, drafts, heads, kv, dim, page, dtype, cache, token_major=False, seed=0, pad=2, spread=1.0, extra=0):
        import torch
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.context, self.drafts, self.lens = context, drafts, [a + b for a, b in zip(context, drafts)]
        self.heads, self.kv, self.dim, self.page, self.cache = heads, kv, dim, page, cache
        held = [-(-n // page) for n in self.lens]
        pages = sum(held) + 2
        order = random.Random(seed).sample(range(pages), pages)
        self.table = torch.full((len(context), max(held + [1]) + extra), -1, dtype=torch.int32)
        for r, n in enumerate(held):
            for i in range(n):
                self.table[r, i] = order.pop()
        shape = (pages, page, kv, dim) if token_major else (pages, kv, page, dim)
        big = 40.0 if cache == "f8" else 1.0
        self.k, self.v = ((torch.randn(shape, device="cuda", generator=self.g) * big * spread).clamp(-440, 440).to(_dt(cache))
                          for _ in range(2))
        if token_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.ks = self.vs = None
        if cache == "f8":
            self.ks, self.vs = ((0.5 + torch.rand(kv, device="cuda", generator=self.g)) / 40 for _ in range(2))
        self.starts = [0]
        for n in drafts:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1] + pad
        self.q = (torch.randn((self.tokens, heads, dim), device="cuda", generator=self.g) * 2).to(_dt(dtype))

    def call(self, bits=None, words=1, **kw):
        mask = None if bits is None else _words(bits + [0] * (self.tokens - len(bits)), words)
        return mx.paged_tree_attention(self.q, self.k, self.v, self.table.cuda(), _i32(self.lens), _i32(self.starts), mask,
                                       k_scale=self.ks, v_scale=self.vs, **kw)

    def sees(self, r, bits, words):
        """[drafts, len] of what the nodes of row r see."""
        import torch
        n, c = self.drafts[r], self.context[r]
        got = torch.zeros((n, c + n), dtype=torch.bool)
        got[:, :c] = True
        for i in range(n):
            for j in range(n):
                got[i, c + j] = j <= i if bits is None else bool(j < 64 * words and bits[self.starts[r] + i] >> j & 1)
        return got.cuda()

    def values(self, store, scale, r):
        """[len, kv, dim] of a row's keys or values (64 bits)."""
        import torch
        n = self.lens[r]
        at = torch.arange(n)
        t = self.table[r, at // self.page].long().cuda()
        x = store.view(torch.uint8)[t, :, (at % self.page).cuda()].view(store.dtype) if self.cache == "f8" else store[t, :, (at % self.page).cuda()]
        x = x.double()
        return x if scale is None else x * scale.double()[None, :, None]

    def check(self, got, lse, bits=None, words=1, scale=None, odt="f32", dtype="bf16"):
        import torch
        got, group = got.double(), self.heads // self.kv
        scale = self.dim ** -0.5 if scale is None else scale
        half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[odt]
        parts = 2.0 ** -15 if dtype == "bf16" and self.cache == "bf16" and odt != "f32" else 2.0 ** -21
        assert not got[self.starts[-1]:].any()
        assert (lse[self.starts[-1]:] == -math.inf).all()
        for r, n in enumerate(self.drafts):
            if n == 0:
                continue
            a = self.starts[r]
            sees = self.sees(r, bits, words)
            k, v = self.values(self.k, self.ks, r), self.values(self.v, self.vs, r)
            q = self.q[a:a + n].double().view(n, self.kv, group, self.dim)
            s = torch.stack([q[:, h].reshape(n * group, self.dim) @ k[:, h].t() for h in range(self.kv)]).view(self.kv, n, group, -1) * scale
            size = torch.stack([q[:, h].reshape(n * group, self.dim).abs() @ k[:, h].abs().t() for h in range(self.kv)])
            size = size.view(self.kv, n, group, -1).masked_fill(~sees[None, :, None], 0.0).amax(-1) * abs(scale)  # [kv, n, group]
            s = s.masked_fill(~sees[None, :, None], -math.inf)
            ref = torch.softmax(s, -1).nan_to_num(0.0)
            ref = torch.stack([ref[h].reshape(n * group, -1) @ v[:, h] for h in range(self.kv)]).view(self.kv, n, group, self.dim)
            top = torch.stack([v[:, h].abs().amax() for h in range(self.kv)]).view(-1, 1, 1, 1)
            # a score is off by 2^-24 of the sum of its magnitudes for each product and five more roundings, its weight by that
            # much relative, the exponential (2^-22) and its parts; sums of weights add one rounding for each 32 tokens and wavefront
            own = (self.dim + 8) * 2.0 ** -24 * size + 2.0 ** -21 + parts + (self.lens[r] / 16 + 64) * 2.0 ** -24
            tol = 2 * own[..., None] * top + half * ref.abs() + (2.0 ** -25 if odt == "f16" else 0)
            have = got[a:a + n].view(n, self.kv, group, self.dim).permute(1, 0, 2, 3)
            off = (have - ref).abs() / tol
            assert off.max().item() <= 1, (r, off.max().item())
            want = torch.logsumexp(s, -1)
            have = lse[a:a + n].double().view(n, self.kv, group).permute(1, 0, 2)
            none = want == -math.inf
            assert torch.equal(have == -math.inf, none)
            off = (have - want).abs() / (own + 2.0 ** -21 * want.abs())
            assert off[~none].numel() == 0 or off[~none].max().item() <= 1


CASES = [("bf16", "bf16", 8, 2, 128, 16, False), ("f16", "f16", 32, 4, 64, 16, False), ("bf16", "f8", 16, 2, 128, 32, False),
         ("f16", "f8", 8, 8, 64, 7, True), ("bf16", "bf16", 7, 1, 256, 5, True), ("f16", "f16", 4, 4, 80, 64, True),
         ("bf16", "bf16", 6, 3, 8, 1, False), ("bf16", "f8", 10, 2, 112, 16, True), ("f16", "f8", 4, 2, 256, 16, False),
         ("bf16", "bf16", 40, 1, 96, 24, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,heads,kv,dim,page,token_major", CASES)
@pytest.mark.parametrize("nodes", [1, 3, 9, 30, 70, 150])
def test_trees(dtype, cache, heads, kv, dim, page, token_major, nodes):
    rng = random.Random(nodes * 31 + dim)
    drafts = [nodes, rng.randrange(1, nodes + 1), 0, nodes, 1, rng.randrange(1, nodes + 1)]
    context = [rng.randrange(0, 300), 0, 5, 64 * rng.randrange(1, 4) - nodes % 64, 777, 128]
    b = Batch(context, drafts, heads, kv, dim, page, dtype, cache, token_major, seed=nodes)
    words = -(-nodes // 64)
    bits = []
    for n in drafts:
        bits += _tree(n, rng)[1]
    b.check(*b.call(bits, words, out_dtype=_dt("f32"), return_lse=True), bits, words, dtype=dtype)
    got, lse = b.call(bits, words, return_lse=True)
    b.check(got, lse, bits, words, odt=dtype, dtype=dtype)
    b.check(*b.call(out_dtype=_dt("f32"), return_lse=True), dtype=dtype)  # a chain


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,heads,kv,dim", [("bf16", "bf16", 32, 8, 128), ("f16", "f16", 8, 1, 64), ("bf16", "f8", 16, 2, 128),
                                                     ("f16", "f16", 6, 2, 256), ("bf16", "bf16", 64, 2, 128)])
@pytest.mark.parametrize("drafts", [[3], [5, 12], [40], [100, 7, 64]])
def test_long_rows_are_cut(dtype, cache, heads, kv, dim, drafts):
    rng = random.Random(len(drafts))
    context = [rng.randrange(2500, 5000) for _ in drafts]
    if len(context) > 1:
        context[1] = 3
    b = Batch(context, drafts, heads, kv, dim, 16, dtype, cache, seed=3, pad=0 if len(drafts) == 1 else 3)
    words, bits = 2, []
    for n in drafts:
        bits += _tree(n, rng)[1]
    b.check(*b.call(bits, words, out_dtype=_dt("f32"), return_lse=True), bits, words, dtype=dtype)
    b.check(*b.call(out_dtype=_dt("f32"), return_lse=True), dtype=dtype)
    # the same bits again, and on another stream
    import torch
    want = b.call(bits, words)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = b.call(bits, words, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(b.call(bits, words), want)


@pytest.mark.gpu
def test_many_rows_and_long_chains():
    rng = random.Random(8)
    rows = 600
    b = Batch([rng.randrange(0, 90) for _ in range(rows)], [rng.randrange(0, 5) for _ in range(rows)], 8, 2, 64, 16, "bf16", "bf16", seed=4)
    b.check(*b.call(out_dtype=_dt("f32"), return_lse=True))
    b = Batch([0, 1000], [700, 300], 8, 2, 128, 16, "bf16", "bf16", seed=5)
    b.check(*b.call(out_dtype=_dt("f32"), return_lse=True))
    b = Batch([0], [1500], 4, 4, 64, 64, "f16", "f16", seed=5)
    b.check(*b.call(out_dtype=_dt("f32"), return_lse=True), dtype="f16")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8"), ("f16", "f8")])
@pytest.mark.parametrize("extra", [0, 500])  # rows of the table's length, many of its tiles empty
def test_many_columns_of_long_rows(dtype, cache, extra):
    """More than 128 columns of rows of more than 512 tokens: masks, a chain, values that are not finite, bad pages."""
    import torch
    rng = random.Random(extra)
    context, drafts = [611, 1300, 0, 64], [40, 65, 130, 0]
    b = Batch(context, drafts, 16, 2, 128, 16, dtype, cache, seed=12, extra=extra)
    bits = []
    for n in drafts:
        bits += _tree(n, rng)[1]
    for odt in ("f32", dtype):
        b.check(*b.call(bits, 3, out_dtype=_dt(odt), return_lse=True), bits, 3, odt=odt, dtype=dtype)
        b.check(*b.call(out_dtype=_dt(odt), return_lse=True), odt=odt, dtype=dtype)
    want = b.call(bits, 3)
    for node in (0, 17, 39):  # of row 0: NaN in a value, then in a key
        at = b.context[0] + node
        pg, t = int(b.table[0, at // 16]), at % 16
        for store in (b.v, b.k):
            keep = store[pg, 1, t].clone()
            store[pg, 1, t, 77] = math.nan
            got = b.call(bits, 3)
            for i in range(40):
                if bits[i] >> node & 1:
                    cell = got[i, 8:, 77] if store is b.v else got[i, 8:]
                    assert torch.isnan(cell).all()
                    cell.copy_(want[i, 8:, 77] if store is b.v else want[i, 8:])
            assert torch.equal(got, want)
            store[pg, 1, t] = keep
    b.table[1, :] = -1
    got = b.call(bits, 3)
    assert not got[40:105].any()
    got[40:105] = want[40:105]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,dim", [("bf16", "bf16", 128), ("f16", "f16", 112), ("bf16", "f8", 128), ("f16", "f8", 64), ("bf16", "bf16", 64)])
@pytest.mark.parametrize("pages,extra", [(30, 0), (36, 0), (36, 700)])  # tiles shared by four and eight wavefronts, cut rows
def test_many_rows_of_wide_trees(dtype, cache, dim, pages, extra):
    import torch
    rng = random.Random(pages)
    rows = 60
    drafts = [rng.randrange(56, 65) for _ in range(rows)]
    context = [rng.randrange(0, 16 * pages - 64) for _ in range(rows)]
    drafts[7], drafts[30], context[9], context[10] = 0, 1, 0, 16 * pages - drafts[10]
    b = Batch(context, drafts, 16, 2, dim, 16, dtype, cache, seed=14, extra=extra)
    bits = []
    for n in drafts:
        bits += _tree(n, rng)[1]
    b.check(*b.call(bits, 1, out_dtype=_dt("f32"), return_lse=True), bits, 1, dtype=dtype)
    b.check(*b.call(bits, 1, return_lse=True), bits, 1, odt=dtype, dtype=dtype)
    b.check(*b.call(out_dtype=_dt("f32"), return_lse=True), dtype=dtype)
    want = b.call(bits, 1)
    a, c = b.starts[20], b.context[20]
    for node in (0, 50):
        pg, t = int(b.table[20, (c + node) // 16]), (c + node) % 16
        for store in (b.v, b.k):
            keep = store[pg, 1, t].clone()
            store[pg, 1, t, 3] = math.nan
            got = b.call(bits, 1)
            for i in range(drafts[20]):
                if bits[a + i] >> node & 1:
                    cell = got[a + i, 8:, 3] if store is b.v else got[a + i, 8:]
                    assert torch.isnan(cell).all()
                    cell.copy_(want[a + i, 8:, 3] if store is b.v else want[a + i, 8:])
            assert torch.equal(got, want)
            store[pg, 1, t] = keep


@pytest.mark.gpu
def test_as_many_rows_as_a_call_takes():
    """MLXR_PAGED_MAX_ROWS rows, and about as many as are cut."""
    import torch
    rng = random.Random(1)
    for rows, dim, extra in ((4096, 256, 0), (1900, 128, 480)):
        b = Batch([rng.randrange(0, 30) for _ in range(rows)], [r % 3 for r in range(rows)], 2, 1, dim, 16, "bf16", "bf16", seed=13, extra=extra)
        whole, lse = b.call(out_dtype=_dt("f32"), return_lse=True)
        some = [0, 1, 2, 1047, rows - 2, rows - 1]
        c = Batch([1] * 6, [b.drafts[r] for r in some], 2, 1, dim, 16, "bf16", "bf16", seed=13)
        c.k, c.v, c.table, c.lens, c.context = b.k, b.v, b.table[some], [b.lens[r] for r in some], [b.context[r] for r in some]
        c.q = torch.cat([b.q[b.starts[r]:b.starts[r + 1]] for r in some] + [b.q[-2:]])
        c.check(torch.cat([whole[b.starts[r]:b.starts[r + 1]] for r in some] + [whole[-2:]]),
                torch.cat([lse[b.starts[r]:b.starts[r + 1]] for r in some] + [lse[-2:]]))


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 200])  # one launch; cut
@pytest.mark.parametrize("dtype,heads,kv,dim", [("bf16", 8, 2, 128), ("f16", 16, 1, 64), ("bf16", 2, 2, 256)])
def test_masks_of_any_shape(dtype, heads, kv, dim, extra):
    """Masks that are no trees: nothing, one far node, everything, later nodes; without context nothing leaves zeros."""
    rng = random.Random(dim)
    drafts, context = [9, 70, 5], [0, 0, 40]
    b = Batch(context, drafts, heads, kv, dim, 16, dtype, dtype, seed=6, extra=extra)
    bits = []
    for n in drafts:
        bits += [0, 1 << (n - 1), (1 << n) - 1] + [rng.getrandbits(n) for _ in range(n - 3)]
    bits = [v | rng.getrandbits(60) << 70 for v in bits]  # bits past the row's nodes mean nothing
    got, lse = b.call(bits, 3, out_dtype=_dt("f32"), return_lse=True)
    b.check(got, lse, bits, 3, dtype=dtype)
    assert not got[0].any() and not got[9].any() and got[79].any()
    got, lse = b.call(bits, 1, out_dtype=_dt("f32"), return_lse=True)  # nodes from 64 on are seen by none
    b.check(got, lse, bits, 1, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 200])
@pytest.mark.parametrize("dtype,cache,heads,kv,dim", [("bf16", "bf16", 8, 2, 128), ("f16", "f16", 32, 1, 64), ("bf16", "f8", 8, 2, 128)])
def test_what_is_not_seen_does_not_count(dtype, cache, heads, kv, dim, extra):
    """NaN and infinities in a node reach those that see it and no others; those behind the row's tokens reach nobody."""
    import torch
    b = Batch([37, 100], [20, 33], heads, kv, dim, 16, dtype, cache, seed=7, extra=extra)
    rng = random.Random(1)
    bits = []
    for n in b.drafts:
        bits += _tree(n, rng)[1]
    want, lse = b.call(bits, 1, return_lse=True)
    bad = math.nan if cache == "f8" else math.inf
    for r, node, value in ((0, 4, math.nan), (1, 9, bad)):
        at = b.context[r] + node
        pg, t = int(b.table[r, at // 16]), at % 16
        keep = b.v[pg, 0, t].clone()
        b.v[pg, 0, t, dim // 2 + 1] = value
        got = b.call(bits, 1)
        group, a = heads // kv, b.starts[r]
        for i in range(b.drafts[r]):
            sees = bits[a + i] >> node & 1
            cell = got[a + i, :group, dim // 2 + 1]
            if sees:
                assert (cell == math.inf).all() if value == math.inf else torch.isnan(cell).all()
                got[a + i, :group, dim // 2 + 1] = want[a + i, :group, dim // 2 + 1]
        assert torch.equal(got, want)
        b.v[pg, 0, t] = keep
        keep = b.k[pg, 0, t].clone()
        b.k[pg, 0, t] = math.nan
        got = b.call(bits, 1)
        for i in range(b.drafts[r]):
            if bits[a + i] >> node & 1:
                got[a + i, :group] = want[a + i, :group]
        assert torch.equal(got, want)
        b.k[pg, 0, t] = keep
    # behind the last token, and in pages of nobody
    used = {int(p) for p in b.table.flatten() if p >= 0}
    for pg in set(range(b.k.shape[0])) - used:
        b.k[pg], b.v[pg] = math.nan, math.nan
    for r, n in enumerate(b.lens):
        if n % 16:
            pg = int(b.table[r, n // 16])
            b.k[pg, :, n % 16:], b.v[pg, :, n % 16:] = math.nan, math.nan
    got, l2 = b.call(bits, 1, return_lse=True)
    assert torch.equal(got, want) and torch.equal(l2, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,heads,dim", [("bf16", "bf16", 8, 128), ("f16", "f8", 14, 128), ("f16", "f16", 8, 64), ("bf16", "bf16", 4, 256)])
@pytest.mark.parametrize("nodes,context,extra", [(1100, 0, 0), (700, 437, 0), (700, 70, 900), (65, 300, 100)])
def test_chains_of_any_length(dtype, cache, heads, dim, nodes, context, extra):
    """Nodes see themselves and what is before them, to the token: NaN in a node's value or key reaches it and those behind it only; a
    row of more nodes than tokens has its first nodes before the first token."""
    import torch
    b = Batch([context, 5, 0], [nodes, 1, 130], heads, 2, dim, 16, dtype, cache, seed=15, extra=extra)
    b.check(*b.call(out_dtype=_dt("f32"), return_lse=True), dtype=dtype)
    want, group = b.call(), heads // 2
    for node in (0, 1, nodes // 2, nodes // 2 + 63, nodes - 1):
        if node >= nodes:
            continue
        pg, t = int(b.table[0, (context + node) // 16]), (context + node) % 16
        for store in (b.v, b.k):
            keep = store[pg, 1, t].clone()
            store[pg, 1, t, 5] = math.nan
            got = b.call()
            assert torch.isnan(got[node:nodes, group:, 5]).all() and not torch.isnan(got[:node]).any()
            got[node:nodes, group:] = torch.where(torch.isnan(got[node:nodes, group:]), want[node:nodes, group:], got[node:nodes, group:])
            assert torch.equal(got, want)
            store[pg, 1, t] = keep
    b.lens[0] = max(nodes - 30, 1)  # the first nodes are in no cache: they see nothing, the others what is there
    gone = nodes - b.lens[0]
    got, lse = b.call(out_dtype=_dt("f32"), return_lse=True)
    assert not got[:gone].any() and (lse[:gone] == -math.inf).all() and torch.isfinite(lse[gone:nodes]).all()
    c = Batch([0], [nodes - gone], heads, 2, dim, 16, dtype, cache, seed=15, pad=0)
    c.k, c.v, c.ks, c.vs, c.table, c.q = b.k, b.v, b.ks, b.vs, b.table[:1], b.q[gone:nodes].contiguous()
    c.check(got[gone:nodes], lse[gone:nodes], dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 200])
def test_bad_pages_lengths_and_starts(extra):
    """Tokens of pages outside the cache are left out; a row whose tokens all are, or that has none, gives zeros; lengths past
    the table are taken as the table's; a row of more nodes than tokens has nodes before its first token."""
    import torch
    b = Batch([40, 30, 20, 64], [4, 5, 6, 7], 8, 2, 128, 16, "bf16", "bf16", seed=9, extra=extra)
    bits = [(1 << 7) - 1] * b.starts[-1]
    table = b.table.clone()
    b.table[0, 1], b.table[1, :] = b.k.shape[0], -1
    got, lse = b.call(bits, 1, out_dtype=_dt("f32"), return_lse=True)
    assert not got[4:9].any() and (lse[4:9] == -math.inf).all()
    # row 0 without positions 16 .. 31: as if its row were two pages
    c = Batch([24], [4], 8, 2, 128, 16, "bf16", "bf16", seed=9)
    c.k, c.v, c.q = b.k, b.v, b.q[:6]
    c.table = torch.cat([table[:1, :1], table[:1, 2:3]], 1)
    want = c.call([15] * 4, 1, out_dtype=_dt("f32"))
    assert (got[:4] - want[:4]).abs().max().item() < 1e-5
    b.table = table
    b.lens = [-3, 0, 4, 1 << 30]
    got, lse = b.call(bits, 1, out_dtype=_dt("f32"), return_lse=True)
    assert not got[:9].any() and (lse[:9] == -math.inf).all()
    assert torch.isfinite(got).all() and got[9:15].any()  # nodes 2 .. 5 at positions 0 .. 3
    c = Batch([0], [4], 8, 2, 128, 16, "bf16", "bf16", seed=9)
    c.k, c.v, c.table, c.q = b.k, b.v, table[2:3], torch.cat([b.q[9:15]])
    c.starts, c.tokens, c.drafts = [0, 4], 6, [4]
    want = c.call([15] * 4, 1, out_dtype=_dt("f32"))
    assert (got[9:13] - want[:4]).abs().max().item() < 1e-5


@pytest.mark.gpu
def test_strides_and_outputs():
    import torch
    b = Batch([100, 9], [5, 12], 8, 2, 64, 16, "bf16", "bf16", seed=10)
    bits = [(1 << 12) - 1] * 17
    want = b.call(bits, 1)
    wide = torch.zeros((b.tokens, 3, 8, 72), dtype=torch.bfloat16, device="cuda")
    wide[:, 1, :, :64] = b.q
    b.q = wide[:, 1, :, :64]
    assert torch.equal(b.call(bits, 1), want)
    odd = torch.zeros((b.tokens, 8, 65), dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = b.q
    b.q = odd[..., 1:]
    assert torch.equal(b.call(bits, 1), want)
    out = torch.full((b.tokens + 1, 8, 64), 3.0, dtype=torch.float16, device="cuda")
    assert b.call(bits, 1, out=out[:-1]).data_ptr() == out.data_ptr() and (out[-1] == 3).all()
    assert torch.allclose(out[:-1].float(), want.float(), atol=2e-2)
    table = torch.full((2, 300), 7, dtype=torch.int32)
    table[:, 5:5 + b.table.shape[1]] = b.table
    b.table = table[:, 5:5 + b.table.shape[1]]
    assert torch.equal(b.call(bits, 1), want)


@pytest.mark.gpu
def test_past_four_gigabytes():
    """Pages, heads and tokens far apart: offsets past 32 bits."""
    import torch
    room = torch.empty(9 << 30, dtype=torch.uint8, device="cuda").view(torch.bfloat16)
    k = room.as_strided((2, 2, 16, 64), (1 << 31, 1 << 30, 64, 1))
    v = room.as_strided((2, 2, 16, 64), (1 << 31, 1 << 30, 64, 1), 4096)
    g = torch.Generator(device="cuda").manual_seed(1)
    k.copy_(torch.randn(k.shape, device="cuda", generator=g)), v.copy_(torch.randn(v.shape, device="cuda", generator=g))
    q = torch.randn((6, 4, 64), device="cuda", generator=g).bfloat16()
    table, lens, starts = _i32([[1, 0]]), _i32([30]), _i32([0, 6])
    assert torch.equal(mx.paged_tree_attention(q, k, v, table, lens, starts),
                       mx.paged_tree_attention(q, k.contiguous(), v.contiguous(), table, lens, starts))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [8, 300])
def test_in_a_graph(width):
    """A captured call follows lengths, starts and masks that change between replays."""
    import torch
    b = Batch([90, 17], [6, 9], 8, 2, 128, 16, "bf16", "bf16", seed=11, extra=width - 7)
    table, lens, starts = b.table.cuda(), _i32(b.lens), _i32(b.starts)
    mask = _words([(1 << 9) - 1] * b.tokens, 1)

    def call():
        return mx.paged_tree_attention(b.q, b.k, b.v, table, lens, starts, mask)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for ln, st, bits in ((b.lens, b.starts, 511), ([50, 26], [0, 3, 12], 7), ([96, 3], [0, 15, 15], 0x7fff), ([0, 26], [0, 0, 0], 1)):
        lens.copy_(_i32(ln)), starts.copy_(_i32(st)), mask.copy_(_words([bits] * b.tokens, 1))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        assert torch.equal(got, call())


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,words", [(1, 1), (5, 1), (64, 1), (65, 2), (130, 1), (300, 5), (5000, 3)])
def test_tree_masks(nodes, words):
    rng = random.Random(nodes)
    drafts = [nodes, 0, rng.randrange(1, nodes + 1), 1]
    parents, bits, depth = [], [], []
    for n in drafts:
        p, b = _tree(n, rng) if n < 1000 else ([i - 1 if i % 3 else max(i - 3000, -1) for i in range(n)], None)
        if b is None:
            b = []
            for i, x in enumerate(p):
                b.append((b[x] if x >= 0 else 0) | 1 << i)
        d = []
        for i, x in enumerate(p):
            d.append(d[x] + 1 if x >= 0 else 0)
        if n > 3:
            i = n - 1  # no parent before it: a root
            p[i], b[i], d[i] = n + 5, 1 << i, 0
        parents, bits, depth = parents + p, bits + b, depth + d
    starts = [0]
    for n in drafts:
        starts.append(starts[-1] + n)
    at = [j + 10 * r for r, n in enumerate(drafts) for j in range(n)]
    pad = [0, 1]
    mask, pos = mx.tree_mask(_i32(parents + pad), _i32(starts), words, positions=_i32(at + [-1, -1]))
    low = [v & (1 << 64 * words) - 1 for v in bits]
    assert mask.tolist() == _words(low + [0, 0], words).tolist()
    want = [10 * r + depth[starts[r] + j] for r, n in enumerate(drafts) for j in range(n)]
    assert pos.tolist() == want + [-1, -1]
    assert mx.tree_mask(_i32(parents + pad), _i32(starts), words)[1].tolist() == depth + [-1, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 200])
@pytest.mark.parametrize("dtype,cache,heads,kv,dim,large", [("bf16", "bf16", 8, 2, 128, 3e38), ("f16", "f16", 8, 2, 128, 65504.0), ("bf16", "f8", 8, 2, 128, 448.0),
                                                          ("f16", "f16", 64, 2, 64, 65504.0), ("bf16", "bf16", 16, 1, 256, 1e38)])
def test_large_values_that_are_not_seen_do_not_count(dtype, cache, heads, kv, dim, large, extra):
    """The largest finite values in nodes: those that do not see them get the bits that zeros there give."""
    import torch
    b = Batch([37, 700], [20, 33], heads, kv, dim, 16, dtype, cache, seed=17, extra=extra)
    rng = random.Random(2)
    bits = []
    for n in b.drafts:
        bits += _tree(n, rng)[1]
    for mask in (bits, None):  # trees and chains
        for r, node in ((0, 7), (1, 0), (1, 20)):
            pg, t = (int(b.table[r, (b.context[r] + node) // 16]), (b.context[r] + node) % 16)
            keep, a = b.v[pg, :, t].clone(), b.starts[r]
            got = []
            for value in (0.0, large):
                b.v[pg, :, t] = value
                got.append(b.call(mask, 1, out_dtype=_dt("f32")))
            b.v[pg, :, t] = keep
            unseen = [i for i in range(b.starts[-1]) if not a <= i < b.starts[r + 1] or not (bits[i] >> node & 1 if mask else node <= i - a)]
            assert torch.equal(got[0][unseen], got[1][unseen]) and len(unseen) < b.starts[-1]


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 500])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (16, 1, 64)])
def test_tokens_of_no_weight_add_nothing(heads, kv, dim, extra):
    """Values of one at 4000 tokens whose weights are below 2^-40 of the largest add at most that much to what zeros there give: less
    than the products keep of a weight (2^-22 of the largest), however many they are."""
    import torch
    b = Batch([4000], [5], heads, kv, dim, 16, "f16", "f16", seed=18, extra=extra)
    b.k.zero_(), b.v.zero_(), b.q.zero_()
    b.q[..., 0] = 1.0
    page = b.table[0, 100 // 16]
    b.k[..., 0] = -40.0
    b.k[page, :, 100 % 16, 0] = 0.0  # token 100 has all the weight: the others exp(-40) = 2^-57 of it
    b.v[page, :, 100 % 16, 1] = 1.0
    want = b.call(scale=1.0, out_dtype=_dt("f32"))
    assert (want[:5, :, 1] == 1).all()
    b.v[..., 2] = 1.0
    b.v[page, :, 100 % 16, 2] = 0.0
    got = b.call(scale=1.0, out_dtype=_dt("f32"))
    assert torch.equal(got[..., 1], want[..., 1]) and got[..., 2].abs().max().item() <= 4000 * 2.0 ** -40


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,heads,kv,dim", [("bf16", "bf16", 32, 8, 128), ("f16", "f16", 8, 1, 64), ("bf16", "f8", 16, 2, 128), ("f16", "f8", 16, 4, 64),
                                                     ("f16", "f16", 6, 2, 256), ("bf16", "bf16", 16, 1, 112)])
@pytest.mark.parametrize("drafts,context,extra", [([3], [70], 0), ([9, 40], [100, 64], 0), ([150], [600], 0), ([20, 65], [2000, 64], 300)])
def test_16_bit_outputs_are_the_32_bit_ones_rounded(dtype, cache, heads, kv, dim, drafts, context, extra):
    """Nothing within depends on the output's type."""
    rng = random.Random(dim)
    b = Batch(context, drafts, heads, kv, dim, 16, dtype, cache, seed=19, extra=extra)
    bits = []
    for n in drafts:
        bits += _tree(n, rng)[1]
    import torch
    for mask in (bits, None):
        got = b.call(mask, 3, out_dtype=_dt("f32"))
        for odt in ("bf16", "f16"):
            assert torch.equal(b.call(mask, 3, out_dtype=_dt(odt)), got.to(_dt(odt)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8"), ("f16", "f8")])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("nodes,context,extra", [(1, 64, 0), (9, 100, 0), (40, 700, 0), (70, 700, 0), (9, 100, 300), (70, 2000, 300)])
def test_weights_keep_their_bits(dtype, cache, heads, kv, dim, nodes, context, extra):
    """Values that are one at one token each read single weights off, relative to token 0's.  Scores are exact (products of a few bits),
    above -4, and 0 at the first token of each tile, which the weights are relative to.  A weight is off by ln 2 times what its exponent is (2^-23 of 4
    for the scale times log2(e) in fp32, 2^-22 for the rounding of the sum), the exponential's 2^-23, as is token 0's, 2^-22 for its parts and
    2^-24 for each of two outputs: 2.5 * 2^-21.  One part less would be off by 2^-12 or 2^-17."""
    import torch
    b = Batch([context], [nodes], heads, kv, dim, 16, dtype, cache, seed=20, extra=extra, pad=0)
    b.ks = b.vs = None
    t = torch.arange(b.lens[0])
    page, at, j = b.table[0, t // 16].long().cuda(), (t % 16).cuda(), (t % 32).cuda()
    keys, values = (torch.zeros((len(t), kv, dim), device="cuda") for _ in range(2))
    keys[..., 0], keys[..., 1] = -(j // 8)[:, None].float(), -(j % 8)[:, None] / 8
    values[t[:64], :, t[:64]] = 1.0
    for store, x in ((b.k, keys), (b.v, values)):
        whole = torch.zeros(store.shape, device="cuda")
        whole[page, :, at] = x
        store.copy_(whole.to(store.dtype))
    q = 0.5 + torch.arange(nodes * heads, device="cuda").view(nodes, heads) * 37 % 128 / 256
    b.q.zero_()
    b.q[..., 0] = b.q[..., 1] = q.to(b.q.dtype)
    scale = float(torch.tensor(math.log(2.0)))
    want = torch.exp(-scale * q.double()[..., None] * (torch.arange(64, device="cuda") % 32).double() / 8)
    for mask in (None, [(1 << nodes) - 1] * nodes):
        got = b.call(mask, 2, scale=scale, out_dtype=_dt("f32")).double()
        off = (got[..., :64] / got[..., :1] / want - 1).abs()
        assert off.max().item() <= 2.5 * 2.0 ** -21, off.max().item() * 2.0 ** 21


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,extra", [(1, 0), (1, 300), (260, 0), (700, 0)])  # cut differently; a workgroup for each block of columns
@pytest.mark.parametrize("low", [5, 1500])  # the infinite value's token, at the start and before the middle
def test_an_infinite_value_counts_however_far_below(dtype, rows, extra, low):
    """Scores of 0 up to a token with an infinite value, of 400 behind: the output is infinite where the row is one workgroup's and
    where it is cut between them."""
    import torch
    b = Batch([2900] + [4] * (rows - 1), [3] * rows, 4, 1, 128, 16, dtype, dtype, seed=21, extra=extra)
    t = torch.arange(b.lens[0])
    page, at = b.table[0, t // 16].long().cuda(), (t % 16).cuda()
    b.q.zero_()
    b.q[..., 0] = 20.0
    b.k[page, :, at] = 0.0
    high = (t > 1600).cuda()
    b.k[page[high], :, at[high], 0] = 20.0
    want = b.call(scale=1.0, out_dtype=_dt("f32"))
    b.v[page[low], :, at[low], 7] = math.inf
    got = b.call(scale=1.0, out_dtype=_dt("f32"))
    assert (got[:3, :, 7] == math.inf).all()
    got[:3, :, 7] = want[:3, :, 7]
    assert torch.equal(got, want) and torch.isfinite(want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [0, 300])
@pytest.mark.parametrize("dtype,cache,heads,kv,dim", [("bf16", "bf16", 8, 2, 128), ("f16", "f16", 16, 1, 64), ("bf16", "f8", 8, 2, 128)])
@pytest.mark.parametrize("cut", [1, 5, 37, 60])
def test_starts_past_the_tokens(dtype, cache, heads, kv, dim, cut, extra):
    """page_resize lists no more tokens than it is given places for, but counts all in starts and lengths: the listed queries of the row
    where the list ends are its first nodes, and what was not written (NaN here) reaches nobody."""
    import torch
    rng = random.Random(cut)
    whole = Batch([30, 300, 7], [20, 40, 3], heads, kv, dim, 16, dtype, cache, seed=22, extra=extra, pad=0)
    b = Batch(whole.context, [min(n, max(0, cut - s)) for n, s in zip(whole.drafts, whole.starts)], heads, kv, dim, 16, dtype, cache, seed=22, pad=0)
    b.k, b.v, b.ks, b.vs, b.table, b.q = whole.k, whole.v, whole.ks, whole.vs, whole.table, whole.q[:cut].contiguous()
    for r, n in enumerate(b.drafts):
        for i in range(n, whole.drafts[r]):
            pg, t = int(b.table[r, (b.context[r] + i) // 16]), (b.context[r] + i) % 16
            b.k[pg, :, t], b.v[pg, :, t] = math.nan, math.nan
    bits = []
    for n in b.drafts:
        bits += _tree(n, rng)[1]
    for listed in (bits, None):
        mask = None if listed is None else _words(listed, 1)
        got = mx.paged_tree_attention(b.q, b.k, b.v, b.table.cuda(), _i32(whole.lens), _i32(whole.starts), mask, k_scale=b.ks, v_scale=b.vs,
                                      out_dtype=_dt("f32"), return_lse=True)
        b.check(*got, listed, 1, dtype=dtype)


@pytest.mark.gpu
def test_a_list_shorter_than_the_drafts():
    """The same through PagedKVCache.resize: the chain that there is room for gives what it gives alone."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(23)
    k, v = (torch.randn((12, 2, 64), device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn((9, 4, 64), device="cuda", generator=g).bfloat16()
    got = []
    for want in (9, 14):  # of the second no more than 9 are listed
        cache = mx.PagedKVCache(1, 8, 16, 2, 64, 1, 64)
        cache.k.fill_(math.nan), cache.v.fill_(math.nan)
        first = cache.resize(_i32([3]), 3)
        cache.append(0, k[9:], v[9:], first.slots)
        grown = cache.resize(_i32([3 + want]), 9)
        cache.append(0, k[:9], v[:9], grown.slots)
        assert grown.starts.tolist() == [0, want]
        got.append(cache.attend_tree(0, q, grown.starts))
    assert torch.isfinite(got[0]).all() and torch.equal(*got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache,heads,kv,dim", [("bf16", "bf16", 8, 2, 128), ("f16", "f16", 16, 2, 64), ("bf16", "f8", 64, 2, 128), ("f16", "f8", 8, 4, 256)])
@pytest.mark.parametrize("scale", [-0.07, 0.0, -0.0, 0.2, 1e-30])
@pytest.mark.parametrize("context,extra", [([45, 7], 0), ([2500, 7], 200)])
def test_scales_of_any_sign(dtype, cache, heads, kv, dim, scale, context, extra):
    """Negative scales, none at all, and of an e4m3 cache one negative scale among the keys' and one among the values'."""
    rng = random.Random(3)
    b = Batch(context, [21, 40], heads, kv, dim, 16, dtype, cache, seed=24, extra=extra)
    if cache == "f8":
        b.ks[0] *= -1
        b.vs[1] *= -1
    bits = []
    for n in b.drafts:
        bits += _tree(n, rng)[1]
    b.check(*b.call(bits, 1, scale=scale, out_dtype=_dt("f32"), return_lse=True), bits, 1, scale=scale, dtype=dtype)
    b.check(*b.call(scale=scale, out_dtype=_dt("f32"), return_lse=True), scale=scale, dtype=dtype)


@pytest.mark.gpu
def test_masks_of_too_many_words_are_refused():
    """Before memory for them is asked for."""
    for words in (65, 1 << 30, 0, -1):
        with pytest.raises(mx.QGemmError):
            mx.tree_mask(_i32([-1] * 4096), _i32([0, 4096]), words)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["bf16", "f16", "f8"])
def test_a_new_cache_holds_nothing_of_the_memorys_last_owner(cache):
    import torch
    for _ in range(3):
        old = [torch.full((2, 60, 2, 16, 128), math.nan, device="cuda").to(_dt(cache)) for _ in range(2)]
        del old
        c = mx.PagedKVCache(2, 60, 16, 2, 128, 2, 400, dtype=_dt(cache))
        assert not c.k.float().any() and not c.v.float().any()
        c.resize(_i32([40, 7]), 3)
        q = torch.ones((2, 4, 128), dtype=torch.float16 if cache == "f16" else torch.bfloat16, device="cuda")
        assert not c.attend(0, q).any()
