"""Paged key-value cache: page tables, writes and decode attention against plain float64 forms."""
import ctypes
import math

import pytest

import mlxr_amd as mx
from mlxr_amd import paged

P = ctypes.c_void_p


# ------------------------------------------------------------------------------ refusals (no GPU)

def _cache(**kw):
    c = dict(k_dev=64, v_dev=128, k_scale_dev=None, v_scale_dev=None, k0=2048 * 8, k1=2048, k2=128, v0=2048 * 8, v1=2048,
             v2=128, dtype=mx.BF16, num_pages=10, page_size=16, kv_heads=8, head_dim=128)
    c.update(kw)
    return paged.Cache(**c)


BAD_CACHES = [
    (dict(k_dev=None), -1, "null buffer"), (dict(dtype=0), -1, "cache dtype"), (dict(dtype=4), -1, "cache dtype"),
    (dict(num_pages=0), -1, "positive"), (dict(page_size=0), -1, "positive"), (dict(kv_heads=-1), -1, "positive"),
    (dict(head_dim=0), -1, "positive"), (dict(head_dim=12), -3, "multiple of 8"), (dict(head_dim=264), -3, "at most 256"),
    (dict(head_dim=72, dtype=3), -3, "multiple of 16"), (dict(k0=2047), -3, "strides"), (dict(v2=-128), -3, "strides"),
    (dict(k2=8, dtype=3), -3, "strides"), (dict(v_dev=8), -1, "addresses"),
    (dict(num_pages=1 << 28, page_size=8), -3, "at most"),
]


@pytest.mark.parametrize("change,code,text", BAD_CACHES)
def test_cache_refusals(change, code, text):
    c = _cache(**change)
    L = paged._lib()
    assert L.mlxr_paged_append(ctypes.byref(c), 1, P(64), 1024, 128, P(64), 1024, 128, mx.BF16, P(64), None) == code
    assert text in L.mlxr_qgemm_last_error().decode()
    n = ctypes.c_size_t()
    assert L.mlxr_paged_attention_workspace_size(ctypes.byref(c), 1, 8, 4, ctypes.byref(n)) == code


def test_append_refusals():
    c, L = _cache(), paged._lib()

    def call(tokens=1, k=64, kt=1024, kh=128, v=64, dt=mx.BF16, slots=64):
        return L.mlxr_paged_append(ctypes.byref(c), tokens, P(k), kt, kh, P(v), 1024, 128, dt, P(slots), None)
    assert call(tokens=-1) == -1
    assert call(tokens=0) == 0
    assert call(k=0) == -1 and call(slots=0) == -1 and call(v=0) == -1
    assert call(dt=3) == -1
    assert call(kt=1023) == -3 and call(kh=4) == -3 and call(k=72) == -3
    assert L.mlxr_paged_append(None, 1, P(64), 1024, 128, P(64), 1024, 128, mx.BF16, P(64), None) == -1


def test_attention_refusals():
    L = paged._lib()

    def call(c=None, rows=1, heads=32, q=64, qdt=mx.BF16, qr=4096, qh=128, table=64, width=4, lens=64, window=0, out=64,
             odt=mx.BF16, ws=64, nb=1 << 40):
        c = c or _cache()
        return L.mlxr_paged_attention(ctypes.byref(c), rows, heads, P(q), qdt, qr, qh, P(table), width, width, P(lens), 0.1,
                                      window, P(out), odt, None, P(ws), nb, None)
    assert call(rows=-1) == -1 and call(heads=0) == -1 and call(rows=0) == 0
    assert call(rows=1 << 24) == -3 and call(heads=33) == -3
    assert call(qdt=mx.F32) == -1 and call(qdt=mx.F16) == -1 and call(odt=3) == -1 and call(window=-1) == -1
    for name in ("q", "table", "lens", "out"):
        assert call(**{name: 0}) == -1, name
    assert call(width=0) == -1 and call(width=100, ws=0) == -1
    assert call(q=72) == -3 and call(out=72) == -3 and call(qr=4095) == -3 and call(qh=4) == -3 and call(ws=72) == -3
    assert call(width=1 << 30) == -3
    assert call(c=_cache(k0=1 << 31)) == -3 and call(c=_cache(v2=1 << 31)) == -3
    assert call(width=100, nb=16) == -1 and "workspace" in L.mlxr_qgemm_last_error().decode()
    n = ctypes.c_size_t()
    c = _cache()
    assert L.mlxr_paged_attention_workspace_size(ctypes.byref(c), 1, 32, 4, None) == -1
    assert L.mlxr_paged_attention_workspace_size(ctypes.byref(c), 1, 32, 0, ctypes.byref(n)) == -1
    assert L.mlxr_paged_attention_workspace_size(ctypes.byref(c), 1, 32, 4, ctypes.byref(n)) == 0 and n.value == 0
    assert L.mlxr_paged_attention_workspace_size(ctypes.byref(c), 1, 32, 400, ctypes.byref(n)) == 0 and n.value > 0


def test_attention_limits():
    """Just within the limits, and just past them."""
    L, n = paged._lib(), ctypes.c_size_t()

    def size(rows=1, heads=8, width=4, **change):
        return L.mlxr_paged_attention_workspace_size(ctypes.byref(_cache(**change)), rows, heads, width, ctypes.byref(n))
    assert size(rows=(1 << 21) - 8) == 0 and size(rows=(1 << 21) - 7) == -3
    assert size(heads=(1 << 24) - 64) == 0 and size(heads=(1 << 24) - 56) == -3
    assert size(k0=(1 << 31) - 8) == 0 and size(k0=1 << 31) == -3 and size(v2=(1 << 31) - 8) == 0 and size(v2=1 << 31) == -3
    assert size(width=(1 << 27) - 65) == 0 and size(width=(1 << 27) - 63) == -3


def test_resize_refusals():
    L = paged._lib()

    def call(rows=2, page=16, pages=10, table=64, stride=4, width=4, lens=64, want=128, free=64, count=64, lens_out=256,
             count_out=320, starts=64, slots=64, positions=64, tokens=3, refused=64):
        return L.mlxr_page_resize(rows, page, pages, P(table), stride, width, P(lens), P(want), P(free), P(count),
                                  P(lens_out), P(count_out), P(starts), P(slots), P(positions), tokens, P(refused), None)
    assert call(rows=-1) == -1 and call(page=0) == -1 and call(pages=0) == -1 and call(width=0) == -1 and call(tokens=-1) == -1
    for name in ("table", "lens", "want", "free", "count", "lens_out", "count_out", "starts", "slots", "positions", "refused"):
        assert call(**{name: 0}) == -1, name
    assert call(rows=4097) == -3 and call(stride=3) == -3 and call(pages=1 << 28) == -3
    assert call(rows=4096, width=1 << 16, stride=1 << 16) == -3
    assert call(lens_out=64) == -1 and call(count_out=64) == -1


def test_wrapper_refusals():
    import torch
    t = torch.zeros((2, 3), dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(mx.QGemmError, match="on a GPU"):
        mx.page_resize(t, one, one, one, one, 16, 1)
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    q = torch.zeros((2, 8, 64), dtype=torch.bfloat16)
    with pytest.raises(mx.QGemmError, match="on one GPU"):
        mx.paged_attention(q, k, k, t, one)
    with pytest.raises(mx.QGemmError, match="one shape"):
        mx.paged_attention(q, k, k[:2], t, one)
    with pytest.raises(mx.QGemmError, match="positive"):
        mx.PagedKVCache(1, 0, 16, 8, 128, 4, 64)


# ------------------------------------------------------------------------------ page tables

class Pool:
    """The definition of page_resize, row by row on lists."""

    def __init__(self, table, lens, free):
        self.table, self.lens, self.free = [list(r) for r in table], list(lens), list(free)

    def resize(self, want, page, width, tokens):
        def pages(n):
            return -(-n // page)
        stack = list(self.free)
        give = []
        for r, w in enumerate(want):
            if 0 <= w <= width * page and pages(w) < pages(self.lens[r]):
                give += self.table[r][pages(w):pages(self.lens[r])]
        stack += give
        asked, refused, slots, positions, starts, lens, got = 0, 0, [], [], [0], [], 0
        for r, w in enumerate(want):
            have = self.lens[r]
            ok = 0 <= w <= width * page
            need = pages(w) - pages(have) if ok else 0
            if need > 0:
                asked += need
                ok = asked <= len(stack)
                if ok:
                    for i in range(need):
                        self.table[r][pages(have) + i] = stack[len(stack) - 1 - got]
                        got += 1
            refused += not ok
            lens.append(w if ok else have)
            for t in range(have, lens[r]):
                slots.append(self.table[r][t // page] * page + t % page)
                positions.append(t)
            starts.append(len(slots))
        self.lens, self.free = lens, stack[:len(stack) - got]
        pad = [-1] * max(0, tokens - len(slots))
        return starts, (slots + pad)[:tokens], (positions + pad)[:tokens], refused


def _resize_case(cuda, rows, width, page, pages, steps, tokens, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    i32 = dict(dtype=torch.int32, device=cuda)
    table = torch.full((rows, width + 3), -7, **i32)[:, :width]  # rows further apart than they are wide
    free = torch.tensor(order, **i32)
    count = torch.tensor([pages], **i32)
    lens = torch.zeros(rows, **i32)
    pool = Pool(table.tolist(), lens.tolist(), order)
    for step in range(steps):
        kind = step % 4
        if kind == 0:  # prompts
            want = torch.randint(0, width * page + 1, (rows,), generator=g)
        elif kind == 1:  # a token each
            want = lens.cpu().long() + 1
        elif kind == 2:  # some end, some grow, some shrink by a few
            want = (lens.cpu().long() + torch.randint(-5, 9, (rows,), generator=g)).clamp(min=0)
            want[torch.rand(rows, generator=g) < 0.3] = 0
        else:  # out of range in places
            want = torch.randint(0, width * page + 1, (rows,), generator=g)
            want[::5] = -1
            want[1::7] = width * page + 1
        r = mx.page_resize(table, lens, want.to(**i32), free, count, page, tokens)
        starts, slots, positions, refused = pool.resize(want.tolist(), page, width, tokens)
        assert r.lens.tolist() == pool.lens
        assert r.free_count.tolist() == [len(pool.free)]
        assert free[:len(pool.free)].tolist() == pool.free
        assert r.starts.tolist() == starts
        assert r.slots.tolist() == slots and r.positions.tolist() == positions
        assert r.refused.tolist() == [refused]
        assert table.tolist() == pool.table
        lens, count = r.lens, r.free_count


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,page,pages,tokens", [
    (1, 1, 1, 1, 1), (1, 5, 16, 3, 80), (3, 4, 5, 9, 64), (17, 12, 16, 100, 3000), (64, 9, 8, 200, 70),
    (257, 6, 3, 700, 5000), (1025, 3, 16, 2000, 50000), (4096, 2, 4, 5000, 40000), (96, 64, 16, 4000, 100000),
    (5, 7, 16, 40, 0),
])
def test_resize_equals_the_definition(cuda, rows, width, page, pages, tokens):
    _resize_case(cuda, rows, width, page, pages, 9, tokens, rows * 31 + width)


@pytest.mark.gpu
@pytest.mark.parametrize("page,pages,width", [(2 ** 31 - 1, 1, 1), (2 ** 30, 1, 1), (1, 2000, 2000)])
def test_resize_at_the_ends_of_the_page_sizes(cuda, page, pages, width):
    """A page of all the tokens that 32 bits count, and pages of one token."""
    import torch
    most = width * page
    table = torch.full((1, width), -1, dtype=torch.int32, device=cuda)
    free = torch.arange(pages, dtype=torch.int32, device=cuda)

    def i32(*v):
        return torch.tensor(v, dtype=torch.int32, device=cuda)
    r = mx.page_resize(table, i32(0), i32(most), free, i32(pages), page, 3)
    assert r.lens.tolist() == [most] and r.free_count.tolist() == [0] and r.refused.tolist() == [0]
    assert r.starts.tolist() == [0, most] and r.positions.tolist() == [0, 1, 2]
    assert r.slots.tolist() == ([0, 1, 2] if page > 1 else [pages - 1, pages - 2, pages - 3])
    r = mx.page_resize(table, r.lens, i32(1), free, r.free_count, page, 3)
    assert r.lens.tolist() == [1] and r.free_count.tolist() == [pages - 1] and r.slots.tolist() == [-1] * 3
    r = mx.page_resize(table, r.lens, i32(0), free, r.free_count, page, 0)
    assert r.lens.tolist() == [0] and sorted(free.tolist()) == list(range(pages)) and r.free_count.tolist() == [pages]


@pytest.mark.gpu
def test_resize_of_no_rows(cuda):
    import torch
    i32 = dict(dtype=torch.int32, device=cuda)
    none = torch.zeros(0, **i32)
    r = mx.page_resize(torch.zeros((0, 4), **i32), none, none, torch.arange(6, **i32), torch.tensor([6], **i32), 16, 3)
    assert r.starts.tolist() == [0] and r.slots.tolist() == [-1] * 3 and r.free_count.tolist() == [6] and r.refused.tolist() == [0]


# ------------------------------------------------------------------------------ writes

def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}[name]


def _bits(t):
    import torch
    return t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16).cpu()


def _store(cuda, pages, heads, page, dim, dtype, token_major):
    """A store whose bytes are all 0x7f.. (NaN in every type), in either memory order."""
    import torch
    shape = (pages, page, heads, dim) if token_major else (pages, heads, page, dim)
    t = torch.empty(shape, dtype=_dt(dtype), device=cuda)
    t.view(torch.uint8).fill_(0x7f)
    if dtype != "f8":
        t.fill_(float("nan"))
    return t.permute(0, 2, 1, 3) if token_major else t


@pytest.mark.gpu
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cache", ["f16", "bf16", "f8"])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,page,token_major", [(1, 1, 16, 1, False), (37, 3, 80, 16, True), (300, 8, 128, 5, False)])
def test_append(cuda, x, cache, scaled, tokens, heads, dim, page, token_major):
    import torch
    g = torch.Generator().manual_seed(tokens + dim)
    pages = -(-2 * tokens // page) + 1
    new = [(torch.randn(tokens, heads, dim, generator=g) * s).to(_dt(x)).to(cuda) for s in (1.0, 200.0)]
    for t in new:
        t.view(-1)[:4] = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0])
    scale = [torch.rand(heads, generator=g).to(cuda) + 0.25 for _ in range(2)] if scaled else [None, None]
    stores = [_store(cuda, pages, heads, page, dim, cache, token_major) for _ in range(2)]
    want = [s.clone() for s in stores]
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    if tokens > 3:
        slots[1], slots[2], slots[3] = -1, pages * page, -(1 << 31)
    mx.paged_append(new[0], new[1], stores[0], stores[1], slots.to(cuda), *scale)
    for n, s, w, f in zip(new, stores, want, scale):
        v = n.float().cpu()
        if f is not None:
            v = v / f.cpu().view(1, -1, 1)
        if cache == "f8":
            v = v.clamp(-448, 448)  # NaN stays
        v = v.to(_dt(cache))
        w = w.cpu()
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                w[slot // page, :, slot % page] = v[t]
        got, ref = s.float().cpu(), w.float()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(got.nan_to_num(0.0), ref.nan_to_num(0.0))


@pytest.mark.gpu
def test_append_rounds_every_e4m3_value_and_middle(cuda):
    """All e4m3 values, the middles between neighbours and what lies beside those: nearest, ties to even."""
    import torch
    v = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (v[1:] + v[:-1]) / 2
    x = torch.cat([v, mid, torch.nextafter(mid, mid * 0), torch.nextafter(mid, mid * 2), torch.tensor([448.1, 1e30, 1e-30])])
    x = torch.cat([x, -x])
    x = torch.cat([x, torch.zeros(-x.numel() % 16)]).view(1, 1, -1)
    for at in range(0, x.shape[2], 256):
        part = x[:, :, at:at + 256].contiguous()
        k, s = part.to(cuda), torch.empty((1, 1, 1, part.shape[2]), dtype=torch.float8_e4m3fn, device=cuda)
        mx.paged_append(k, k, s, torch.empty_like(s), torch.zeros(1, dtype=torch.int32, device=cuda))
        assert torch.equal(s.float().cpu().view(-1), part.clamp(-448, 448).to(torch.float8_e4m3fn).float().view(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["bf16", "f16", "f8"])
def test_append_divides_as_division_does(cuda, cache):
    """Quotients over the whole range of fp32, infinite and NaN ones, scales of zero, subnormal and infinite."""
    import torch
    g = torch.Generator().manual_seed(7)
    scales = torch.cat([torch.tensor([0.0, -0.0, 1e-44, 1e-38, 3e38, float("inf"), float("nan"), -0.3, 1.0, 3.0]),
                        (torch.rand(54, generator=g) * 2 - 1) * 2.0 ** torch.randint(-126, 127, (54,), generator=g)])
    x = (torch.rand(40, 64, 64, generator=g) * 2 - 1) * 2.0 ** torch.randint(-140, 127, (40, 64, 64), generator=g)
    x[1] = torch.rand(64, 64, generator=g) * scales[:, None] * 3
    x[0, :, :6] = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), 3.4e38])
    store = torch.zeros((1, 64, 40, 64), dtype=_dt(cache), device=cuda)
    slots = torch.arange(40, dtype=torch.int32, device=cuda)
    s = scales.to(cuda)
    mx.paged_append(x.to(cuda), x.to(cuda), store, torch.empty_like(store), slots, s, s)
    q = x / scales[None, :, None]
    want = (q.clamp(-448, 448) if cache == "f8" else q).to(_dt(cache)).float()
    got = store[0].permute(1, 0, 2).float().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0, 1e39, -1e39), want.nan_to_num(0.0, 1e39, -1e39))


@pytest.mark.gpu
def test_append_of_every_bf16_value_divided_to_e4m3(cuda):
    """All 65536 values by scales of ordinary size, those among them whose multiples lie next to middles of e4m3 values; zeros
    keep their sign."""
    import torch
    g = torch.Generator().manual_seed(8)
    near = [(2 ** 20 * m + e) * 2.0 ** (k - 23) for m in range(9, 16) for e in (-3, -1, 1, 2) for k in (-6, 5)]
    scales = torch.tensor((near + [1.0, -0.125, 3.0, 448.0])[:60] + [2.0 ** -39, 2.0 ** 39, 2.0 ** -41, 2.0 ** 41])
    assert scales.shape == (64,)
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)[torch.randperm(65536, generator=g)]
    x = x.view(1024, 1, 64).expand(1024, 64, 64)
    store = torch.zeros((32, 64, 32, 64), dtype=torch.float8_e4m3fn, device=cuda)
    slots = torch.arange(1024, dtype=torch.int32, device=cuda)
    s = scales.to(cuda)
    mx.paged_append(x.to(cuda), x.to(cuda), store, torch.empty_like(store), slots, s, s)
    want = (x.float() / scales[None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    got = store.permute(0, 2, 1, 3).reshape(1024, 64, 64).cpu()
    nan = torch.isnan(want.float())
    assert torch.equal(torch.isnan(got.float()), nan)
    assert torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


@pytest.mark.gpu
def test_append_takes_slices_of_a_fused_projection(cuda):
    import torch
    heads, dim, n, page, pages = 4, 64, 9, 16, 3
    fused = torch.randn(n, 5 * heads * dim, device=cuda).to(torch.bfloat16)
    k, v = (fused[:, i * heads * dim:(i + 1) * heads * dim].view(n, heads, dim) for i in (3, 4))
    layers = torch.zeros((2, 2, pages, heads, page, dim), dtype=torch.bfloat16, device=cuda)
    slots = torch.arange(20, 20 + n, dtype=torch.int32, device=cuda)
    mx.paged_append(k, v, layers[1, 0], layers[1, 1], slots)
    flat = layers.permute(0, 1, 2, 4, 3, 5).reshape(2, 2, pages * page, heads, dim)
    assert torch.equal(flat[1, 0, 20:20 + n], k) and torch.equal(flat[1, 1, 20:20 + n], v)
    assert not flat[0].any() and not flat[1, :, :20].any() and not flat[1, :, 20 + n:].any()
    odd = fused[:, 1:1 + heads * dim].view(n, heads, dim)  # rows off 16 bytes: copied first
    mx.paged_append(odd, odd, layers[0, 0], layers[0, 1], slots)
    assert torch.equal(layers[0, 0].permute(0, 2, 1, 3).reshape(pages * page, heads, dim)[20:20 + n], odd)


# ------------------------------------------------------------------------------ attention

def _fill(cuda, lens, heads, dim, page, cache, token_major, seed, spread=1.0):
    """Stores that hold NaN wherever no row has a token, the table, and the rows' keys and values in
    float64 (lists of [len, heads, dim])."""
    import torch
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lens]
    pages, width = sum(held) + 2, max(max(held), 1) + 1
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    table[:, -1] = 1 << 30
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    both, rows = [], []
    for which in range(2):
        s = torch.full((pages, heads, page, dim), float("nan"))
        mine = []
        for r, n in enumerate(lens):
            v = (torch.randn(n, heads, dim, generator=g) * spread).to(_dt(cache)).float()
            full = torch.full((held[r] * page, heads, dim), float("nan"))
            full[:n] = v
            if held[r]:
                s[table[r, :held[r]].long()] = full.view(held[r], page, heads, dim).permute(0, 2, 1, 3)
            mine.append(v.double())
        s = s.to(_dt(cache)).to(cuda)
        if token_major:
            s = s.view(torch.uint8).view(pages, heads, page, -1).permute(0, 2, 1, 3).contiguous().view(_dt(cache)) \
                .permute(0, 2, 1, 3)
        both.append(s)
        rows.append(mine)
    return both, table.to(cuda), rows


def _attend64(q, keys, values, lens, window, scale, ks=None, vs=None):
    """(out, lse) of the definition in float64, and the largest |value| of each row."""
    import torch
    q = q.double().cpu()
    rows, heads, dim = q.shape
    kv = keys[0].shape[1]
    out, lse = torch.zeros_like(q), torch.full((rows, heads), -math.inf, dtype=torch.float64)
    for r, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        if n - first <= 0:
            continue
        for h in range(heads):
            j = h // (heads // kv)
            k, v = keys[r][first:n, j], values[r][first:n, j]
            s = (k @ q[r, h]) * (scale * (1.0 if ks is None else float(ks[j])))
            lse[r, h] = torch.logsumexp(s, 0)
            out[r, h] = torch.softmax(s, 0) @ v * (1.0 if vs is None else float(vs[j]))
    return out, lse


def _check(got, ref, values, lens, odt, vs=None):
    """Weights are off by up to about 2^-13 relative: a score of size up to ~100 (in units of log2) is
    rounded to fp32 and summed over at most 256 products of fp32 accumulation (256 * 2^-24 of the
    sum of magnitudes, ~100), the weight itself to 2^-17 (bf16 in two parts) or better.  An average
    of values is then off by twice that times the largest value; the output is rounded once."""
    import torch
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[odt]
    worst = 0.0
    for r, n in enumerate(lens):
        if n <= 0:
            assert not got[r].any()
            continue
        top = float(values[r].abs().max()) * (1.0 if vs is None else float(vs.max()))
        tol = 2.0 ** -10 * top * 0.25 + half * ref[r].abs() + (2.0 ** -25 if odt == "f16" else 0.0)
        worst = max(worst, float(((got[r] - ref[r]).abs() / tol).max()))
    assert worst <= 1.0, worst


def _run(cuda, lens, heads, kv, dim, page, dtype, cache, window=0, token_major=False, out="f32", seed=0, spread=1.0, scale=None):
    import torch
    g = torch.Generator().manual_seed(seed + 5)
    (k, v), table, (keys, values) = _fill(cuda, lens, kv, dim, page, cache, token_major, seed, spread)
    q = (torch.randn(len(lens), heads, dim, generator=g) * 2).to(_dt(dtype)).to(cuda)
    ks = vs = None
    if cache == "f8":
        ks, vs = torch.rand(kv, generator=g) + 0.5, torch.rand(kv, generator=g) + 0.5
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    sc = dim ** -0.5 if scale is None else scale
    got, lse = mx.paged_attention(q, k, v, table, lt, scale=scale, window=window, out_dtype=_dt(out), return_lse=True,
                                  k_scale=None if ks is None else ks.to(cuda), v_scale=None if vs is None else vs.to(cuda))
    ref, ref_lse = _attend64(q, keys, values, lens, window, sc, ks, vs)
    _check(got, ref, values, lens, out, vs)
    lse = lse.double().cpu()
    for r, n in enumerate(lens):
        if n <= 0:
            assert (lse[r] == -math.inf).all()
        else:
            assert float((lse[r] - ref_lse[r]).abs().max()) <= 2.0 ** -12 * max(1.0, float(ref_lse[r].abs().max()))


LENS = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 64, 100, 257, 1000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8"), ("f16", "f8")])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (32, 4, 64, 16), (4, 4, 256, 32), (7, 1, 80, 8), (33, 1, 128, 24),
                                               (16, 1, 16, 16), (10, 2, 208, 5), (3, 3, 48, 1), (20, 4, 128, 7)])
@pytest.mark.parametrize("token_major", [False, True])
def test_attention(cuda, dtype, cache, heads, kv, dim, page, token_major):
    _run(cuda, LENS, heads, kv, dim, page, dtype, cache, token_major=token_major, seed=heads + dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [8, 24, 40, 56, 72, 80, 88, 96, 104, 120, 136, 248])
def test_attention_dims_of_eight(cuda, dim):
    _run(cuda, [1, 40, 333, 0], 6, 2, dim, 16, "bf16", "bf16", seed=dim)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 8, 31, 32, 33, 100, 5000])
@pytest.mark.parametrize("page", [16, 3])
def test_attention_window(cuda, window, page):
    _run(cuda, LENS, 8, 2, 64, page, "bf16", "bf16", window=window, seed=window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8")])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (33, 1, 128, 8), (4, 4, 256, 6), (6, 2, 80, 16)])
@pytest.mark.parametrize("window", [1100, 2049, 4000])
def test_attention_window_of_cut_rows(cuda, dtype, cache, heads, kv, dim, page, window):
    """Windows of more than 256 KiB a head of few rows: the rows are cut, and what is in the window is joined; rows shorter
    than it, and empty ones, among them.  Then the same rows behind a table that could hold many more."""
    import torch
    lens = [5000, 0, 700, 3001, 1, window, window + 1]
    g = torch.Generator().manual_seed(window)
    (k, v), table, (keys, values) = _fill(cuda, lens, kv, dim, page, cache, page == 8, window + dim)
    q = torch.randn(len(lens), heads, dim, generator=g).to(_dt(dtype)).to(cuda)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    ref, ref_lse = _attend64(q, keys, values, lens, window, dim ** -0.5)
    for t in (table, torch.nn.functional.pad(table, (0, 30000 // page), value=-1)):
        got, lse = mx.paged_attention(q, k, v, t, lt, window=window, out_dtype=torch.float32, return_lse=True)
        _check(got, ref, values, lens, "f32")
        assert (lse[1] == -math.inf).all()
        held = [r for r, n in enumerate(lens) if n]
        assert float((lse[held].double().cpu() - ref_lse[held]).abs().max()) < 1e-3

@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_attention_output_types(cuda, out):
    _run(cuda, [5, 0, 700], 8, 2, 128, 16, "bf16", "bf16", out=out)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1], [0], [5], [40000], [9000, 1], [0, 0, 20000, 3, 0], [33] * 300, [0] * 40 + [12000]])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_split_over_the_length(cuda, lens, dtype):
    _run(cuda, lens, 8, 2, 64, 16, dtype, dtype, seed=len(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8")])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (33, 1, 64, 8), (40, 2, 80, 5), (4, 4, 256, 32)])
def test_attention_cut_and_uncut(cuda, dtype, cache, heads, kv, dim, page):
    """The same rows behind a table that holds little more than they need and one that could hold 40000 tokens."""
    import torch
    lens = [0, 1, 33, 150, 64]
    (k, v), table, (keys, values) = _fill(cuda, lens, kv, dim, page, cache, False, 11)
    wide = torch.full((len(lens), 40000 // page), -5, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table
    q = torch.randn(len(lens), heads, dim, device=cuda).to(_dt(dtype))
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    ref, ref_lse = _attend64(q, keys, values, lens, 0, dim ** -0.5)
    for t in (table, wide):
        got, lse = mx.paged_attention(q, k, v, t, lt, out_dtype=torch.float32, return_lse=True)
        _check(got, ref, values, lens, "f32")
        assert (lse[0] == -math.inf).all() and float((lse[1:].double().cpu() - ref_lse[1:]).abs().max()) < 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8"), ("f16", "f8")])
@pytest.mark.parametrize("heads,dim,page,window", [(16, 16, 8, 0), (32, 48, 16, 0), (16, 64, 16, 0), (32, 64, 40, 37), (16, 80, 16, 0),
                                                   (16, 96, 8, 300), (32, 112, 32, 0), (48, 128, 16, 0), (16, 128, 64, 100), (16, 256, 16, 0),
                                                   (16, 80, 6, 0)])
@pytest.mark.parametrize("token_major", [False, True])
def test_attention_that_fills_the_device(cuda, dtype, cache, heads, dim, page, window, token_major):
    """As many kv heads of all rows as there are CUs: keys go through LDS where pages allow it."""
    _run(cuda, LENS, heads, 16, dim, page, dtype, cache, window=window, token_major=token_major, seed=heads + dim + page)


@pytest.mark.gpu
def test_attention_of_many_rows(cuda):
    _run(cuda, [(i * 5) % 40 for i in range(5000)], 2, 1, 64, 16, "bf16", "bf16")
    _run(cuda, [(i * 7) % 50 for i in range(2500)], 4, 2, 64, 8, "bf16", "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_sharp_and_flat_scores(cuda, dtype):
    _run(cuda, [3000, 17], 4, 1, 128, 16, dtype, dtype, spread=1.5, scale=0.35)  # one token takes nearly all
    _run(cuda, [3000, 17], 4, 1, 128, 16, dtype, dtype, scale=0.0)  # the mean


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_of_one_large_and_many_tiny_weights(cuda, dtype):
    """One score 11.5 above 30000 equal ones: together they outweigh it only in the sum, each is 2^-17."""
    import torch
    n, dim = 30000, 64
    k = torch.zeros((n // 16 + 1, 1, 16, dim), dtype=_dt(dtype), device=cuda)
    v = torch.ones_like(k)
    k[0, 0, 3, 0] = 11.5
    v[0, 0, 3] = -1.0
    q = torch.zeros((1, 1, dim), dtype=_dt(dtype), device=cuda)
    q[0, 0, 0] = 1.0
    table = torch.arange(k.shape[0], dtype=torch.int32, device=cuda).view(1, -1)
    got = mx.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device=cuda), scale=1.0, out_dtype=torch.float32)
    w = math.exp(11.5)
    assert abs(float(got[0, 0, 0]) - (n - 1 - w) / (n - 1 + w)) < 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8"), ("f16", "f8")])
@pytest.mark.parametrize("dim", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("pages", [0, 2500])
def test_attention_weights_have_the_bits_of_fp32(cuda, dtype, cache, dim, pages):
    """Value t is 1 in dim t and 0 elsewhere, so an output element is one weight: off by 2^-19 of itself at most.
    Scores lie in [-1, 1], so that in units of log2 (below 1.5, with f16's shift of 14 below 16) the scale, the score
    and the two sums of the exponent are off by 2 * 2^-24 * 1.5 + 2 * 2^-21, times ln 2; the exponential, its parts, the sum of
    dim weights, two rescalings and the division by 2^-23, 2^-22, 2^-22, 2^-22 and 2^-22: 2^-19 in all."""
    import torch
    g = torch.Generator().manual_seed(dim)
    page, heads = 16, 4
    held = -(-dim // page)
    s = (torch.randint(-128, 129, (dim,), generator=g) / 128.0).to(_dt(cache))
    k, v = torch.zeros(2, held * page, dim)
    k[:dim, 0] = s.float()
    v[torch.arange(dim), torch.arange(dim)] = 1.0
    k, v = (t.view(held, 1, page, dim).to(_dt(cache)).to(cuda) for t in (k, v))
    q = torch.zeros(1, heads, dim)
    q[0, :, 0] = torch.tensor([1.0, 0.5, -1.0, 0.75])
    table = torch.full((1, max(held, pages)), -1, dtype=torch.int32, device=cuda)
    table[0, :held] = torch.arange(held, dtype=torch.int32, device=cuda)
    got = mx.paged_attention(q.to(_dt(dtype)).to(cuda), k, v, table, torch.tensor([dim], dtype=torch.int32, device=cuda), scale=1.0,
                             out_dtype=torch.float32)[0].double().cpu()
    ref = torch.softmax(q[0, :, :1].double() * s.double()[None, :], 1)
    assert float(((got - ref).abs() / ref).max()) <= 2.0 ** -19


@pytest.mark.gpu
def test_attention_infinite_scores(cuda):
    """Scores of -inf have no weight, wherever they lie; a row of nothing else, or with +inf, is NaN as by
    the formula; other rows are not touched."""
    import torch
    n, dim, page = 600, 64, 16
    k = torch.zeros((3 * 38, 1, page, dim), dtype=torch.bfloat16, device=cuda)
    v = torch.randn(k.shape, device=cuda).to(torch.bfloat16)
    flat = k.view(3, 38 * page, dim)
    flat[0, :300, 0] = float("-inf")
    flat[1, :n, 0] = float("-inf")
    flat[2, 77, 0] = float("inf")
    q = torch.ones((4, 2, dim), dtype=torch.bfloat16, device=cuda)
    table = torch.arange(3 * 38, dtype=torch.int32, device=cuda).view(3, 38)
    table = torch.cat([table, table[:1]])
    lens = torch.tensor([n, n, n, 300], dtype=torch.int32, device=cuda)
    got = mx.paged_attention(q, k, v, table, lens, out_dtype=torch.float32).cpu()
    mean = v.view(3, -1, dim)[0, 300:n].double().mean(0).cpu()
    assert float((got[0] - mean).abs().max()) < 1e-4
    assert torch.isnan(got[1]).all() and torch.isnan(got[2]).all() and torch.isnan(got[3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("width", [5, 400])
def test_attention_infinite_values(cuda, dtype, width):
    """An infinite value makes its dimension of the output infinite, not NaN; NaN values make it NaN; the other
    dimensions and rows stay as they are."""
    import torch
    n, dim = 70, 64
    k = torch.randn((10, 1, 16, dim), device=cuda).to(_dt(dtype))
    v = torch.randn((10, 1, 16, dim), device=cuda).to(_dt(dtype))
    q = torch.randn((2, 3, dim), device=cuda).to(_dt(dtype))
    table = torch.full((2, width), -1, dtype=torch.int32, device=cuda)
    table[:, :5] = torch.arange(10, dtype=torch.int32, device=cuda).view(2, 5)
    lens = torch.tensor([n, n], dtype=torch.int32, device=cuda)
    plain = mx.paged_attention(q, k, v, table, lens, out_dtype=torch.float32)
    v[1, 0, 3, 5], v[2, 0, 0, 7], v[0, 0, 9, 8] = float("inf"), float("-inf"), float("nan")
    got = mx.paged_attention(q, k, v, table, lens, out_dtype=torch.float32)
    assert (got[0, :, 5] == float("inf")).all() and (got[0, :, 7] == float("-inf")).all() and torch.isnan(got[0, :, 8]).all()
    got[0, :, [5, 7, 8]] = plain[0, :, [5, 7, 8]]
    assert torch.equal(got, plain)


@pytest.mark.gpu
def test_single_places_have_any_stride(cuda):
    """Stores of one page, one head or one token, whose strides torch may have set to anything."""
    import torch
    q = torch.randn(1, 2, 64, device=cuda).to(torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32, device=cuda)
    zero = torch.zeros(1, dtype=torch.int32, device=cuda)
    for shape in ((1, 1, 16, 64), (3, 1, 8, 64), (4, 2, 1, 64), (1, 1, 1, 64)):
        k, v = torch.randn(2, *shape, device=cuda).to(torch.bfloat16)
        odd = [torch.as_strided(t, shape, [s if n > 1 else 3 for s, n in zip(t.stride(), shape)]) for t in (k, v)]
        mx.paged_append(q[:, :shape[1]], q[:, :shape[1]], *odd, zero)
        assert torch.equal(k[0, :, 0], q[0, :shape[1]])
        table = torch.as_strided(zero, (1, 1), (0, 1))
        a = mx.paged_attention(q, *odd, table, one)
        assert torch.equal(a, mx.paged_attention(q, k, v, table, one))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 6])
def test_attention_leaves_pages_outside_the_cache_out(cuda, page):
    import torch
    lens = [100, 3 * page]
    (k, v), table, (keys, values) = _fill(cuda, lens, 2, 64, page, "bf16", False, 3)
    bad = {0: [1, 3], 1: [0, 1, 2]}
    kept = []
    for r, pages in bad.items():
        for j in pages:
            table[r, j] = [-1, 1 << 30, k.shape[0]][j % 3]
        kept.append([t for t in range(lens[r]) if t // page not in pages])
    q = torch.randn(2, 4, 64, device=cuda).to(torch.bfloat16)
    got = mx.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=cuda), out_dtype=torch.float32)
    ref, _ = _attend64(q[:1], [keys[0][kept[0]]], [values[0][kept[0]]], [len(kept[0])], 0, 0.125)
    _check(got[:1], ref, values[:1], lens[:1], "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["bf16", "f8"])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 64, 16), (20, 1, 128, 8), (4, 2, 80, 6), (2, 2, 256, 16)])
@pytest.mark.parametrize("width", [0, 40000])
@pytest.mark.parametrize("window", [0, 33])
def test_attention_rows_without_a_page_in_the_cache(cuda, cache, heads, kv, dim, page, width, window):
    """Rows that have a length, but none of whose tokens (none of whose window) lies in the cache, are empty: zeros, -inf."""
    import torch
    lens = [100, 3 * page, 700, 650, 90, 1]
    (k, v), table, (keys, values) = _fill(cuda, lens, kv, dim, page, cache, False, 21)
    table = torch.nn.functional.pad(table, (0, max(0, width // page - table.shape[1])), value=-1)
    table[1, :3] = torch.tensor([-1, k.shape[0], 1 << 30], dtype=torch.int32, device=cuda)  # none
    table[3, :] = -5  # none of many
    table[2, (lens[2] - 33) // page:] = -1  # none of the window's
    kept = (lens[2] - 33) // page * page
    empty = [1, 3] + ([2] if window else [])
    q = torch.randn(len(lens), heads, dim, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    vs = torch.full((kv,), 2.0, device=cuda) if cache == "f8" else None
    got, lse = mx.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=cuda), window=window,
                                  v_scale=vs, out_dtype=torch.float32, return_lse=True)
    assert not got[empty].any() and (lse[empty] == -math.inf).all()
    if not window:  # what is left of row 2
        keys[2], values[2], lens[2] = keys[2][:kept], values[2][:kept], kept
    rest = [r for r in range(len(lens)) if r not in empty]
    ref, ref_lse = _attend64(q[rest], [keys[r] for r in rest], [values[r] for r in rest], [lens[r] for r in rest], window, dim ** -0.5, vs=vs)
    _check(got[rest], ref, [values[r] for r in rest], [lens[r] for r in rest], "f32", vs)
    assert float((lse[rest].double().cpu() - ref_lse).abs().max()) < 1e-3


@pytest.mark.gpu
def test_attention_lengths_past_the_table_and_negative(cuda):
    import torch
    (k, v), table, (keys, values) = _fill(cuda, [64, 64, 5], 2, 64, 16, "bf16", False, 4)
    q = torch.randn(3, 4, 64, device=cuda).to(torch.bfloat16)
    lens = torch.tensor([64, 1 << 30, -3], dtype=torch.int32, device=cuda)
    got = mx.paged_attention(q, k, v, table[:, :4], lens, out_dtype=torch.float32)
    ref, _ = _attend64(q, keys, values, [64, 64, 0], 0, 0.125)
    _check(got, ref, values, [64, 64, 0], "f32")


@pytest.mark.gpu
def test_attention_strides(cuda):
    """Queries from a fused projection, stores that are one layer of a larger tensor with keys and
    values side by side, a table that is a part of a wider one: the same bits as of copies."""
    import torch
    heads, kv, dim, page, pages = 8, 2, 64, 16, 30
    fused = torch.randn(3, (heads + 2 * kv) * dim, device=cuda).to(torch.float16)
    q = fused[:, :heads * dim].view(3, heads, dim)
    both = torch.randn(2, pages, 2, page, kv, dim, device=cuda).to(torch.float16)
    k, v = (both[1, :, i].permute(0, 2, 1, 3) for i in (0, 1))
    wide = torch.stack([torch.randperm(pages, device=cuda) for _ in range(3)]).to(torch.int32)
    lens = torch.tensor([100, 1, 77], dtype=torch.int32, device=cuda)
    a = mx.paged_attention(q, k, v, wide[:, 5:15], lens)
    b = mx.paged_attention(q.contiguous(), k.contiguous(), v.contiguous(), wide[:, 5:15].contiguous(), lens)
    assert torch.equal(a, b)
    odd = torch.randn(3 * heads * dim + 1, device=cuda).to(torch.float16)[1:].view(3, heads, dim)  # off 16 bytes
    assert torch.equal(mx.paged_attention(odd, k, v, wide, lens), mx.paged_attention(odd.clone(), k, v, wide, lens))


@pytest.mark.gpu
def test_attention_past_four_gigabytes(cuda):
    """Pages whose addresses lie more than 2^32 elements into the stores."""
    import torch
    heads, kv, dim, page = 8, 8, 128, 16
    pages = (1 << 32) // (kv * dim * page) + 200
    k = torch.empty((pages, kv, page, dim), dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    n = 1000
    held = -(-n // page)
    ids = torch.arange(pages - held, pages).flip(0)
    ids[5] = 0
    small = torch.randn(2, held, kv, page, dim, device=cuda).to(torch.bfloat16)
    k[ids.to(cuda)], v[ids.to(cuda)] = small[0], small[1]
    q = torch.randn(1, heads, dim, device=cuda).to(torch.bfloat16)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    a = mx.paged_attention(q, k, v, ids.to(torch.int32).to(cuda).view(1, -1), lens)
    b = mx.paged_attention(q, small[0], small[1], torch.arange(held, dtype=torch.int32, device=cuda).view(1, -1), lens)
    assert torch.equal(a, b)
    slots = torch.tensor([pages * page - 1], dtype=torch.int32, device=cuda)
    mx.paged_append(q, q, k, v, slots)
    assert torch.equal(k[pages - 1, :, page - 1], q[0]) and torch.equal(v[pages - 1, :, page - 1], q[0])


@pytest.mark.gpu
def test_attention_repeats_its_bits_and_on_another_stream(cuda):
    import torch
    lens = [5000, 0, 33, 1200]
    (k, v), table, _ = _fill(cuda, lens, 2, 128, 16, "bf16", False, 9)
    q = torch.randn(4, 8, 128, device=cuda).to(torch.bfloat16)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    first = mx.paged_attention(q, k, v, table, lt)
    for _ in range(5):
        assert torch.equal(mx.paged_attention(q, k, v, table, lt), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = [mx.paged_attention(q, k, v, table, lt, stream=s) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(t, first) for t in got)


@pytest.mark.gpu
def test_cache_step_in_a_graph(cuda):
    """A decode step (resize, append, attend) captured once and replayed, the lengths growing on the
    device, against the same steps made eagerly."""
    import torch
    heads, kv, dim, page, rows, steps = 4, 2, 64, 16, 3, 40
    torch.manual_seed(2)
    inputs = torch.randn(steps, rows, heads + 2 * kv, dim, device=cuda).to(torch.bfloat16)

    def fresh():
        return mx.PagedKVCache(1, 20, page, kv, dim, rows, 100, device=cuda)

    def step(c, x):
        r = mx.page_resize(c.table, c.lens, c.lens + 1, c.free, c.free_count, page, rows)
        mx.paged_append(x[:, heads:heads + kv], x[:, heads + kv:], c.k[0], c.v[0], r.slots)
        out = mx.paged_attention(x[:, :heads], c.k[0], c.v[0], c.table, r.lens)
        c.lens.copy_(r.lens)
        c.free_count.copy_(r.free_count)
        return out
    eager = fresh()
    want = [step(eager, x).clone() for x in inputs]
    c, x = fresh(), inputs[0].clone()
    lens, count, table, free = c.lens.clone(), c.free_count.clone(), c.table.clone(), c.free.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c, x)
    torch.cuda.current_stream().wait_stream(side)
    c.lens.copy_(lens), c.free_count.copy_(count), c.table.copy_(table), c.free.copy_(free)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c, x)
    c.lens.copy_(lens), c.free_count.copy_(count), c.table.copy_(table), c.free.copy_(free)
    for i in range(steps):
        x.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
    assert c.lens.tolist() == [steps] * rows and c.lens.tolist() == eager.lens.tolist()


@pytest.mark.gpu
def test_paged_cache_class_in_a_graph(cuda):
    """A step through the class's methods, captured once: every replay goes on from where the one before it left the rows."""
    import torch
    heads, kv, dim, page, rows, steps = 4, 2, 64, 16, 3, 40
    torch.manual_seed(3)
    inputs = torch.randn(steps, rows, heads + 2 * kv, dim, device=cuda).to(torch.bfloat16)

    def step(c, x):
        r = c.resize(c.lens + 1, rows)
        c.append(0, x[:, heads:heads + kv], x[:, heads + kv:], r.slots)
        return c.attend(0, x[:, :heads]), r
    eager = mx.PagedKVCache(1, 20, page, kv, dim, rows, 100, device=cuda)
    want = [(out.clone(), r.slots.tolist(), r.positions.tolist()) for out, r in (step(eager, x) for x in inputs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(mx.PagedKVCache(1, 20, page, kv, dim, rows, 100, device=cuda), inputs[0])
    torch.cuda.current_stream().wait_stream(side)
    c, x = mx.PagedKVCache(1, 20, page, kv, dim, rows, 100, device=cuda), inputs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, r = step(c, x)
    for i in range(steps):
        x.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert r.positions.tolist() == [i] * rows == want[i][2], i
        assert r.slots.tolist() == want[i][1] and torch.equal(out, want[i][0]), i
        assert c.lens.tolist() == [i + 1] * rows
    assert int(c.free_count) == int(eager.free_count) and c.table.tolist() == eager.table.tolist()


@pytest.mark.gpu
def test_paged_cache_class(cuda):
    import torch
    rows, kv, heads, dim, page = 3, 2, 4, 64, 8
    c = mx.PagedKVCache(2, 12, page, kv, dim, rows, 40, device=cuda)
    torch.manual_seed(1)
    held = [[[] for _ in range(rows)] for _ in range(2)]
    for want in ([5, 0, 17], [6, 9, 18], [0, 10, 19], [3, 11, 0], [30, 0, 40]):
        before = c.lens.tolist()
        r = c.resize(torch.tensor(want, dtype=torch.int32, device=cuda), 128)
        assert r.refused.tolist() == [0]
        n = int(r.starts[-1])
        for layer in range(2):
            k, v = torch.randn(2, 128, kv, dim, device=cuda).to(torch.bfloat16)
            c.append(layer, k, v, r.slots)
            st = r.starts.tolist()
            for i in range(rows):
                held[layer][i] = held[layer][i][:want[i]] + [(k[t].double().cpu(), v[t].double().cpu()) for t in range(st[i], st[i + 1])]
            q = torch.randn(rows, heads, dim, device=cuda).to(torch.bfloat16)
            got = c.attend(layer, q, out_dtype=torch.float32)
            empty = torch.zeros(0, kv, dim, dtype=torch.float64)
            keys = [torch.stack([x[0] for x in h]) if h else empty for h in held[layer]]
            values = [torch.stack([x[1] for x in h]) if h else empty for h in held[layer]]
            ref, _ = _attend64(q, keys, values, want, 0, dim ** -0.5)
            _check(got, ref, values, want, "f32")
        assert c.lens.tolist() == want and n == sum(max(0, w - b) for w, b in zip(want, before))
        assert int(c.free_count) == 12 - sum(-(-w // page) for w in want)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [128, 256])
def test_attention_of_as_many_rows_as_are_cut(cuda, dim):
    """4096 rows of a table that could hold long ones: their tiles are summed up beside the keys in LDS; 4097 rows are not cut."""
    import torch
    lens = [(i * 11) % 70 for i in range(4097)]
    (k, v), table, (keys, values) = _fill(cuda, lens, 1, dim, 16, "bf16", False, 3, 1.0)
    wide = torch.nn.functional.pad(table, (0, 300), value=-1)
    q = torch.randn(4097, 2, dim, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(cuda)
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)
    ref, _ = _attend64(q, keys, values, lens, 0, dim ** -0.5)
    for n in (4096, 4097):
        got = mx.paged_attention(q[:n], k, v, wide[:n], lt[:n], out_dtype=torch.float32)
        _check(got, ref[:n], values[:n], lens[:n], "f32")


@pytest.mark.gpu
def test_attend_with_a_bound_on_the_lengths(cuda):
    """A bound that holds changes the split, not the result; what lies past one that does not is left out."""
    import torch
    c = mx.PagedKVCache(1, 600, 8, 2, 64, 2, 2400, device=cuda)
    r = c.resize(torch.tensor([37, 5], dtype=torch.int32, device=cuda), 64)
    torch.manual_seed(2)
    k, v = torch.randn(2, 64, 2, 64, device=cuda).to(torch.bfloat16)
    c.append(0, k, v, r.slots)
    q = torch.randn(2, 4, 64, device=cuda).to(torch.bfloat16)
    keys, values = ([t[:37].double().cpu(), t[37:42].double().cpu()] for t in (k, v))
    for longest, lens in ((None, [37, 5]), (37, [37, 5]), (40, [37, 5]), (16, [16, 5]), (0, [8, 5])):
        got = c.attend(0, q, longest=longest, out_dtype=torch.float32)
        ref, _ = _attend64(q, [t[:n] for t, n in zip(keys, lens)], [t[:n] for t, n in zip(values, lens)], lens, 0, 0.125)
        _check(got, ref, [t[:n] for t, n in zip(values, lens)], lens, "f32")


@pytest.mark.gpu
def test_wrapper_refusals_on_the_gpu(cuda):
    import torch
    i32 = dict(dtype=torch.int32, device=cuda)
    t, two, one = torch.zeros((2, 3), **i32), torch.zeros(2, **i32), torch.ones(1, **i32)
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, device=cuda)
    q = torch.zeros((2, 8, 64), dtype=torch.bfloat16, device=cuda)

    def refused(match, code, call, *args, **kw):
        with pytest.raises(mx.QGemmError, match=match) as e:
            call(*args, **kw)
        assert e.value.code == code
    refused("table must", -1, mx.page_resize, t.long(), two, two, one, one, 16, 1)
    refused("table must", -1, mx.page_resize, t.t(), two, two, one, one, 16, 1)
    refused("lens must", -3, mx.page_resize, t, one, two, one, one, 16, 1)
    refused("want must", -1, mx.page_resize, t, two, two.float(), one, one, 16, 1)
    refused("want must", -1, mx.page_resize, t, two, two.cpu(), one, one, 16, 1)
    refused("free_count must", -3, mx.page_resize, t, two, two, one, two, 16, 1)
    refused("tokens must not", -1, mx.page_resize, t, two, two, one, one, 16, -1)
    refused("page_size must", -1, mx.page_resize, t, two, two, one, one, 0, 1)
    refused("queries must be", -3, mx.paged_attention, q[..., :32], k, k, t, two)
    refused("on the cache's GPU", -1, mx.paged_attention, q.cpu(), k, k, t, two)
    refused("must have the cache's type", -1, mx.paged_attention, q.half(), k, k, t, two)
    refused("unsupported dtype", -1, mx.paged_attention, q, k.float(), k.float(), t, two)
    refused("one row per query", -3, mx.paged_attention, q, k, k, t[:1], two)
    refused("lens must", -3, mx.paged_attention, q, k, k, t, one)
    refused("multiple of kv_heads", -3, mx.paged_attention, q[:, :7], k, k, t, two)
    refused("window must not", -1, mx.paged_attention, q, k, k, t, two, window=-1)
    refused("window must not", -1, mx.paged_attention, q, k, k, t, two, window=1 << 32)
    refused("out must be", -1, mx.paged_attention, q, k, k, t, two, out=q[:1])
    refused("k_scale must", -3, mx.paged_attention, q, k, k, t, two, k_scale=torch.ones(3, device=cuda))
    refused("last dimension", -3, mx.paged_attention, q, k.transpose(2, 3), k.transpose(2, 3), t, two)
    refused("keys and values must be", -3, mx.paged_append, q, q, k, k, two)
    refused("one dtype", -1, mx.paged_append, q[:, :2], q[:, :2].float(), k, k, two)
    refused("slots must", -3, mx.paged_append, q[:, :2], q[:, :2], k, k, one)
    odd = torch.zeros(4 * 2 * 16 * 64 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(4, 2, 16, 64)
    refused("multiples of 16 bytes", -1, mx.paged_attention, q, odd, odd, t, two)
    empty = mx.paged_attention(q[:0], k, k, t[:0], two[:0])
    assert empty.shape == (0, 8, 64)
    mx.paged_append(q[:0, :2], q[:0, :2], k, k, two[:0])


@pytest.mark.gpu
def test_concurrent_calls_from_host_threads(cuda):
    """Four host threads, each with a stream of its own, make calls of every operator of the cache at once: the
    results of the same calls made alone, bit for bit."""
    import threading
    import torch
    lens = [3000, 0, 33, 1200]
    cases = []
    for cache, dim, page in (("bf16", 128, 16), ("f8", 64, 16), ("bf16", 256, 6)):
        (k, v), table, _ = _fill(cuda, lens, 2, dim, page, cache, False, dim)
        cases.append((k, v, table, torch.randn(4, 8, dim, device=cuda).to(torch.bfloat16)))
    lt = torch.tensor(lens, dtype=torch.int32, device=cuda)

    def work(stream):
        """Attention of the given stores, then resizes, writes and attention of a cache of the thread's own."""
        got = [mx.paged_attention(q, k, v, t, lt, stream=stream) for k, v, t, q in cases]
        got += [mx.paged_attention(q, k, v, t[:, :5], lt, window=40, stream=stream) for k, v, t, q in cases]
        with torch.cuda.stream(stream):
            c = mx.PagedKVCache(1, 60, 16, 2, 128, 4, 400, device=cuda)
            rows = torch.arange(128 * 2 * 128, device=cuda).view(128, 2, 128).remainder(63).sub(31).to(torch.bfloat16)
        for n in (1, 17, 90, 3):
            with torch.cuda.stream(stream):
                want = torch.arange(4, dtype=torch.int32, device=cuda) * n
            r = c.resize(want, 128, stream=stream)
            c.append(0, rows, rows, r.slots, stream=stream)
            got += [c.attend(0, cases[0][3], stream=stream), r.slots, r.positions, r.lens]
        stream.synchronize()
        return got
    want = work(torch.cuda.Stream())
    errors = []

    def thread():
        torch.cuda.set_device(cuda)
        stream = torch.cuda.Stream()
        for _ in range(5):
            if not all(torch.equal(a, b) for a, b in zip(work(stream), want)):
                errors.append("mismatch")
    threads = [threading.Thread(target=thread) for _ in range(4)]
    torch.cuda.synchronize()
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
