"""Tokens moved within a paged cache: accepted paths of drafted trees, copies and forks, against lists."""
import ctypes
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

def test_move_refusals():
    L = paged._lib()

    def accept(c=None, layers=2, kl=1 << 20, vl=1 << 20, rows=2, table=64, width=4, lens=64, starts=64, path=64, depth=3, counts=64,
               out=128):
        return L.mlxr_paged_accept(ctypes.byref(c or _cache()), layers, kl, vl, rows, P(table), width, width, P(lens), P(starts),
                                   P(path), depth, depth, P(counts), P(out), None)
    assert accept(rows=-1) == -1 and accept(depth=-1) == -1 and accept(width=0) == -1 and accept(layers=0) == -1
    assert accept(rows=0) == 0 and accept(rows=4097) == -3 and accept(width=1 << 28) == -3
    for name in ("table", "lens", "starts", "path", "counts", "out"):
        assert accept(**{name: 0}) == -1, name
    assert accept(out=64) == -1
    assert accept(kl=-8) == -3 and accept(vl=9) == -3 and accept(layers=1 << 20) == -3 and accept(c=_cache(head_dim=12)) == -3

    def copy(c=None, layers=2, kl=1 << 20, tokens=3, src=64, dst=128):
        return L.mlxr_paged_copy(ctypes.byref(c or _cache()), layers, kl, kl, tokens, P(src), P(dst), None)
    assert copy(tokens=-1) == -1 and copy(tokens=0) == 0 and copy(src=0) == -1 and copy(dst=0) == -1 and copy(tokens=(1 << 27) + 1) == -3
    assert copy(kl=4) == -3 and copy(layers=0) == -1 and copy(layers=40000) == -3 and copy(c=_cache(k_dev=None)) == -1

    def fork(rows=2, tokens=3, width=4, **at):
        p = dict(table=64, sources=64, starts=64, slots=64, positions=64)
        p.update(at)
        return L.mlxr_paged_fork(ctypes.byref(_cache()), 1, 0, 0, rows, P(p["table"]), width, width, P(p["sources"]), P(p["starts"]),
                                 P(p["slots"]), P(p["positions"]), tokens, None)
    assert fork(rows=-1) == -1 and fork(tokens=-1) == -1 and fork(width=0) == -1 and fork(rows=0) == 0 and fork(tokens=0) == 0
    assert fork(tokens=(1 << 27) + 1) == -3
    for name in ("table", "sources", "starts", "slots", "positions"):
        assert fork(**{name: 0}) == -1, name


def test_wrapper_refusals():
    import torch
    k, t = torch.zeros((2, 4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((2, 3), dtype=torch.int32)
    one = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(mx.QGemmError, match="on one GPU"):
        mx.paged_accept(k, k, t, one, one, t, one)
    with pytest.raises(mx.QGemmError, match="one shape"):
        mx.paged_copy(k, k[:1], one, one)
    with pytest.raises(mx.QGemmError, match="layers"):
        mx.paged_copy(k[0, 0], k[0, 0], one, one)


# ------------------------------------------------------------------------------ the kernels

def _stores(layers, pages, kv, page, dim, kind, token_major, seed):
    """Two stores whose bytes are random."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    size = {"f8": 1}.get(kind, 2)
    dt = {"f8": torch.float8_e4m3fn, "bf16": torch.bfloat16, "f16": torch.float16}[kind]
    got = []
    for _ in range(2):
        shape = (layers, pages, page, kv, dim * size) if token_major else (layers, pages, kv, page, dim * size)
        b = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g).view(dt)
        got.append(b.transpose(2, 3) if token_major else b)
    return got


def _bytes(t):
    import torch
    return t.contiguous().view(torch.uint8).cpu()


def _tables(lens, page, pages, seed, wide=0):
    import torch
    rng = random.Random(seed)
    order = rng.sample(range(pages), pages)
    wide = max([wide, 1] + [-(-n // page) for n in lens])
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    for r, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[r, i] = order.pop()
    return table


def _kept(n, path, count):
    got, last = [], -1
    for p in path[:max(count, 0)]:
        if not last < p < n:
            break
        got.append(p)
        last = p
    return got


LAYOUTS = [("bf16", 8, 128, 16, False), ("bf16", 3, 80, 5, True), ("f16", 1, 8, 1, False), ("f8", 2, 16, 64, True), ("f8", 8, 256, 16, False)]


def _i32(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("kind,kv,dim,page,token_major", LAYOUTS)
@pytest.mark.parametrize("depth,nodes", [(1, 1), (3, 7), (12, 64), (20, 25), (300, 600)])
def test_accept(kind, kv, dim, page, token_major, depth, nodes):
    import torch
    rng = random.Random(depth * 100 + page)
    rows, layers = 9, 3
    n = [rng.randrange(1, nodes + 1) for _ in range(rows)]
    n[3], n[5] = 0, nodes
    context = [rng.randrange(0, 40) for _ in range(rows)]
    context[0] = 0
    lens = [a + b for a, b in zip(context, n)]
    path = []
    for r in range(rows):
        p = sorted(rng.sample(range(n[r]), min(n[r], depth)))
        path.append(p + [-1] * (depth - len(p)))
    counts = [rng.randrange(0, depth + 1) for _ in range(rows)]
    counts[5], counts[6], counts[7] = depth, depth + 5, -2
    if depth > 2:
        path[2][1] = path[2][0]       # does not ascend
        path[4][depth // 2] = n[4]    # no node
        counts[2] = counts[4] = depth
        path[1][0], counts[1] = -1, depth
    pages = sum(-(-m // page) for m in lens) + 2
    k, v = _stores(layers, pages, kv, page, dim, kind, token_major, depth)
    table = _tables(lens, page, pages, 7)
    starts = [0]
    for m in n:
        starts.append(starts[-1] + m)
    before = [_bytes(k), _bytes(v)]
    got = mx.paged_accept(k, v, table.cuda(), _i32(lens), _i32(starts), _i32(path), _i32(counts))
    want = []
    for b in before:
        b = b.clone()
        for r in range(rows):
            at = lambda t: (int(table[r, t // page]), t % page)  # noqa: E731
            for j, p in enumerate(_kept(n[r], path[r], min(counts[r], depth))):
                (sp, st), (dp, d) = at(context[r] + p), at(context[r] + j)
                b[:, dp, :, d] = b[:, sp, :, st]
        want.append(b)
    assert got.tolist() == [context[r] + len(_kept(n[r], path[r], min(counts[r], depth))) for r in range(rows)]
    assert torch.equal(_bytes(k), want[0]) and torch.equal(_bytes(v), want[1])


@pytest.mark.gpu
def test_accept_leaves_out_bad_pages_and_lengths():
    import torch
    k, v = _stores(2, 6, 2, 4, 64, "bf16", False, 3)
    table = torch.tensor([[0, 99], [2, -1], [3, 4]], dtype=torch.int32)
    lens, starts = [8, 8, 2], [0, 6, 12, 17]  # the last row claims five drafts of two tokens
    path, counts = [[1, 5], [0, 1], [3, 4]], [2, 2, 2]
    before = [_bytes(k), _bytes(v)]
    got = mx.paged_accept(k, v, table.cuda(), _i32(lens), _i32(starts), _i32(path), _i32(counts))
    assert got.tolist() == [4, 4, 0]
    for t, b in zip((k, v), before):
        b[:, 0, :, 2] = b[:, 0, :, 3]  # row 0: node 1 from position 3 to 2; node 5 lies in a page outside the cache
        assert torch.equal(_bytes(t), b)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,kv,dim,page,token_major", LAYOUTS)
@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 500])
def test_copy(kind, kv, dim, page, token_major, tokens):
    import torch
    layers = 2
    pages = 2 * tokens // page + 3
    k, v = _stores(layers, pages, kv, page, dim, kind, token_major, tokens)
    rng = random.Random(tokens)
    slots = rng.sample(range(pages * page), 2 * tokens)
    src, dst = slots[:tokens], slots[tokens:]
    src = [rng.choice(src) for _ in src]  # one to many
    if tokens > 10:
        dst[3], src[5], dst[7], src[9] = -1, -7, pages * page, 1 << 30
    before = [_bytes(k), _bytes(v)]
    mx.paged_copy(k, v, _i32(src), _i32(dst))
    for t, b in zip((k, v), before):
        old = b.clone()
        for s, d in zip(src, dst):
            if 0 <= s < pages * page and 0 <= d < pages * page:
                b[:, d // page, :, d % page] = old[:, s // page, :, s % page]
        assert torch.equal(_bytes(t), b)
    one = [t[1] for t in (k, v)]  # one layer's stores, and none to copy
    mx.paged_copy(*one, _i32([]), _i32([]))


@pytest.mark.gpu
def test_cache_forks_accepts_and_frees():
    """A row becomes three; drafts of all of them are appended, a path of each is accepted, the pages of the others go back."""
    import torch
    page, layers, kv, dim = 4, 2, 2, 64
    c = mx.PagedKVCache(layers, 40, page, kv, dim, 5, 64)
    content = {}  # (row, position) -> value in every place

    def append(grown, value_of):
        starts, pos = grown.starts.tolist(), grown.positions.tolist()
        n = len(pos)
        x = torch.zeros((n, kv, dim), device="cuda", dtype=torch.bfloat16)
        for r in range(5):
            for t in range(starts[r], starts[r + 1]):
                content[r, pos[t]] = value_of(r, pos[t])
                x[t] = content[r, pos[t]]
        for i in range(layers):
            c.append(i, x + i, x - i, grown.slots)

    def check():
        lens, table = c.lens.tolist(), c.table.tolist()
        used = []
        for r in range(5):
            held = table[r][:-(-lens[r] // page)]
            used += held
            for t in range(lens[r]):
                for i in range(layers):
                    assert (c.k[i, held[t // page], :, t % page] == content[r, t] + i).all(), (r, t)
                    assert (c.v[i, held[t // page], :, t % page] == content[r, t] - i).all(), (r, t)
        left = c.free[:c.free_count.item()].tolist()
        assert sorted(used + left) == list(range(40))

    append(c.resize(_i32([10, 0, 3, 0, 0]), 20), lambda r, t: 10 * r + t)
    check()
    c.fork(_i32([0, 5, 2, -7, 1 << 30]), 30)  # itself, and no rows
    check()
    with pytest.raises(mx.QGemmError, match="sources"):
        c.fork(_i32([-1, 0]), 30)
    with pytest.raises(mx.QGemmError, match="sources"):
        c.fork(_i32([-1] * 5).long(), 30)
    grown = c.fork(_i32([-1, 0, -1, 0, 2]), 30)
    assert c.lens.tolist() == [10, 10, 3, 10, 3] and grown.refused.item() == 0
    for r, s, n in ((1, 0, 10), (3, 0, 10), (4, 2, 3)):
        for t in range(n):
            content[r, t] = content[s, t]
    check()
    drafts = [6, 5, 0, 7, 9]
    grown = c.resize(_i32([n + d for n, d in zip([10, 10, 3, 10, 3], drafts)]), 32)
    append(grown, lambda r, t: 100 + 20 * r + t)
    check()
    path, counts = [[0, 2, 5], [4, -1, -1], [0, 0, 0], [1, 3, 6], [2, 7, 8]], [3, 1, 2, 2, 3]
    old = dict(content)
    c.accept(grown, _i32(path), _i32(counts))
    base = [10, 10, 3, 10, 3]
    kept = [3, 1, 0, 2, 3]
    for r in range(5):
        for j in range(kept[r]):
            content[r, base[r] + j] = old[r, base[r] + path[r][j]]
    assert c.lens.tolist() == [b + n for b, n in zip(base, kept)]
    check()
    c.resize(_i32([0, 0, 0, 0, 0]), 0)
    assert c.free_count.item() == 40


@pytest.mark.gpu
def test_moves_in_a_graph_and_on_other_streams():
    import torch
    k, v = _stores(2, 20, 2, 4, 64, "bf16", False, 9)
    table, lens = _tables([11, 7], 4, 20, 1).cuda(), _i32([11, 7])
    starts, path, counts = _i32([0, 6, 10]), _i32([[2, 3, 5], [1, 3, 0]]), _i32([3, 2])
    src, dst = _i32([60, 61, 62]), _i32([77, 3, 78])
    k0, v0 = k.clone(), v.clone()
    want = mx.paged_accept(k, v, table, lens, starts, path, counts)
    kw, vw = k.clone(), v.clone()
    side = torch.cuda.Stream()
    k.copy_(k0), v.copy_(v0)
    side.wait_stream(torch.cuda.current_stream())
    got = mx.paged_accept(k, v, table, lens, starts, path, counts, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(_bytes(k), _bytes(kw)) and torch.equal(_bytes(v), _bytes(vw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = mx.paged_accept(k, v, table, lens, starts, path, counts)
        mx.paged_copy(k, v, src, dst)
    for _ in range(3):
        k.copy_(k0), v.copy_(v0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
        k1, v1 = k.clone(), v.clone()
        k.copy_(kw), v.copy_(vw)
        mx.paged_copy(k, v, src, dst)
        assert torch.equal(_bytes(k), _bytes(k1)) and torch.equal(_bytes(v), _bytes(v1))
