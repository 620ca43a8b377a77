"""Low-rank adapters beside shared projections (lora_apply) against the formula in float64."""
import ctypes
import math

import pytest

import mlxr_amd as mx
from mlxr_amd import lora

P = ctypes.c_void_p


# ------------------------------------------------------------------------------ refusals (no GPU)

def test_refusals():
    L = lora._lib()

    def call(count=1, tokens=4, K=256, adapters=3, rank=16, x=64, dt=mx.BF16, xs=256, ids=64, ws=64, nb=1 << 40, a=64, b=64,
             y=64, out=64, N=32, ydt=mx.BF16):
        items = (lora.Item * max(1, count))(*[lora.Item(a, b, y, out, N, ydt)] * max(1, count))
        return L.mlxr_lora_apply(count, items, tokens, K, adapters, rank, P(x), dt, xs, P(ids), None, None, P(ws), nb, None)
    assert call(count=0) == 0 and call(tokens=0) == 0
    assert call(count=-1) == -1 and call(tokens=-1) == -1 and call(K=0) == -1 and call(adapters=0) == -1 and call(rank=0) == -1
    assert call(adapters=4097) == -3 and call(rank=12) == -3 and call(rank=136) == -3 and call(K=252) == -3
    assert call(tokens=(1 << 24) + 1) == -3
    assert call(dt=mx.F32) == -1 and call(dt=3) == -1
    for name in ("x", "ids", "a", "b", "y", "out"):
        assert call(**{name: 0 if name in ("x", "ids") else None}) == -1, name
    assert call(tokens=300, ws=0) == -1
    assert call(xs=252) == -3 and call(x=72) == -3 and call(ws=72) == -3 and call(a=72) == -3 and call(b=72) == -3
    assert call(N=0) == -1 and call(ydt=3) == -1
    assert call(tokens=300, nb=16) == -1 and "workspace" in L.mlxr_qgemm_last_error().decode()
    n = ctypes.c_size_t()
    item = (lora.Item * 1)(lora.Item(None, None, None, None, 32, mx.BF16))
    bad = (lora.Item * 1)(lora.Item(None, None, None, None, 0, mx.BF16))

    def size(count=1, items=item, tokens=4, rank=16, out=ctypes.byref(n)):
        return L.mlxr_lora_workspace_size(count, items, tokens, 256, 3, rank, out)
    assert size(out=None) == -1 and size(rank=17) == -3 and size(items=None) == -1 and size(items=bad) == -1
    assert size(count=0) == 0 and n.value == 0
    assert size() == 0 and n.value == 0  # one launch
    assert size(tokens=300) == 0 and n.value > 0


def test_limits():
    """The largest sizes the workspace of which is told, and those just past them."""
    L, n = lora._lib(), ctypes.c_size_t()
    item = (lora.Item * 1)(lora.Item(None, None, None, None, 32, mx.BF16))

    def size(tokens=300, K=256, adapters=3, rank=16):
        return L.mlxr_lora_workspace_size(1, item, tokens, K, adapters, rank, ctypes.byref(n))
    assert size(tokens=1 << 20) == 0 and size(tokens=(1 << 20) + 1) == -3
    assert size(adapters=4096) == 0 and size(adapters=4097) == -3
    assert size(rank=128) == 0 and size(rank=136) == -3
    assert size(K=1 << 28) == 0 and size(K=(1 << 28) + 8) == -3


def test_sizes_that_indexes_would_not_hold_are_refused():
    L = lora._lib()
    for N, K in ((32, (1 << 28) + 8), ((1 << 28) + 1, 256)):
        item = (lora.Item * 1)(lora.Item(64, 64, 64, 64, N, mx.BF16))
        assert L.mlxr_lora_apply(1, item, 4, K, 3, 16, P(64), mx.BF16, K, P(64), None, None, P(64), 1 << 40, None) in (-1, -3)


def test_wrapper_refusals():
    import torch
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    with pytest.raises(mx.QGemmError, match="on a GPU"):
        mx.lora_apply(x, torch.zeros(4, dtype=torch.int32), [], [], [])
    with pytest.raises(mx.QGemmError, match="multiple of 8"):
        mx.LoraBank(4, 16, 32, 100, device="cpu")
    bank = mx.LoraBank(4, 12, 32, 64, device="cpu")
    assert bank.a.shape == (4, 16, 64) and bank.b.shape == (4, 32, 16)
    with pytest.raises(mx.QGemmError, match="up to 12"):
        bank.load(0, torch.zeros(13, 64), torch.zeros(32, 13))
    bank.load(2, torch.ones(5, 64), torch.ones(32, 5), 0.5)
    assert bank.ranks.tolist() == [0, 0, 5, 0] and bank.scales.tolist() == [0, 0, 0.5, 0]


# ------------------------------------------------------------------------------ values

def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _make(cuda, tokens, K, adapters, rank, widths, dtype, ydt, seed, ids=None, ranks=None):
    """Inputs whose A and B hold NaN past each adapter's rank."""
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, K, generator=g).to(_dt(dtype))
    if ids is None:
        ids = torch.randint(-1, adapters, (tokens,), generator=g)
    ids = torch.as_tensor(ids).to(torch.int32)
    ranks = torch.randint(0, rank + 1, (adapters,), generator=g) if ranks is None else torch.as_tensor(ranks)
    a, b, y = [], [], []
    for n in widths:
        A, B = torch.randn(adapters, rank, K, generator=g) * K ** -0.5, torch.randn(adapters, n, rank, generator=g) * 0.3
        for i, r in enumerate(ranks.tolist()):
            A[i, r:] = float("nan")
            B[i, :, r:] = float("nan")
        a.append(A.to(_dt(dtype))), b.append(B.to(_dt(dtype))), y.append(torch.randn(tokens, n, generator=g).to(_dt(ydt)))
    scales = torch.rand(adapters, generator=g) + 0.5
    return x, ids, a, b, y, scales, ranks.to(torch.int32)


def _formula(x, ids, A, B, y, scales, ranks):
    """(result, what the error of the products is measured by) in float64."""
    import torch
    x, y = x.double(), y.double()
    out, size = y.clone(), torch.zeros_like(y)
    for i in set(ids.tolist()):
        if 0 <= i < A.shape[0]:
            r, rows = int(ranks[i]), torch.nonzero(ids == i)[:, 0]
            a, b, s = A[i, :r].double(), B[i, :, :r].double(), float(scales[i])
            out[rows] += s * (x[rows] @ a.t() @ b.t())
            size[rows] = s * (x[rows].abs() @ a.abs().t() @ b.abs().t())
    return out, size


def _check(got, x, ids, A, B, y, scales, ranks, ydt):
    """The products' fp32 sums of K and of rank terms are off by at most (K + rank + 64) 2^-24 of the sum of
    magnitudes (64: joins of partial sums), h enters the second product with 2^-16; then one sum with y and one
    rounding to y's type."""
    import torch
    ref, size = _formula(x, ids, A, B, y, scales, ranks)
    got = got.double().cpu()
    half = {"f32": 2.0 ** -23, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[ydt]
    tol = ((A.shape[2] + A.shape[1] + 64) * 2.0 ** -24 + 2.0 ** -16) * size * 1.01 + half * ref.abs() + 2.0 ** -25
    assert torch.isfinite(got).all()
    bad = ((got - ref).abs() / tol).max()
    assert float(bad) <= 1.0, float(bad)


def _run(cuda, tokens, K, adapters, rank, widths, dtype="bf16", ydt=None, seed=0, **kw):
    ydt = ydt or dtype
    x, ids, a, b, y, scales, ranks = _make(cuda, tokens, K, adapters, rank, widths, dtype, ydt, seed, **kw)
    got = mx.lora_apply(x.to(cuda), ids.to(cuda), [t.to(cuda) for t in a], [t.to(cuda) for t in b], [t.to(cuda) for t in y],
                        scales.to(cuda), ranks.to(cuda))
    for o, A, B, t in zip(got, a, b, y):
        _check(o, x, ids, A, B, t, scales, ranks, ydt)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,K,adapters,rank,widths", [
    (1, 8, 1, 8, [1]), (1, 4096, 3, 16, [64]), (2, 264, 2, 8, [65, 3]), (8, 2048, 16, 16, [2048, 256, 256]),
    (15, 520, 4, 24, [100]), (16, 1024, 1, 32, [257]), (17, 1024, 2, 40, [130, 64, 7, 12, 33]), (61, 2048, 24, 64, [500, 500]),
    (100, 1000, 5, 128, [300]), (333, 256, 300, 8, [72]), (700, 512, 6, 16, [640]), (2048, 256, 3, 32, [96, 1024]),
    (200, 4096, 20, 16, [2048]), (3, 8192, 4, 32, [1000, 24]), (64, 4096, 3, 8, [14336]), (257, 2048, 2, 120, [520]),
])
def test_lora(cuda, dtype, tokens, K, adapters, rank, widths):
    _run(cuda, tokens, K, adapters, rank, widths, dtype, seed=tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,ydt", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("tokens,K,adapters,rank,N", [
    (256, 4352, 1, 16, 43693), (256, 2560, 1, 32, 43776), (256, 128, 1, 64, 43693), (256, 128, 1, 128, 21851),
    (300, 64, 60, 16, 24208), (300, 64, 60, 16, 24203), (300, 64, 60, 64, 12107), (300, 64, 60, 128, 6101)])
def test_lora_of_wide_projections(cuda, dtype, ydt, tokens, K, adapters, rank, N):
    """Two to four steps of columns to a workgroup of the second product, for each of its forms: rows of B of the step
    after on their way, their place in LDS used again, widths that end inside a lane's columns."""
    ids = [(7 * t) % (adapters + 1) - 1 if t < 120 else adapters - 1 for t in range(tokens)]
    _run(cuda, tokens, K, adapters, rank, [N], dtype, ydt, seed=rank, ids=ids)


@pytest.mark.gpu
@pytest.mark.parametrize("ydt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_lora_output_types(cuda, dtype, ydt):
    _run(cuda, 37, 512, 4, 16, [130, 64], dtype, ydt)


@pytest.mark.gpu
@pytest.mark.parametrize("ydt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,K,rank", [(40, 512, 64), (40, 512, 128), (100, 4608, 16), (64, 2560, 32), (300, 128, 8), (300, 128, 32),
                                           (300, 128, 64), (300, 128, 128)])
def test_lora_output_types_of_two_launches(cuda, dtype, ydt, tokens, K, rank):
    """Every kernel of the second product, at widths whose rows start at any element and end inside a lane's columns."""
    _run(cuda, tokens, K, 4, rank, [640, 131, 1025], dtype, ydt, seed=rank)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,K,rank", [(9, 256, 16), (40, 512, 64), (300, 128, 32)])
def test_lora_of_outputs_of_different_types(cuda, tokens, K, rank):
    import torch
    x, ids, a, b, y, scales, ranks = _make(cuda, tokens, K, 5, rank, [96, 72, 130, 40, 33], "bf16", "f32", 4)
    types = ["f32", "bf16", "f16", "bf16", "f32"]
    y = [t.to(_dt(name)) for t, name in zip(y, types)]
    got = mx.lora_apply(x.to(cuda), ids.to(cuda), [t.to(cuda) for t in a], [t.to(cuda) for t in b], [t.to(cuda) for t in y],
                        scales.to(cuda), ranks.to(cuda))
    for o, A, B, t, name in zip(got, a, b, y, types):
        assert o.dtype is _dt(name)
        _check(o, x, ids, A, B, t, scales, ranks, name)

@pytest.mark.gpu
@pytest.mark.parametrize("ids", [[-1] * 40, [2] * 40, [3, 4, -5, 1 << 30] * 10, list(range(40)), [0] * 16 + [1] * 24, [0] * 17 + [-1] * 23])
def test_lora_ids(cuda, ids):
    _run(cuda, 40, 320, 41 if max(ids) == 39 else 3, 16, [96], ids=ids, ranks=[16] * (41 if max(ids) == 39 else 3))


@pytest.mark.gpu
@pytest.mark.parametrize("ranks", [[0, 0, 0], [1, 7, 9], [16, 15, 3], [2, 0, 16]])
def test_lora_ranks(cuda, ranks):
    _run(cuda, 30, 256, 3, 16, [64], ranks=ranks)


@pytest.mark.gpu
def test_lora_of_many_adapters(cuda):
    _run(cuda, 500, 64, 4096, 8, [40], seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,rank", [(40, 16), (40, 32), (256, 64), (256, 128), (260, 128)])
def test_lora_of_the_most_adapters(cuda, tokens, rank):
    """A counter for each of 4096 adapters beside the LDS of every kernel; tokens that share adapters and that do not."""
    _run(cuda, tokens, 64, 4096, rank, [24], seed=rank, ids=[(t * 1237) % 4097 - 1 if t % 3 else 4095 for t in range(tokens)])

@pytest.mark.gpu
def test_lora_f16_products_outside_its_range(cuda):
    """x . A^T far above 65504 and far below 2^-24 in f16: the products between are held in fp32."""
    import torch
    for size_a, size_b in ((3e4, 1e-4), (1e-7, 60.0)):
        x, ids, a, b, y, scales, ranks = _make(cuda, 9, 2048, 2, 16, [80], "f16", "f32", 3, ranks=[16, 16])
        a[0], b[0] = (a[0].float() * size_a).to(torch.float16), (b[0].float() * size_b).to(torch.float16)
        x = (x.float() * (8 if size_a > 1 else 0.5)).to(torch.float16)
        got = mx.lora_apply(x.to(cuda), ids.to(cuda), [a[0].to(cuda)], [b[0].to(cuda)], [y[0].to(cuda)], scales.to(cuda),
                            ranks.to(cuda))
        _check(got[0], x, ids, a[0], b[0], y[0], scales, ranks, "f32")


@pytest.mark.gpu
def test_lora_in_place_strided_and_on_another_stream(cuda):
    import torch
    x, ids, a, b, y, scales, ranks = _make(cuda, 50, 256, 4, 16, [72, 64], "bf16", "bf16", 5)
    dev = lambda t: t.to(cuda)  # noqa: E731
    ids, a, b, y, scales, ranks = dev(ids), list(map(dev, a)), list(map(dev, b)), list(map(dev, y)), dev(scales), dev(ranks)
    want = mx.lora_apply(dev(x), ids, a, b, y, scales, ranks)
    wide = torch.zeros(50, 400, dtype=torch.bfloat16, device=cuda)
    wide[:, 64:320] = dev(x)
    odd = torch.zeros(50, 401, dtype=torch.bfloat16, device=cuda)
    odd[:, 3:259] = dev(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for xs in (wide[:, 64:320], odd[:, 3:259]):
        for stream in (None, s):
            got = mx.lora_apply(xs, ids, a, b, y, scales, ranks, stream=stream)
            torch.cuda.current_stream().wait_stream(s)
            assert all(torch.equal(g, w) for g, w in zip(got, want))
            s.wait_stream(torch.cuda.current_stream())
    mine = [t.clone() for t in y]
    assert mx.lora_apply(dev(x), ids, a, b, mine, scales, ranks, outs=mine)[0] is mine[0]
    assert all(torch.equal(g, w) for g, w in zip(mine, want))
    with pytest.raises(mx.QGemmError, match="x's dtype"):
        mx.lora_apply(dev(x), ids, [t.half() for t in a], b, y, scales, ranks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,K,rank", [(3, 64, 8), (20, 2048, 64), (300, 256, 32)])
def test_infinite_b_gives_infinity(cuda, dtype, tokens, K, rank):
    """An infinite element of B: an infinite output of h's sign, whatever h's bits past 16 (0 among them), not NaN."""
    import torch
    x, ids, a, b, y, scales, ranks = _make(cuda, tokens, K, 3, rank, [40], dtype, dtype, 5)
    ids = torch.arange(tokens, dtype=torch.int32) % 3
    a, b = [t.nan_to_num(0.0) for t in a], [t.nan_to_num(0.0) for t in b]
    x[::2] = x[::2].round()  # every other token: h is a small multiple of a power of two, its low part 0
    a[0] = (a[0] * 16).round() / 4
    ranks[:], scales[:] = rank, 0.5
    for i in range(3):
        b[0][i, 7 + i, i], b[0][i, 20, 3] = math.inf, -math.inf
    got = mx.lora_apply(x.to(cuda), ids.to(cuda), [a[0].to(cuda)], [b[0].to(cuda)], [y[0].to(cuda)], scales.to(cuda),
                        ranks.to(cuda))[0].double().cpu()
    for t in range(tokens):
        i = int(ids[t])
        h = a[0][i].double() @ x[t].double()
        for n, r, sign in ((7 + i, i, 1.0), (20, 3, -1.0)):
            if abs(float(h[r])) > 1e-3:
                assert float(got[t, n]) == math.copysign(math.inf, sign * float(h[r])), (t, n)
            elif float(h[r]) == 0:
                assert math.isnan(float(got[t, n]))
        rest = [n for n in range(40) if n not in (7 + i, 20)]
        assert torch.isfinite(got[t, rest]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,rank", [(3, 8), (20, 64), (300, 32), (300, 8), (20, 24)])
@pytest.mark.parametrize("short", [0, 3])
def test_infinite_sums_of_the_first_product(cuda, dtype, tokens, rank, short):
    """An infinite element of x: infinite outputs, and NaN where B is 0; NaN in x: NaN; the tokens beside them stay as
    they are; also where the adapter uses less than the bank's rank, or that is no multiple of 16."""
    import torch
    g = torch.Generator().manual_seed(rank)
    x = torch.rand(tokens, 64, generator=g) + 0.5
    a, b = torch.rand(1, rank, 64, generator=g) + 0.5, torch.rand(1, 40, rank, generator=g) + 0.5
    b[0, 7, 1] = 0.0
    ranks = torch.tensor([rank - short], dtype=torch.int32, device=cuda)
    ids = torch.zeros(tokens, dtype=torch.int32, device=cuda)
    dev = lambda t: t.to(_dt(dtype)).to(cuda)  # noqa: E731

    def run():
        return mx.lora_apply(dev(x), ids, [dev(a)], [dev(b)], [torch.zeros(tokens, 40, device=cuda)], ranks=ranks)[0].cpu()
    plain = run()
    assert torch.isfinite(plain).all()
    x[1, 9], x[2, 9] = math.inf, math.nan
    got = run()
    assert torch.isnan(got[1, 7]) and (got[1, [n for n in range(40) if n != 7]] == math.inf).all() and torch.isnan(got[2]).all()
    rest = [t for t in range(tokens) if t not in (1, 2)]
    assert torch.equal(got[rest], plain[rest])


def _one_hot(adapters, N, rank):
    """B whose row j picks rank j, row rank + j the difference of ranks j and j + 1."""
    import torch
    b = torch.zeros(adapters, N, rank)
    b[:, :rank] = torch.eye(rank)
    b[:, rank:2 * rank - 1] = torch.eye(rank)[:-1] - torch.eye(rank)[1:]
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,K,rank", [(5, 64, 8), (5, 64, 16), (33, 64, 32), (20, 64, 64), (20, 64, 128), (100, 8192, 16), (100, 4096, 32),
                                           (300, 64, 8), (300, 64, 16), (300, 64, 32), (300, 64, 64), (300, 64, 128)])
def test_lora_keeps_the_sums_of_the_first_product(cuda, dtype, tokens, K, rank):
    """x and A are integers of up to 8 bits, so x . A^T has up to 22 and is exact in fp32; B shows it, and differences of its
    ranks.  What the second product takes of it is off by 2^-22 of each rank at most (f16; bf16 holds it all), the fp32 sum of
    two by 2^-24 of them."""
    import torch
    g = torch.Generator().manual_seed(rank + K)
    top = 255 if K == 64 else 15
    x, a = torch.randint(top // 2, top + 1, (tokens, K), generator=g), torch.randint(top // 2, top + 1, (3, rank, K), generator=g)
    a *= torch.randint(0, 2, (3, rank, 1), generator=g) * 2 - 1
    N = 2 * rank + 3
    ids = torch.randint(-1, 3, (tokens,), generator=g).to(torch.int32)
    dev = lambda t: t.to(_dt(dtype)).to(cuda)  # noqa: E731
    got = mx.lora_apply(dev(x), ids.to(cuda), [dev(a)], [dev(_one_hot(3, N, rank))], [torch.zeros(tokens, N, device=cuda)])[0].double().cpu()
    h = torch.einsum("tk,trk->tr", x.double(), a.double()[ids.clamp(min=0).long()]) * (ids >= 0)[:, None]
    assert float(h.abs().max()) < 1 << 24
    ref, size = torch.zeros(2, tokens, N, dtype=torch.float64)
    ref[:, :rank], size[:, :rank] = h, h.abs()
    ref[:, rank:2 * rank - 1], size[:, rank:2 * rank - 1] = h[:, :-1] - h[:, 1:], h[:, :-1].abs() + h[:, 1:].abs()
    assert ((got - ref).abs() <= 2.0 ** -21 * size).all(), float(((got - ref).abs() / size.clamp(min=1)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,K,rank", [(5, 64, 16), (33, 64, 32), (20, 64, 64), (20, 64, 128), (100, 8192, 16), (300, 64, 8), (300, 64, 16),
                                           (300, 64, 32), (300, 64, 64), (300, 64, 128)])
def test_lora_ranks_of_a_token_far_apart(cuda, dtype, tokens, K, rank):
    """x . A^T of 2^16 in one rank and 2^-22 in another of the same token: each is held relative to itself (2^-20), not to
    the largest; among tokens of the same adapter whose ranks are alike, and whose results they do not touch."""
    import torch
    g = torch.Generator().manual_seed(rank + K)
    x = torch.randint(1, 8, (tokens, K), generator=g)
    a = torch.randint(-7, 8, (2, rank, K), generator=g).double()
    a[:, :, K // 2:] *= 2.0 ** (10 - 2.0 * (torch.arange(rank) % 17))[None, :, None]
    alike = torch.rand(tokens, generator=g) < 0.6
    x[alike, K // 2:], x[~alike, :K // 2] = 0, 0
    N = 2 * rank
    ids = torch.randint(-1, 2, (tokens,), generator=g).to(torch.int32)
    dev = lambda t: t.to(_dt(dtype)).to(cuda)  # noqa: E731
    b, y = dev(_one_hot(2, N, rank)), torch.zeros(tokens, N, device=cuda)
    scales = torch.tensor([1.0, 3.0], device=cuda)
    got = mx.lora_apply(dev(x), ids.to(cuda), [dev(a)], [b], [y], scales)[0]
    i = ids.clamp(min=0).long()
    h = torch.einsum("tk,trk->tr", x.double(), a[i]) * ((ids >= 0) * torch.where(i > 0, 3.0, 1.0))[:, None]
    assert ((got[:, :rank].double().cpu() - h).abs() <= 2.0 ** -20 * h.abs()).all()
    step = (h[:, :-1] - h[:, 1:]).abs(), h[:, :-1].abs() + h[:, 1:].abs()
    assert ((got[:, rank:2 * rank - 1].double().cpu().abs() - step[0]).abs() <= 2.0 ** -20 * step[1]).all()
    x[~alike] = 0
    again = mx.lora_apply(dev(x), ids.to(cuda), [dev(a)], [b], [y], scales)[0]
    assert torch.equal(again[alike.to(cuda)], got[alike.to(cuda)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,rank", [(3, 8), (20, 64), (300, 32)])
def test_infinite_b_beside_infinite_sums(cuda, dtype, tokens, rank):
    """The product of an infinite x . A^T and an infinite element of B is infinite."""
    import torch
    g = torch.Generator().manual_seed(rank)
    x = torch.rand(tokens, 64, generator=g) + 0.5
    a, b = torch.rand(1, rank, 64, generator=g) + 0.5, torch.rand(1, 40, rank, generator=g) + 0.5
    b[0, 6, 1], b[0, 7, 1] = math.inf, 0.0
    ids = torch.zeros(tokens, dtype=torch.int32, device=cuda)
    dev = lambda t: t.to(_dt(dtype)).to(cuda)  # noqa: E731

    def run():
        return mx.lora_apply(dev(x), ids, [dev(a)], [dev(b)], [torch.zeros(tokens, 40, device=cuda)])[0].cpu()
    plain = run()
    assert (plain[:, 6] == math.inf).all() and torch.isfinite(plain[:, 7:]).all()
    x[1, 9], x[2, 9] = math.inf, math.nan
    got = run()
    assert torch.isnan(got[1, 7]) and (got[1, [n for n in range(40) if n != 7]] == math.inf).all() and torch.isnan(got[2]).all()
    rest = [t for t in range(tokens) if t not in (1, 2)]
    assert torch.equal(got[rest], plain[rest])


@pytest.mark.gpu
def test_lora_bank(cuda):
    import torch
    bank = mx.LoraBank(3, 20, 96, 256, device=cuda)
    torch.manual_seed(4)
    parts = []
    for i, r in enumerate((4, 20, 9)):
        A, B = torch.randn(r, 256) / 16, torch.randn(96, r) / 4
        bank.load(i, A, B, 0.5 * i + 1)
        parts.append((A.to(torch.bfloat16).double(), B.to(torch.bfloat16).double(), 0.5 * i + 1))
    x, y = torch.randn(7, 256).to(torch.bfloat16), torch.randn(7, 96)
    ids = torch.tensor([2, 0, -1, 1, 1, 2, 0], dtype=torch.int32)
    got = bank.apply(x.to(cuda), ids.to(cuda), y.to(cuda))
    for t, i in enumerate(ids.tolist()):
        ref = y[t].double()
        if i >= 0:
            A, B, s = parts[i]
            ref = ref + s * (x[t].double() @ A.t() @ B.t())
        assert float((got[t].double().cpu() - ref).abs().max()) < 1e-3


@pytest.mark.gpu
def test_linear_with_adapters(cuda):
    """Linear(x, lora, ids) is its projection plus each token's adapter; without them nothing changes."""
    import torch
    K, N = 512, 384
    lin = mx.Linear(K, N, bias=True).load_weight(mx.synth_gguf(mx.QuantType.Q4_K, N, K, 3), mx.QuantType.Q4_K, device=cuda)
    lin.set_bias(torch.linspace(-1, 1, N, device=cuda))
    bank = mx.LoraBank(2, 8, N, K, device=cuda)
    bank.load(0, torch.randn(8, K) / 20, torch.randn(N, 8)).load(1, torch.randn(3, K) / 20, torch.randn(N, 3), 2.0)
    x = torch.randn(2, 5, K, device=cuda).to(torch.bfloat16)
    ids = torch.tensor([0, 1, -1, 1, 0, 0, -1, 1, 1, 0], dtype=torch.int32, device=cuda)
    y = lin(x)
    got = lin(x, lora=bank, adapter_ids=ids)
    want = mx.lora_apply(x.view(10, K), ids, [bank.a], [bank.b], [y.view(10, N)], bank.scales, bank.ranks)[0]
    assert got.shape == (2, 5, N) and torch.equal(got.view(10, N), want) and not torch.equal(got, y)
    assert torch.equal(got.view(10, N)[[2, 6]], y.view(10, N)[[2, 6]])
    with pytest.raises(mx.QGemmError, match="together"):
        lin(x, lora=bank)
    with pytest.raises(mx.QGemmError, match="do not match"):
        lin(x, lora=mx.LoraBank(2, 8, N, 256, device=cuda), adapter_ids=ids)


@pytest.mark.gpu
def test_mlp_taken_apart_for_adapters(cuda):
    """Gate and up with adapters, gating, down with adapters; tokens without one get what the layer gives them, within the
    bf16 rounding of gate and up (2^-8 each, about 2^-8 of the output's norm together as they are independent; bound 2^-6)."""
    import torch
    K, inter, tokens = 512, 768, 6
    torch.manual_seed(6)
    mlp = mx.MLP(K, inter)
    banks = {}
    for i, (name, n, k) in enumerate((("gate", inter, K), ("up", inter, K), ("down", K, inter))):
        getattr(mlp, name + "_proj").load_weight(mx.synth_gguf(mx.QuantType.Q4_K, n, k, 60 + i), mx.QuantType.Q4_K, device=cuda)
        banks[name] = mx.LoraBank(2, 8, n, k, device=cuda)
        for j in range(2):
            banks[name].load(j, torch.randn(8, k) * k ** -0.5, torch.randn(n, 8) * 0.2, 1.0 + j)
    gate, up, down = banks["gate"], banks["up"], banks["down"]
    x = torch.randn(tokens, K).to(torch.bfloat16).to(cuda)
    ids = torch.tensor([0, 1, -1, 1, -1, 0], dtype=torch.int32, device=cuda)
    g, u = mx.q_gemm_dequant_grouped(x, [mlp.gate_proj.weight, mlp.up_proj.weight])
    mx.lora_apply(x, ids, [gate.a, up.a], [gate.b, up.b], [g, u], gate.scales, gate.ranks, outs=[g, u])
    got = mlp.down_proj(mx.swiglu(g, u, out=g), lora=down, adapter_ids=ids).double().cpu()

    def project(h, name, i):
        out = h @ mx.dequantize(getattr(mlp, name + "_proj").weight).double().cpu().t()
        bank = banks[name]
        if i >= 0:
            out = out + float(bank.scales[i]) * (h @ bank.a[i].double().cpu().t() @ bank.b[i].double().cpu().t())
        return out
    for t, i in enumerate(ids.tolist()):
        h = x[t].double().cpu()
        ref = project(torch.nn.functional.silu(project(h, "gate", i)) * project(h, "up", i), "down", i)
        assert float((got[t] - ref).norm() / ref.norm()) < 2.0 ** -6
    plain = mlp(x).double().cpu()
    none = [t for t, i in enumerate(ids.tolist()) if i < 0]
    assert float((got[none] - plain[none]).norm() / plain[none].norm()) < 2.0 ** -6

@pytest.mark.gpu
def test_concurrent_calls_from_host_threads(cuda):
    """Four host threads, each with a stream of its own, make calls of every kernel at once: the results of the same
    calls made alone, bit for bit."""
    import threading
    import torch
    cases = []
    for tokens, K, rank, dtype in ((9, 256, 16, "bf16"), (40, 512, 64, "f16"), (300, 128, 32, "bf16"), (300, 128, 128, "f16")):
        x, ids, a, b, y, scales, ranks = _make(cuda, tokens, K, 5, rank, [96, 1030], dtype, dtype, rank)
        dev = lambda v: [t.to(cuda) for t in v]  # noqa: E731
        cases.append((x.to(cuda), ids.to(cuda), dev(a), dev(b), dev(y), scales.to(cuda), ranks.to(cuda)))
    want = [mx.lora_apply(*c) for c in cases]
    torch.cuda.synchronize()
    errors = []

    def thread(t):
        torch.cuda.set_device(cuda)
        stream = torch.cuda.Stream()
        for rep in range(20):
            i = (t + rep) % len(cases)
            got = mx.lora_apply(*cases[i], stream=stream)
            stream.synchronize()
            if not all(torch.equal(g, w) for g, w in zip(got, want[i])):
                errors.append((t, i))
    threads = [threading.Thread(target=thread, args=(t,)) for t in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
