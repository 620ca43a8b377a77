"""RMS norm, rows in 8 bits and block-scaled products against plain float64 forms."""
import ctypes
import math

import pytest

import mlxr_amd as mx
from mlxr_amd import fp8

P = ctypes.c_void_p
TOP, BLOCK = 448.0, 128


# ------------------------------------------------------------------------------ refusals (no GPU)

def test_norm_refusals():
    L = fp8._lib()

    def call(rows=2, K=64, x=64, xt=mx.BF16, xs=64, res=0, rs=64, w=64, wt=mx.BF16, eps=1e-5, total=0, out=64, ot=mx.BF16,
             scales=0):
        return L.mlxr_rms_norm(rows, K, P(x), xt, xs, P(res), rs, P(w), wt, eps, P(total), P(out), ot, P(scales), None)
    assert call(rows=-1) == -1 and call(K=0) == -1 and call(rows=0) == 0
    assert call(K=(1 << 28) + 1) == -3 and call(rows=1 << 30, K=1 << 20) == -3
    assert call(xs=-64) == -3 and call(res=64, rs=-64) == -3
    assert call(xt=3) == -1 and call(wt=7) == -1 and call(ot=5) == -1
    assert call(x=0) == -1 and call(out=0) == -1
    assert call(ot=3) == -1 and call(scales=64) == -1 and "8 bits" in L.mlxr_qgemm_last_error().decode()
    assert call(eps=-1.0) == -1 and call(eps=math.nan) == -1

    def rows(n=2, K=64, x=64, xt=mx.BF16, xs=64, out=64, scales=64):
        return L.mlxr_quantize_fp8(n, K, P(x), xt, xs, P(out), P(scales), None)
    assert rows(n=-1) == -1 and rows(K=0) == -1 and rows(n=0) == 0 and rows(xt=3) == -1 and rows(xs=-1) == -3
    assert rows(x=0) == -1 and rows(out=0) == -1 and rows(scales=0) == -1

    def weight(N=2, K=64, w=64, wt=mx.BF16, out=64, scales=64):
        return L.mlxr_quantize_fp8_weight(N, K, P(w), wt, P(out), P(scales), None)
    assert weight(N=0) == -1 and weight(K=0) == -1 and weight(wt=3) == -1 and weight(N=1 << 28, K=1 << 28) == -3
    assert weight(w=0) == -1 and weight(out=0) == -1 and weight(scales=0) == -1


def test_matmul_refusals():
    L, n = fp8._lib(), ctypes.c_size_t()

    def call(M=2, N=64, K=64, x=64, xs=64, w=64, ws=64, bias=0, bt=mx.F32, y=64, yt=mx.BF16, space=0, nb=0):
        return L.mlxr_fp8_matmul(M, N, K, P(x), P(xs), P(w), P(ws), P(bias), bt, P(y), yt, P(space), nb, None)
    assert call(M=-1) == -1 and call(N=0) == -1 and call(K=0) == -1 and call(M=0) == 0
    assert call(K=72) == -3 and call(N=(1 << 26) + 1) == -3 and call(K=(1 << 22) + 16) == -3 and call(M=1 << 20, N=1 << 20) == -3
    assert call(yt=3) == -1 and call(bias=64, bt=9) == -1
    for name in ("x", "xs", "w", "ws", "y"):
        assert call(**{name: 0}) == -1, name
    assert call(x=72) == -3 and call(w=72) == -3 and call(y=72) == -3 and call(space=72, nb=1 << 40) == -3
    assert L.mlxr_fp8_matmul_workspace_size(2, 64, 64, mx.BF16, None) == -1
    assert L.mlxr_fp8_matmul_workspace_size(2, 64, 72, mx.BF16, ctypes.byref(n)) == -3
    assert L.mlxr_fp8_matmul_workspace_size(2, 64, 64, 3, ctypes.byref(n)) == -1
    assert L.mlxr_fp8_matmul_workspace_size(0, 64, 64, mx.BF16, ctypes.byref(n)) == 0 and n.value == 0
    assert L.mlxr_fp8_matmul_workspace_size(100, 1024, 8192, mx.BF16, ctypes.byref(n)) == 0
    if n.value:
        assert call(M=100, N=1024, K=8192, space=64, nb=n.value - 1) == -1


def test_wrapper_refusals():
    import torch
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    for fn in (lambda: mx.rms_norm(x), lambda: mx.quantize_fp8(x), lambda: mx.quantize_fp8_weight(x),
               lambda: mx.Fp8Weight(x.to(torch.float8_e4m3fn), torch.ones((1, 1))), lambda: mx.fp8_matmul(x, x)):
        with pytest.raises(mx.QGemmError):
            fn()


# ------------------------------------------------------------------------------ norms

def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _types():
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


def _near(got, want, dtype, own=0.0):
    """Rounding once (half a step) and `own` (relative to each value) of the computation before it."""
    import torch
    tiny = torch.finfo(dtype).smallest_normal * _half_step(dtype) * 2
    off = (got.double() - want).abs() - (want.abs() * (_half_step(dtype) + own) + tiny)
    assert off.max().item() <= 0, off.max().item()


def _norm64(x, weight, eps, residual):
    s = x.double() + (residual.double() if residual is not None else 0)
    y = s / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    return (y if weight is None else y * weight.double()), s


def _norm_own(K, dtype):
    """Relative error before the last rounding: the sum in fp32 (half a step of it, relative to s, only where both are
    fp32: sums of 16-bit values cancel with an error of 2^-24 of the larger, so it is counted apart), at most log2 K + 8 additions of positive
    squares on the way to the mean, halved by the root, and six roundings."""
    return (0.5 * (math.log2(K) + 64) + 8) * 2.0 ** -24


SIZES = [(1, 64), (3, 8), (5, 128), (1, 4096), (7, 200), (33, 256), (2, 512), (9, 1000), (4, 1024), (600, 2048), (5, 2560), (513, 4096),
         (520, 5120), (3, 8192), (515, 8192), (4, 9000), (514, 12000), (2, 16384), (3, 20000), (513, 32768), (2, 40000), (3, 77),
         (2, 1), (5, 129), (3, 4099), (600, 501), (5, 2047), (700, 8191), (3, 12345), (2, 32767), (3, 32769)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_norm(rows, K, kind):
    import torch
    dt, g = _types()[kind], _gen(rows * 7 + K)
    x = (torch.randn((rows, K), device="cuda", generator=g) * 4).to(dt)
    r = torch.randn((rows, K), device="cuda", generator=g).to(dt)
    for weight, residual in ((torch.randn(K, device="cuda", generator=g).to(dt), None), (None, r),
                             (torch.randn(K, device="cuda", generator=g), r)):
        got = mx.rms_norm(x, weight, eps=1e-5, residual=residual)
        y, s = _norm64(x, weight, 1e-5, residual)
        if residual is not None:
            got, total = got
            _near(total, s, dt, 2.0 ** -24)
        # an element of the sum is off by half a step of fp32, relative to itself
        _near(got, y, dt, _norm_own(K, dt) + 2.0 ** -24)
        wide = mx.rms_norm(x, weight, eps=1e-5, residual=residual, out_dtype=torch.float32)
        _near(wide if residual is None else wide[0], y, torch.float32, _norm_own(K, dt) + 2.0 ** -24)


def _eight64(y):
    """Scales and y / scale (64 bits) of blocks of 128 of rows."""
    import torch
    m, k = y.shape
    b = torch.nn.functional.pad(y, (0, -k % BLOCK)).view(m, -1, BLOCK)
    top = b.abs().amax(-1)
    return torch.where(top > 0, top / TOP, torch.ones_like(top)), k


def _check_eight(got, y, own):
    """got (Fp8Rows) against y [M, K] in 64 bits: scales to half a step of fp32 and `own`; values at most half a step of e4m3
    from y, its steps below the normal numbers being 2^-9."""
    import torch
    scale, k = _eight64(y)
    _near(got.scales, scale, torch.float32, own)
    each = got.scales.double().repeat_interleave(BLOCK, 1)[:, :k]
    want, have = y / each, got.data.double()
    # half a step of e4m3: 2^-4 of the value, or 2^-10; `own` may move a value over a border between two roundings
    off = (have - want).abs() - (want.abs() * (2.0 ** -4 + 2 * own + 2.0 ** -23)).clamp(min=2.0 ** -10 * (1 + 2.0 ** -20))
    assert off.max().item() <= 0, off.max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_eight_bits(rows, K, kind):
    import torch
    dt, g = _types()[kind], _gen(rows * 5 + K)
    x = (torch.randn((rows, K), device="cuda", generator=g) * 4).to(dt)
    x[0, :max(1, K // 3)] = 0  # blocks of zeros
    q = mx.quantize_fp8(x)
    _check_eight(q, x.double(), 0.0)
    # without a norm every bit is known: fp32 scales, division and rounding to nearest even
    b = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).view(rows, -1, BLOCK)
    top = b.abs().amax(-1)
    scale = torch.where(top > 0, top / torch.full_like(top, TOP), torch.ones_like(top))
    assert torch.equal(q.scales, scale)
    want = (b / scale[..., None]).to(torch.float8_e4m3fn).view(rows, -1)[:, :K]
    assert torch.equal(q.data.view(torch.uint8), want.contiguous().view(torch.uint8))
    r, w = torch.randn((rows, K), device="cuda", generator=g).to(dt), torch.randn(K, device="cuda", generator=g).to(dt)
    got, total = mx.rms_norm(x, w, residual=r, quantize=True)
    y, s = _norm64(x, w, 1e-5, r)
    _near(total, s, dt, 2.0 ** -24)
    _check_eight(got, y, _norm_own(K, dt) + 2.0 ** -24)


@pytest.mark.gpu
def test_norm_strides_shapes_and_streams():
    import torch
    g = _gen(1)
    wide = torch.randn((9, 5, 300), device="cuda", generator=g).bfloat16()
    w = torch.randn(128, device="cuda", generator=g).bfloat16()
    for x in (wide[:, 2, 7:135], wide[:, :, 8:136], wide.transpose(0, 1)[..., :128], wide[::2, 0, 128:256], wide[0, 0, :128],
              wide[:, :, 40:168].expand(9, 5, 128), wide[:1, 0, :128].expand(6, 128)):
        y, _ = _norm64(x, w, 1e-5, None)
        got = mx.rms_norm(x, w)
        assert got.shape == x.shape
        _near(got, y, torch.bfloat16, _norm_own(128, None))
        q = mx.quantize_fp8(x)
        _check_eight(q, x.reshape(-1, 128).double(), 0.0)
    x = torch.randn((50, 4096), device="cuda", generator=g).half()
    want, side = mx.rms_norm(x), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = mx.rms_norm(x, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    assert mx.rms_norm(x[:0]).shape == (0, 4096) and mx.quantize_fp8(x[:0]).scales.shape == (0, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [128, 4096, 4100, 333, 9001])
def test_norm_in_place(K):
    """The sum over the residual, the output over x: the C entry allows both."""
    import torch
    g = _gen(K)
    x, r = (torch.randn((300, K), device="cuda", generator=g).bfloat16() for _ in range(2))
    want, total = mx.rms_norm(x, residual=r)
    x2, r2 = x.clone(), r.clone()
    assert fp8._lib().mlxr_rms_norm(300, K, x2.data_ptr(), mx.BF16, K, r2.data_ptr(), K, None, 0, 1e-5, r2.data_ptr(), x2.data_ptr(),
                                    mx.BF16, None, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(x2, want) and torch.equal(r2, total)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [256, 4096, 300])
def test_eight_bits_of_extreme_values(K):
    import torch
    x = torch.ones((6, K), device="cuda")
    x[0, 3] = math.nan       # stays NaN, counts in no maximum
    x[1, 5] = math.inf       # its block has an infinite scale
    x[2, :128] = 1e-45       # below what a normal scale can hold
    x[3] = 3e38
    x[4] = -0.0
    x[5, :128] = torch.linspace(-448, 448, 128, device="cuda")
    q = mx.quantize_fp8(x)
    v, s = q.data.float(), q.scales
    assert torch.isnan(v[0, 3]) and torch.equal(s[0], torch.ones_like(s[0]) / torch.full_like(s[0], TOP))
    assert (v[0, :3] == 448).all() and (v[0, 4:128] == 448).all()
    assert s[1, 0] == math.inf and torch.isnan(v[1, 5]) and (v[1, :5] == 0).all() and (v[1, 128:] == 448).all()
    assert s[2, 0] == torch.finfo(torch.float32).smallest_normal and (v[2, :128] == 0).all()
    assert (v[3] == 448).all() and torch.isfinite(s[3]).all()
    assert (v[4] == 0).all() and (s[4] == 1).all()
    assert v[5, 0] == -448 and v[5, 127] == 448 and s[5, 0] == 1


# ------------------------------------------------------------------------------ products

def _weights(n, k, seed, dtype=None):
    import torch
    g = _gen(seed)
    data = (torch.randn((n, k), device="cuda", generator=g) * 60).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    scales = (0.5 + torch.rand((-(-n // BLOCK), -(-k // BLOCK)), device="cuda", generator=g)) * 0.02 * k ** -0.5
    return mx.Fp8Weight(data, scales)


def _activations(m, k, seed):
    import torch
    g = _gen(seed + 1)
    data = (torch.randn((m, k), device="cuda", generator=g) * 100).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return mx.Fp8Rows(data, 0.001 + 0.01 * torch.rand((m, -(-k // BLOCK)), device="cuda", generator=g))


def _full(data, scales, by_rows):
    s = scales.double()
    if by_rows:
        s = s.repeat_interleave(BLOCK, 0)[:data.shape[0]]
    return data.double() * s.repeat_interleave(BLOCK, 1)[:, :data.shape[1]]


def _dropped(x, w):
    """What the matrix instruction of 8 bits may drop: of eight neighbouring products (bytes k / 8) it keeps multiples of
    2^-13 of the power of two of the largest, so each of the seven others loses less than 2^-13 of the largest."""
    import torch
    m, n, k = x.data.shape[0], w.N, w.K
    xd, wd = x.data.float().abs(), w.data.float().abs()
    got = torch.zeros((m, n), device="cuda", dtype=torch.float64)
    for at in range(0, k, BLOCK):
        top = torch.zeros((m, n), device="cuda")
        for g in range(at, min(k, at + BLOCK), 8):
            most = torch.zeros((m, n), device="cuda")
            for i in range(g, g + 8):
                most = torch.maximum(most, xd[:, i:i + 1] * wd[:, i])
            top += most
        got += top.double() * x.scales[:, at // BLOCK, None].double() * \
            w.scales[:, at // BLOCK].double().repeat_interleave(BLOCK)[:n]
    return got * 7 * 2.0 ** -13


def _check_product(y, x, w, bias, dtype):
    """Each output: half a step of its type, and of the sum of the magnitudes that it adds up 2^-24 for each of the block's 128
    products (their order is the hardware's), the block's scale (3) and each block and the bias (2); for 16-bit outputs also what
    the instruction drops."""
    import torch
    xd, wd = _full(x.data, x.scales, False), _full(w.data, w.scales, True)
    want, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    own = (BLOCK + 5 + math.ceil(w.K / BLOCK)) * 2.0 ** -24
    most = want.abs() * _half_step(dtype) + size * own + torch.finfo(dtype).smallest_normal
    if dtype is not torch.float32:
        most += _dropped(x, w)
    off = (y.double() - want).abs() - most
    assert off.max().item() <= 0, off.max().item()


# few rows, one tile, ragged tiles, K shorter than a block, ending inside one, long
PRODUCTS = [(1, 16, 16), (1, 4096, 4096), (7, 100, 144), (16, 129, 2048), (17, 64, 512), (31, 1000, 1040), (32, 4096, 1024),
            (33, 256, 128), (33, 4097, 400), (61, 1024, 4096), (64, 64, 8192), (65, 77, 272), (100, 1024, 8192), (128, 128, 128),
            (130, 2050, 1168), (255, 3, 256), (300, 5120, 640), (1000, 513, 384), (1, 5, 28672), (40, 5, 28672), (257, 8200, 1536),
            (2048, 2048, 256), (2049, 8193, 272)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k):
    import torch
    x, w = _activations(m, k, m + n), _weights(n, k, n + k)
    for dtype, bias in ((torch.float32, None), (torch.bfloat16, torch.randn(n, device="cuda", generator=_gen(3)).bfloat16()),
                        (torch.float16, torch.randn(n, device="cuda", generator=_gen(4)))):
        _check_product(mx.fp8_matmul(x, w, bias=bias, out_dtype=dtype), x, w, bias, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", range(1, 8))
@pytest.mark.parametrize("m,n,k,splits", [(1, 5, 16, 1), (33, 300, 528, 1), (260, 517, 1040, 1), (300, 260, 1168, 3), (70, 1000, 2304, 7)])
def test_product_in_every_kernel(kind, m, n, k, splits):
    import torch
    x, w = _activations(m, k, kind), _weights(n, k, kind + 1)
    L = fp8._lib()
    assert L.mlxr_fp8_test_force(8, 1) == -1 and L.mlxr_fp8_test_force(-1, 1) == -1
    assert L.mlxr_fp8_test_force(kind, splits) == 0
    try:
        for dtype, bias in ((torch.float32, None), (torch.bfloat16, torch.randn(n, device="cuda", generator=_gen(3)))):
            _check_product(mx.fp8_matmul(x, w, bias=bias, out_dtype=dtype), x, w, bias, dtype)
    finally:
        L.mlxr_fp8_test_force(0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", range(0, 8))
@pytest.mark.parametrize("m,n,k", [(1, 64, 28672), (17, 100, 400), (61, 257, 2048), (300, 520, 1040), (130, 70, 8192)])
def test_products_of_small_integers_are_exact(kind, m, n, k):
    """Products up to 4 and scales that are powers of two: neither the instruction of 8 bits nor sums in fp32 round anything (sums are
    multiples of 2^-2 below 2^21), so every output is the exact one rounded once.  One product lost or counted twice shows."""
    import torch
    g = _gen(m + k)
    x, w = (torch.randint(-2, 3, (r, k), device="cuda", generator=g).float() for r in (m, n))
    xs = 2.0 ** torch.randint(-1, 2, (m, -(-k // BLOCK)), device="cuda", generator=g)
    ws = 2.0 ** torch.randint(-1, 2, (-(-n // BLOCK), -(-k // BLOCK)), device="cuda", generator=g)
    xq, wq = mx.Fp8Rows(x.to(torch.float8_e4m3fn), xs), mx.Fp8Weight(w.to(torch.float8_e4m3fn), ws)
    want = _full(xq.data, xs, False) @ _full(wq.data, ws, True).t()
    L = fp8._lib()
    for splits in (1, 3):
        assert L.mlxr_fp8_test_force(kind, splits) == 0
        try:
            for dtype in (torch.float32, torch.bfloat16, torch.float16):
                assert torch.equal(mx.fp8_matmul(xq, wq, out_dtype=dtype), want.to(dtype)), dtype
        finally:
            L.mlxr_fp8_test_force(0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(17, 512, 1024), (61, 1024, 8192), (300, 512, 4096), (2048, 2048, 2048), (33, 256, 28672)])
def test_products_of_16_bit_outputs_as_a_whole(m, n, k):
    """The norm of the error: half a step of the output, and of the instruction of 8 bits what it drops of the seven smaller of eight
    products, each a part of 2^-13 of the largest that is evenly spread (2^-13 / sqrt(3) rms) and of either sign: sqrt(7 / 3) 2^-13 of the
    largest, which of eight products of normal numbers is 2.5 times their size on average, beside their sum, sqrt(8) times it: 1.4 * 2^-13,
    so 2^-12 is allowed.  A product lost is sqrt(1 / K), 48 * 2^-13 at 28672."""
    import torch
    x, w = _activations(m, k, m), _weights(n, k, n)
    want = _full(x.data, x.scales, False) @ _full(w.data, w.scales, True).t()
    for dtype in (torch.bfloat16, torch.float16):
        y = mx.fp8_matmul(x, w, out_dtype=dtype).double()
        assert ((y - want).norm() / want.norm()).item() <= _half_step(dtype) + 2.0 ** -12


@pytest.mark.gpu
@pytest.mark.parametrize("kind", range(0, 8))
def test_product_knows_every_code(kind):
    """One-hot rows read single weights off, of every one of the 256 codes (both zeros, the values below the normal ones, NaN)."""
    import torch
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    w = mx.Fp8Weight(codes.view(256, 1).expand(256, 16).contiguous().view(torch.float8_e4m3fn), torch.full((2, 1), 0.5, device="cuda"))
    one = torch.zeros((40, 16), device="cuda")
    one[torch.arange(40), torch.arange(40) % 16] = 1.0
    x = mx.Fp8Rows(one.to(torch.float8_e4m3fn), torch.full((40, 1), 2.0, device="cuda"))
    # 0 times NaN is NaN: codes of one are their value in every row
    want = codes.view(torch.float8_e4m3fn).float().expand(40, 256)
    L = fp8._lib()
    assert L.mlxr_fp8_test_force(kind, 1) == 0
    try:
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            got = mx.fp8_matmul(x, w, out_dtype=dtype).float()
            assert torch.equal(got.nan_to_num(1e9), want.nan_to_num(1e9)), dtype  # 4 bits fit every output type
            back = mx.fp8_matmul(mx.Fp8Rows(w.data, torch.ones((256, 1), device="cuda")), mx.Fp8Weight(x.data, torch.ones((1, 1), device="cuda")), out_dtype=dtype)
            assert torch.equal(back.float().nan_to_num(1e9), want.t().contiguous().nan_to_num(1e9)), dtype
    finally:
        L.mlxr_fp8_test_force(0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 300, 272), (20, 256, 512), (50, 300, 272), (200, 300, 640), (600, 8192, 256)])
def test_product_uses_nothing_outside(m, n, k):
    """NaN before and behind the operands, in rows of others and in scales of blocks that do not exist: none is seen.  A NaN
    within is, in its row or column alone."""
    import torch
    x, w = _activations(m, k, 5), _weights(n, k, 6)
    room = torch.full(((m + 2) * k + 64,), math.nan, device="cuda").to(torch.float8_e4m3fn)
    data = room[16 * (-(-k // 16)):][:m * k].view(m, k)
    data.copy_(x.data)
    wroom = torch.full(((n + 2) * k + 64,), math.nan, device="cuda").to(torch.float8_e4m3fn)
    wdata = wroom[16 * (-(-k // 16)):][:n * k].view(n, k)
    wdata.copy_(w.data)
    out = torch.full((m + 1, n), 7.0, device="cuda", dtype=torch.bfloat16)
    y = mx.fp8_matmul(mx.Fp8Rows(data, x.scales), mx.Fp8Weight(wdata, w.scales), out=out[:m])
    _check_product(y, x, w, None, torch.bfloat16)
    assert (out[m] == 7).all()
    bad = mx.Fp8Rows(x.data.clone(), x.scales)
    bad.data.view(torch.uint8)[m // 2, k - 1] = 0x7f
    y2 = mx.fp8_matmul(bad, w)
    assert torch.isnan(y2[m // 2]).all()
    y2[m // 2] = y[m // 2]
    assert torch.equal(y2, y)


@pytest.mark.gpu
def test_product_of_16_bit_rows_streams_and_graphs():
    import torch
    w = _weights(1000, 1024, 9)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn((3, 20, 1024), device="cuda", generator=_gen(5)).to(dtype)
        y = mx.fp8_matmul(x, w)
        assert y.shape == (3, 20, 1000) and y.dtype is dtype
        _check_product(y.view(60, 1000), mx.quantize_fp8(x), w, None, dtype)
    assert mx.fp8_matmul(x[:0], w).shape == (0, 20, 1000)
    for m in (5, 50, 100):
        x = mx.quantize_fp8(torch.randn((m, 1024), device="cuda", generator=_gen(m)))
        want, side = mx.fp8_matmul(x, w), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = mx.fp8_matmul(x, w, stream=side)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = mx.fp8_matmul(x, w)
        for _ in range(3):
            held.zero_()
            graph.replay()
            other = mx.fp8_matmul(x, w)
            torch.cuda.synchronize()
            assert torch.equal(held, want) and torch.equal(other, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (3, 100, 144), (16, 130, 4096), (7, 300, 400), (33, 5, 128), (100, 64, 28672), (600, 1040, 2048)])
def test_product_of_rows_in_16_and_32_bits(m, n, k, kind):
    """The same bits as quantize_fp8 and the product of its rows, values that are not finite included, of rows that lie apart and
    of their copy; nothing behind or between the rows is seen."""
    import torch
    w = _weights(n, k, m)
    room = torch.full((m + 3, k + 8), math.nan, device="cuda", dtype=_types()[kind])
    x = room[:m, :k]
    x.copy_(torch.randn((m, k), device="cuda", generator=_gen(k)) * 3)
    x[0, :min(k, 128)] = 0
    x[m // 2, k - 1] = 3e4
    bias = torch.randn(n, device="cuda", generator=_gen(1))
    for y in (x, x.contiguous(), x.reshape(1, m, k)):
        for dtype in (torch.float32, torch.bfloat16):
            got = mx.fp8_matmul(y, w, bias, out_dtype=dtype)
            assert torch.equal(got.reshape(m, n), mx.fp8_matmul(mx.quantize_fp8(x), w, bias, out_dtype=dtype))
    x[m - 1, k // 2] = math.nan
    x[0, 1] = math.inf
    got, want = mx.fp8_matmul(x, w), mx.fp8_matmul(mx.quantize_fp8(x), w, out_dtype=x.dtype)
    assert torch.isnan(got[m - 1]).all() and torch.isnan(got[0]).all()
    assert torch.equal(got.nan_to_num(1e4), want.nan_to_num(1e4))


def test_linear_entry_refuses():
    L, n = mx.fp8._lib(), ctypes.c_size_t()
    P = ctypes.c_void_p

    def call(M=2, N=64, K=64, x=64, xt=mx.BF16, w=64, ws=64, bias=0, bt=mx.F32, y=64, yt=mx.BF16, space=64, nb=1 << 20):
        return L.mlxr_fp8_linear(M, N, K, P(x), xt, 64, P(w), P(ws), P(bias), bt, P(y), yt, P(space), nb, None)
    assert call(M=-1) == -1 and call(K=0) == -1 and call(K=72) == -3 and call(yt=3) == -1 and call(xt=3) == -1
    assert call(x=0) == -1 and call(w=0) == -1 and call(ws=0) == -1 and call(y=0) == -1 and call(bias=64, bt=3) == -1
    assert call(w=72) == -3 and call(y=72) == -3 and call(space=72) == -3 and call(space=0) == -1 and call(nb=100) == -1
    assert call(M=0, x=0, space=0, nb=0) == 0
    assert L.mlxr_fp8_linear_workspace_size(2, 64, 64, mx.BF16, None) == -1
    assert L.mlxr_fp8_linear_workspace_size(0, 64, 64, mx.BF16, ctypes.byref(n)) == 0 and n.value == 0
    assert L.mlxr_fp8_linear_workspace_size(5, 64, 144, mx.BF16, ctypes.byref(n)) == 0 and n.value == 768 + 256


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(64, 16), (128, 128), (300, 400), (1000, 1040)])
def test_weights_to_eight_bits(n, k):
    import torch
    w = torch.randn((n, k), device="cuda", generator=_gen(n)).bfloat16()
    q = mx.quantize_fp8_weight(w)
    b = torch.nn.functional.pad(w.float(), (0, -k % BLOCK, 0, -n % BLOCK)).view(-(-n // BLOCK), BLOCK, -1, BLOCK)
    top = b.abs().amax((1, 3))
    assert torch.equal(q.scales, top / torch.full_like(top, TOP))
    want = (b / q.scales[:, None, :, None]).to(torch.float8_e4m3fn).view(-(-n // BLOCK) * BLOCK, -1)[:n, :k]
    assert torch.equal(q.data.view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.gpu
def test_no_rows():
    import torch
    w = _weights(130, 144, 1)
    for shape in ((0, 144), (3, 0, 144)):
        x = torch.zeros(shape, device="cuda", dtype=torch.bfloat16)
        assert mx.rms_norm(x).shape == shape and mx.rms_norm(x, residual=x)[1].shape == shape
        q = mx.quantize_fp8(x)
        assert q.data.shape == (0, 144) and q.scales.shape == (0, 2)
        assert mx.fp8_matmul(x, w).shape == (*shape[:-1], 130) and mx.fp8_matmul(q, w).shape == (0, 130)
        assert mx.Linear(144, 130).load_weight(w)(x).shape == (*shape[:-1], 130)
    strided = torch.zeros((0, 300), device="cuda", dtype=torch.float16)[:, :144]
    assert mx.fp8_matmul(strided, w, out_dtype=torch.float32).shape == (0, 130)
