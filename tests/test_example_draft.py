"""examples/draft_step.py: requests whose drafts are accepted or not get the logits of a dense float64 model, and the
layers with 8-bit weights."""
import importlib.util
import os

import pytest

import mlxr_amd as mx

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "draft_step.py")


def _example():
    spec = importlib.util.spec_from_file_location("draft_step", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _dense_weight(linear):
    w = linear.weight
    s = w.scales.double().repeat_interleave(128, 0)[:w.N].repeat_interleave(128, 1)[:, :w.K]
    return (w.data.double() * s).cpu()


def _dense(ex, model, sequence):
    """Logits after each token of a sequence, without cache or rounding."""
    import torch
    n = len(sequence)

    def norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w.double().cpu()

    def rotate(x):
        half = ex.DIM // 2
        angle = torch.arange(n).double()[:, None] * 10000.0 ** (-torch.arange(half).double() / half)
        c, s = angle.cos(), angle.sin()
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    x = model.embed[torch.tensor(sequence, device=model.device)].double().cpu()
    mask = torch.ones(n, n).tril().bool()
    for lay in model.layers:
        h = norm(x, lay["norm"])
        q, k, v = (h @ _dense_weight(lay[m]).t() for m in ("q", "k", "v"))
        q = rotate(q.view(n, ex.HEADS, ex.DIM).permute(1, 0, 2))
        k = rotate(k.view(n, ex.KV, ex.DIM).permute(1, 0, 2)).repeat_interleave(ex.HEADS // ex.KV, 0)
        v = v.view(n, ex.KV, ex.DIM).permute(1, 0, 2).repeat_interleave(ex.HEADS // ex.KV, 0)
        p = torch.softmax((q @ k.transpose(1, 2) * ex.DIM ** -0.5).masked_fill(~mask, float("-inf")), -1)
        x = x + (p @ v).permute(1, 0, 2).reshape(n, -1) @ _dense_weight(lay["o"]).t()
        h, m = norm(x, lay["mlp_norm"]), lay["mlp"]
        gated = torch.nn.functional.silu(h @ _dense_weight(m.gate_proj).t()) * (h @ _dense_weight(m.up_proj).t())
        x = x + gated @ _dense_weight(m.down_proj).t()
    return norm(x, model.norm) @ _dense_weight(model.head).t()


def _check(ex, model, requests, out):
    """Rows are rounded to e4m3 five times a layer on their way (once more for the head), by at most 2^-4 and 2.6 % rms each,
    three of them one after the other on the longest branch (h, gated rows; q, k and v, o): a branch is off by at most
    sqrt(3) * 2.6 % = 4.5 % of its norm (the gated product of two by sqrt(2) more), and so is their sum of independent errors
    beside the head's own 2.6 %: below 8 % of the logits' norm; bound twice that."""
    prompt = None
    for q, (tokens, logits) in zip(requests, out):
        prompt, n = (q[0], q[1]) if q else (prompt, n)
        assert len(tokens) == len(logits) == n
        ref = _dense(ex, model, prompt + tokens[:-1])[len(prompt) - 1:]
        for t, got, want in zip(tokens, logits, ref):
            got = got.double().cpu()
            assert int(got.argmax()) == t
            assert float((got - want).norm() / want.norm()) < 0.16


@pytest.mark.gpu
def test_drafts_do_not_change_what_is_computed(cuda):
    ex = _example()
    model = ex.Model(cuda)
    plain, passes, cache = ex.serve(model, ex.REQUESTS, guess=lambda s: [])
    _check(ex, model, ex.REQUESTS, plain)
    assert passes == 30 and cache.lens.tolist() == [0] * ex.ROWS and sorted(cache.free.tolist()) == list(range(ex.PAGES))
    out, fewer, cache = ex.serve(model, ex.REQUESTS)
    _check(ex, model, ex.REQUESTS, out)
    assert fewer <= passes and int(cache.free_count) == ex.PAGES

    # drafts that are right for two tokens beside two that are wrong: three tokens a pass where the logits agree
    known = {}
    for q, (tokens, _) in zip(ex.REQUESTS, plain):
        if q:
            known[tuple(q[0])] = q[0] + tokens

    def right(sequence):
        for prompt, whole in known.items():
            if tuple(sequence[:len(prompt)]) == prompt and sequence == whole[:len(sequence)]:
                a, b = (whole[len(sequence):] + [1, 1])[:2]
                return [(-1, (a + 1) % ex.VOCAB), (-1, a), (1, (b + 1) % ex.VOCAB), (1, b)]
        return [(-1, 3)]
    out, third, cache = ex.serve(model, ex.REQUESTS, guess=right)
    _check(ex, model, ex.REQUESTS, out)
    assert third < passes and sorted(cache.free.tolist()) == list(range(ex.PAGES))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3,), (2, 5), (40,)])
def test_layers_with_8_bit_weights(cuda, shape):
    """Linear and MLP give what their parts give."""
    import torch
    g = torch.Generator().manual_seed(1)
    w = lambda n, k: mx.quantize_fp8_weight((torch.randn(n, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(cuda))  # noqa: E731
    lin = mx.Linear(256, 200, bias=True).load_weight(w(200, 256))
    lin.set_bias(torch.randn(200, generator=g).to(cuda))
    x = torch.randn(*shape, 256, generator=g).to(torch.bfloat16).to(cuda)
    x8 = mx.quantize_fp8(x)
    want = mx.fp8_matmul(x8, lin.weight, bias=lin.bias)
    assert torch.equal(lin(x).reshape(-1, 200), want) and torch.equal(lin(x8), want) and lin(x).shape == (*shape, 200)
    with pytest.raises(mx.QGemmError):
        lin(x8, lora=mx.LoraBank(2, 8, 200, 256), adapter_ids=torch.zeros(len(x8.data), dtype=torch.int32, device=cuda))
    with pytest.raises(mx.QGemmError):
        mx.Linear(256, 100).load_weight(w(200, 256))
    mlp = mx.MLP(256, 512)
    for p, n, k in (("gate_proj", 512, 256), ("up_proj", 512, 256), ("down_proj", 256, 512)):
        getattr(mlp, p).load_weight(w(n, k))
    h = mx.swiglu(mx.fp8_matmul(x8, mlp.gate_proj.weight), mx.fp8_matmul(x8, mlp.up_proj.weight))
    want = mx.fp8_matmul(h, mlp.down_proj.weight)
    assert torch.equal(mlp(x).reshape(-1, 256), want) and torch.equal(mlp(x8), want) and mlp(x).shape == x.shape
    assert mlp(x.half()).dtype is torch.float16
    # one of the weights in GGUF blocks
    rng = torch.randint(0, 255, (256 * 16, 34), generator=g, dtype=torch.uint8)
    rng[:, :2] = torch.tensor([0, 0x20], dtype=torch.uint8)
    mlp.down_proj.load_weight(rng.reshape(-1).numpy(), mx.QuantType.Q8_0, device=cuda)
    y = mlp(x)
    assert torch.equal(y.reshape(-1, 256), mlp.down_proj(h)) and torch.isfinite(y).all()
    mlp.up_proj.load_weight(rng[:512 * 8].reshape(-1).numpy(), mx.QuantType.Q8_0, device=cuda)
    assert mlp(x).shape == x.shape
    with pytest.raises(mx.QGemmError):
        mlp(x8)
