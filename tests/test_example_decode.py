"""examples/decode_step.py: requests that enter, generate and leave get the logits of a dense float64 model."""
import importlib.util
import os

import pytest

import mlxr_amd as mx

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_step.py")


def _example():
    spec = importlib.util.spec_from_file_location("decode_step", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _dense(ex, model, sequence, adapter):
    """Logits after each token of a sequence, without cache or rounding."""
    import torch
    w = lambda lin: mx.dequantize(lin.weight).double().cpu()  # noqa: E731
    n = len(sequence)

    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)

    def lora(h, bank):
        if adapter < 0:
            return 0.0
        r = int(bank.ranks[adapter])
        a, b = bank.a[adapter, :r].double().cpu(), bank.b[adapter, :, :r].double().cpu()
        return float(bank.scales[adapter]) * (h @ a.t() @ b.t())

    def rotate(x):
        half = ex.DIM // 2
        angle = torch.arange(n).double()[:, None] * 10000.0 ** (-torch.arange(half).double() / half)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    x = model.embed[torch.tensor(sequence, device=model.device)].double().cpu()
    mask = torch.ones(n, n).tril().bool()
    for lay in model.layers:
        h = norm(x)
        q, k, v = (h @ w(lay[m]).t() + lora(h, lay[m + "_lora"]) for m in ("q", "k", "v"))
        q = rotate(q.view(n, ex.HEADS, ex.DIM)).permute(1, 0, 2)
        k = rotate(k.view(n, ex.KV, ex.DIM)).permute(1, 0, 2).repeat_interleave(ex.HEADS // ex.KV, 0)
        v = v.view(n, ex.KV, ex.DIM).permute(1, 0, 2).repeat_interleave(ex.HEADS // ex.KV, 0)
        p = torch.softmax((q @ k.transpose(1, 2) * ex.DIM ** -0.5).masked_fill(~mask, float("-inf")), -1)
        o = (p @ v).permute(1, 0, 2).reshape(n, -1)
        x = x + o @ w(lay["o"]).t() + lora(o, lay["o_lora"])
        h = norm(x)
        m = lay["mlp"]
        x = x + (torch.nn.functional.silu(h @ w(m.gate_proj).t()) * (h @ w(m.up_proj).t())) @ w(m.down_proj).t()
    return norm(x) @ w(model.head).t()


def test_a_refused_row_has_no_new_token():
    """Its place in the list of slots is that of the next row that has one."""
    import torch
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    # four rows: refused, one token, free, one token at the end of the list
    grown = mx.Resized(i32(16, 6, 0, 40), i32(0), i32(0, 0, 1, 1, 2), i32(85, 39, -1, -1), i32(5, 39, -1, -1), i32(1))
    slots, positions = _example().new_tokens(grown)
    assert slots.tolist() == [-1, 85, -1, 39] and positions.tolist() == [-1, 5, -1, 39]
    # the last row refused: its place lies past the list
    grown = mx.Resized(i32(1, 1, 1, 16), i32(0), i32(0, 1, 2, 3, 3), i32(0, 16, 32, -1), i32(0, 0, 0, -1), i32(1))
    slots, positions = _example().new_tokens(grown)
    assert slots.tolist() == [0, 16, 32, -1] and positions.tolist() == [0, 0, 0, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [3, 5])
def test_requests_wait_for_pages(cuda, pages):
    """A pool too small for the requests that come together: rows wait, the last gives its pages back and starts again;
    every request that fits the pool alone gets the dense model's logits (bound as below), one that does not gets none."""
    ex = _example()
    model = ex.Model(cuda)
    requests = ex.REQUESTS + [([4] * (pages * ex.PAGE), 2, 0)]
    out, cache = ex.serve(model, requests, 400, pages)
    assert out.pop() == ([], [])
    for (prompt, n, adapter), (tokens, logits) in zip(ex.REQUESTS, out):
        assert len(tokens) == n and len(logits) == n
        ref = _dense(ex, model, prompt + tokens[:-1], adapter)[len(prompt) - 1:]
        for got, want in zip(logits, ref):
            assert float((got.double().cpu() - want).norm() / want.norm()) < 0.04
    assert cache.lens.tolist() == [0] * ex.ROWS and sorted(cache.free.tolist()) == list(range(pages))


@pytest.mark.gpu
def test_served_requests_match_a_dense_model(cuda):
    """bf16 activations are rounded about thirty times on the way through the layers (2^-9 rms each, half of them on
    branches beside the residual): about one percent of the logits' norm; bound 4 %."""
    ex = _example()
    model = ex.Model(cuda)
    out, cache = ex.serve(model, ex.REQUESTS, 100)
    for (prompt, n, adapter), (tokens, logits) in zip(ex.REQUESTS, out):
        assert len(tokens) == n and len(logits) == n
        ref = _dense(ex, model, prompt + tokens[:-1], adapter)[len(prompt) - 1:]
        for got, want in zip(logits, ref):
            got = got.double().cpu()
            assert float((got - want).norm() / want.norm()) < 0.04
    assert cache.lens.tolist() == [0] * ex.ROWS and int(cache.free_count) == ex.PAGES
    assert sorted(cache.free.tolist()) == list(range(ex.PAGES))
