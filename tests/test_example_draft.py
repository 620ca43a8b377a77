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


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["8 bits", "gguf", "8 bits and gguf"])
def test_layers_work_on_the_given_stream_alone(cuda, kind):
    """Rows that lie apart are copied, and intermediate results made and freed, on the call's stream: it does not see what the current
    stream still has to do, nor does that stream's later work take their memory."""
    import torch
    g = torch.Generator().manual_seed(2)

    def load(layer, n, k, eight):
        if eight:
            return layer.load_weight(mx.quantize_fp8_weight((torch.randn(n, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(cuda)))
        return layer.load_weight(mx.synth_gguf(mx.QuantType.Q8_0, n, k, n), mx.QuantType.Q8_0, device=cuda)
    lin, mlp = load(mx.Linear(512, 384), 384, 512, kind != "gguf"), mx.MLP(512, 1024)
    load(mlp.gate_proj, 1024, 512, kind != "gguf"), load(mlp.up_proj, 1024, 512, kind == "8 bits"), load(mlp.down_proj, 512, 1024, kind == "8 bits")
    x = torch.randn(70, 2, 512, generator=g).to(torch.bfloat16).to(cuda).transpose(0, 1)
    big = torch.randn(8192, 8192, device=cuda)
    want, side = (lin(x), mlp(x)), torch.cuda.Stream()
    big @ big
    torch.cuda.synchronize()
    for _ in range(3):
        for _ in range(4):
            big @ big  # some 50 ms of the current stream's
        got = lin(x, stream=side), mlp(x, stream=side)
        for n in (70 * 2 * 1024, 70 * 2 * 512, 70 * 2 * 384):  # memory of the sizes that the calls had in between
            torch.full((n,), 7.0, device=cuda, dtype=torch.bfloat16)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [True, False])
def test_projections_of_an_mlp_keep_their_biases(cuda, eight):
    import torch
    g = torch.Generator().manual_seed(3)
    mlp, parts = mx.MLP(256, 512), []
    for name, n, k in (("gate_proj", 512, 256), ("up_proj", 512, 256), ("down_proj", 256, 512)):
        lin = mx.Linear(k, n, bias=True)
        if eight:
            lin.load_weight(mx.quantize_fp8_weight((torch.randn(n, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(cuda)))
        else:
            lin.load_weight(mx.synth_gguf(mx.QuantType.Q8_0, n, k, n + len(name)), mx.QuantType.Q8_0, device=cuda)
        setattr(mlp, name, lin)
        parts.append(lin)
    x = torch.randn(9, 256, generator=g).to(torch.bfloat16).to(cuda)
    with pytest.raises(mx.QGemmError, match="bias not set"):
        mlp(x)
    for lin in parts:
        lin.set_bias(torch.randn(lin.out_features, generator=g).to(cuda))
    gate, up, down = parts
    want = down(mx.swiglu(gate(x), up(x)))
    assert torch.equal(mlp(x), want)
    if eight:
        assert torch.equal(mlp(mx.quantize_fp8(x)), want)
    for lin in parts:
        lin.bias = torch.zeros_like(lin.bias)
    assert not torch.equal(mlp(x), want)


@pytest.mark.gpu
def test_a_captured_pass_follows_its_inputs(cuda):
    """A whole pass (pages, masks, layers, accepted paths, a fork) captured once and replayed with other lengths, trees, tokens and
    paths, the program's own calls in between, gives the bits of the same calls made one by one."""
    import random

    import torch
    ex = _example()
    model = ex.Model(cuda)
    rng = random.Random(5)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    inputs = {"want": i32([0] * ex.ROWS), "tokens": torch.zeros(ex.TOKENS, dtype=torch.int64, device=cuda),
              "parents": i32([-1] * ex.TOKENS), "path": i32([[-1] * ex.DEPTH] * ex.ROWS), "counts": i32([0] * ex.ROWS),
              "sources": i32([-1] * ex.ROWS)}

    def one(cache):
        grown = cache.resize(inputs["want"], ex.TOKENS)
        logits = ex.step(model, cache, inputs["tokens"], inputs["parents"], grown)
        kept = cache.accept(grown, inputs["path"], inputs["counts"])
        forked = cache.fork(inputs["sources"], ex.TOKENS)
        return grown.starts, logits, kept.lens, forked.refused

    def new():
        c = mx.PagedKVCache(ex.LAYERS, ex.PAGES, ex.PAGE, ex.KV, ex.DIM, ex.ROWS, ex.LONGEST, device=cuda)
        c.k.zero_(), c.v.zero_()
        return c
    eager, held = new(), new()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(new())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = one(held)
    lens = [0] * ex.ROWS
    for step in range(6):
        n = [rng.randrange(0, 20) for _ in lens]
        if step == 3:
            lens, n[1], n[2] = [lens[0], 0, 0, lens[3]], 0, 0  # rows 1 and 2 end, and become copies
        want = [a + b for a, b in zip(lens, n)]
        parents, path, counts = [], [], []
        for m in n:
            parents += [rng.randrange(-1, i) if i else -1 for i in range(m)]
            kept = sorted(rng.sample(range(m), rng.randrange(0, m + 1)))
            path.append(kept + [-1] * (ex.DEPTH - len(kept))), counts.append(len(kept))
        inputs["want"].copy_(i32(want)), inputs["path"].copy_(i32(path)), inputs["counts"].copy_(i32(counts))
        inputs["parents"].copy_(i32(parents + [-1] * (ex.TOKENS - len(parents))))
        inputs["tokens"].copy_(torch.randint(0, ex.VOCAB, (ex.TOKENS,), device=cuda))
        inputs["sources"].copy_(i32([-1, 0, 3, -1] if step == 3 else [-1, 9, 2, -5]))
        want_out = [t.clone() for t in one(eager)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want_out, captured):
            assert torch.equal(a, b), step
        for t in ("lens", "table", "free_count"):
            assert torch.equal(getattr(eager, t), getattr(held, t)), (step, t)
        lens = [a + c for a, c in zip(lens, counts)]
        if step == 3:
            lens[1], lens[2] = lens[0], lens[3]
        assert eager.lens.tolist() == lens


@pytest.mark.gpu
def test_calls_of_several_threads_at_once(cuda):
    """Each thread's own stream, inputs and outputs; the library keeps nothing between calls that others could see."""
    import threading

    import torch
    g = torch.Generator(device=cuda).manual_seed(3)
    rnd = lambda *s: torch.randn(s, device=cuda, generator=g)  # noqa: E731
    work = []
    for i, (m, n, k) in enumerate([(5, 512, 1024), (90, 4096, 2048), (40, 256, 8192)]):
        w, x, res = mx.quantize_fp8_weight(rnd(n, k)), rnd(m, k).bfloat16(), rnd(m, k).bfloat16()
        kc, vc = rnd(64 * (i + 1), 2, 16, 128).bfloat16(), rnd(64 * (i + 1), 2, 16, 128).bfloat16()
        rows = 2 * (i + 1)
        table = torch.randperm(64 * (i + 1), device=cuda, generator=g).to(torch.int32).view(rows, 32)
        lens = torch.full((rows,), 400 + 30 * i, dtype=torch.int32, device=cuda)
        starts = torch.arange(0, 7 * rows + 1, 7, dtype=torch.int32, device=cuda)
        q = rnd(7 * rows, 8, 128).bfloat16()
        work.append((w, x, res, kc, vc, table, lens, starts, q))

    def run(job, stream):
        w, x, res, kc, vc, table, lens, starts, q = job
        h, total = mx.rms_norm(x, residual=res, quantize=True, stream=stream)
        return [h.data.view(torch.uint8), h.scales, total, mx.fp8_matmul(h, w, stream=stream), mx.fp8_matmul(x, w, stream=stream),
                *mx.paged_tree_attention(q, kc, vc, table, lens, starts, return_lse=True, stream=stream)]
    wants = [run(job, None) for job in work]
    torch.cuda.synchronize()
    wrong = []

    def loop(i):
        stream = torch.cuda.Stream()
        for _ in range(30):
            got = run(work[i], stream)
            stream.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, wants[i])):
                wrong.append(i)
    threads = [threading.Thread(target=loop, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
