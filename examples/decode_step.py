"""Continuous batching over a quantized decoder: what a serving loop does with this package.

A batch has a fixed number of rows.  Requests enter free rows, feed their prompt a token a step,
generate, and leave; each may have a low-rank adapter of its own.  A step over all rows is

  PagedKVCache.resize        pages and slots for every row's next token (0 frees a row)
  per layer:
    q_gemm_dequant_grouped   q, k, v of the quantized projections
    lora_apply               the rows' adapters on top of them
    PagedKVCache.append      keys and values into the cache
    PagedKVCache.attend      attention over each row's pages
    Linear (+ adapters), MLP output projection and the MLP block
  Linear                     the vocabulary head

with nothing copied to the host but the tokens.  Weights are random (GGUF Q4_K blocks centred on
zero); norms and rotary embeddings are plain torch.  Run: python examples/decode_step.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mlxr_amd as mx  # noqa: E402

HIDDEN, HEADS, KV, DIM, INTER, VOCAB, LAYERS = 512, 8, 2, 64, 1024, 768, 2
ROWS, PAGE, PAGES, LONGEST = 4, 16, 24, 96
ADAPTERS, RANK = 3, 12


def q4k(n, k, seed):
    """Q4_K blocks of weights d * 32 * (q - 7.5), q random in 0 .. 15: scales and mins 32, dmin = 7.5 d."""
    rng = np.random.default_rng(seed)
    w = rng.integers(0, 256, (n * (k // 256), 144), dtype=np.uint8)
    d = np.full(len(w), 0.04 / (32 * 4.61), np.float16)
    w[:, 0:2] = d.view(np.uint8).reshape(-1, 2)
    w[:, 2:4] = (d * np.float16(7.5)).view(np.uint8).reshape(-1, 2)
    w[:, 4:12], w[:, 12:16] = 0xA0, 0  # the six-bit 32 eight times, twice
    return w.reshape(-1)


class Model:
    """Weights as a serving process holds them."""

    def __init__(self, device, seed=0):
        self.device = device
        self.embed = torch.randn(VOCAB, HIDDEN, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(device)
        self.layers = []
        for i in range(LAYERS):
            s = seed + 100 * i
            lay = {}
            for j, (name, n, k) in enumerate((("q", HEADS * DIM, HIDDEN), ("k", KV * DIM, HIDDEN), ("v", KV * DIM, HIDDEN),
                                              ("o", HIDDEN, HEADS * DIM))):
                lay[name] = mx.Linear(k, n).load_weight(q4k(n, k, s + j), mx.QuantType.Q4_K, device=device)
                lay[name + "_lora"] = self._bank(n, k, s + 10 + j)
            lay["mlp"] = mx.MLP(HIDDEN, INTER)
            lay["mlp"].gate_proj.load_weight(q4k(INTER, HIDDEN, s + 5), mx.QuantType.Q4_K, device=device)
            lay["mlp"].up_proj.load_weight(q4k(INTER, HIDDEN, s + 6), mx.QuantType.Q4_K, device=device)
            lay["mlp"].down_proj.load_weight(q4k(HIDDEN, INTER, s + 7), mx.QuantType.Q4_K, device=device)
            self.layers.append(lay)
        self.head = mx.Linear(HIDDEN, VOCAB).load_weight(q4k(VOCAB, HIDDEN, seed + 99), mx.QuantType.Q4_K, device=device)

    def _bank(self, n, k, seed):
        g = torch.Generator().manual_seed(seed)
        bank = mx.LoraBank(ADAPTERS, RANK, n, k, device=self.device)
        for i in range(ADAPTERS):
            r = RANK - 4 * i
            bank.load(i, torch.randn(r, k, generator=g) * k ** -0.5, torch.randn(n, r, generator=g) * 0.1, 0.5 + i)
        return bank


def norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)


def rotate(x, positions):
    """Rotary embedding of x [rows, heads, dim] at the rows' positions."""
    half = x.shape[-1] // 2
    angle = positions.clamp(min=0).float()[:, None] * 10000.0 ** (-torch.arange(half, device=x.device).float() / half)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def new_tokens(grown):
    """Slot and position [rows] of each row's new token, -1 for a row without one: a free row, and one that was refused
    (its place in the list is the next row's).  What such a row computes is written nowhere and read by nobody."""
    first, has = grown.starts[:-1].long(), grown.starts[1:] > grown.starts[:-1]
    at = first.clamp(max=len(grown.slots) - 1)
    return torch.where(has, grown.slots[at], -1), torch.where(has, grown.positions[at], -1)


def step(model, cache, tokens, want, ids):
    """One token for each row: tokens, the lengths after it (0: the row is free) and the adapters [rows], on
    the device.  Returns the logits [rows, VOCAB]; those of a row whose length is not the wanted one mean nothing."""
    slots, positions = new_tokens(cache.resize(want, ROWS))
    x = model.embed[tokens]
    for i, lay in enumerate(model.layers):
        h = norm(x)
        names = ("q", "k", "v")
        y = mx.q_gemm_dequant_grouped(h, [lay[n].weight for n in names])
        banks = [lay[n + "_lora"] for n in names]
        q, k, v = mx.lora_apply(h, ids, [b.a for b in banks], [b.b for b in banks], y, banks[0].scales, banks[0].ranks, outs=y)
        q = rotate(q.view(ROWS, HEADS, DIM), positions)
        k = rotate(k.view(ROWS, KV, DIM), positions)
        cache.append(i, k, v.view(ROWS, KV, DIM), slots)
        o = cache.attend(i, q).view(ROWS, HEADS * DIM)
        x = x + lay["o"](o, lora=lay["o_lora"], adapter_ids=ids)
        x = x + lay["mlp"](norm(x))
    return model.head(norm(x))


def serve(model, requests, steps, pages=PAGES):
    """requests: [(prompt tokens, tokens to generate, adapter)].  Returns each one's generated tokens and the
    logits that chose them, and the cache as it is left.  Where the pool has no page for a row's next token the
    row waits; where no row can go on, the one that came last gives its pages back and starts again later.  A request that
    the tables or the pool cannot hold is not served at all."""
    dev = model.device
    cache = mx.PagedKVCache(LAYERS, pages, PAGE, KV, DIM, ROWS, LONGEST, device=dev)
    held = lambda q: len(requests[q][0]) + requests[q][1] - 1  # noqa: E731  (the last token is not fed)
    waiting = [q for q in range(len(requests)) if held(q) <= min(LONGEST, pages * PAGE)]
    rows, lens = [None] * ROWS, [0] * ROWS  # the request in each, the tokens of it in the cache
    out = [([], []) for _ in requests]
    came = []  # requests in rows, in the order in which they came
    for _ in range(steps):
        # a row that a request left has length 0 in this step (its pages go back) and is taken in the next
        for r, q in enumerate(rows):
            if q is not None and len(out[q][0]) == requests[q][1]:
                came.remove(q)
                rows[r] = None
            elif q is None and lens[r] == 0 and waiting:
                rows[r] = waiting.pop(0)
                came.append(rows[r])
        want, tokens, ids = [0] * ROWS, [0] * ROWS, [-1] * ROWS
        for r, q in enumerate(rows):
            if q is not None:
                prompt, _, ids[r] = requests[q]
                tokens[r], want[r] = (prompt + out[q][0])[lens[r]], lens[r] + 1
        as_dev = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        logits = step(model, cache, as_dev(tokens).long(), as_dev(want), as_dev(ids))
        best, lens = logits.argmax(-1).tolist(), cache.lens.tolist()
        for r, q in enumerate(rows):
            if q is not None and lens[r] == want[r] == len(requests[q][0]) + len(out[q][0]):
                out[q][0].append(best[r])
                out[q][1].append(logits[r].float())
        if not any(want) and not waiting:
            break
        if any(want) and not any(w and n == w for w, n in zip(want, lens)):
            waiting.insert(0, came.pop())  # it will feed its prompt and what it has generated again
            rows[rows.index(waiting[0])] = None
    return out, cache


REQUESTS = [([5, 9, 300, 41], 6, 0), ([7] * 21, 5, -1), ([1, 2, 3], 9, 1), ([640, 11], 4, 2), ([99, 98, 97, 96, 95], 7, 0),
            ([13] * 17, 3, 1)]


def main():
    model = Model(torch.device("cuda:0"))
    for (prompt, n, adapter), (tokens, _) in zip(REQUESTS, serve(model, REQUESTS, 100)[0]):
        print(f"adapter {adapter:2d}  prompt of {len(prompt):2d}  ->  {tokens}")


if __name__ == "__main__":
    main()
