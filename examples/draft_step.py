"""Speculative decoding over a decoder with 8-bit projections: what a serving loop does with drafted tokens.

A pass takes, for each request, the tokens that are certain (its prompt at first, then the last token it
was given) and a tree of guesses of what follows, all at once:

  PagedKVCache.resize          pages and slots for all of them
  tree_mask                    who sees whom, and the tokens' positions in the text
  per layer:
    rms_norm                   with the residual's addition, to 8 bits
    Linear (Fp8Weight)         q, k, v
    PagedKVCache.append, attend_tree
    Linear, rms_norm, MLP
  Linear                       the vocabulary head, at every token
  PagedKVCache.accept          keeps the guesses that came true, gives the others' pages back

PagedKVCache.fork makes a second request that goes on from the same tokens.  Weights are random; rotary embeddings are plain
torch.  Run: python examples/draft_step.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import mlxr_amd as mx  # noqa: E402

HIDDEN, HEADS, KV, DIM, INTER, VOCAB, LAYERS = 512, 8, 2, 64, 1024, 768, 2
ROWS, PAGE, PAGES, LONGEST = 4, 16, 48, 160
TOKENS, DEPTH, WORDS = 96, 32, 1  # of a pass; of an accepted path; of a mask (64 tokens of a row and pass)


class Model:
    """Weights as a serving process holds them."""

    def __init__(self, device, seed=0):
        g = torch.Generator().manual_seed(seed)

        def linear(n, k):
            w = (torch.randn(n, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(device)
            return mx.Linear(k, n).load_weight(mx.quantize_fp8_weight(w))

        def norm():
            return (1 + 0.1 * torch.randn(HIDDEN, generator=g)).to(torch.bfloat16).to(device)
        self.device = device
        self.embed = torch.randn(VOCAB, HIDDEN, generator=g).to(torch.bfloat16).to(device)
        self.layers = []
        for _ in range(LAYERS):
            lay = {"q": linear(HEADS * DIM, HIDDEN), "k": linear(KV * DIM, HIDDEN), "v": linear(KV * DIM, HIDDEN),
                   "o": linear(HIDDEN, HEADS * DIM), "mlp": mx.MLP(HIDDEN, INTER), "norm": norm(), "mlp_norm": norm()}
            for name, n, k in (("gate_proj", INTER, HIDDEN), ("up_proj", INTER, HIDDEN), ("down_proj", HIDDEN, INTER)):
                setattr(lay["mlp"], name, linear(n, k))
            self.layers.append(lay)
        self.norm, self.head = norm(), linear(VOCAB, HIDDEN)


def rotate(x, positions):
    """Rotary embedding of x [tokens, heads, dim] at the tokens' positions."""
    half = x.shape[-1] // 2
    angle = positions.clamp(min=0).float()[:, None] * 10000.0 ** (-torch.arange(half, device=x.device).float() / half)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def step(model, cache, tokens, parents, grown):
    """One pass over tokens [TOKENS] (those past the last row's mean nothing) of trees `parents`, whose slots `grown` lists.
    Returns the logits [TOKENS, VOCAB]."""
    mask, positions = mx.tree_mask(parents, grown.starts, WORDS, positions=grown.positions)
    total, branch = model.embed[tokens], None

    def norm(weight):
        nonlocal total
        if branch is None:
            return mx.rms_norm(total, weight, quantize=True)
        h, total = mx.rms_norm(branch, weight, residual=total, quantize=True)
        return h
    for i, lay in enumerate(model.layers):
        h = norm(lay["norm"])
        q, k, v = (lay[n](h) for n in ("q", "k", "v"))
        q, k = rotate(q.view(-1, HEADS, DIM), positions), rotate(k.view(-1, KV, DIM), positions)
        cache.append(i, k, v.view(-1, KV, DIM), grown.slots)
        branch = lay["o"](cache.attend_tree(i, q, grown.starts, mask).view(-1, HEADS * DIM))
        branch = lay["mlp"](norm(lay["mlp_norm"]))
    return model.head(norm(model.norm))


def repeats(sequence):
    """Guesses of what follows a sequence, as (parent, token), the parent -1 for what follows its last token: what followed the
    last two places where its last token stood before, three tokens of each."""
    got, found = [], 0
    for at in range(len(sequence) - 2, -1, -1):
        if sequence[at] == sequence[-1] and found < 2:
            found += 1
            parent = -1
            for t in sequence[at + 1:at + 4]:
                got.append((parent, t))
                parent = len(got) - 1
    return got


def serve(model, requests, guess=repeats):
    """requests: [(prompt tokens, tokens to generate)], at most ROWS; a request None goes on from the same tokens as the one before it
    (its prompt is copied, not computed).  Returns each one's tokens and the logits that chose them, how many passes
    it took, and the cache as it is left."""
    dev = model.device
    cache = mx.PagedKVCache(LAYERS, PAGES, PAGE, KV, DIM, ROWS, LONGEST, device=dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    out = [([], []) for _ in requests]
    certain = [list(q[0]) if q else [] for q in requests] + [[] for _ in range(ROWS - len(requests))]
    wanted = [q[1] if q else requests[i - 1][1] for i, q in enumerate(requests)] + [0] * (ROWS - len(requests))
    held = [[] for _ in range(ROWS)]  # the tokens whose keys and values the cache holds
    passes = 0
    while any(certain):
        trees = []
        for r in range(ROWS):
            nodes = [(j - 1, t) for j, t in enumerate(certain[r])]
            room = 0 if not certain[r] else max(0, wanted[r] - len(out[r][0]) - 1)
            for p, t in guess(held[r] + certain[r])[:8] if room else []:
                nodes.append((p + len(certain[r]) if p >= 0 else len(certain[r]) - 1, t))
            trees.append(nodes)
        lens = [len(h) + len(t) for h, t in zip(held, trees)]
        flat = [n for t in trees for n in t]
        assert len(flat) <= TOKENS and max(map(len, trees)) <= 64 * WORDS and max(lens) <= LONGEST
        pad = TOKENS - len(flat)
        grown = cache.resize(i32(lens), TOKENS)
        logits = step(model, cache, i32([t for _, t in flat] + [0] * pad).long(), i32([p for p, _ in flat] + [-1] * pad), grown)
        best = logits.argmax(-1).tolist()
        passes += 1
        path, at = [[-1] * DEPTH for _ in range(ROWS)], 0
        counts = [0] * ROWS
        for r, nodes in enumerate(trees):
            if nodes:
                kept = list(range(len(certain[r])))
                while True:  # what the model says after the last kept token; go on while a guess says the same
                    out[r][0].append(best[at + kept[-1]])
                    out[r][1].append(logits[at + kept[-1]].float())
                    child = [j for j, (p, t) in enumerate(nodes) if j >= len(certain[r]) and p == kept[-1] and t == out[r][0][-1]]
                    if len(out[r][0]) == wanted[r] or not child or len(kept) == DEPTH:
                        break
                    kept.append(child[0])
                path[r][:len(kept)], counts[r] = kept, len(kept)
                held[r] += [nodes[j][1] for j in kept]
                certain[r] = [out[r][0][-1]] if len(out[r][0]) < wanted[r] else []
                at += len(nodes)
        cache.accept(grown, i32(path), i32(counts))
        if passes == 1:
            sources = [i - 1 if i < len(requests) and requests[i] is None else -1 for i in range(ROWS)]
            if any(s >= 0 for s in sources):
                cache.fork(i32(sources), ROWS * LONGEST)
                for r, s in enumerate(sources):
                    if s >= 0:
                        held[r], certain[r] = list(held[s]), list(certain[s])
                        out[r][0].extend(out[s][0]), out[r][1].extend(out[s][1])
        ended = [0 if h and not c else len(h) for h, c in zip(held, certain)]
        cache.resize(i32(ended), 0)
        held = [h if n else [] for h, n in zip(held, ended)]
    return out, passes, cache


REQUESTS = [([5, 9, 300, 41, 5, 9], 24), None, ([7] * 21, 30), ([640, 11], 9)]


def main():
    model = Model(torch.device("cuda:0"))
    out, passes, _ = serve(model, REQUESTS)
    for q, (tokens, _) in zip(REQUESTS, out):
        print(f"{'the same' if q is None else f'prompt of {len(q[0]):2d}'}  ->  {tokens}")
    print(f"{sum(len(t) for t, _ in out)} tokens in {passes} passes")


if __name__ == "__main__":
    main()
