"""Performance cases of a decoder's pass over drafted tokens, and of its eight-bit projections.

Speculative decoding feeds a tree of drafted tokens for each request at once: the residual stream is
normed and rounded to eight bits with a scale for each 128 values (``rms_norm``), multiplied with
projections held in eight bits with a scale for each 128 x 128 values (``fp8_matmul``), attention lets
every drafted token see its request's cached tokens and its ancestors in the tree
(``paged_tree_attention``), and the tokens of the accepted path move together in every layer's
cache (``paged_accept``); a request that goes on in several ways is copied to other rows
(``paged_copy``).  A case is one call of one of them.  Model sizes are those of the tests and the
benchmark (TinyLlama, Llama-3-8B, Llama-3-70B) or generic; lengths, trees and paths are ragged.

``run`` is the plain form (elementary torch operations in float32) unless ``own`` is set;
``exact`` is the definition in float64.
"""
import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f8": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "f8": 1}
BLOCK, TOP = 128, 448.0  # values that share a scale, the largest of eight bits
EPS = 1e-5


def _tree(name, rows, heads, kv, dim, longest, nodes, page=16, dtype="bf16", cache="bf16", chain=False, ragged=True,
          token_major=False):
    """Up to `nodes` drafted tokens for each of `rows` requests over up to `longest` cached ones (ragged: spread over
    the range, one row in eleven without drafts).  chain: each sees those before it (no mask)."""
    return {"name": name, "op": "tree", "rows": rows, "heads": heads, "kv": kv, "dim": dim, "longest": longest, "nodes": nodes,
            "page": page, "dtype": dtype, "cache": cache, "chain": chain, "ragged": ragged, "token_major": token_major}


def _accept(name, rows, layers, kv, dim, longest, nodes, depth, page=16, cache="bf16", token_major=False):
    """Paths of up to `depth` of up to `nodes` drafted tokens."""
    return {"name": name, "op": "accept", "rows": rows, "layers": layers, "kv": kv, "dim": dim, "longest": longest,
            "nodes": nodes, "depth": depth, "page": page, "cache": cache, "token_major": token_major}


def _copy(name, tokens, times, layers, kv, dim, page=16, cache="bf16", token_major=False):
    """A request of `tokens` tokens, copied `times` times."""
    return {"name": name, "op": "copy", "tokens": tokens, "times": times, "layers": layers, "kv": kv, "dim": dim, "page": page,
            "cache": cache, "token_major": token_major}


def _norm(name, tokens, hidden, dtype="bf16", residual=True, eight=False, normed=True):
    """eight: to eight bits with scales.  normed: the norm, or only the rounding."""
    return {"name": name, "op": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "residual": residual, "eight": eight,
            "normed": normed}


def _matmul(name, tokens, hidden, out, x="f8", dtype="bf16", bias=False):
    """x: the type of the activations, rounded to eight bits in the call unless they are."""
    return {"name": name, "op": "matmul", "tokens": tokens, "hidden": hidden, "out": out, "x": x, "dtype": dtype, "bias": bias}


def listed():
    return [
        # five drafted tokens of one TinyLlama request: latency counts
        _tree("tree_tiny_m1", 1, 32, 4, 64, 700, 5, dtype="f16", cache="f16", ragged=False),
        # small trees of a batch of Llama-3-8B requests over ragged contexts up to the model's 8192
        _tree("tree_8b_m16", 16, 32, 8, 128, 8192, 16),
        # wide trees of a large model over an eight-bit cache
        _tree("tree_70b_fp8_m8", 8, 64, 8, 128, 16384, 64, page=32, cache="f8"),
        # the next part of one request's prompt: a chain of an odd length
        _tree("chain_8b_513", 1, 32, 8, 128, 6001, 513, page=64, chain=True, ragged=False, token_major=True),
        # the accepted tokens of a batch, in all of Llama-3-8B's layers
        _accept("accept_8b_m64", 64, 32, 8, 128, 100, 16, 6),
        # few requests of a large model with an eight-bit cache
        _accept("accept_70b_fp8_m8", 8, 80, 8, 128, 300, 64, 12, page=32, cache="f8"),
        # a prompt that three more samples go on from
        _copy("fork_8b_1501", 1501, 3, 32, 8, 128),
        # one token's residual stream
        _norm("norm_8b_m1", 1, 4096),
        # those of a large model's prompts, to eight bits for the projections
        _norm("norm_70b_fp8_m2048", 2048, 8192, eight=True),
        # a few drafted tokens through an attention projection, rounded in the call
        _matmul("fp8_8b_o_m7", 7, 4096, 4096, x="bf16"),
        # the drafts of a batch through a large model's gate
        _matmul("fp8_70b_gate_m61", 61, 8192, 28672),
        # prompts through a gate
        _matmul("fp8_8b_gate_m2048", 2048, 4096, 14336),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {}
    for c in listed():
        for k, v in work(c).items():
            most[c["op"], k] = max(most.get((c["op"], k), 0), v)
    most["accept", "bytes"] = most["copy", "bytes"]
    while True:
        op = rng.choice(["tree", "tree", "accept", "copy", "norm", "matmul", "matmul"])
        kv, dim = rng.choice([1, 2, 4, 8, 8, 8, 10, 32]), rng.choice([64, 80, 112, 128, 128, 128, 256])
        if op == "tree":
            dtype, chain = rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.25
            c = _tree("", _log(rng, 1, 64), kv * rng.choice([1, 2, 4, 4, 7, 8]), kv, dim, _log(rng, 1, 32768),
                      _log(rng, 1, 700) if chain else _log(rng, 1, 200), rng.choice([16, 16, 32, 64, 128]), dtype,
                      rng.choice([dtype, dtype, "f8"]), chain, rng.random() < 0.8, rng.random() < 0.3)
            held = c["rows"] * (c["longest"] + c["nodes"])
            if held * c["heads"] * c["nodes"] > 8 * 16384 * 64 * 64 or held * kv * dim > 1 << 28:  # what the plain form holds
                continue
        elif op == "accept":
            nodes = _log(rng, 2, 200)
            c = _accept("", _log(rng, 1, 128), rng.randrange(1, 81), kv, dim, _log(rng, 16, 500), nodes,
                        rng.randrange(1, min(nodes, 16) + 1), rng.choice([16, 16, 32, 64]), rng.choice(["bf16", "f16", "f8"]),
                        rng.random() < 0.3)
            if c["rows"] * (c["longest"] + nodes) * c["layers"] * kv * dim > 1 << 29:
                continue
        elif op == "copy":
            c = _copy("", _log(rng, 1, 6000), rng.randrange(1, 8), rng.randrange(1, 81), kv, dim, rng.choice([16, 16, 32, 64]),
                      rng.choice(["bf16", "f16", "f8"]), rng.random() < 0.3)
            if c["tokens"] * (c["times"] + 1) * c["layers"] * kv * dim > 1 << 29:
                continue
        elif op == "norm":
            hidden = rng.choice([2048, 2560, 3584, 4096, 5120, 6656, 8192, _log(rng, 64, 16384)])
            c = _norm("", _log(rng, 1, 4096), hidden, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.5,
                      rng.random() < 0.5)
            if c["eight"] and not c["residual"] and rng.random() < 0.5:
                c["normed"] = False
        else:
            sizes = [1024, 2048, 2560, 4096, 5120, 8192, 14336, 16 * _log(rng, 16, 900)]
            c = _matmul("", _log(rng, 1, 2048), rng.choice(sizes), rng.choice(sizes + [_log(rng, 100, 28672)]),
                        rng.choice(["f8", "f8", "bf16", "f16"]), rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.3)
        del c["name"]
        if all(v <= most[op, k] for k, v in work(c).items()):
            return c


# ------------------------------------------------------------------------------ the inputs

def _rng(seed, *ids):
    s = int(seed)
    for i in ids:
        s = (s * 1000003 + int(i) + 12345) % (1 << 62)
    return torch.Generator().manual_seed(s)


def _dev(seed, *ids):
    return torch.Generator(device="cuda").manual_seed(int(_rng(seed, 77, *ids).initial_seed()))


def _normal(shape, dtype, g, scale=1.0):
    """N(0, scale) in dtype, made a slice at a time so that long caches need no float32 copy."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    step = 1 << 26
    for at in range(0, flat.numel(), step):
        part = flat[at:at + step]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=g) * scale)
    return t


def _store(lead, pages, c, g, scale=1.0):
    """A key or value store [*lead, pages, kv, page, dim], in the case's memory order."""
    if c["token_major"]:
        return _normal((*lead, pages, c["page"], c["kv"], c["dim"]), DTYPE[c["cache"]], g, scale).transpose(-3, -2)
    return _normal((*lead, pages, c["kv"], c["page"], c["dim"]), DTYPE[c["cache"]], g, scale)


def _counts(c, seed):
    """(cached tokens, drafted tokens) of the rows: the longest first, then ragged.  The drafts are the case's, so that
    outputs have one shape."""
    rows = c["rows"]
    if not c.get("ragged", True):
        return [c["longest"]] * rows, [c["nodes"]] * rows
    context = [int(c["longest"] * s) for s in torch.rand(rows, generator=_rng(seed, 1)).tolist()]
    drafts = [max(1, int(round(c["nodes"] * (0.25 + 0.75 * s)))) for s in torch.rand(rows, generator=_rng(0, 9)).tolist()]
    for r in range(10, rows, 11):
        drafts[r] = 0
    context[0], drafts[0] = c["longest"], c["nodes"]
    return context, drafts


def _tables(c, lens, seed):
    """Page tables [rows, width] of rows of these lengths, and the pages of a pool that holds every row at its longest."""
    held = [-(-n // c["page"]) for n in lens]
    wide = max(1, *held)
    pages = len(lens) * wide + 3
    order = torch.randperm(pages, generator=_rng(seed, 3)).to(torch.int32)
    table = torch.full((len(lens), wide), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    return table, pages


def _starts(drafts):
    return torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(drafts).cumsum(0)]).to(torch.int32)


def _parents(n, seed, r):
    """A tree of n nodes: children come after their parents, -1 is the last cached token.  Wide at the root, as drafts are."""
    u = torch.rand(n, generator=_rng(seed, 21, r)).tolist()
    return [int(i * x * x) - 1 if i else -1 for i, x in enumerate(u)]


def _mask(c, drafts, tokens, seed):
    """[tokens, words]: bit b of word w says that a token sees node 64 w + b of its row's tree."""
    words = -(-c["nodes"] // 64)
    got = torch.zeros((tokens, words), dtype=torch.int64)
    at = 0
    for r, n in enumerate(drafts):
        seen = []
        for i, p in enumerate(_parents(n, seed, r)):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            for w in range(words):
                v = seen[-1] >> 64 * w & (1 << 64) - 1
                got[at + i, w] = v - (1 << 64) if v >> 63 else v
        at += n
    return got


def prepare(case, seed):
    return {"tree": _prepare_tree, "accept": _prepare_accept, "copy": _prepare_copy, "norm": _prepare_norm,
            "matmul": _prepare_matmul}[case["op"]](case, seed)


def _prepare_tree(c, seed):
    g = _dev(seed, 2)
    context, drafts = _counts(c, seed)
    lens = [a + b for a, b in zip(context, drafts)]
    table, pages = _tables(c, lens, seed)
    eight = c["cache"] == "f8"
    ks, vs = ((0.01 + 0.04 * torch.rand(c["kv"], device="cuda", generator=g)) if eight else None for _ in range(2))
    # values stored in eight bits use the type's range; scores spread by about 2.5 either way
    k, v = (_store((), pages, c, g, 40.0 if eight else 1.0) for _ in range(2))
    tokens = sum(drafts) + 3  # the last ones are padding
    q = _normal((tokens, c["heads"], c["dim"]), DTYPE[c["dtype"]], g, 2.5)
    return {"case": c, "q": q, "k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table.cuda(),
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "starts": _starts(drafts).cuda(),
            "mask": None if c["chain"] else _mask(c, drafts, tokens, seed).cuda()}


def _paths(c, drafts, seed):
    """Accepted nodes [rows, depth] of each tree, ascending, and how many of them."""
    path, counts = torch.full((c["rows"], c["depth"]), -1, dtype=torch.int32), []
    u = torch.rand(c["rows"], c["depth"] + 1, generator=_rng(seed, 23)).tolist()
    for r, n in enumerate(drafts):
        want, at = min(n, 1 + int(c["depth"] * u[r][-1])), -1
        for j in range(want):
            at += 1 + int((n - at - 1 - (want - j) + 1) * u[r][j] ** 2)
            path[r, j] = at
        counts.append(want)
    return path, torch.tensor(counts, dtype=torch.int32)


def _prepare_accept(c, seed):
    g = _dev(seed, 4)
    context, drafts = _counts(c, seed)
    lens = [a + b for a, b in zip(context, drafts)]
    table, pages = _tables(c, lens, seed)
    path, counts = _paths(c, drafts, seed)
    k, v = (_store((c["layers"],), pages, c, g) for _ in range(2))
    return {"case": c, "k": k, "v": v, "table": table.cuda(), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "starts": _starts(drafts).cuda(), "path": path.cuda(), "counts": counts.cuda()}


def _prepare_copy(c, seed):
    g, n, times = _dev(seed, 5), c["tokens"], c["times"]
    table, pages = _tables(c, [n] * (times + 1), seed)
    at = torch.arange(n)
    slots = table[:, at // c["page"]] * c["page"] + at % c["page"]  # [rows, tokens]
    src, dst = slots[0].repeat(times), slots[1:].reshape(-1).clone()
    dst[11::37] = -1  # padding of a batch
    k, v = (_store((c["layers"],), pages, c, g) for _ in range(2))
    return {"case": c, "k": k, "v": v, "src": src.to(torch.int32).cuda(), "dst": dst.to(torch.int32).cuda()}


def _prepare_norm(c, seed):
    g, shape, dt = _dev(seed, 6), (c["tokens"], c["hidden"]), DTYPE[c["dtype"]]
    # a residual stream has a few dims that are far larger than the others
    wide = torch.where(torch.rand(c["hidden"], device="cuda", generator=g) < 0.01, 30.0, 1.0)
    x = (torch.randn(shape, device="cuda", generator=g) * wide).to(dt)
    return {"case": c, "x": x, "residual": _normal(shape, dt, g, 3.0) if c["residual"] else None,
            "weight": (1 + 0.2 * torch.randn(c["hidden"], device="cuda", generator=g)).to(dt) if c["normed"] else None}


def _blocks(x):
    """[rows, blocks, 128] of x [rows, n], zeros past n."""
    rows, n = x.shape
    return torch.nn.functional.pad(x, (0, -n % BLOCK)).view(rows, -1, BLOCK)


def _plain_eight(x):
    """x [rows, n] (float32) in eight bits with a scale for each 128 values of a row."""
    b = _blocks(x)
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / torch.full_like(top, TOP), torch.ones_like(top))  # divided, not times 1 / 448
    q = (b / scale).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return q.reshape(x.shape[0], -1)[:, :x.shape[1]].contiguous(), scale[..., 0].contiguous()


def _prepare_matmul(c, seed):
    g, m, k, n = _dev(seed, 8), c["tokens"], c["hidden"], c["out"]
    s = {"case": c, "bias": _normal((n,), torch.float32, g) if c["bias"] else None}
    x = _normal((m, k), DTYPE["bf16" if c["x"] == "f8" else c["x"]], g)
    if c["x"] == "f8":
        s["x"], s["x_scale"] = _plain_eight(x.float())
    else:
        s["x"], s["x_scale"] = x, None
    s["w"] = _normal((n, k), torch.float8_e4m3fn, g, 60.0)
    s["w_scale"] = (0.5 + torch.rand((-(-n // BLOCK), -(-k // BLOCK)), device="cuda", generator=g)) * (0.01 * k ** -0.5)
    return s


# ------------------------------------------------------------------------------ the passes

def run(s):
    op = s["case"]["op"]
    if own:
        return {"tree": _own_tree, "accept": _own_accept, "copy": _own_copy, "norm": _own_norm, "matmul": _own_matmul}[op](s)
    return {"tree": _plain_tree, "accept": _plain_accept, "copy": _plain_copy, "norm": _plain_norm, "matmul": _plain_matmul}[op](s)


def _own_tree(s):
    import mlxr_amd as mx
    return mx.paged_tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"], s["mask"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"])


def _own_accept(s):
    import mlxr_amd as mx
    return [mx.paged_accept(s["k"], s["v"], s["table"], s["lens"], s["starts"], s["path"], s["counts"]), s["k"], s["v"]]


def _own_copy(s):
    import mlxr_amd as mx
    mx.paged_copy(s["k"], s["v"], s["src"], s["dst"])
    return [s["k"], s["v"]]


def _own_norm(s):
    import mlxr_amd as mx
    c = s["case"]
    if not c["normed"]:
        return list(mx.quantize_fp8(s["x"]))
    got = mx.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"], quantize=c["eight"])
    y, total = got if c["residual"] else (got, None)
    return [*(y if c["eight"] else [y]), *([total] if c["residual"] else [])]


def _own_matmul(s):
    import mlxr_amd as mx
    x = s["x"] if s["x_scale"] is None else mx.Fp8Rows(s["x"], s["x_scale"])
    return mx.fp8_matmul(x, mx.Fp8Weight(s["w"], s["w_scale"]), bias=s["bias"], out_dtype=DTYPE[s["case"]["dtype"]])


def _gather(store, table):
    """[rows, kv, positions, dim] of a store by its table, in float32."""
    rows, wide = table.shape
    at = table.clamp(min=0).long()
    got = store.view(torch.uint8)[at].view(store.dtype) if store.element_size() == 1 else store[at]
    return got.float().permute(0, 2, 1, 3, 4).reshape(rows, store.shape[1], wide * store.shape[2], store.shape[3])


def _plain_tree(s):
    c, q, starts = s["case"], s["q"], s["starts"].long()
    rows, kv, group, dim, n = c["rows"], c["kv"], c["heads"] // c["kv"], c["dim"], c["nodes"]
    count = starts[1:] - starts[:-1]
    context = s["lens"].long() - count
    node = torch.arange(n, device=q.device)
    token = torch.where(node < count[:, None], starts[:-1, None] + node, q.shape[0] - 1)  # [rows, n]; a padding token past a row's
    place = torch.arange(s["table"].shape[1] * c["page"], device=q.device)
    of = place - context[:, None]  # [rows, places]: the node that lies there
    if s["mask"] is None:
        sees = of[:, None, :] <= node[:, None]
    else:
        at = of.clamp(0, n - 1)[:, None, :].expand(-1, n, -1)
        sees = (of < 0)[:, None, :] | (s["mask"][token].gather(2, at // 64) >> at % 64 & 1).bool()
    sees = sees & (of < count[:, None])[:, None, :]
    score = (q.float()[token].view(rows, n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(rows, kv, group * n, dim)
             @ _gather(s["k"], s["table"]).transpose(2, 3)).view(rows, kv, group, n, -1) * dim ** -0.5
    if s["k_scale"] is not None:
        score = score * s["k_scale"].view(1, -1, 1, 1, 1)
    score = score.masked_fill(~sees[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    v = _gather(s["v"], s["table"]).masked_fill((of >= count[:, None])[:, None, :, None], 0.0)
    total = p.sum(-1, keepdim=True)
    out = (p.view(rows, kv, group * n, -1) @ v).view(rows, kv, group, n, dim) / torch.where(total > 0, total, 1.0)
    if s["v_scale"] is not None:
        out = out * s["v_scale"].view(1, -1, 1, 1, 1)
    out = out.permute(0, 3, 1, 2, 4).reshape(rows, n, c["heads"], dim)
    real = node < count[:, None]
    got = torch.zeros_like(q)
    got[token[real]] = out[real].to(q.dtype)
    return got


def _plain_move(store, src, dst):
    """Tokens at slots src to slots dst, in every layer."""
    page = store.shape[3]
    t = store.view(torch.uint8) if store.element_size() == 1 else store
    t[:, dst // page, :, dst % page] = t[:, src // page, :, src % page]


def _plain_accept(s):
    c, starts, path = s["case"], s["starts"].long(), s["path"].long()
    count = starts[1:] - starts[:-1]
    context = s["lens"].long() - count
    j = torch.arange(path.shape[1], device=path.device)
    before = torch.cat([path.new_full((c["rows"], 1), -1), path[:, :-1]], 1)
    ok = ((j < s["counts"].long()[:, None]) & (path > before) & (path < count[:, None])).long().cumprod(1).bool()
    row = torch.arange(c["rows"], device=path.device)[:, None].expand_as(path)[ok]

    def slots(position):
        return s["table"][row, position // c["page"]].long() * c["page"] + position % c["page"]

    src, dst = slots((context[:, None] + path)[ok]), slots((context[:, None] + j)[ok])
    for store in (s["k"], s["v"]):
        _plain_move(store, src, dst)
    return [(context + ok.sum(1)).to(torch.int32), s["k"], s["v"]]


def _plain_copy(s):
    ok = (s["src"] >= 0) & (s["dst"] >= 0)
    src, dst = s["src"][ok].long(), s["dst"][ok].long()
    for store in (s["k"], s["v"]):
        _plain_move(store, src, dst)
    return [s["k"], s["v"]]


def _plain_norm(s):
    c, x = s["case"], s["x"].float()
    total = x + s["residual"].float() if c["residual"] else x
    y = total
    if c["normed"]:
        y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    y = list(_plain_eight(y)) if c["eight"] else [y.to(s["x"].dtype)]
    return [*y, *([total.to(s["x"].dtype)] if c["residual"] else [])]


def _plain_matmul(s):
    x, xs = (s["x"], s["x_scale"]) if s["x_scale"] is not None else _plain_eight(s["x"].float())
    n, k = s["w"].shape
    x = x.float() * xs.repeat_interleave(BLOCK, 1)[:, :k]
    w = s["w"].float() * s["w_scale"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    return (y if s["bias"] is None else y + s["bias"]).to(DTYPE[s["case"]["dtype"]])


# ------------------------------------------------------------------------------ the counts

def work(case):
    c = case
    if c["op"] == "tree":
        context, drafts = _counts(c, 0)
        # a node sees its context, itself and its ancestors: of the drafted tokens half, or their logarithm
        pairs = sum(n * (a + (n / 2 if c["chain"] else math.log2(n + 1))) for a, n in zip(context, drafts))
        held = sum(a + n for a, n in zip(context, drafts) if n)
        return {"bytes": 2 * held * c["kv"] * c["dim"] * SIZE[c["cache"]] + 2 * sum(drafts) * c["heads"] * c["dim"] * SIZE[c["dtype"]],
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    if c["op"] == "accept":
        _, drafts = _counts(c, 0)
        path, _ = _paths(c, drafts, 0)
        moved = int((path > torch.arange(c["depth"])).sum())
        return {"bytes": 4 * moved * c["layers"] * c["kv"] * c["dim"] * SIZE[c["cache"]] + 4 * path.numel(), "flops": 0}
    if c["op"] == "copy":
        each = 2 * c["layers"] * c["kv"] * c["dim"] * SIZE[c["cache"]]
        return {"bytes": c["tokens"] * (c["times"] + 1) * each, "flops": 0}
    if c["op"] == "norm":
        n, size = c["tokens"] * c["hidden"], SIZE[c["dtype"]]
        out = n + 4 * c["tokens"] * -(-c["hidden"] // BLOCK) if c["eight"] else n * size
        return {"bytes": n * size * (3 if c["residual"] else 1) + out + c["hidden"] * size, "flops": 4 * n}
    m, k, n = c["tokens"], c["hidden"], c["out"]
    x = m * k * SIZE[c["x"]] + (4 * m * -(-k // BLOCK) if c["x"] == "f8" else 0)
    return {"bytes": n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK) + x + m * n * SIZE[c["dtype"]], "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "accept": _exact_accept, "copy": _exact_copy, "norm": _exact_norm,
            "matmul": _exact_matmul}[case["op"]](case, s)


def _exact_tree(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, lens, mask = s["starts"].tolist(), s["lens"].tolist(), None if s["mask"] is None else s["mask"].tolist()
    group = c["heads"] // c["kv"]
    for r in range(c["rows"]):
        a, b, held = starts[r], starts[r + 1], lens[r]
        if a == b:
            continue
        sees = torch.ones((b - a, held), dtype=torch.bool)
        tree = sees[:, held - (b - a):]
        if mask is None:
            tree.copy_(torch.tril(tree))
        else:
            for i in range(b - a):
                words = mask[a + i]
                for j in range(b - a):
                    tree[i, j] = bool(words[j >> 6] >> (j & 63) & 1)
        sees = sees.cuda()
        pages = s["table"][r, :-(-held // c["page"])].long()
        for h in range(c["kv"]):
            k, v = (torch.cat([p for p in t[:, h].view(torch.uint8)[pages].view(t.dtype)] if t.element_size() == 1
                              else [p for p in t[pages, h]])[:held].double() for t in (s["k"], s["v"]))
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            for g in range(h * group, (h + 1) * group):
                score = (s["q"][a:b, g].double() @ k.t() / math.sqrt(c["dim"])).masked_fill_(~sees, -math.inf)
                out[a:b, g] = torch.softmax(score, -1) @ v
    return out


def _exact_accept(c, s):
    starts, lens, path, counts = (s[k].tolist() for k in ("starts", "lens", "path", "counts"))
    got = []
    for r in range(c["rows"]):
        n, kept, last = starts[r + 1] - starts[r], 0, -1
        while kept < min(counts[r], c["depth"]) and last < path[r][kept] < n:
            last = path[r][kept]
            kept += 1
        got.append(lens[r] - n + kept)
    return [torch.tensor(got, dtype=torch.int32), None, None]  # the stores hold copies


def _exact_copy(c, s):
    return None  # copies


def _exact_eight(y):
    """y / scale before its rounding, and the scales (float32 values: what is rounded goes by them)."""
    rows, n = y.shape
    scale = torch.ones((rows, -(-n // BLOCK)), dtype=torch.float64, device=y.device)
    for b in range(scale.shape[1]):
        top = y[:, b * BLOCK:(b + 1) * BLOCK].abs().max(1).values
        scale[:, b] = torch.where(top > 0, top / TOP, 1.0).float().double()
    return torch.stack([y[:, i] / scale[:, i // BLOCK] for i in range(n)], 1), scale


def _exact_norm(c, s):
    total = s["x"].double() + (s["residual"].double() if c["residual"] else 0)
    y = total
    if c["normed"]:
        y = total / torch.sqrt((total * total).sum(1, keepdim=True) / c["hidden"] + EPS) * s["weight"].double()
    return [*(_exact_eight(y) if c["eight"] else [y]), *([total] if c["residual"] else [])]


def _exact_matmul(c, s):
    n, k = s["w"].shape
    x, xs = s["x"].double(), s["x_scale"]
    if xs is None:
        x, xs = _exact_eight(x)
        x = x.float().clamp(-TOP, TOP).to(torch.float8_e4m3fn).double()
    y = torch.zeros((c["tokens"], n), dtype=torch.float64, device="cuda")
    at = torch.arange(n, device="cuda") // BLOCK
    for b in range(xs.shape[1]):
        part = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        y += (x[:, part] @ s["w"][:, part].double().t()) * xs[:, b:b + 1].double() * s["w_scale"][at, b].double()
    return y if s["bias"] is None else y + s["bias"].double()
