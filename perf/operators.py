"""Performance cases of the serving operators that stand beside the quantized projections.

A decode step over many requests brings every request's pages up to its new length
(``page_resize``), adds the requests' low-rank adapters to the shared projections
(``lora_apply``), writes the new keys and values into the paged cache (``paged_append``) and
attends over it (``paged_attention``).  A case is one call of one of them, as such a step makes
it.  Model sizes are those of the tests and the benchmark (TinyLlama, Llama-3-8B, Llama-3-70B)
or generic; lengths, pages and adapters are drawn ragged, with empty rows among them.

``run`` is the plain form (elementary torch operations in float32) unless ``own`` is set;
``exact`` is the definition in float64.
"""
import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f8": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "f8": 1}


def _attention(name, rows, heads, kv, dim, longest, page, dtype="bf16", cache="bf16", window=0, ragged=True,
               token_major=False):
    """One new token for each of `rows` requests; lengths up to `longest` (ragged: spread over the
    range, one in eleven rows empty).  token_major: a page holds [token, head, dim]."""
    return {"name": name, "op": "attention", "rows": rows, "heads": heads, "kv": kv, "dim": dim, "longest": longest,
            "page": page, "dtype": dtype, "cache": cache, "window": window, "ragged": ragged, "token_major": token_major}


def _append(name, tokens, kv, dim, pages, page, dtype="bf16", cache="bf16", token_major=False):
    return {"name": name, "op": "append", "tokens": tokens, "kv": kv, "dim": dim, "pages": pages, "page": page,
            "dtype": dtype, "cache": cache, "token_major": token_major}


def _resize(name, rows, longest, page, grow, turnover):
    """grow: tokens each running request gains; turnover: share of the rows that change: half of
    them end (all pages go back), half are admitted with a prompt."""
    return {"name": name, "op": "resize", "rows": rows, "longest": longest, "page": page, "grow": grow, "turnover": turnover}


def _lora(name, tokens, adapters, rank, hidden, outs, dtype="bf16", none=0.1, run=1):
    """outs: widths of the projections that share x, "a,b,...".  run: neighbouring tokens of one
    adapter (a prompt); none: share of the tokens without an adapter."""
    return {"name": name, "op": "lora", "tokens": tokens, "adapters": adapters, "rank": rank, "hidden": hidden,
            "outs": outs, "dtype": dtype, "none": none, "run": run}


def listed():
    return [
        # one TinyLlama request early in its answer: latency counts
        _attention("attn_tiny_m1", 1, 32, 4, 64, 700, 16, dtype="f16", cache="f16", ragged=False),
        # a decode batch of Llama-3-8B over ragged contexts up to the model's 8192
        _attention("attn_8b_m64", 64, 32, 8, 128, 8192, 16),
        # one request with a very long context: all the work is in one row
        _attention("attn_8b_long", 1, 32, 8, 128, 120001, 16, ragged=False),
        # a large model's batch over an eight-bit cache
        _attention("attn_70b_fp8_m32", 32, 64, 8, 128, 16384, 32, cache="f8"),
        # as many key heads as heads, a sliding window, pages laid out by token
        _attention("attn_mha_window_m17", 17, 32, 32, 80, 6000, 64, window=1024, token_major=True),
        # the new keys and values of a decode batch
        _append("append_8b_m64", 64, 8, 128, 4096, 16),
        # those of a prompt, rounded to eight bits
        _append("append_8b_prompt_fp8", 4099, 8, 128, 1024, 32, cache="f8"),
        # every request of a full batch gains a token
        _resize("pages_decode_m256", 256, 8192, 16, 1, 0.0),
        # requests end and prompts are admitted beside running ones
        _resize("pages_admit_m96", 96, 16384, 16, 1, 0.5),
        # q/k/v of a small decode batch, an adapter for nearly every request
        _lora("lora_8b_qkv_m8", 8, 16, 16, 4096, "4096,1024,1024", none=0.0),
        # gate and up of a large model for a full batch, high ranks
        _lora("lora_70b_gate_up_m61", 61, 24, 64, 8192, "28672,28672"),
        # gate and up over prompts of several requests
        _lora("lora_8b_gate_up_m2048", 2048, 6, 32, 4096, "14336,14336", run=341),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), work(c)["bytes"])
    while True:
        op = rng.choice(["attention", "attention", "append", "resize", "lora", "lora"])
        if op == "attention":
            kv, dim = rng.choice([1, 2, 4, 8, 8, 8, 10, 32]), rng.choice([64, 80, 112, 128, 128, 128, 256])
            dtype = rng.choice(["bf16", "bf16", "f16"])
            c = _attention("", _log(rng, 1, 128), kv * rng.choice([1, 2, 4, 4, 7, 8]), kv, dim, _log(rng, 1, 131072),
                           rng.choice([16, 16, 32, 64, 128]), dtype, rng.choice([dtype, dtype, "f8"]),
                           rng.choice([0, 0, 0, rng.randrange(1, 5000)]), rng.random() < 0.8, rng.random() < 0.3)
            if c["rows"] * c["longest"] * kv * dim > 64 * 8192 * 8 * 128:  # what the plain form has to gather
                continue
        elif op == "append":
            dtype, page = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([16, 16, 32, 64])
            c = _append("", _log(rng, 1, 4099), rng.choice([1, 2, 4, 8, 8, 32]), rng.choice([64, 80, 128, 128, 256]), 0, page,
                        dtype, rng.choice(["bf16", "f16", "f8"]), rng.random() < 0.3)
            c["pages"] = max(64, 8192 // page, 2 * -(-c["tokens"] // page))
            if c["pages"] * page * c["kv"] * c["dim"] > 1 << 27:
                continue
        elif op == "resize":
            c = _resize("", _log(rng, 1, 1024), _log(rng, 16, 16384), rng.choice([8, 16, 16, 32, 64]),
                        rng.choice([1, 1, rng.randrange(2, 9)]), rng.choice([0.0, 0.1, 0.5, 1.0]))
            if c["rows"] * c["longest"] > 256 * 8192:
                continue
        else:
            tokens, hidden = _log(rng, 1, 2048), rng.choice([2048, 2560, 3584, 4096, 5120, 6656, 8192])
            outs = [rng.choice([1024, 4096, 14336, 16 * (2 * _log(rng, 32, 448) + 1)]) for _ in range(rng.choice([1, 2, 3]))]
            if rng.random() < 0.3:
                outs[-1] += rng.randrange(1, 64)
            adapters, rank = _log(rng, 1, 64), rng.choice([8, 16, 16, 32, 64, 24])
            if adapters * rank > 2048:  # what the plain form multiplies every token with
                continue
            c = _lora("", tokens, adapters, rank, hidden, ",".join(map(str, outs)), rng.choice(["bf16", "bf16", "f16"]),
                      rng.choice([0.0, 0.1, 0.5]), rng.choice([1, 1, max(1, tokens // 5)]))
        del c["name"]
        if work(c)["bytes"] <= most[op]:
            return c


# ------------------------------------------------------------------------------ the inputs

def _rng(seed, *ids):
    s = int(seed)
    for i in ids:
        s = (s * 1000003 + int(i) + 12345) % (1 << 62)
    return torch.Generator().manual_seed(s)


def _dev(seed, *ids):
    return torch.Generator(device="cuda").manual_seed(int(_rng(seed, 77, *ids).initial_seed()))


def _lengths(c, seed):
    """Lengths of the rows of an attention case (host): the longest first, then ragged."""
    n, g = c["longest"], _rng(seed, 1)
    if not c["ragged"]:
        return [n] * c["rows"]
    share = torch.rand(c["rows"], generator=g).tolist()
    got = [max(1, int(n * s)) for s in share]
    for r in range(c["rows"]):
        if r % 11 == 10:
            got[r] = 0
    got[0] = n
    return got


def _normal(shape, dtype, g, scale=1.0):
    """N(0, scale) in dtype, made a slice at a time so that long caches need no float32 copy."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    step = 1 << 26
    for at in range(0, flat.numel(), step):
        part = flat[at:at + step]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=g) * scale)
    return t


def _store(pages, c, g, scale=1.0):
    """A key or value store [pages, kv, page, dim], in the case's memory order."""
    if c["token_major"]:
        return _normal((pages, c["page"], c["kv"], c["dim"]), DTYPE[c["cache"]], g, scale).permute(0, 2, 1, 3)
    return _normal((pages, c["kv"], c["page"], c["dim"]), DTYPE[c["cache"]], g, scale)


def prepare(case, seed):
    return {"attention": _prepare_attention, "append": _prepare_append, "resize": _prepare_resize,
            "lora": _prepare_lora}[case["op"]](case, seed)


def _scales(c, g):
    """What the cache's values are multiplied with, for each kv head (eight-bit caches)."""
    if c["cache"] != "f8":
        return None, None
    return (0.01 + 0.04 * torch.rand(c["kv"], device="cuda", generator=g),
            0.01 + 0.04 * torch.rand(c["kv"], device="cuda", generator=g))


def _prepare_attention(c, seed):
    lens, g = _lengths(c, seed), _dev(seed, 2)
    page = c["page"]
    held = [-(-n // page) for n in lens]
    wide = max(held)
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=_rng(seed, 3)).to(torch.int32)
    table = torch.full((c["rows"], wide), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    ks, vs = _scales(c, g)
    # values stored in eight bits use the type's range; scores spread by about 2.5 either way
    k = _store(pages, c, g, 40.0 if ks is not None else 1.0)
    v = _store(pages, c, g, 40.0 if ks is not None else 1.0)
    q = _normal((c["rows"], c["heads"], c["dim"]), DTYPE[c["dtype"]], g, 2.5)
    return {"case": c, "q": q, "k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table.cuda(),
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}


def _prepare_append(c, seed):
    g, n = _dev(seed, 4), c["tokens"]
    k, v = (_normal((n, c["kv"], c["dim"]), DTYPE[c["dtype"]], g) for _ in range(2))
    ks, vs = _scales(c, g)
    slots = torch.randperm(c["pages"] * c["page"], generator=_rng(seed, 5))[:n].to(torch.int32)
    slots[10::23] = -1  # padding of a batch
    return {"case": c, "new_k": k, "new_v": v, "k": _store(c["pages"], c, g), "v": _store(c["pages"], c, g),
            "k_scale": ks, "v_scale": vs, "slots": slots.cuda()}


def _resize_plan(c, seed):
    """(lengths held, lengths wanted) of the rows."""
    g = _rng(seed, 6)
    have = (torch.rand(c["rows"], generator=g) * (c["longest"] - c["grow"])).to(torch.int64).clamp_(min=1).tolist()
    other = (torch.rand(c["rows"], generator=g) * c["longest"]).to(torch.int64).clamp_(min=1).tolist()
    draw_ = torch.rand(c["rows"], generator=g).tolist()
    want = [min(n + c["grow"], c["longest"]) for n in have]
    for r in range(c["rows"]):
        if draw_[r] < c["turnover"] / 2:  # ends
            want[r] = 0
        elif draw_[r] < c["turnover"]:  # is admitted
            have[r], want[r] = 0, other[r]
    return have, want


def _prepare_resize(c, seed):
    have, want = _resize_plan(c, seed)
    page, wide = c["page"], -(-c["longest"] // c["page"])
    held = [-(-n // page) for n in have]
    pages = c["rows"] * wide  # a pool that holds every row at its longest
    order = torch.randperm(pages, generator=_rng(seed, 7)).to(torch.int32)
    table = torch.full((c["rows"], wide), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    free = torch.full((pages,), -1, dtype=torch.int32)
    free[:pages - at] = order[at:]
    # places for the new tokens: the running rows' and twice the prompts that are admitted on average
    tokens = c["rows"] * c["grow"] + int(c["turnover"] * c["rows"] * c["longest"] / 2) + 5
    return {"case": c, "table": table.cuda(), "free": free.cuda(), "tokens": tokens,
            "free_count": torch.tensor([pages - at], dtype=torch.int32, device="cuda"),
            "lens": torch.tensor(have, dtype=torch.int32, device="cuda"),
            "want": torch.tensor(want, dtype=torch.int32, device="cuda")}


def _widths(c):
    return [int(n) for n in c["outs"].split(",")]


def _adapter_ids(c, seed):
    g, n = _rng(seed, 8), c["tokens"]
    ids = torch.randint(0, c["adapters"], (-(-n // c["run"]),), generator=g)
    ids[torch.rand(ids.numel(), generator=g) < c["none"]] = -1
    return ids.repeat_interleave(c["run"])[:n].to(torch.int32)


def _ranks(c, seed):
    """Adapters have their own ranks, up to the bank's."""
    return [c["rank"] if i % 3 else max(1, c["rank"] // 2) for i in range(c["adapters"])]


def _prepare_lora(c, seed):
    g, dt, k, r = _dev(seed, 9), DTYPE[c["dtype"]], c["hidden"], c["rank"]
    return {"case": c, "x": _normal((c["tokens"], k), dt, g), "ids": _adapter_ids(c, seed).cuda(),
            "a": [_normal((c["adapters"], r, k), dt, g, k ** -0.5) for _ in _widths(c)],
            "b": [_normal((c["adapters"], n, r), dt, g, 0.5 * r ** -0.5) for n in _widths(c)],
            "y": [_normal((c["tokens"], n), dt, g) for n in _widths(c)],
            "scales": 0.5 + torch.rand(c["adapters"], device="cuda", generator=g),
            "ranks": torch.tensor(_ranks(c, seed), dtype=torch.int32, device="cuda")}


# ------------------------------------------------------------------------------ the passes

def run(s):
    op = s["case"]["op"]
    if own:
        return {"attention": _own_attention, "append": _own_append, "resize": _own_resize, "lora": _own_lora}[op](s)
    return {"attention": _plain_attention, "append": _plain_append, "resize": _plain_resize, "lora": _plain_lora}[op](s)


def _own_attention(s):
    import mlxr_amd as mx
    return mx.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                              window=s["case"]["window"])


def _own_append(s):
    import mlxr_amd as mx
    mx.paged_append(s["new_k"], s["new_v"], s["k"], s["v"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return [s["k"], s["v"]]


def _own_resize(s):
    import mlxr_amd as mx
    r = mx.page_resize(s["table"], s["lens"], s["want"], s["free"], s["free_count"], s["case"]["page"], s["tokens"])
    return [s["table"], s["free"], r.lens, r.free_count, r.starts, r.slots, r.positions, r.refused]


def _own_lora(s):
    import mlxr_amd as mx
    return mx.lora_apply(s["x"], s["ids"], s["a"], s["b"], s["y"], scales=s["scales"], ranks=s["ranks"])


def _stored(t):
    """The values a store's elements stand for, before their head's scale."""
    return t.to(torch.float32)


def _gather(store, table):
    """[rows, kv, positions, dim] of a store by its table, in float32."""
    rows, wide = table.shape
    at = table.clamp(min=0).long()
    got = store.view(torch.uint8)[at].view(torch.float8_e4m3fn) if store.element_size() == 1 else store[at]
    got = _stored(got)  # [rows, wide, kv, page, dim]
    return got.permute(0, 2, 1, 3, 4).reshape(rows, store.shape[1], wide * store.shape[2], store.shape[3])


def _plain_attention(s):
    c, q, lens = s["case"], s["q"], s["lens"].long()
    rows, group = c["rows"], c["heads"] // c["kv"]
    scale = c["dim"] ** -0.5
    at = torch.arange(s["table"].shape[1] * c["page"], device=q.device)
    first = (lens - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(lens)
    keep = (at[None, :] < lens[:, None]) & (at[None, :] >= first[:, None])
    score = q.float().view(rows, c["kv"], group, c["dim"]) @ _gather(s["k"], s["table"]).transpose(2, 3) * scale
    if s["k_scale"] is not None:
        score = score * s["k_scale"].view(1, -1, 1, 1)
    score = score.masked_fill(~keep[:, None, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    v = _gather(s["v"], s["table"]).masked_fill(~keep[:, None, :, None], 0.0)
    out = (p @ v) / p.sum(-1, keepdim=True)
    if s["v_scale"] is not None:
        out = out * s["v_scale"].view(1, -1, 1, 1)
    out = out.masked_fill((lens == 0)[:, None, None, None], 0.0)
    return out.reshape(rows, c["heads"], c["dim"]).to(q.dtype)


def _plain_append(s):
    page = s["case"]["page"]
    at = (s["slots"] >= 0).nonzero()[:, 0]
    slots = s["slots"][at].long()
    for new, store, scale in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
        x = new.float()[at]
        if scale is not None:
            x = (x / scale.view(1, -1, 1)).clamp(-448.0, 448.0)
            store.view(torch.uint8)[slots // page, :, slots % page] = x.to(store.dtype).view(torch.uint8)
        else:
            store[slots // page, :, slots % page] = (x.clamp(-448.0, 448.0) if store.element_size() == 1 else x).to(store.dtype)
    return [s["k"], s["v"]]


def _plain_resize(s):
    page, have, want = s["case"]["page"], s["lens"].long(), s["want"].long()
    rows, wide = s["table"].shape
    pages, count = s["free"].numel(), s["free_count"].long()
    held, asked = (have + page - 1) // page, (want + page - 1) // page
    fits = asked <= wide
    need = torch.where(fits, (asked - held).clamp(min=0), 0)
    give = (held - asked).clamp(min=0)
    stack = count + give.sum()
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= stack))
    taken = torch.where(granted, need, 0)
    new_lens = torch.where(granted, want, have)
    col = torch.arange(wide, device=have.device)[None, :]
    # pages that go back, in the order of the rows, onto the stack
    back = (col >= asked[:, None]) & (col < held[:, None])
    place = torch.where(back, count + (give.cumsum(0) - give)[:, None] + col - asked[:, None], pages)
    free = torch.cat([s["free"], s["free"].new_zeros(1)])
    free = free.scatter(0, place.reshape(-1), s["table"].reshape(-1))
    # pages taken from its top
    out = granted[:, None] & (col >= held[:, None]) & (col < asked[:, None])
    place = torch.where(out, stack - 1 - ((upto - need)[:, None] + col - held[:, None]), pages)
    table = torch.where(out, free[place], s["table"])
    gained = (new_lens - have).clamp(min=0)
    ends = gained.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(s["tokens"], device=have.device)
    row = torch.searchsorted(ends, t, right=True).clamp(max=rows - 1)
    pos = have[row] + t - starts[row]
    real = t < ends[-1]
    at = torch.where(real, pos // page, 0)
    slots = torch.where(real, table[row, at].long() * page + pos % page, -1)
    pos = torch.where(real, pos, -1)
    i32 = torch.int32
    return [table, free[:-1], new_lens.to(i32), (stack - taken.sum()).to(i32), starts.to(i32), slots.to(i32), pos.to(i32),
            (~granted).sum().view(1).to(i32)]


def _plain_lora(s):
    c, x, ids = s["case"], s["x"].float(), s["ids"].long()
    n, r = c["adapters"], c["rank"]
    mine = ids[:, None] == torch.arange(n, device=x.device)[None, :]  # [tokens, adapters]
    in_rank = torch.arange(r, device=x.device)[None, :] < s["ranks"][:, None]  # [adapters, rank]
    keep = (mine[:, :, None] & in_rank[None]).reshape(-1, n * r)
    got = []
    weight = s["scales"].repeat_interleave(r)
    for a, b, y in zip(s["a"], s["b"], s["y"]):
        h = x @ a.float().view(n * r, -1).t()
        h = torch.where(keep, h * weight, 0.0)
        d = h @ b.float().transpose(1, 2).reshape(n * r, -1)
        got.append((y.float() + d).to(y.dtype))
    return got


# ------------------------------------------------------------------------------ the counts

def work(case):
    c = case
    if c["op"] == "attention":
        lens = _lengths(c, 0)
        seen = sum(min(n, c["window"]) if c["window"] else n for n in lens)
        return {"bytes": 2 * seen * c["kv"] * c["dim"] * SIZE[c["cache"]] + 2 * c["rows"] * c["heads"] * c["dim"] * SIZE[c["dtype"]],
                "flops": 4 * seen * c["heads"] * c["dim"]}
    if c["op"] == "append":
        n = c["tokens"] * c["kv"] * c["dim"]
        return {"bytes": 2 * n * (SIZE[c["dtype"]] + SIZE[c["cache"]]) + 4 * c["tokens"], "flops": 2 * n}
    if c["op"] == "resize":
        have, want = _resize_plan(c, 0)
        page = c["page"]
        moved = sum(abs(-(-w // page) + -h // page) for w, h in zip(want, have))
        gained = sum(max(0, w - h) for w, h in zip(want, have))
        return {"bytes": 16 * c["rows"] + 8 * moved + 8 * gained, "flops": 10 * c["rows"] + 2 * gained}
    ids = _adapter_ids(c, 0)
    ranks = _ranks(c, 0)
    used = set(ids.tolist()) - {-1}
    k, wide = c["hidden"], _widths(c)
    rank_rows = sum(ranks[i] for i in used)
    flops = sum(2 * ranks[i] for i in ids.tolist() if i >= 0) * (k * len(wide) + sum(wide))
    return {"bytes": SIZE[c["dtype"]] * (c["tokens"] * (k + 2 * sum(wide)) + rank_rows * (k * len(wide) + sum(wide))), "flops": flops}


# ------------------------------------------------------------------------------ the definition

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "resize":
        return None  # whole numbers
    return {"attention": _exact_attention, "append": _exact_append, "lora": _exact_lora}[case["op"]](s)


def _exact_attention(s):
    c, lens = s["case"], s["lens"].tolist()
    page, group = c["page"], c["heads"] // c["kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda")
        page_of = s["table"][r, at // page].long()
        for h in range(c["kv"]):
            k = s["k"].view(torch.uint8)[page_of, h, at % page].view(s["k"].dtype) if c["cache"] == "f8" else s["k"][page_of, h, at % page]
            v = s["v"].view(torch.uint8)[page_of, h, at % page].view(s["v"].dtype) if c["cache"] == "f8" else s["v"][page_of, h, at % page]
            k, v = k.to(torch.float32).double(), v.to(torch.float32).double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            q = s["q"][r, h * group:(h + 1) * group].double()
            w = torch.softmax((q @ k.t()) / math.sqrt(c["dim"]), dim=-1)
            out[r, h * group:(h + 1) * group] = w @ v
    return out


def _exact_append(s):
    c, page = s["case"], s["case"]["page"]
    got = []
    for new, store, scale in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
        full = store.to(torch.float32).double()
        for t, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                x = new[t].double()
                if scale is not None:
                    x = (x / scale.double()[:, None]).clamp(-448.0, 448.0)
                full[slot // page, :, slot % page] = x
        got.append(full)
    return got


def _exact_lora(s):
    ids, ranks = s["ids"].tolist(), s["ranks"].tolist()
    got = []
    for a, b, y in zip(s["a"], s["b"], s["y"]):
        out = y.double()
        for i in set(ids) - {-1}:
            rows = torch.tensor([t for t, j in enumerate(ids) if j == i], device="cuda")
            h = s["x"][rows].double() @ a[i, :ranks[i]].double().t()
            out[rows] += float(s["scales"][i]) * (h @ b[i, :, :ranks[i]].double().t())
        got.append(out)
    return got
