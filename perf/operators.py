"""The operators that answer many prompts at once: keys and values appended to a cache in pages, attention of new tokens (one, a
chunk, a whole prompt) over that cache, and the choice of the next token from its logits.

A case is a dict of plain values. "op" is one of
    append    new rows of k and v go to the pages of their sequences; with a rotation, q and k are turned by their positions on the way
    attend    every sequence's new tokens attend to all its positions up to their own, read from its pages
    sample    temperature, top-k, top-p and min-p on rows of logits, one given random number to a row
append and attend:
    dtype, heads, kv_heads, size (of a head), page (positions to a page), seqs, longest (positions of the longest sequence), new (most
    new tokens of a sequence), idle (whether some sequences have no new token), spare (rows behind the last sequence's), heads_first
    (pages laid out [kv_heads][page][size] rather than [page][kv_heads][size]); append: rot (features that are turned, 0 for none),
    neighbours (features 2 i and 2 i + 1 turned together, not i and i + rot / 2); attend: cap (soft cap of the scores, 0 for none)
sample:
    dtype, rows, vocab, pick: "greedy", "plain", "topk", "topp", "minp" or "mixed" (each row its own)
The lengths follow from the case alone; the values, and where the pages lie, from the seed.
With `own`, run issues its work on the library's stream, which neither waits for torch's nor is waited for by it: prepare ends with what it
made being there, and whoever reads run's outputs with torch waits for the device first.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_GOLDEN, _ROOT = 0.6180339887498949, 0.4142135623730951


def _paged(op, dtype, heads, kv_heads, size, page, seqs, longest, new, idle=False, spare=0, heads_first=False, **more):
    c = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, size=size, page=page, seqs=seqs, longest=longest, new=new, idle=idle,
             spare=spare, heads_first=heads_first)
    c.update({"rot": 0, "neighbours": False} if op == "append" else {"cap": 0.0})
    c.update(more)
    return c


def _sample(dtype, rows, vocab, pick):
    return dict(op="sample", dtype=dtype, rows=rows, vocab=vocab, pick=pick)


def listed():
    return [
        # one token of one sequence of the model defaults (8 heads of 32, 256 positions) in fp32: all latency
        dict(_paged("append", "f32", 8, 8, 32, 16, 1, 250, 1), name="append-one-8x32"),
        # a token each for a batch of sequences, heads shared by four, turned by position
        dict(_paged("append", "bf16", 32, 8, 128, 64, 192, 2048, 1, rot=128, spare=5), name="append-tokens-32x128"),
        # ragged prompts of the GPT-2-small shape written to their pages for the first time
        dict(_paged("append", "bf16", 12, 12, 64, 16, 20, 1024, 1024, idle=True), name="append-prompts-12x64"),
        # large prompts in fp32, partly turned features, neighbouring ones together, pages of an odd size
        dict(_paged("append", "f32", 16, 4, 128, 33, 8, 4000, 4000, rot=64, neighbours=True, heads_first=True), name="append-prompts-16x128"),
        # one token of one sequence of the GPT-2-small shape near the end of its context: all latency
        dict(_paged("attend", "bf16", 12, 12, 64, 16, 1, 777, 1, cap=30.0), name="attend-one-12x64"),
        # a token each of a batch of the 384-wide model in fp32, head size 48
        dict(_paged("attend", "f32", 8, 8, 48, 16, 20, 512, 1, cap=30.0, spare=3), name="attend-tokens-8x48"),
        # a token each of long ragged contexts, heads shared by four: the cache is read once
        dict(_paged("attend", "bf16", 32, 8, 128, 64, 24, 24000, 1), name="attend-tokens-32x128"),
        # ragged prompts of the GPT-2-small shape in fp32, the scores capped, on pages of an odd size
        dict(_paged("attend", "f32", 12, 12, 64, 24, 16, 1024, 1024, idle=True, cap=30.0), name="attend-prompts-12x64"),
        # a chunk of a long prompt behind what is cached of it, heads shared by four
        dict(_paged("attend", "bf16", 32, 8, 128, 64, 2, 16384, 2048, heads_first=True), name="attend-chunks-32x128"),
        # the next token of one sequence as the sampling defaults choose it (temperature 0.8, top 40)
        dict(_sample("f32", 1, 50304, "topk"), name="sample-one-50304"),
        # a small batch of byte-level logits, nucleus
        dict(_sample("f32", 20, 4096, "topp"), name="sample-tokens-4096"),
        # a large batch over a large vocabulary, every row with a choice of its own
        dict(_sample("bf16", 160, 131072, "mixed"), name="sample-mixed-131072"),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "sample", "sample"])
    while True:
        dtype = rng.choice(["f32", "bf16"])
        if op == "sample":
            c = _sample(dtype, spread(1, 256), spread(64, 131072), rng.choice(["greedy", "plain", "topk", "topp", "minp", "mixed", "mixed"]))
            if c["rows"] * c["vocab"] <= 160 * 131072:
                return c
            continue
        kv_heads, group = rng.randint(1, 16), rng.choice([1, 1, 1, 2, 3, 4, 8])
        longest = spread(1, 24000)
        new = rng.choice([1, 1, rng.randint(1, 16), spread(1, 2048), longest])
        c = _paged(op, dtype, kv_heads * group, kv_heads, 8 * rng.randint(1, 16), rng.choice([1, 13, 16, 16, 32, 33, 64, 64, 100, 128, 256]),
                   spread(1, 192), longest, min(new, longest), rng.random() < 0.3, rng.choice([0, 0, 7]), rng.random() < 0.4)
        if op == "append":
            c["rot"] = rng.choice([0, c["size"], 2 * rng.randint(1, c["size"] // 2)])
            c["neighbours"] = rng.random() < 0.4
        else:
            c["cap"] = rng.choice([0.0, 30.0, 5.0])
        w, rows = work(c), sum(_lengths(c)[1])
        positions = sum(-(-n // c["page"]) * c["page"] for n in _lengths(c)[0])
        if c["heads"] > 64 or rows > 32768 or positions * kv_heads * c["size"] > 3.0e8:
            continue
        # the plain form's scores and gathered keys in fp32, and the time of what is listed
        padded = c["seqs"] * longest * max(kv_heads * c["size"] * 2, c["heads"] * max(_lengths(c)[1]))
        if op == "attend" and (padded > 1.2e9 or w["flops"] > (5e11 if dtype == "bf16" else 1e11)):
            continue
        return c


def _lengths(c):
    """(positions, new tokens) of every sequence: the first is the longest, the others are spread below it."""
    lens, news = [], []
    for s in range(c["seqs"]):
        n = 1 + int((c["longest"] - 1) * (1.0 - (s * _GOLDEN) % 1.0))
        m = n if c["new"] == c["longest"] else 1 + int((c["new"] - 1) * (1.0 - (s * _ROOT) % 1.0))
        lens.append(n)
        news.append(0 if c["idle"] and s % 5 == 4 else min(m, n))
    return lens, news


def work(case):
    c = case
    if c["op"] == "sample":
        values = c["rows"] * c["vocab"]
        return {"bytes": float(values * (4 if c["dtype"] == "f32" else 2) + 28 * c["rows"]), "flops": 4.0 * values}
    lens, news = _lengths(c)
    size, rows, kv = (4 if c["dtype"] == "f32" else 2), sum(news), c["kv_heads"] * c["size"]
    table = 4 * sum(-(-n // c["page"]) for n in lens)
    if c["op"] == "append":
        turned = c["heads"] * c["size"] if c["rot"] else 0
        nbytes = size * rows * (4 * kv + 2 * turned) + (4 * rows * c["rot"] if c["rot"] else 0) + min(table, 4 * rows)
        return {"bytes": float(nbytes), "flops": 3.0 * rows * (c["rot"] * (c["heads"] + c["kv_heads"]))}
    pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lens, news))
    read = sum(n for n, m in zip(lens, news) if m)
    return {"bytes": float(size * (2 * read * kv + 2 * rows * c["heads"] * c["size"]) + 4 * rows * c["heads"] + table),
            "flops": 4.0 * pairs * c["heads"] * c["size"]}


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if c["op"] == "sample":
        # logits of a trained model: a Zipf-like law over ids in no order, noise on top
        rows, vocab = c["rows"], c["vocab"]
        rank = torch.rand(rows, vocab, generator=g, device="cuda").argsort(1)
        logits = (normal(rows, vocab) - 1.1 * torch.log1p(rank.float())).to(dtype)
        rand = torch.rand(5, rows, generator=g, device="cuda")
        off = torch.zeros(rows, device="cuda")
        mixed = c["pick"] == "mixed"
        on = {k: (rand[0] * 5).int() == i if mixed else torch.full((rows,), c["pick"] == k, device="cuda")
              for i, k in enumerate(("greedy", "plain", "topk", "topp", "minp"))}
        both = on["topk"] | (on["topp"] & (rand[3] < 0.3) if mixed else on["greedy"])
        s = {"case": dict(c), "logits": logits, "uniform": rand[1].contiguous(),
             "temperature": torch.where(on["greedy"], off, 0.8 if not mixed else 0.5 + rand[2]),
             "top_k": torch.where(both, torch.full_like(off, 40.0) if not mixed else 1 + 200 * rand[3], off).int(),
             "top_p": torch.where(on["topp"], 0.9 if not mixed else 0.5 + 0.49 * rand[4], off + 1),
             "min_p": torch.where(on["minp"], 0.05 if not mixed else 0.2 * rand[4] + 0.001, off),
             "tokens": torch.zeros(rows, dtype=torch.int32, device="cuda"), "logprobs": torch.zeros(rows, device="cuda")}
        torch.cuda.synchronize()
        return s

    lens, news = _lengths(c)
    H, Hk, D, page, seqs = c["heads"], c["kv_heads"], c["size"], c["page"], c["seqs"]
    need = [-(-n // page) for n in lens]
    pages, width, rows = sum(need) + 3, max(need), sum(news) + c["spare"]
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).int()
    table, at = torch.zeros(seqs, width, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = free[at:at + n]
        at += n
    starts = torch.tensor([0] + news).cumsum(0).int()
    shape = (pages, Hk, page, D) if c["heads_first"] else (pages, page, Hk, D)
    qkv = normal(rows, (H + 2 * Hk) * D).to(dtype)                  # one product leaves q, k and v of a row side by side
    s = {"case": dict(c), "qkv": qkv, "k": normal(*shape).to(dtype), "v": normal(*shape).to(dtype), "table": table.cuda(), "starts": starts.cuda(),
         "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "out": torch.zeros(rows, H, D, dtype=dtype, device="cuda")}
    if c["op"] == "attend":
        s["lse"] = torch.zeros(rows, H, device="cuda")
        s["scale"], s["most"] = 1.0 / math.sqrt(D), max(news)
        if H == Hk and c["cap"]:
            qkv.mul_(1.5)
    elif c["rot"]:
        angles = torch.outer(torch.arange(c["longest"], dtype=torch.float64),
                             10000.0 ** (-2.0 * torch.arange(c["rot"] // 2, dtype=torch.float64) / c["rot"]))
        s["rotary"] = torch.cat([angles.cos(), angles.sin()], 1).float().cuda()
    torch.cuda.synchronize()
    return s


def _split(s):
    c = s["case"]
    H, Hk, D = c["heads"], c["kv_heads"], c["size"]
    rows = s["qkv"].shape[0]
    q, k, v = s["qkv"].split([H * D, Hk * D, Hk * D], 1)
    return q.view(rows, H, D), k.view(rows, Hk, D), v.view(rows, Hk, D)


# ---------------------------------------------------------------------------------------------- plain forms
def _places(s):
    """(sequence, position) of every new row."""
    starts = s["starts"].long()
    row = torch.arange(s["qkv"].shape[0] - s["case"]["spare"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, s["lens"].long()[seq] - starts[seq + 1] + row


def _by_position(s, name):
    """[pages, page, kv_heads, size] whichever way the pages are laid out: a view."""
    return s[name].transpose(1, 2) if s["case"]["heads_first"] else s[name]


def _turn(x, cos, sin, rot, neighbours):
    x = x.float()
    if neighbours:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(s):
    c = s["case"]
    q, k, v = _split(s)
    seq, position = _places(s)
    rows = seq.shape[0]
    page = s["table"].long()[seq, position // c["page"]]
    q, k, v = q[:rows], k[:rows], v[:rows]
    if c["rot"]:
        cos, sin = s["rotary"][position][:, None].split(c["rot"] // 2, -1)
        s["out"][:rows] = _turn(q, cos, sin, c["rot"], c["neighbours"]).to(q.dtype)
        k = _turn(k, cos, sin, c["rot"], c["neighbours"]).to(k.dtype)
    _by_position(s, "k")[page, position % c["page"]] = k
    _by_position(s, "v")[page, position % c["page"]] = v
    return {"k": s["k"], "v": s["v"], "q": s["out"]} if c["rot"] else {"k": s["k"], "v": s["v"]}


def _plain_attend(s):
    c = s["case"]
    H, Hk, D, seqs = c["heads"], c["kv_heads"], c["size"], c["seqs"]
    lens, starts = s["lens"].long(), s["starts"].long()
    longest, most = s["table"].shape[1] * c["page"], s["most"]
    q = _split(s)[0]
    seq, position = _places(s)
    token = torch.arange(seq.shape[0], device="cuda") - starts[seq]
    # every sequence padded to the longest: [seqs, kv_heads, queries of all heads of the group, size] and [seqs, kv_heads, positions, size]
    padded = torch.zeros(seqs, most, H, D, device="cuda")
    padded[seq, token] = q[:seq.shape[0]].float()
    padded = padded.view(seqs, most, Hk, H // Hk, D).permute(0, 2, 1, 3, 4).reshape(seqs, Hk, most * (H // Hk), D)
    keys, values = (_by_position(s, n)[s["table"].long()].float().reshape(seqs, longest, Hk, D).transpose(1, 2).contiguous() for n in ("k", "v"))
    at = torch.arange(longest, device="cuda")
    values = values * (at < lens[:, None]).float()[:, None, :, None]
    scores = torch.matmul(padded, keys.transpose(2, 3).contiguous()).mul_(s["scale"])
    if c["cap"] > 0:
        scores = scores.div_(c["cap"]).tanh_().mul_(c["cap"])
    limit = torch.full((seqs, most), -1, device="cuda")
    limit[seq, token] = position
    seen = at <= limit.repeat_interleave(H // Hk, 1)[:, :, None]
    scores.masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), torch.zeros_like(top), top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, values).div_(total.clamp_min(1e-30))
    lse = (top + total.log()).view(seqs, Hk, most, H // Hk).permute(0, 2, 1, 3).reshape(seqs, most, H)
    out = out.view(seqs, Hk, most, H // Hk, D).permute(0, 2, 1, 3, 4).reshape(seqs, most, H, D)
    s["out"][:seq.shape[0]] = out[seq, token].to(q.dtype)
    s["lse"][:seq.shape[0]] = lse[seq, token]
    return {"out": s["out"], "lse": s["lse"]}


def _plain_sample(s):
    logits, temperature = s["logits"].double(), s["temperature"].double()[:, None]
    vocab = logits.shape[1]
    greedy = ~(temperature > 0)
    k, p, m = s["top_k"].long()[:, None], s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    sorted_, order = torch.sort(logits, dim=1, descending=True, stable=True)
    weights = torch.exp((sorted_ - sorted_[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    kth = sorted_.gather(1, k.clamp(1, vocab) - 1)
    weights = torch.where((k > 0) & (k < vocab) & (sorted_ < kth), torch.zeros_like(weights), weights)
    mass = weights.cumsum(1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    nucleus = (p > 0) & (p < 1)
    kept = ~(nucleus & (before >= p * mass[:, -1:])) & ~((m > 0) & (weights < m.clamp_max(1)))
    weights = torch.where(kept, weights, torch.zeros_like(weights))
    by_index = torch.zeros_like(weights).scatter_(1, order, weights)
    total = weights.sum(1, keepdim=True)
    target = s["uniform"].double()[:, None] * total
    # the first whose running mass passes the target; the last that is kept where rounding leaves none
    places = torch.arange(vocab, device="cuda")
    down = torch.minimum((weights.cumsum(1) <= target).sum(1, keepdim=True), (places * (weights > 0)).amax(1, keepdim=True))
    across = torch.minimum((by_index.cumsum(1) <= target).sum(1, keepdim=True), (places * (by_index > 0)).amax(1, keepdim=True))
    token = torch.where(greedy, order[:, :1], torch.where(nucleus, order.gather(1, down), across))
    logprob = torch.where(greedy, torch.zeros_like(total), (by_index.gather(1, token) / total).log())
    return {"tokens": token[:, 0].int(), "logprobs": logprob[:, 0].float()}


# ---------------------------------------------------------------------------------------------- the framework's operators
_library = None


def _entry_points():
    global _library
    if _library is None:
        from alpha2_amd import _ffi
        _ffi.check(_ffi.load().ah_init(0))
        _library = _ffi
    return _library


def _pages(ffi, s):
    c, k = s["case"], s["k"]
    a, b = (1, 2) if not c["heads_first"] else (2, 1)
    return ffi.AhPages({"f32": ffi.F32, "bf16": ffi.BF16}[c["dtype"]], c["kv_heads"], c["size"], c["page"], c["seqs"], s["table"].shape[1],
                       k.shape[0], k.stride(0), k.stride(a), k.stride(b), k.data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(),
                       s["starts"].data_ptr(), s["lens"].data_ptr())


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[c["op"]](s)
    ffi = _entry_points()
    lib = ffi.load()
    if c["op"] == "sample":
        rows, vocab = s["logits"].shape
        ffi.check(lib.ah_sample(ffi.AhSample({"f32": ffi.F32, "bf16": ffi.BF16}[c["dtype"]], vocab, rows, vocab, s["logits"].data_ptr(),
                                             s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(),
                                             s["uniform"].data_ptr(), s["tokens"].data_ptr(), s["logprobs"].data_ptr())))
        return {"tokens": s["tokens"], "logprobs": s["logprobs"]}
    H, Hk, D = c["heads"], c["kv_heads"], c["size"]
    rows, row = s["qkv"].shape
    q, esize = s["qkv"].data_ptr(), s["qkv"].element_size()
    if c["op"] == "append":
        rot = c["rot"]
        ffi.check(lib.ah_paged_append(_pages(ffi, s), ffi.AhPagedAppend(
            rows, H, rot, c["longest"] if rot else 0, int(c["neighbours"]), 0, row, D, row, D, row, D, H * D, D, q if rot else 0, q + H * D * esize,
            q + (H + Hk) * D * esize, s["out"].data_ptr() if rot else 0, s["rotary"].data_ptr() if rot else 0)))
        return {"k": s["k"], "v": s["v"], "q": s["out"]} if rot else {"k": s["k"], "v": s["v"]}
    ffi.check(lib.ah_paged_attention(_pages(ffi, s), ffi.AhPagedAttention(rows, H, s["scale"], c["cap"], row, D, H * D, D, q, s["out"].data_ptr(),
                                                                          s["lse"].data_ptr())))
    return {"out": s["out"], "lse": s["lse"]}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _sequences(s):
    """(positions' page, positions' row in it, first new row, row behind the last new one) of every sequence."""
    c, table = s["case"], s["table"].cpu()
    lens, news = _lengths(c)
    at = 0
    for i, (n, m) in enumerate(zip(lens, news)):
        places = torch.arange(n)
        yield table[i][places // c["page"]].long().cuda(), (places % c["page"]).cuda(), at, at + m
        at += m


def _exact_append(s):
    c = s["case"]
    rot, order = c["rot"], (0, 2, 1, 3) if c["heads_first"] else (0, 1, 2, 3)
    q, k, v = (t.double() for t in _split(s))
    caches = [s[n].double().permute(order).contiguous() for n in ("k", "v")]
    turned = torch.zeros_like(q)
    # features as complex numbers: a turn by an angle is a product
    first = torch.arange(0, rot, 2) if c["neighbours"] else torch.arange(rot // 2)
    second = first + 1 if c["neighbours"] else first + rot // 2
    for page, row, a, b in _sequences(s):
        if a == b:
            continue
        kk, qq, n = k[a:b].clone(), q[a:b].clone(), page.shape[0]
        if rot:
            table = s["rotary"][n - (b - a):n].double()
            unit = torch.complex(table[:, :rot // 2], table[:, rot // 2:])[:, None]
            for x in (kk, qq):
                z = torch.complex(x[..., first], x[..., second]) * unit
                x[..., first], x[..., second] = z.real, z.imag
        turned[a:b] = qq
        for cache, new in zip(caches, (kk, v[a:b])):
            cache[page[n - (b - a):], row[n - (b - a):]] = new
    k, v = (x.permute(order).contiguous() for x in caches)
    return {"k": k, "v": v, "q": turned} if rot else {"k": k, "v": v}


def _exact_attend(s):
    c = s["case"]
    H, Hk = c["heads"], c["kv_heads"]
    q = _split(s)[0].double()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    for page, row, a, b in _sequences(s):
        n, m = page.shape[0], b - a
        if m == 0:
            continue
        hidden = torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None]
        for h in range(H):
            kh = h // (H // Hk)
            key, value = (s[x][page, kh, row] if c["heads_first"] else s[x][page, row, kh] for x in ("k", "v"))
            score = q[a:b, h] @ key.double().t().contiguous() * s["scale"]
            if c["cap"] > 0:
                score = c["cap"] * torch.tanh(score / c["cap"])
            score = torch.where(hidden, torch.full_like(score, -math.inf), score)
            lse[a:b, h] = torch.logsumexp(score, 1)
            out[a:b, h] = torch.exp(score - lse[a:b, h][:, None]) @ value.double()
    return {"out": out, "lse": lse}


def _exact_sample(s):
    import numpy as np
    rows, found = s["logits"].shape[0], []
    host = {n: s[n].double().cpu().numpy() for n in ("logits", "temperature", "top_k", "top_p", "min_p", "uniform")}
    for r in range(rows):
        l, t, k, p, m, u = (host[n][r] for n in ("logits", "temperature", "top_k", "top_p", "min_p", "uniform"))
        if t <= 0:
            found.append(0.0)
            continue
        ids = np.argsort(-l, kind="stable")
        if 0 < k < l.size:
            ids = ids[l[ids] >= l[ids[int(k) - 1]]]
        w = np.exp((l[ids] - l.max()) / t)
        keep = w >= min(m, 1.0) if m > 0 else np.ones(w.size, bool)
        if 0 < p < 1:
            keep &= np.arange(w.size) <= np.searchsorted(np.cumsum(w), p * np.sum(w))
        ids, w = ids[keep], w[keep]
        if not 0 < p < 1:
            back = np.argsort(ids)
            ids, w = ids[back], w[back]
        total = np.cumsum(w)
        found.append(math.log(w[min(np.searchsorted(total, u * total[-1], side="right"), w.size - 1)] / total[-1]))
    return {"tokens": None, "logprobs": torch.tensor(found, dtype=torch.float64)}
