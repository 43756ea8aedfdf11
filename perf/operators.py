"""A paged KV cache in 8 bits and the attention that reads it, on the calls of a serving iteration.

The cache holds, for each token, KV head and of key and value, ``head_dim`` numbers of 8 bits (e4m3 or whole numbers) and one fp32
scale; a cached value is number times scale. Four operators:

``append``  norms of queries and keys per head (where the model has them), rotation, and the write into the cache; what was written is
            read back, as a chunk of a prompt is in front of its attention
``read``    pages of the cache as bf16 pages
``decode``  attention of one query token per request over its cached tokens
``shared``  the same where all requests of the batch see one prefix, whose pages are listed once
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
LARGEST = {"e4m3": 448.0, "int8": 127.0}     # largest number of the type: what a vector's largest entry becomes
DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ---- cases -------------------------------------------------------------------------------------------------------
def _append(name, tokens, requests, past, heads, kv_heads, dim, kind, norm):
    return dict(name=name, op="append", tokens=tokens, requests=requests, past=past, heads=heads, kv_heads=kv_heads, dim=dim, kind=kind,
                norm=norm)


def _read(name, pages, kv_heads, dim, kind):
    return dict(name=name, op="read", pages=pages, kv_heads=kv_heads, dim=dim, kind=kind)


def _decode(name, requests, lo, hi, heads, kv_heads, dim, kind):
    return dict(name=name, op="decode", requests=requests, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, dim=dim, kind=kind)


def _shared(name, requests, prefix, lo, hi, heads, kv_heads, dim, kind):
    return dict(name=name, op="shared", requests=requests, prefix=prefix, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, dim=dim,
                kind=kind)


def listed():
    return [
        # one user's chat, deep in a long conversation: a single token of a model with normed heads
        _append("append 1", 1, 1, 100000, 32, 8, 128, "e4m3", True),
        # the steady state's decoded tokens of a large model
        _append("append 683 int8", 683, 683, 1300, 64, 8, 128, "int8", False),
        # a full dense batch of prompts
        _append("append 2048", 2048, 3, 0, 32, 8, 128, "e4m3", True),
        # a few hundred cached tokens in front of the next chunk of a short prompt
        _read("read 37 int8", 37, 4, 64, "int8"),
        # a long document's cached tokens in front of its next chunk
        _read("read 4096", 4096, 8, 128, "e4m3"),
        # one user's chat: a single query
        _decode("decode 1", 1, 900, 900, 32, 8, 128, "e4m3"),
        # light online traffic, contexts of very different length
        _decode("decode 24", 24, 100, 6000, 32, 8, 128, "e4m3"),
        # offline generation, wider groups
        _decode("decode 256 int8", 256, 200, 2000, 64, 8, 128, "int8"),
        # the steady state of 1024-token prompts and 512-token answers
        _decode("decode 683", 683, 1024, 1536, 32, 8, 128, "e4m3"),
        # a handful of chats behind one system prompt of odd length
        _shared("shared 16 x 1999", 16, 1999, 1, 200, 32, 8, 128, "e4m3"),
        # a batch job that asks many questions of one document
        _shared("shared 256 x 8192", 256, 8192, 20, 400, 32, 8, 128, "e4m3"),
        # agents of a large model behind a long common context
        _shared("shared 64 x 32768 int8", 64, 32768, 50, 1000, 64, 8, 128, "int8"),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["append", "read", "decode", "decode", "shared", "shared"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (64, 8, 128), (32, 32, 128), (28, 4, 128), (40, 10, 128), (16, 1, 128), (24, 8, 64),
                                       (12, 12, 64), (9, 3, 64)])
    kind = rng.choice(["e4m3", "int8"])
    if op == "append":
        requests = log(1, 700)
        tokens = requests if rng.random() < 0.4 else max(requests, log(1, 2048))
        c = _append("", tokens, requests, rng.choice([0, log(1, 100000)]) if requests < 64 else log(1, 3000), heads, kv_heads, dim, kind,
                    rng.random() < 0.5)
    elif op == "read":
        c = _read("", log(1, 4096), min(kv_heads, 8), dim, kind)
    elif op == "decode":
        hi = log(2, 8000)
        lo = max(1, int(hi * rng.choice([0.01, 0.1, 0.5, 1.0])))
        most = 683 * 1280 * 8 * 128 // (hi * kv_heads * dim)
        c = _decode("", log(1, max(1, min(683, most))), lo, hi, heads, kv_heads, dim, kind)
    else:
        prefix = log(20, 32768)
        requests = log(2, max(2, min(400, 64 * 64 * 32768 // (prefix * heads))))
        hi = log(1, 600)
        c = _shared("", requests, prefix, max(1, hi // rng.choice([1, 3, 20])), hi, heads, kv_heads, dim, kind)
    del c["name"]
    return c


def _lengths(case):
    """Cached tokens of each request, the newest included."""
    r = random.Random("%d %d %d" % (case["requests"], case["lo"], case["hi"]))
    lo, hi = math.log(case["lo"]), math.log(case["hi"])
    return [int(round(math.exp(r.uniform(lo, hi)))) for _ in range(case["requests"])]


def _spans(case):
    """(cached tokens before, new tokens) of each request."""
    r = random.Random("%d %d %d" % (case["tokens"], case["requests"], case["past"]))
    n, k = case["tokens"], case["requests"]
    cuts = sorted(r.sample(range(1, n), k - 1)) if k > 1 else []
    counts = [b - a for a, b in zip([0] + cuts, cuts + [n])]
    return [(r.randint(case["past"] // 2, case["past"]), c) for c in counts]


# ---- inputs --------------------------------------------------------------------------------------------------------
def _pages(lengths, g, first=0):
    """Page lists of requests over a pool in random order: indptr, indices, tokens in the last page."""
    counts = [-(-n // PAGE) for n in lengths]
    ptr = [0]
    for c in counts:
        ptr.append(ptr[-1] + c)
    order = first + torch.randperm(ptr[-1], generator=g, device="cuda")
    last = [n - (c - 1) * PAGE if c else 0 for n, c in zip(lengths, counts)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return dict(kv_indptr=i32(ptr), kv_indices=order.to(torch.int32), kv_last=i32(last), num_pages=ptr[-1])


def _filled(pages, case, g):
    """A pool as the write leaves it: vectors of normal numbers whose size differs from token to token, quantised."""
    kind, dim = case["kind"], case["dim"]
    shape = (pages, 2, case["kv_heads"], PAGE)
    pool = torch.empty(*shape, dim, dtype=DTYPES[kind], device="cuda")
    scale = torch.empty(shape, dtype=torch.float32, device="cuda")
    for a in range(0, pages, 4096):
        n = min(4096, pages - a)
        x = torch.randn((n, *shape[1:], dim), generator=g, device="cuda")
        x *= torch.empty((n, *shape[1:], 1), device="cuda").uniform_(0.5, 1.5, generator=g)
        scale[a:a + n] = x.abs().amax(-1) / LARGEST[kind]
        x /= scale[a:a + n, ..., None]
        pool[a:a + n] = (x.round() if kind == "int8" else x.clamp(-448, 448)).to(DTYPES[kind])
    return pool, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s, std=1.0, mean=0.0: torch.empty(*s, device="cuda").normal_(mean, std, generator=g).to(torch.bfloat16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    s = {"case": case}
    dim, kv = case["dim"], case["kv_heads"]
    if case["op"] == "read":
        # a request's pages, spread over a pool with others' pages between them
        n = case["pages"]
        s["pool"], s["scale"] = _filled(n + n // 4 + 1, case, g)
        s["pages"] = torch.randperm(n + n // 4 + 1, generator=g, device="cuda")[:n].to(torch.int32)
        s["out"] = torch.empty(n, 2, kv, PAGE, dim, dtype=torch.bfloat16, device="cuda")
        return s
    heads = case["heads"]
    if case["op"] == "append":
        spans, T = _spans(case), case["tokens"]
        # pages from the first one with a new token on; the earlier part of a long context keeps its place in the list only
        s.update(_pages([p + n for p, n in spans], g))
        at, used = s["kv_indptr"].tolist(), []
        for (p, n), a in zip(spans, at):
            used += range(a + p // PAGE, a + (p + n - 1) // PAGE + 1)
        used = torch.tensor(used, device="cuda")
        s["kv_indices"] = torch.full_like(s["kv_indices"], 0)
        s["kv_indices"][used] = torch.randperm(len(used), generator=g, device="cuda").to(torch.int32)
        s["pages"] = s["kv_indices"][used].contiguous()
        s["pool"], s["scale"] = _filled(len(used), case, g)
        s["out"] = torch.empty(len(used), 2, kv, PAGE, dim, dtype=torch.bfloat16, device="cuda")
        s["qkv"] = normal(T, (heads + 2 * kv) * dim, std=2.0)        # columns: keys, values, queries
        s["q"] = torch.empty(T, heads * dim, dtype=torch.bfloat16, device="cuda")
        s["positions"] = i32([p + i for p, n in spans for i in range(n)])
        s["token_req"] = i32([r for r, (_, n) in enumerate(spans) for _ in range(n)])
        s["inv_freq"] = (500000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)).float()
        s["q_norm"], s["k_norm"] = (normal(dim, std=0.1, mean=1.0) if case["norm"] else None for _ in range(2))
        return s
    lengths = _lengths(case)
    prefix = -(-case["prefix"] // PAGE) if case["op"] == "shared" else 0
    s.update(_pages(lengths, g, prefix))
    s["most"] = max(lengths)
    if prefix:
        s["prefix_pages"] = torch.randperm(prefix, generator=g, device="cuda").to(torch.int32)
    s["pool"], s["scale"] = _filled(prefix + s["num_pages"], case, g)
    s["q"] = normal(case["requests"], heads * dim)
    s["out"] = torch.empty_like(s["q"])
    s["qo_indptr"] = torch.arange(case["requests"] + 1, dtype=torch.int32, device="cuda")
    if own:
        from nanoflow_b200 import ops

        s["workspace"] = ops.decode_workspace_q8(requests=case["requests"], q_heads=heads, kv_heads=kv, head_dim=dim,
                                                 prefix_len=case.get("prefix", 0))
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _normed(x, w):
    if w is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _append_plain(s):
    case = s["case"]
    H, G, d, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    x = s["qkv"].float().view(T, 2 * G + H, d)
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    k = _rotated(_normed(x[:, :G], s["k_norm"]), cos, sin)
    q = _rotated(_normed(x[:, 2 * G:], s["q_norm"]), cos, sin)
    s["q"].copy_(q.reshape(T, H * d))
    pos = s["positions"].long()
    page = s["kv_indices"][s["kv_indptr"].long()[s["token_req"].long()] + pos // PAGE].long()
    new = torch.stack((k, x[:, G:2 * G]), 1)                                       # [T, 2, kv heads, dim]
    scale = new.abs().amax(-1) / LARGEST[case["kind"]]
    number = new / scale.clamp_min(1e-30)[..., None]
    number = number.round() if case["kind"] == "int8" else number.clamp(-448, 448)
    s["pool"][page, :, :, pos % PAGE] = number.to(s["pool"].dtype)
    s["scale"][page, :, :, pos % PAGE] = scale
    s["out"].copy_(s["pool"][s["pages"].long()].float() * s["scale"][s["pages"].long()][..., None])
    return {"q": s["q"], "cache": s["out"], "scale": s["scale"]}


def _prefix_values(s):
    """Keys and values of the shared tokens, [kv heads, tokens, dim]."""
    at = s["prefix_pages"].long()
    x = (s["pool"][at].float() * s["scale"][at][..., None]).permute(1, 2, 0, 3, 4)
    return x.reshape(2, x.shape[1], -1, x.shape[-1])[:, :, :s["case"]["prefix"]]


def _attend_plain(s):
    case = s["case"]
    H, G, d, R = case["heads"], case["kv_heads"], case["dim"], case["requests"]
    ptr = s["kv_indptr"].long()
    count = ptr[1:] - ptr[:-1]
    length = (count - 1).clamp_min(0) * PAGE + s["kv_last"]
    slot = torch.arange(-(-s["most"] // PAGE), device="cuda")
    entry = (ptr[:-1, None] + slot).clamp_max(s["kv_indices"].numel() - 1)
    page = s["kv_indices"][entry].long()                                          # [requests, pages]
    kv = s["pool"][page].float() * s["scale"][page][..., None]                    # [requests, pages, 2, kv heads, 16, dim]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, R, G, -1, d)
    q = s["q"].float().view(R, G, H // G, d) * d ** -0.5
    score = q @ kv[0].transpose(-1, -2)                                           # [requests, kv heads, group, tokens]
    score = score.masked_fill((torch.arange(kv.shape[3], device="cuda") >= length[:, None])[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    if case["op"] == "shared":
        pk, pv = _prefix_values(s)
        front = q.transpose(0, 1).reshape(G, -1, d) @ pk.transpose(-1, -2)        # [kv heads, requests x group, tokens]
        front = front.view(G, R, H // G, -1).transpose(0, 1)
        most = torch.maximum(most, front.amax(-1, keepdim=True))
        front = (front - most).exp()
    p = (score - most).exp()
    total, o = p.sum(-1, keepdim=True), p @ kv[1]
    if case["op"] == "shared":
        total = total + front.sum(-1, keepdim=True)
        o = o + (front.transpose(0, 1).reshape(G, -1, front.shape[-1]) @ pv).view(G, R, H // G, d).transpose(0, 1)
    s["out"].copy_((o / total).reshape(R, H * d))
    return s["out"]


def _plain(s):
    if s["case"]["op"] == "append":
        return _append_plain(s)
    if s["case"]["op"] == "read":
        at = s["pages"].long()
        s["out"].copy_(s["pool"][at].float() * s["scale"][at][..., None])
        return s["out"]
    return _attend_plain(s)


# ---- the framework's calls ---------------------------------------------------------------------------------------
def _own(s):
    from nanoflow_b200 import ops

    case = s["case"]
    if case["op"] == "read":
        return ops.kv_read_q8(s["pool"], s["scale"], s["pages"], out=s["out"])
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        ops.rope_append_q8(s["qkv"], s["q"], s["pool"], s["scale"], s["inv_freq"], s["positions"], s["token_req"], s["kv_indptr"],
                           s["kv_indices"], q_heads=H, kv_heads=G, head_dim=d, q_off=2 * G * d, k_off=0, v_off=G * d,
                           q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
        ops.kv_read_q8(s["pool"], s["scale"], s["pages"], out=s["out"])
        return {"q": s["q"], "cache": s["out"], "scale": s["scale"]}
    lists = (s["qo_indptr"], s["kv_indptr"], s["kv_indices"], s["kv_last"])
    if case["op"] == "decode":
        return ops.attn_decode_q8(s["q"], s["out"], s["pool"], s["scale"], *lists, q_heads=H, req_begin=0, req_count=case["requests"],
                                  workspace=s["workspace"])
    return ops.attn_decode_shared_q8(s["q"], s["out"], s["pool"], s["scale"], *lists, s["prefix_pages"], case["prefix"], q_heads=H,
                                     req_begin=0, req_count=case["requests"], workspace=s["workspace"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- work ------------------------------------------------------------------------------------------------------------
def work(case):
    d, G = case["dim"], case["kv_heads"]
    token = 2 * G * (d + 4)                     # one cached token
    if case["op"] == "read":
        return {"bytes": case["pages"] * (PAGE * (token + 4 * G * d) + 4), "flops": 2 * case["pages"] * PAGE * G * d}
    H = case["heads"]
    if case["op"] == "append":
        T = case["tokens"]
        pages = sum((p + n - 1) // PAGE - p // PAGE + 1 for p, n in _spans(case))
        other = pages * PAGE - T                # tokens that the written pages held already are read back too
        return {"bytes": T * ((H + 2 * G) * d * 2 + H * d * 2 + token) + other * token + pages * PAGE * 4 * G * d, "flops": 12 * T * (H + 2 * G) * d}
    lengths = _lengths(case)
    seen = sum(lengths) + case.get("prefix", 0)
    pairs = sum(lengths) + case["requests"] * case.get("prefix", 0)
    return {"bytes": seen * token + 4 * case["requests"] * H * d, "flops": 4 * pairs * H * d}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def _nearest(x, kind):
    """The number of the type nearest to x (of two, the even one)."""
    if kind == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)   # three bits behind the leading one; 2^-9 at the least
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    d, G = case["dim"], case["kv_heads"]
    f = torch.float64
    if case["op"] == "read":
        out = torch.empty(s["out"].shape, dtype=f, device="cuda")
        for side in (0, 1):
            out[:, side] = torch.einsum("pgtd,pgt->pgtd", s["pool"].to(f)[s["pages"].long(), side], s["scale"].to(f)[s["pages"].long(), side])
        return out
    H = case["heads"]
    if case["op"] == "append":
        T, half = case["tokens"], d // 2
        pos = s["positions"].to(f)
        i = torch.arange(half, device="cuda")
        turn = torch.polar(torch.ones((T, half), dtype=f, device="cuda"), torch.outer(pos, s["inv_freq"].to(f)))
        rows = s["qkv"].to(f)

        def head(first, w):
            x = rows[:, first:first + d]
            if w is not None:
                x = w.to(f) * x / torch.sqrt((x * x).sum(1, keepdim=True) / d + 1e-6)
            z = torch.complex(x[:, i], x[:, i + half]) * turn
            return torch.cat((z.real, z.imag), 1)

        q = torch.cat([head((2 * G + h) * d, s["q_norm"]) for h in range(H)], 1)
        pool, scale = s["pool"].to(f), s["scale"].to(f)
        at = s["positions"].tolist()
        first, req, listed_pages = s["kv_indptr"].tolist(), s["token_req"].tolist(), s["kv_indices"].tolist()
        page = torch.tensor([listed_pages[first[r] + p // PAGE] for r, p in zip(req, at)], device="cuda")
        slot = torch.tensor([p % PAGE for p in at], device="cuda")
        for h in range(G):
            for side, x in ((0, head(h * d, s["k_norm"])), (1, rows[:, (G + h) * d:(G + h + 1) * d])):
                unit = x.abs().max(1).values / LARGEST[case["kind"]]
                scale[page, side, h, slot] = unit
                pool[page, side, h, slot] = _nearest(x / unit[:, None], case["kind"])
        order = s["pages"].long()
        return {"q": q, "cache": pool[order] * scale[order].unsqueeze(-1), "scale": scale}
    group = H // G
    out = torch.empty(case["requests"], H, d, dtype=f, device="cuda")
    q = s["q"].to(f).view(-1, H, d)
    front = [torch.cat([_tokens(s, int(p), G, d) for p in s["prefix_pages"].tolist()], 2)[:, :, :case["prefix"]]] if case["op"] == "shared" else []
    first, listed_pages = s["kv_indptr"].tolist(), s["kv_indices"]
    for r, n in enumerate(_lengths(case)):
        at = listed_pages[first[r]:first[r + 1]].long()
        kv = s["pool"][at].to(f) * s["scale"][at].to(f).unsqueeze(-1)
        kv = torch.cat(list(kv), 2)[:, :, :n] if len(at) else kv.new_empty(2, G, 0, d)
        kv = torch.cat(front + [kv], 2)
        for h in range(G):
            p = torch.softmax(q[r, h * group:(h + 1) * group] @ kv[0, h].T / math.sqrt(d), 1)
            out[r, h * group:(h + 1) * group] = p @ kv[1, h]
    return out.view(case["requests"], H * d)


def _tokens(s, page, G, d):
    return s["pool"][page].to(torch.float64) * s["scale"][page].to(torch.float64).unsqueeze(-1)
