"""Drafted tokens checked by the model, on the GPU from the page lists to the cache: operators of a serving step in which each request
brings a tree (or a chain) of drafted tokens instead of one.

Four operators:

``tables``  page tables that grow by the step's tokens, with the lists that the step's kernels read (page lists, positions, the place of
            each token in the cache), and give the dropped tokens' pages back
``rotate``  rotary positions (pairs that lie next to each other or half apart, the whole head or a part of it, frequencies scaled for
            long contexts) of queries and keys, and the write into the tokens' places in the cache
``attend``  attention of the drafted tokens over the cached ones: each sees its request's context and its own branch
``commit``  masks and positions of trees, the branch that the model agrees with, and its cached keys and values moved to the front
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16


# ---- cases -------------------------------------------------------------------------------------------------------
def _tables(name, requests, lo, hi, most_new):
    return dict(name=name, op="tables", requests=requests, lo=lo, hi=hi, most_new=most_new)


def _rotate(name, tokens, far, heads, kv_heads, dim, rot, interleaved, scaling):
    return dict(name=name, op="rotate", tokens=tokens, far=far, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, interleaved=interleaved,
                scaling=scaling)


def _attend(name, requests, lo, hi, nodes, same, chain, heads, kv_heads, dim):
    return dict(name=name, op="attend", requests=requests, lo=lo, hi=hi, nodes=nodes, same=same, chain=chain, heads=heads, kv_heads=kv_heads,
                dim=dim)


def _commit(name, requests, nodes, same, layers, kv_heads, dim):
    return dict(name=name, op="commit", requests=requests, nodes=nodes, same=same, layers=layers, kv_heads=kv_heads, dim=dim)


def listed():
    return [
        # one user's chat with a small tree
        _tables("tables 1", 1, 2000, 2000, 26),
        # online traffic, contexts and drafts of very different length
        _tables("tables 256", 256, 100, 6000, 60),
        # the steady state of a large offline batch with short chains
        _tables("tables 2048", 2048, 500, 4000, 8),
        # one user's small tree, a model that rotates neighbours in half of each head
        _rotate("rotate 26 interleaved", 26, 4000, 32, 8, 128, 64, True, "none"),
        # some hundred requests' chains, deep in contexts beyond the trained ones
        _rotate("rotate 1215 yarn", 1215, 120000, 64, 8, 128, 128, False, "yarn"),
        # a full dense batch with prompts among the drafts
        _rotate("rotate 8192", 8192, 8000, 32, 8, 128, 128, False, "llama3"),
        # one user's chat with a small tree
        _attend("attend 1 x 26", 1, 2000, 2000, 26, True, False, 32, 8, 128),
        # online traffic with chains of up to five
        _attend("attend 64 x 5", 64, 200, 4000, 5, False, True, 32, 8, 128),
        # a batch of a large model with full trees
        _attend("attend 32 x 64", 32, 1000, 8000, 64, True, False, 64, 8, 128),
        # one request of a very long document, a full tree
        _attend("attend 1 x 60 far", 1, 100000, 100000, 60, True, False, 32, 8, 128),
        # one user's small tree, all layers of a small model
        _commit("commit 1 x 26", 1, 26, True, 32, 8, 128),
        # online traffic, trees of different size, all layers
        _commit("commit 48 x 60", 48, 60, False, 32, 8, 128),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["tables", "rotate", "attend", "attend", "attend", "commit"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (64, 8, 128), (32, 32, 128), (28, 4, 128), (40, 10, 128), (16, 1, 128), (24, 8, 64),
                                       (12, 12, 64), (9, 3, 64), (64, 8, 64)])
    if op == "tables":
        hi = log(1, 20000)
        requests = log(1, max(1, min(2048, 2048 * 2000 // hi)))
        c = _tables("", requests, max(1, hi // rng.choice([1, 2, 10, 100])), hi, log(1, 128))
    elif op == "rotate":
        rot = dim if rng.random() < 0.5 else rng.choice([dim // 2, dim // 4, 3 * dim // 4, 20])
        c = _rotate("", log(1, 8192), log(10, 1000000), heads, kv_heads, dim, rot, rng.random() < 0.5,
                    rng.choice(["none", "linear", "llama3", "yarn"]))
        if c["tokens"] * (heads + 2 * kv_heads) * dim > 8192 * 48 * 128:
            c["tokens"] = 8192 * 48 * 128 // ((heads + 2 * kv_heads) * dim)
    elif op == "attend":
        nodes, hi = log(1, 128), log(1, 100000)
        lo = max(1, int(hi * rng.choice([0.01, 0.1, 0.5, 1.0])))
        most = min(32 * 64 * 64 * 3600 * 128 // (nodes * heads * dim * (hi + nodes)), 8 * 100000 * 128 // (kv_heads * dim * (hi + nodes)))
        c = _attend("", log(1, max(1, min(256, most))), lo, hi, nodes, rng.random() < 0.5, rng.random() < 0.3, heads, kv_heads, dim)
    else:
        nodes = log(1, 128)
        layers = log(1, 32)
        most = 48 * 60 * 32 * 8 * 128 // (nodes * layers * kv_heads * dim)
        c = _commit("", log(1, max(1, min(256, most))), nodes, rng.random() < 0.5, layers, kv_heads, dim)
    del c["name"]
    return c


def _lengths(case):
    """Cached tokens of each request in front of the step."""
    r = random.Random("%d %d %d" % (case["requests"], case["lo"], case["hi"]))
    lo, hi = math.log(case["lo"]), math.log(case["hi"])
    return [int(round(math.exp(r.uniform(lo, hi)))) for _ in range(case["requests"])]


def _counts(case):
    """Drafted tokens of each request, the last one that is sure (the tree's root) among them."""
    r = random.Random("%d %d" % (case["requests"], case["nodes"]))
    return [case["nodes"] if case["same"] else r.randint(1, case["nodes"]) for _ in range(case["requests"])]


def _new(case):
    r = random.Random("%d %d" % (case["requests"], case["most_new"]))
    return [r.randint(1, case["most_new"]) for _ in range(case["requests"])]


# ---- inputs --------------------------------------------------------------------------------------------------------
def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(counts):
    ptr = [0]
    for c in counts:
        ptr.append(ptr[-1] + c)
    return ptr


def _parents(counts, chain, g):
    """A tree per request: node 0 is its root, a later node hangs on one of the few in front of it or (in wide trees) on any of them."""
    ptr = _starts(counts)
    start = torch.repeat_interleave(_i32(ptr[:-1]), _i32(counts).long(), output_size=ptr[-1])
    node = torch.arange(ptr[-1], device="cuda", dtype=torch.int32) - start
    if chain:
        return node - 1
    back = torch.empty(ptr[-1], device="cuda").uniform_(0, 1, generator=g)
    back = torch.where(back < 0.5, torch.ones_like(back), (back * 2 - 1) * node.clamp_min(1))      # half of them go on with the node before
    return (node - back.int().clamp_min(1)).clamp_min(-1).minimum(node - 1)


def _padded(s, parents):
    """[requests, nodes]: which places hold a node, the row of each, its parent (-1: none)."""
    start, end = s["qo_indptr"][:-1].long(), s["qo_indptr"][1:].long()
    node = torch.arange(s["most"], device="cuda")
    live = node < (end - start)[:, None]
    row = (start[:, None] + node).clamp_max(parents.numel() - 1)
    return live, row, torch.where(live, parents[row].long(), -1)


def _branches(parent, live):
    """[requests, nodes, nodes]: whether the second node is the first or one that it descends from."""
    n = parent.shape[1]
    step = (parent[:, :, None] == torch.arange(n, device=parent.device)) | torch.eye(n, dtype=torch.bool, device=parent.device)
    seen = (step & live[:, :, None]).float()
    for _ in range(max(1, (n - 1).bit_length())):
        seen = (seen @ seen).clamp_max(1)
    return seen > 0


def _words(seen, live, words):
    """Rows of bits, 64 to a word, of the live nodes."""
    n = seen.shape[-1]
    seen = torch.nn.functional.pad(seen, (0, words * 64 - n)).long().view(*seen.shape[:2], words, 64)
    return (seen << torch.arange(64, device=seen.device)).sum(-1)[live]


def _frequencies(case):
    """Inverse frequencies and the factor of cosines and sines, from the model's configuration."""
    rot, theta = case["rot"], 500000.0
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    wave = 2 * math.pi / f
    if case["scaling"] == "linear":
        return (f / 4).float(), 1.0
    if case["scaling"] == "llama3":
        smooth = ((8192 / wave - 1) / 3).clamp(0, 1)
        return ((1 - smooth) * f / 8 + smooth * f).float(), 1.0
    if case["scaling"] == "yarn":
        at = lambda turns: rot * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64, device="cuda") - low) / max(high - low, 0.001)).clamp(0, 1)
        return (f / 16 * ramp + f * (1 - ramp)).float(), 0.1 * math.log(16) + 1
    return f.float(), 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s, std=1.0: torch.empty(*s, device="cuda").normal_(0, std, generator=g).to(torch.bfloat16)
    s = {"case": case}
    if case["op"] == "tables":
        lengths, new = _lengths(case), _new(case)
        R, rows = case["requests"], case["requests"] + case["requests"] // 3 + 5          # other requests wait in between
        pages = [-(-n // PAGE) for n in lengths]
        per_row = -(-(max(lengths) + max(new)) // PAGE) + 3
        total = [-(-(a + b) // PAGE) for a, b in zip(lengths, new)]
        num_pages = sum(total) + 64
        s["rows"] = torch.randperm(rows, generator=g, device="cuda")[:R].to(torch.int32)
        s["new"] = _i32(new)
        s["lengths"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["lengths"][s["rows"].long()] = _i32(lengths)
        order = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
        used = sum(pages)
        s["table"] = torch.zeros(rows, per_row, dtype=torch.int32, device="cuda")
        held = torch.arange(per_row, device="cuda") < _i32(pages)[:, None]
        mine = torch.zeros(R, per_row, dtype=torch.int32, device="cuda")
        mine[held] = order[:used]
        s["table"][s["rows"].long()] = mine
        s["free_pages"] = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
        s["free_pages"][:num_pages - used] = order[used:]
        s["free_count"] = _i32([num_pages - used])
        zeros = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
        s["lists"] = dict(qo_indptr=zeros(R + 1), kv_indptr=zeros(R + 1), kv_indices=zeros(sum(total) + 7), kv_last_page_len=zeros(R),
                          positions=zeros(sum(new) + 5), token_req=zeros(sum(new) + 5), slots=zeros(sum(new) + 5))
        if own:
            from nanoflow_b200 import ops

            s["tables"] = ops.PageTables(s["table"], s["lengths"], s["free_pages"], s["free_count"])
            s["batch"] = ops.BatchLists(**s["lists"])
        return s
    dim, kv = case["dim"], case["kv_heads"]
    if case["op"] == "rotate":
        T, heads = case["tokens"], case["heads"]
        pages = -(-T // PAGE) + 3
        s["qkv"] = normal(T, (heads + 2 * kv) * dim, std=2.0)        # columns: queries, keys, values
        s["q"] = torch.empty(T, heads * dim, dtype=torch.bfloat16, device="cuda")
        s["pool"] = torch.zeros(pages, 2, kv, PAGE, dim, dtype=torch.bfloat16, device="cuda")
        s["slots"] = torch.randperm(pages * PAGE, generator=g, device="cuda")[:T].to(torch.int32)
        s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda").to(torch.int32)
        s["inv_freq"], s["factor"] = _frequencies(case)
        return s
    counts = _counts(case)
    s["most"], ptr = max(counts), _starts(counts)
    s["qo_indptr"] = _i32(ptr)
    words = -(-s["most"] // 64)
    s["parents"] = _parents(counts, case.get("chain", False), g)
    if case["op"] == "attend":
        heads = case["heads"]
        lengths = [a + b for a, b in zip(_lengths(case), counts)]
        pages = [-(-n // PAGE) for n in lengths]
        s["kv_indptr"], s["kv_last"] = _i32(_starts(pages)), _i32([n - (c - 1) * PAGE for n, c in zip(lengths, pages)])
        s["kv_indices"] = torch.randperm(sum(pages), generator=g, device="cuda").to(torch.int32)
        s["most_kv"] = max(lengths)
        s["pool"] = torch.empty(sum(pages), 2, kv, PAGE, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        s["q"] = normal(ptr[-1], heads * dim)
        s["out"] = torch.empty_like(s["q"])
        live, _, parent = _padded(s, s["parents"])
        s["tree"] = _words(_branches(parent, live), live, words)
        if own:
            from nanoflow_b200 import ops

            s["workspace"] = ops.tree_workspace(q_heads=heads, kv_heads=kv, head_dim=dim)
        return s
    T, R = ptr[-1], case["requests"]
    pages = -(-T // PAGE) + 2
    s["pool"] = torch.empty(case["layers"], pages, 2, kv, PAGE, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    s["pools"] = list(s["pool"])                 # a layer each
    s["slots"] = torch.randperm(pages * PAGE, generator=g, device="cuda")[:T].to(torch.int32)
    at = torch.repeat_interleave(torch.arange(R, device="cuda"), _i32(counts).long(), output_size=T)
    first = torch.randint(0, 100000, (R,), generator=g, device="cuda")
    s["positions"] = (first[at] + torch.arange(T, device="cuda") - s["qo_indptr"].long()[at]).to(torch.int32)
    s["tokens"] = torch.randint(0, 32000, (T,), generator=g, device="cuda").to(torch.int32)
    # what the model says behind each node: most of the time what one of its children holds, so that branches of some length agree
    s["targets"] = torch.randint(0, 32000, (T,), generator=g, device="cuda").to(torch.int32)
    asked = (s["parents"] >= 0) & (torch.empty(T, device="cuda").uniform_(generator=g) < 0.7)
    child = torch.where(asked, torch.arange(T, device="cuda"), T)
    first = torch.full((T,), T, device="cuda").scatter_reduce_(0, s["qo_indptr"].long()[at] + s["parents"].clamp_min(0), child, "amin")
    s["targets"] = torch.where(first < T, s["tokens"][first.clamp_max(T - 1)], s["targets"])
    s["tree"] = torch.zeros(T, words, dtype=torch.int64, device="cuda")
    s["path"] = torch.zeros(R, s["most"], dtype=torch.int32, device="cuda")
    s["counts"], s["next"], s["dropped"] = (torch.zeros(R, dtype=torch.int32, device="cuda") for _ in range(3))
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _up(n):
    return (n + (PAGE - 1)) // PAGE


def _spread(start, n, size):
    """Of each of `size` places: the request whose start .. start + n - 1 holds it (the last one where none does), and its index there."""
    place = torch.arange(size, device="cuda")
    at = (torch.searchsorted(start + n, place, right=True)).clamp_max(len(n) - 1)
    return at, place - start[at]


def _tables_plain(s):
    rows, new, li = s["rows"].long(), s["new"].long(), s["lists"]
    old = s["lengths"][rows].long()
    length = old + new
    had, pages = _up(old), _up(length)
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    qo, kv = torch.cat((zero, new.cumsum(0))), torch.cat((zero, pages.cumsum(0)))
    taken = pages - had
    before = taken.cumsum(0) - taken
    # new pages: from the top of the free ones, in the order of the requests
    at, i = _spread(kv[:-1], pages, li["kv_indices"].numel())
    live = i < pages[at]
    fresh = live & (i >= had[at])
    top = s["free_count"].long() - 1 - (before[at] + i - had[at])
    entry = s["table"][rows[at], i.clamp_max(s["table"].shape[1] - 1)]
    page = torch.where(fresh, s["free_pages"][top.clamp(0, s["free_pages"].numel() - 1)], entry)
    li["kv_indices"].copy_(torch.where(live, page, li["kv_indices"]))
    held = torch.arange(s["table"].shape[1], device="cuda")
    source = s["free_pages"][(s["free_count"].long() - 1 - (before[:, None] + held - had[:, None])).clamp(0, s["free_pages"].numel() - 1)]
    s["table"][rows] = torch.where((held >= had[:, None]) & (held < pages[:, None]), source, s["table"][rows])
    li["qo_indptr"].copy_(qo)
    li["kv_indptr"].copy_(kv)
    li["kv_last_page_len"].copy_(length - (pages - 1).clamp_min(0) * PAGE)
    at, i = _spread(qo[:-1], new, li["slots"].numel())
    live = i < new[at]
    pos = old[at] + i
    slot = s["table"][rows[at], (pos // PAGE).clamp_max(s["table"].shape[1] - 1)].long() * PAGE + pos % PAGE
    li["positions"].copy_(torch.where(live, pos, 0))
    li["token_req"].copy_(torch.where(live, at, -1))
    li["slots"].copy_(torch.where(live, slot, -1))
    grown = s["lengths"].clone()
    grown[rows] = length.int()
    s["free_count"] -= taken.sum().int()
    # the step's tokens are dropped again: their pages go back, the first one to the top
    at, i = _spread(before, taken, s["free_pages"].numel())
    live = i < taken[at]
    total = taken.sum()
    back = s["table"][rows[at], (had[at] + i).clamp(0, s["table"].shape[1] - 1)]
    place = torch.where(live, s["free_count"].long() + total - 1 - torch.arange(len(live), device="cuda"), s["free_pages"].numel())
    s["free_pages"] = torch.cat((s["free_pages"], zero.int())).scatter_(0, place, back)[:-1]
    s["free_count"] += total.int()
    return {**li, "grown": grown, "table": s["table"], "lengths": s["lengths"], "free_pages": s["free_pages"], "free_count": s["free_count"]}


def _turned(x, cos, sin, case):
    r, x1 = case["rot"], x[..., case["rot"]:]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x1), -1)
    a, b = x[..., :r // 2], x[..., r // 2:r]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x1), -1)


def _rotate_plain(s):
    case = s["case"]
    H, G, d, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    x = s["qkv"].float().view(T, H + 2 * G, d)
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = (angle.cos() * s["factor"]).float()[:, None], (angle.sin() * s["factor"]).float()[:, None]
    s["q"].copy_(_turned(x[:, :H], cos, sin, case).reshape(T, H * d))
    slot = s["slots"].long()
    s["pool"][slot // PAGE, 0, :, slot % PAGE] = _turned(x[:, H:H + G], cos, sin, case).to(torch.bfloat16)
    s["pool"][slot // PAGE, 1, :, slot % PAGE] = x[:, H + G:].to(torch.bfloat16)
    return {"q": s["q"], "pool": s["pool"]}


def _attend_plain(s):
    case = s["case"]
    H, G, d, R, n = case["heads"], case["kv_heads"], case["dim"], case["requests"], s["most"]
    ptr = s["kv_indptr"].long()
    length = (ptr[1:] - ptr[:-1] - 1) * PAGE + s["kv_last"]
    entry = (ptr[:-1, None] + torch.arange(_up(s["most_kv"]), device="cuda")).clamp_max(s["kv_indices"].numel() - 1)
    kv = s["pool"][s["kv_indices"][entry].long()].float()                         # [requests, pages, 2, kv heads, 16, dim]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, R, G, -1, d)
    live, row, _ = _padded(s, s["parents"])
    q = s["q"].float()[row].view(R, n, G, H // G, d).transpose(1, 2).reshape(R, G, -1, d) * d ** -0.5
    score = (q @ kv[0].transpose(-1, -2)).view(R, G, n, H // G, -1)
    token = torch.arange(kv.shape[3], device="cuda")
    draft = token - (length - live.sum(1))[:, None]                               # [requests, tokens]: which drafted token, if it is one
    word = s["tree"][row][torch.arange(R, device="cuda")[:, None, None], torch.arange(n, device="cuda")[:, None],
                          (draft.clamp(0, n - 1) // 64)[:, None]]                   # [requests, nodes, tokens]
    sees = (draft < 0)[:, None] | ((draft < live.sum(1)[:, None])[:, None] & ((word >> (draft.clamp(0, n - 1) % 64)[:, None] & 1) > 0))
    kv[1].masked_fill_((token >= length[:, None])[:, None, :, None], 0)
    score = score.masked_fill(~sees[:, None, :, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(R, G, -1, p.shape[-1]) @ kv[1]).view(R, G, n, H // G, d) / total
    s["out"].copy_(o.permute(0, 2, 1, 3, 4).reshape(R, n, H * d)[live])
    return s["out"]


def _commit_plain(s):
    R, n = s["case"]["requests"], s["most"]
    live, row, parent = _padded(s, s["parents"])
    seen = _branches(parent, live)
    s["tree"].copy_(_words(seen, live, s["tree"].shape[1]))
    depth = seen.sum(-1) - 1
    s["positions"].copy_((s["positions"][row[:, :1]] + depth)[live])
    # a node agrees if it is the first child of its parent that holds what the model says behind that
    node = torch.arange(n, device="cuda")
    token, said = s["tokens"][row], s["targets"][row].gather(1, parent.clamp_min(0))
    right = live & (parent >= 0) & (token == said)
    twin = (parent[:, :, None] == parent[:, None]) & right[:, None] & (node < node[:, None])
    agrees = (right & ~twin.any(-1)) | (live & (node == 0))
    kept = live & ~(seen & ~agrees[:, None]).any(-1)
    count = kept.sum(-1)
    path = torch.where(kept, node, n).sort(-1).values
    s["path"].copy_(torch.where(node < count[:, None], path, -1))
    s["counts"].copy_(count)
    s["dropped"].copy_(live.sum(-1) - count)
    last = path.gather(1, (count - 1)[:, None]).squeeze(1)
    s["next"].copy_(s["targets"][s["qo_indptr"][:-1].long() + last])
    slot = s["slots"].long()[row]
    moves = (node < count[:, None]) & live
    to = torch.where(moves, slot, slot[:, :1]).flatten()
    source = torch.where(moves, slot.gather(1, path.clamp_max(n - 1)), slot[:, :1]).flatten()
    s["pool"][:, to // PAGE, :, :, to % PAGE] = s["pool"][:, source // PAGE, :, :, source % PAGE]
    return {k: s[k] for k in ("tree", "positions", "path", "counts", "dropped", "next", "pool")}


_PLAIN = {"tables": _tables_plain, "rotate": _rotate_plain, "attend": _attend_plain, "commit": _commit_plain}


# ---- the framework's calls ---------------------------------------------------------------------------------------
def _own(s):
    from nanoflow_b200 import ops

    case = s["case"]
    if case["op"] == "tables":
        ops.tables_grow(s["tables"], s["rows"], s["new"], s["batch"])
        grown = s["lengths"].clone()
        ops.tables_trim(s["tables"], s["rows"], s["new"])
        return {**s["lists"], "grown": grown, "table": s["table"], "lengths": s["lengths"], "free_pages": s["free_pages"],
                "free_count": s["free_count"]}
    G, d = case["kv_heads"], case["dim"]
    if case["op"] == "rotate":
        H = case["heads"]
        ops.rope_append_slots(s["qkv"], s["q"], s["pool"], s["inv_freq"], s["positions"], s["slots"], q_heads=H, kv_heads=G, head_dim=d,
                              q_off=0, k_off=H * d, v_off=(H + G) * d, interleaved=case["interleaved"], factor=s["factor"])
        return {"q": s["q"], "pool": s["pool"]}
    if case["op"] == "attend":
        return ops.attn_tree(s["q"], s["out"], s["pool"], s["qo_indptr"], s["kv_indptr"], s["kv_indices"], s["kv_last"], s["tree"],
                             q_heads=case["heads"], workspace=s["workspace"])
    ops.tree_masks(s["parents"], s["qo_indptr"], s["tree"], positions=s["positions"])
    ops.tree_accept(s["tokens"], s["parents"], s["targets"], s["qo_indptr"], s["path"], s["counts"], s["next"], dropped=s["dropped"])
    ops.kv_keep(s["pools"], s["slots"], s["path"], s["counts"], s["qo_indptr"])
    return {k: s[k] for k in ("tree", "positions", "path", "counts", "dropped", "next", "pool")}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- work ------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "tables":
        lengths, new = _lengths(case), _new(case)
        pages = sum(-(-(a + b) // PAGE) for a, b in zip(lengths, new))
        fresh = sum(-(-(a + b) // PAGE) - -(-a // PAGE) for a, b in zip(lengths, new))
        # read: rows, new tokens, lengths, pages; written: the lists, fresh pages into the table and back, lengths twice
        return {"bytes": case["requests"] * 4 * 8 + pages * 8 + sum(new) * 12 + fresh * 12, "flops": pages}
    d, G = case["dim"], case["kv_heads"]
    if case["op"] == "rotate":
        T, H = case["tokens"], case["heads"]
        return {"bytes": T * ((H + 2 * G) * d * 4 + 8), "flops": 3 * T * (H + G) * case["rot"]}
    counts = _counts(case)
    T = sum(counts)
    if case["op"] == "attend":
        H = case["heads"]
        lengths = [a + b for a, b in zip(_lengths(case), counts)]
        return {"bytes": sum(lengths) * 4 * G * d + 4 * T * H * d, "flops": 4 * sum(a * b for a, b in zip(lengths, counts)) * H * d}
    # each node's parent, token, target, mask and position, and a few of its vectors moved (a third of the tree's depth, say)
    words = -(-max(counts) // 64)
    moved = sum(min(c, 4) for c in counts) * case["layers"] * 2 * G * d * 2
    return {"bytes": T * (20 + 8 * words) + 2 * moved, "flops": T}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("tables", "commit"):       # whole numbers, and copies of what was there
        return None
    s = prepare(case, seed)
    f, H, G, d = torch.float64, case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotate":
        r = case["rot"]
        first = torch.arange(0, r, 2, device="cuda") if case["interleaved"] else torch.arange(r // 2, device="cuda")
        second = first + 1 if case["interleaved"] else first + r // 2
        turn = torch.polar(torch.full((1, 1), s["factor"], dtype=f, device="cuda"), torch.outer(s["positions"].to(f), s["inv_freq"].to(f)))
        q, pool = s["qkv"][:, :H * d].to(f), s["pool"].to(f)

        def turned(x):
            x = x.clone()
            z = torch.complex(x[:, first], x[:, second]) * turn
            x[:, first], x[:, second] = z.real, z.imag
            return x

        q = torch.cat([turned(q[:, h * d:(h + 1) * d]) for h in range(H)], 1)
        page, slot = torch.div(s["slots"].long(), PAGE, rounding_mode="floor"), s["slots"].long() % PAGE
        for h in range(G):
            pool[page, 0, h, slot] = turned(s["qkv"][:, (H + h) * d:(H + h + 1) * d].to(f))
            pool[page, 1, h, slot] = s["qkv"][:, (H + G + h) * d:(H + G + h + 1) * d].to(f)
        return {"q": q, "pool": pool}
    counts = _counts(case)
    lengths = [a + b for a, b in zip(_lengths(case), counts)]
    if sum(a * b for a, b in zip(lengths, counts)) * H * d > 4e11:
        return None
    group, parents = H // G, s["parents"].tolist()
    q, out = s["q"].to(f).view(-1, H, d), torch.empty(sum(counts), H, d, dtype=f, device="cuda")
    rows, pages = s["qo_indptr"].tolist(), s["kv_indptr"].tolist()
    for r, (n, length) in enumerate(zip(counts, lengths)):
        branch = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            j = i
            while j >= 0:
                branch[i, j] = True
                j = parents[rows[r] + j]
        hidden = torch.zeros(n, length, dtype=torch.bool, device="cuda")
        hidden[:, length - n:] = ~branch.to("cuda")
        own_pages = s["kv_indices"][pages[r]:pages[r + 1]].long()
        for h in range(G):
            k, v = (s["pool"][own_pages, side, h].reshape(-1, d)[:length].to(f) for side in (0, 1))
            for a in range(rows[r], rows[r] + n, 64):
                b = min(a + 64, rows[r] + n)
                score = (q[a:b, h * group:(h + 1) * group] @ k.T / math.sqrt(d)).masked_fill(hidden[a - rows[r]:b - rows[r], None], -math.inf)
                out[a:b, h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out.view(-1, H * d)
