"""A step in which each request brings drafted tokens (a tree of them, or a chain) that the model checks at once: page tables and lists
built on the GPU, rotation and cache write by slot, attention of the drafted tokens, and the accepted branch in the cache.

One step, for the requests in rows ``rows`` of the tables, ``new_tokens`` tokens each (the last sure one and what is drafted behind it)::

    tables_grow(tables, rows, new_tokens, lists)                            # pages, lists, slots
    tree_masks(parents, lists.qo_indptr, mask, positions=lists.positions)   # who descends from whom (chains: not needed)
    for each layer:
        rope_append_slots(qkv, q, pool, inv_freq, lists.positions, lists.slots, ...)
        attn_tree(q, out, pool, lists.qo_indptr, ..., mask, ...)
    tree_accept(tokens, parents, targets, lists.qo_indptr, path, counts, next_tokens, dropped=dropped)
    kv_keep(pools, lists.slots, path, counts, lists.qo_indptr)              # all layers
    tables_trim(tables, rows, dropped)

Caches are the bf16 pools ``[num_pages, 2, kv_heads, 16, head_dim]`` of :func:`nanoflow_b200.ops.rope_append` and
:func:`nanoflow_b200.ops.attn_decode`. A token's slot is ``page * 16 + place in the page``. Nothing here waits for the GPU, and all calls can
be captured into a CUDA graph; lists longer than a step needs hold tokens of no request and requests of nothing, which the other calls
leave alone (of a request of nothing, :func:`tree_accept` says so).

No tensor that a call writes may overlap another one of its tensors. Lists that are none are reported in ``status`` and touch nothing
outside the call's tensors. Requests of a call, and entries of a list, number up to 2^31 - 2^20. ``early_start`` (EARLY_*): kernels may be
launched while the one before them on the stream still runs, and wait for it there; 0 keeps the SMs free until then, for another stream's
kernels beside it.
"""
from __future__ import annotations

import ctypes
import math
from ctypes import c_float, c_int, c_longlong, c_void_p, Structure, byref
from dataclasses import dataclass, field
from typing import Optional, Sequence, Tuple

import torch

from . import EARLY_FIRST, EARLY_FURTHER, lib

PAGE = 16
TREE_NODES = 512              # tokens of a request that masks and paths reach


class TablesParams(Structure):
    _fields_ = [(n, c_void_p) for n in ("table", "lengths", "free_pages", "free_count", "ticket", "rows", "tokens", "qo_indptr", "kv_indptr",
                                        "kv_indices", "kv_last_page_len", "positions", "token_req", "slots")] + \
               [(n, c_int) for n in ("requests", "max_requests", "max_pages", "num_pages", "num_indices", "num_tokens", "early_start")] + \
               [("status", c_void_p)] + [(n, c_int) for n in ("num_qo", "num_kv", "num_last")]


class RopeSlotsParams(Structure):
    _fields_ = [("qkv", c_void_p), ("ld_qkv", c_longlong), ("q_off", c_int), ("k_off", c_int), ("v_off", c_int), ("q_out", c_void_p),
                ("kv_pool", c_void_p), ("inv_freq", c_void_p), ("positions", c_void_p), ("slots", c_void_p), ("factor", c_float),
                ("T", c_int), ("q_heads", c_int), ("kv_heads", c_int), ("head_dim", c_int), ("pairs", c_int), ("interleaved", c_int),
                ("num_pages", c_int), ("early_start", c_int), ("status", c_void_p)]


class AttnTreeParams(Structure):
    _fields_ = [("q", c_void_p), ("ld_q", c_longlong), ("out", c_void_p), ("ld_out", c_longlong), ("kv_pool", c_void_p), ("qo_indptr", c_void_p),
                ("kv_indptr", c_void_p), ("kv_indices", c_void_p), ("kv_last_page_len", c_void_p), ("tree", c_void_p), ("q_heads", c_int),
                ("kv_heads", c_int), ("head_dim", c_int), ("num_pages", c_int), ("num_tokens", c_int), ("num_indices", c_int),
                ("req_begin", c_int), ("req_count", c_int), ("words", c_int), ("sm_scale", c_float), ("num_ctas", c_int), ("early_start", c_int),
                ("workspace", c_void_p), ("workspace_bytes", c_longlong), ("status", c_void_p), ("request_tokens", c_int), ("listed", c_int)]


class TreeMasksParams(Structure):
    _fields_ = [("parents", c_void_p), ("qo_indptr", c_void_p), ("mask", c_void_p), ("positions", c_void_p), ("requests", c_int),
                ("num_tokens", c_int), ("words", c_int), ("early_start", c_int), ("status", c_void_p)]


class TreeAcceptParams(Structure):
    _fields_ = [(n, c_void_p) for n in ("tokens", "parents", "targets", "qo_indptr", "path", "counts", "next_tokens", "dropped")] + \
               [("requests", c_int), ("num_tokens", c_int), ("max_path", c_int), ("early_start", c_int), ("status", c_void_p)]


class KvKeepParams(Structure):
    _fields_ = [("pools", c_void_p * 64), ("num_pools", c_int), ("slots", c_void_p), ("path", c_void_p), ("counts", c_void_p),
                ("qo_indptr", c_void_p), ("requests", c_int), ("num_tokens", c_int), ("max_path", c_int), ("num_pages", c_int),
                ("kv_heads", c_int), ("head_dim", c_int), ("early_start", c_int), ("status", c_void_p)]


@dataclass
class PageTables:
    """Pages of requests. ``table[row, i]``: page of the row's tokens 16 i to 16 i + 15; ``lengths[row]``: its tokens; the first
    ``free_count`` entries of ``free_pages``: pages that nobody has, taken from the end. All int32 on the GPU. Up to 65536 rows."""

    table: torch.Tensor
    lengths: torch.Tensor
    free_pages: torch.Tensor
    free_count: torch.Tensor
    ticket: torch.Tensor = field(default=None, repr=False)     # the calls' own, zero between them

    def __post_init__(self):
        if self.ticket is None:
            self.ticket = torch.zeros(1, dtype=torch.int32, device=self.table.device)


@dataclass
class BatchLists:
    """What :func:`tables_grow` writes, int32: lists of the batch's requests as ``attn_decode`` and :func:`attn_tree` read them, and
    of each new token its position, its request (-1: none) and its slot (-1: none)."""

    qo_indptr: torch.Tensor           # [requests at most + 1]
    kv_indptr: torch.Tensor           # [requests at most + 1]
    kv_indices: torch.Tensor          # [pages at most]
    kv_last_page_len: torch.Tensor    # [requests at most]
    positions: torch.Tensor           # [tokens at most]
    token_req: torch.Tensor
    slots: torch.Tensor


def page_tables(rows: int, max_pages: int, num_pages: int, device="cuda") -> PageTables:
    """Tables of ``rows`` requests of up to ``max_pages`` pages each, all of the cache's ``num_pages`` pages free, lowest first."""
    i32 = dict(dtype=torch.int32, device=device)
    return PageTables(torch.zeros(rows, max_pages, **i32), torch.zeros(rows, **i32), torch.arange(num_pages - 1, -1, -1, **i32),
                      torch.full((1,), num_pages, **i32))


def batch_lists(requests: int, tokens: int, pages: int, device="cuda") -> BatchLists:
    """Lists of up to ``requests`` requests with up to ``tokens`` new tokens and ``pages`` pages in all."""
    i32 = dict(dtype=torch.int32, device=device)
    return BatchLists(torch.zeros(requests + 1, **i32), torch.zeros(requests + 1, **i32), torch.zeros(pages, **i32), torch.zeros(requests, **i32),
                      torch.zeros(tokens, **i32), torch.full((tokens,), -1, **i32), torch.full((tokens,), -1, **i32))


_calls_module = None


def _calls():
    """The extension module that checks and launches, connected to the kernel library (once). Raises if either is not built."""
    global _calls_module
    if _calls_module is None:
        try:
            from . import _draft
        except ImportError as e:
            raise RuntimeError("nanoflow_b200/ops/_draft is missing: run `python -m nanoflow_b200.ops.build`") from e
        _draft.connect(*(ctypes.cast(getattr(lib(), f), c_void_p).value
                         for f in ("nfk_tables_grow", "nfk_tables_trim", "nfk_rope_slots", "nfk_attn_tree", "nfk_tree_masks", "nfk_tree_accept",
                                   "nfk_kv_keep")))
        _calls_module = _draft
    return _calls_module


def tables_grow(tables: PageTables, rows: torch.Tensor, new_tokens: torch.Tensor, lists: BatchLists, *, status: Optional[torch.Tensor] = None,
                early_start: int = EARLY_FIRST) -> BatchLists:
    """Request i of the batch, in row ``rows[i]``, grows by ``new_tokens[i]`` tokens: pages are taken for them, requests in their order,
    and the lists are written: to their ends, tokens of no request and requests of nothing behind the last ones, but for ``lists.kv_indices``,
    which behind the last page is left as it was.

    Nothing changes, all lists are empty, and ``status`` says so, if a row does not exist or comes twice, a number is negative, or something
    does not fit: a row's pages, the free pages, the lists. Up to 4096 requests."""
    _calls().grow(tables.table, tables.lengths, tables.free_pages, tables.free_count, tables.ticket, rows, new_tokens, lists.qo_indptr,
                  lists.kv_indptr, lists.kv_indices, lists.kv_last_page_len, lists.positions, lists.token_req, lists.slots, status, early_start)
    return lists


def tables_trim(tables: PageTables, rows: torch.Tensor, dropped: torch.Tensor, *, status: Optional[torch.Tensor] = None,
                early_start: int = EARLY_FIRST) -> None:
    """The last ``dropped[i]`` tokens of row ``rows[i]`` go (all of them, if it has fewer), and pages that hold none any more are free
    again: the first one will be taken first. ``dropped`` has an entry per row (a slice, where :func:`tree_accept` wrote one for each place
    of longer lists). Refusals as in :func:`tables_grow`."""
    _calls().trim(tables.table, tables.lengths, tables.free_pages, tables.free_count, tables.ticket, rows, dropped, status, early_start)


def rope_frequencies(rot_dim: int, theta: float, scaling: Optional[dict] = None, *, length: Optional[int] = None,
                     max_position: Optional[int] = None, device="cuda") -> Tuple[torch.Tensor, float]:
    """Inverse frequencies (fp32 ``[rot_dim / 2]``) and the factor of cosines and sines for :func:`rope_append_slots`, from a model's
    configuration (``rope_scaling`` of its config.json). Types: none, ``linear``, ``dynamic`` (by ``length``, above ``max_position``), ``llama3``,
    ``yarn``, ``longrope`` (short or long factors by ``length``). An entry that is None is as if it were not there."""
    if rot_dim < 2 or rot_dim % 2:
        raise RuntimeError("rope_frequencies: rot_dim must be even")
    if not theta > 1:
        raise RuntimeError("rope_frequencies: theta must be above 1")
    scaling = {name: value for name, value in (scaling or {}).items() if value is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim
    inv, out = theta ** -i, 1.0
    original = scaling.get("original_max_position_embeddings") or max_position
    if kind not in ("default", "linear", "dynamic", "llama3", "yarn", "longrope"):
        raise RuntimeError(f"rope_frequencies: unknown scaling {kind}")
    if kind in ("dynamic", "yarn", "longrope") and not original:
        raise RuntimeError(f"rope_frequencies: {kind} needs max_position or original_max_position_embeddings")
    needed = {"linear": ("factor",), "dynamic": ("factor",), "llama3": ("factor",), "longrope": ("short_factor", "long_factor"),
              "yarn": () if max_position else ("factor",)}
    for name in needed.get(kind, ()):
        if name not in scaling:
            raise RuntimeError(f"rope_frequencies: {kind} needs {name}")
    sizes = dict(scaling, max_position=max_position)
    for name in ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings", "max_position", "beta_fast", "beta_slow"):
        absent = (None,) if name in ("factor", "low_freq_factor", "high_freq_factor") else (None, 0)
        if sizes.get(name) not in absent and not 0 < float(sizes[name]) < math.inf:
            raise RuntimeError(f"rope_frequencies: {name} must be positive")
    if kind == "llama3" and not float(scaling.get("low_freq_factor", 1)) < float(scaling.get("high_freq_factor", 4)):
        raise RuntimeError("rope_frequencies: low_freq_factor must be below high_freq_factor")
    if kind == "dynamic" and rot_dim == 2:
        raise RuntimeError("rope_frequencies: dynamic has no form for a single pair")
    if kind == "longrope" and not len(scaling["short_factor"]) == len(scaling["long_factor"]) == rot_dim // 2:
        raise RuntimeError("rope_frequencies: longrope needs a factor for each pair")
    if kind == "longrope" and not (all(0 < float(f) < math.inf for f in (*scaling["short_factor"], *scaling["long_factor"])) and original > 1):
        raise RuntimeError("rope_frequencies: longrope's factors must be positive, and its original length above 1")
    if kind == "linear":
        inv = inv / float(scaling["factor"])
    elif kind == "dynamic":
        factor, most = float(scaling["factor"]), float(max_position or original)
        grown = factor * max(length or 0, most) / most - (factor - 1)
        inv = (theta * grown ** (rot_dim / (rot_dim - 2))) ** -i
    elif kind == "llama3":
        from .reference import rope_inv_freq

        inv = rope_inv_freq(rot_dim, theta, scaling).double()
    elif kind == "yarn":
        factor = float(scaling.get("factor") or (max_position / original))
        by = lambda m: 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0
        out = scaling.get("attention_factor")
        if out is None:
            m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
            out = by(m) / by(m_all) if m and m_all else by(1)
        at = lambda turns: rot_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = at(scaling.get("beta_fast") or 32), at(scaling.get("beta_slow") or 1)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rot_dim - 1)
        if low == high:
            high += 0.001
        ramp = ((torch.arange(rot_dim // 2, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
    elif kind == "longrope":
        factors = scaling["long_factor"] if (length or 0) > original else scaling["short_factor"]
        inv = inv / torch.tensor(factors, dtype=torch.float64)
        out = scaling.get("attention_factor")
        if out is None:
            factor = float(scaling.get("factor") or (max_position or original) / original)
            out = math.sqrt(1 + math.log(factor) / math.log(original)) if factor > 1 else 1.0
    return inv.float().to(device), float(out)


def rope_append_slots(qkv: torch.Tensor, q_out: torch.Tensor, kv_pool: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor,
                      slots: torch.Tensor, *, q_heads: int, kv_heads: int, head_dim: int, q_off: int, k_off: int, v_off: int,
                      interleaved: bool = False, factor: float = 1.0, status: Optional[torch.Tensor] = None,
                      early_start: int = EARLY_FIRST) -> None:
    """:func:`nanoflow_b200.ops.rope_append` by slot, for rotations of any layout: q rotated to ``q_out``, k rotated and v to their tokens'
    slots of the bf16 cache.

    ``inv_freq`` (fp32) has an entry per pair that turns: head_dim / 2, or fewer where only the first 2 ``len(inv_freq)`` elements of a
    head do. Pairs are elements i and i + ``len(inv_freq)``, or 2 i and 2 i + 1 where ``interleaved``. ``factor`` multiplies cosines and
    sines (:func:`rope_frequencies`). Angles are formed in 64 bits.
    Tokens with a negative slot are not cached; one whose slot does not exist is reported. Two tokens must not have the same slot."""
    _calls().rope(qkv, q_out, kv_pool, inv_freq, positions, slots, q_heads, kv_heads, head_dim, q_off, k_off, v_off, interleaved, factor, status,
                  early_start)


def tree_workspace(*, q_heads: int, kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """Workspace of :func:`attn_tree` calls with these heads, whatever their batch. What it holds before a call does not matter. Calls that
    may run at the same time (two streams, two captured graphs) each need their own."""
    p = AttnTreeParams(q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim)
    fn = lib().nfk_attn_tree_workspace
    fn.restype = c_longlong
    device = torch.device(device)
    if device.type == "cuda" and device.index is not None and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            n = fn(byref(p))
    else:
        n = fn(byref(p))
    if n <= 0 or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads or q_heads // kv_heads > 128:
        raise RuntimeError("tree_workspace: unsupported sizes (head_dim 64 or 128, up to 128 query heads per KV head)")
    return torch.empty(n, dtype=torch.uint8, device=device)


def attn_tree(q: torch.Tensor, out: torch.Tensor, kv_pool: torch.Tensor, qo_indptr: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
              kv_last_page_len: torch.Tensor, tree: Optional[torch.Tensor] = None, *, q_heads: int, workspace: torch.Tensor, req_begin: int = 0,
              req_count: Optional[int] = None, sm_scale: Optional[float] = None, num_ctas: int = 0, request_tokens: int = 0,
              status: Optional[torch.Tensor] = None, early_start: int = EARLY_FIRST | EARLY_FURTHER) -> torch.Tensor:
    """Attention of the n_r query tokens of each request over its cached tokens, of which the last n_r are the query tokens themselves: all
    of them see what is cached in front, and token i sees token j of the request where bit j of ``tree`` (int64 ``[tokens, words]``, up to 8
    words, the row of token i) is set. ``tree=None``: a chain, i sees j up to itself.

    ``q`` and ``out``: bf16 ``[tokens, q_heads * head_dim]``, rows may be strided. Requests [req_begin, req_begin + req_count), all that
    ``kv_last_page_len`` lists by default; rows of other requests, and rows behind the last one, are left as they were. A row that sees
    nothing gets zeros, one that only sees scores of minus infinity NaN; infinities and NaN in cached tokens that a row does not see do not
    reach it. Results do not depend on what else runs, or on the workspace's contents; they may differ in their last bits between batches.

    Reported in ``status``: page numbers that are none (page 0 is read instead), lists that are none (no rows, or rows of zeros), fewer
    cached than query tokens (rows of zeros). ``workspace``: :func:`tree_workspace`. ``num_ctas``: CTA budget of each kernel.

    ``request_tokens``: about how many query tokens a request has, for the choice between the forms for few and for many rows (any number
    gives right results). 0: the rows of ``q`` for each listed request, which is too many where ``q`` has room for more than a step brings, as in
    a captured graph: there short requests take up to a quarter longer.

    Chains can also be run by :func:`nanoflow_b200.ops.attn_prefill`, where the host knows the tokens of each request and cuts them into items.
    With 32 query and 8 KV heads of 128 that is the faster one for many requests of 16 tokens and more, or little in front (32 requests of 64
    behind 4000: 157 us and 165; 4 of 512 with nothing in front: 25 and 67), and this one for few requests with long contexts, which it cuts (one
    of 60 behind 100000: 120 us and 1460; one of 26 behind 2000: 16 and 31)."""
    _calls().attend(q, out, kv_pool, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, tree, q_heads, req_begin, req_count, sm_scale, num_ctas,
                    workspace, status, early_start, request_tokens)
    return out


def tree_masks(parents: torch.Tensor, qo_indptr: torch.Tensor, mask: torch.Tensor, *, positions: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None, early_start: int = EARLY_FIRST) -> torch.Tensor:
    """``mask`` (int64 ``[tokens, words]``) = bits of each token and of those that it descends from. ``parents[t]``: place of t's parent among
    its request's tokens, in front of its own; -1: none (anything else is reported and taken for it). ``positions``: of which each request's
    first is right; the others become that plus the token's depth. Tokens behind a mask's last bit (64 a word, up to 512) see none of the others
    and are reported; rows of tokens of no request are left as they were."""
    _calls().masks(parents, qo_indptr, mask, positions, status, early_start)
    return mask


def tree_accept(tokens: torch.Tensor, parents: torch.Tensor, targets: torch.Tensor, qo_indptr: torch.Tensor, path: torch.Tensor,
                counts: torch.Tensor, next_tokens: torch.Tensor, *, dropped: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None,
                early_start: int = EARLY_FIRST) -> None:
    """The branch that the model agrees with, greedily: from a request's token 0 (the last sure one) on to the first child that holds
    ``targets`` of its parent, the model's choice behind it. ``path[r]`` (``[requests, places]``): the places of the tokens on it, -1
    behind the last; ``counts[r]``: how many (``places`` at most); ``next_tokens[r]``: the target of the last one, -1 for a request without tokens;
    ``dropped[r]``: how many tokens are not on it. Tokens behind a request's 512th are dropped and reported."""
    _calls().accept(tokens, parents, targets, qo_indptr, path, counts, next_tokens, dropped, status, early_start)


def kv_keep(kv_pools: Sequence[torch.Tensor], slots: torch.Tensor, path: torch.Tensor, counts: torch.Tensor, qo_indptr: torch.Tensor, *,
            status: Optional[torch.Tensor] = None, early_start: int = EARLY_FIRST) -> None:
    """In every pool (a list, a layer each, of one size): keys and values of request r's token ``path[r, k]`` go to the slot of its token
    k, for k < ``counts[r]``, so that the accepted branch lies behind its context without gaps. ``path[r, k] >= k``, as :func:`tree_accept`
    gives it; an entry that is none, or slots that do not exist, are reported and not moved. Slots of the batch's tokens must differ."""
    _calls().keep(kv_pools, slots, path, counts, qo_indptr, status, early_start)
