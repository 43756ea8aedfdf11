"""A paged KV cache in 8 bits: the write into it, attention over it, and its pages as bf16.

The cache of a layer is a pool ``[num_pages, 2, kv_heads, 16, head_dim]`` of ``float8_e4m3fn`` or ``int8`` numbers and a scale
for every vector, ``[num_pages, 2, kv_heads, 16]`` in fp32; a cached value is number * scale. Pages, page lists and the calls
have the form of the bf16 cache (:func:`nanoflow_b200.ops.rope_append`, :func:`nanoflow_b200.ops.attn_decode`), at half the bytes.

No tensor that a call writes (outputs, the workspace, the cache in the write, ``status``) may overlap another one of its tensors.

``early_start`` (EARLY_*) of the calls: their kernels may be launched while the one before them on the stream still runs, and wait
for it there; 0 keeps the SMs free until then, for another stream's kernels beside it.
"""
from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_longlong, c_void_p, Structure, byref
from typing import Optional, Tuple

import torch

from . import EARLY_FIRST, EARLY_FURTHER, lib

PAGE = 16
KINDS = {torch.float8_e4m3fn: 0, torch.int8: 1}


class RopeAppendQ8Params(Structure):
    _fields_ = [("qkv", c_void_p), ("ld_qkv", c_longlong), ("q_off", c_int), ("k_off", c_int), ("v_off", c_int),
                ("q_out", c_void_p), ("kv_pool", c_void_p), ("kv_scale", c_void_p), ("inv_freq", c_void_p),
                ("cos_sin", c_void_p), ("positions", c_void_p), ("token_req", c_void_p), ("kv_indptr", c_void_p),
                ("kv_indices", c_void_p), ("q_norm", c_void_p), ("k_norm", c_void_p), ("eps", c_float), ("T", c_int),
                ("q_heads", c_int), ("kv_heads", c_int), ("head_dim", c_int), ("num_pages", c_int), ("num_reqs", c_int),
                ("num_indices", c_int), ("kind", c_int), ("early_start", c_int), ("status", c_void_p)]


class KvReadQ8Params(Structure):
    _fields_ = [("kv_pool", c_void_p), ("kv_scale", c_void_p), ("out", c_void_p), ("page_ids", c_void_p), ("n_pages", c_int),
                ("kv_heads", c_int), ("head_dim", c_int), ("num_pages", c_int), ("kind", c_int),
                ("early_start", c_int), ("status", c_void_p)]


class AttnQ8Params(Structure):
    _fields_ = [("q", c_void_p), ("out", c_void_p), ("kv_pool", c_void_p), ("kv_scale", c_void_p), ("qo_indptr", c_void_p),
                ("kv_indptr", c_void_p), ("kv_indices", c_void_p), ("kv_last_page_len", c_void_p), ("prefix_pages", c_void_p),
                ("q_heads", c_int), ("kv_heads", c_int), ("head_dim", c_int), ("num_pages", c_int), ("num_tokens", c_int),
                ("num_indices", c_int), ("req_begin", c_int), ("req_count", c_int), ("prefix_len", c_int), ("kind", c_int),
                ("sm_scale", c_float), ("num_ctas", c_int), ("early_start", c_int), ("workspace", c_void_p), ("workspace_bytes", c_longlong),
                ("status", c_void_p)]


def kv_pool_q8(num_pages: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float8_e4m3fn,
               device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """The pool and the scales of one layer, zeros."""
    if dtype not in KINDS:
        raise RuntimeError(f"kv_pool_q8: numbers are float8_e4m3fn or int8, not {dtype}")
    shape = (num_pages, 2, kv_heads, PAGE)
    pool = torch.zeros((*shape, head_dim), dtype=torch.int8, device=device).view(dtype)
    return pool, torch.zeros(shape, dtype=torch.float32, device=device)


_calls_module = None


def _calls():
    """The extension module that checks and launches, connected to the kernel library (once). Raises if either is not built."""
    global _calls_module
    if _calls_module is None:
        try:
            from . import _cache_q8
        except ImportError as e:
            raise RuntimeError("nanoflow_b200/ops/_cache_q8 is missing: run `python -m nanoflow_b200.ops.build`") from e
        _cache_q8.connect(*(ctypes.cast(getattr(lib(), f), c_void_p).value
                            for f in ("nfk_rope_append_q8", "nfk_kv_read_q8", "nfk_attn_decode_q8")))
        _calls_module = _cache_q8
    return _calls_module


def rope_append_q8(qkv: torch.Tensor, q_out: torch.Tensor, kv_pool: torch.Tensor, kv_scale: torch.Tensor, inv_freq: torch.Tensor,
                   positions: torch.Tensor, token_req: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor, *,
                   q_heads: int, kv_heads: int, head_dim: int, q_off: int, k_off: int, v_off: int,
                   q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   cos_sin: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None, early_start: int = EARLY_FIRST) -> None:
    """:func:`nanoflow_b200.ops.rope_append` into the 8-bit cache: rotate q and k, write q to ``q_out`` (bf16) and k and v, each
    vector with its own scale (largest magnitude / 448 or / 127), into their page slots.

    ``q_norm`` / ``k_norm`` (bf16 ``[head_dim]``): RMS norm of every query / key head in front of the rotation, with ``eps``.
    ``cos_sin``: the iteration's table from ``rope_table``; without it angles are computed here, in 64 bits.
    Two tokens of a call must not have the same place (request and position, or pages that two requests share). A vector with an
    infinity or NaN, or a key that rotation takes beyond fp32, is cached as NaN, one whose largest magnitude is below 2^-80 as zeros. A
    token whose page does not exist is not cached and reported in ``status``."""
    _calls().rope_append(qkv, q_out, kv_pool, kv_scale, inv_freq, positions, token_req, kv_indptr, kv_indices, q_heads, kv_heads, head_dim,
                         q_off, k_off, v_off, q_norm, k_norm, eps, cos_sin, status, early_start)


def kv_read_q8(kv_pool: torch.Tensor, kv_scale: torch.Tensor, page_ids: torch.Tensor, *, out: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None, early_start: int = EARLY_FIRST) -> torch.Tensor:
    """``out[i]`` = the bf16 values of page ``page_ids[i]``: a pool that ``attn_prefill`` reads with the page list 0, 1, 2, ...
    Pages that do not exist are reported in ``status`` and leave their place in ``out`` as it was."""
    if out is None:
        out = torch.empty((page_ids.numel(), *kv_pool.shape[1:]), dtype=torch.bfloat16, device=kv_pool.device)
    _calls().read(kv_pool, kv_scale, page_ids, out, status, early_start)
    return out


def decode_workspace_q8(*, requests: int, q_heads: int, kv_heads: int, head_dim: int, prefix_len: int = 0,
                        device="cuda") -> torch.Tensor:
    """Workspace of ``attn_decode_q8`` and ``attn_decode_shared_q8`` calls with these heads, of up to ``requests`` requests and
    ``prefix_len`` tokens of prefix. What it holds before a call does not matter. Calls that may run at the same time (two streams,
    two captured graphs) each need their own."""
    p = AttnQ8Params(q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, req_count=requests, prefix_len=prefix_len)
    fn = lib().nfk_attn_q8_workspace
    fn.restype = c_longlong
    device = torch.device(device)
    if device.type == "cuda" and device.index is not None and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            n = fn(byref(p))
    else:
        n = fn(byref(p))
    if n <= 0:
        raise RuntimeError("decode_workspace_q8: unsupported sizes (head_dim 64 or 128, up to 16 query heads per KV head, counts of 32 bits)")
    return torch.empty(n, dtype=torch.uint8, device=device)


def attn_decode_q8(q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, *, q_heads: int, req_begin: int,
                   req_count: int, workspace: torch.Tensor, sm_scale: Optional[float] = None, num_ctas: int = 0,
                   status: Optional[torch.Tensor] = None, early_start: int = EARLY_FIRST | EARLY_FURTHER) -> torch.Tensor:
    """:func:`nanoflow_b200.ops.attn_decode` over the 8-bit cache: single-query attention for requests [req_begin, req_begin +
    req_count), each with a row of ``q`` of its own. Contexts are cut over the CTAs by their pages, whatever their lengths. Requests
    without pages get zeros; rows of other requests are left as they were. ``workspace``: :func:`decode_workspace_q8`. ``num_ctas``: CTA
    budget of each kernel, 0 = all that fit.

    Reported in ``status``: page numbers that are none (page 0 is read instead), rows that are none (left out), page lists that fall or
    leave ``kv_indices`` (as if there were no pages). Small batches, by ``kv_indices.numel()``, take one launch instead of two; with a list
    that is longer than its pages sums may differ in their last bits. Values whose scale is more than 2^20 below the request's largest
    lose bits of their weights; scores that fp32 does not hold give NaN."""
    _calls().decode("attn_decode_q8", q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, None, 0, q_heads,
                    req_begin, req_count, sm_scale, num_ctas, workspace, status, early_start)
    return out


def attn_decode_shared_q8(q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, prefix_pages: torch.Tensor,
                          prefix_len: int, *, q_heads: int, req_begin: int, req_count: int, workspace: torch.Tensor,
                          sm_scale: Optional[float] = None, num_ctas: int = 0,
                          status: Optional[torch.Tensor] = None, early_start: int = EARLY_FIRST | EARLY_FURTHER) -> torch.Tensor:
    """:func:`attn_decode_q8` for requests that all see the same first ``prefix_len`` tokens, those of ``prefix_pages``; their own
    page lists hold what comes after (or nothing). The prefix is read once for all of them. If a wait in its kernel runs out
    (``status``), the rows that it has part in are NaN."""
    _calls().decode("attn_decode_shared_q8", q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, prefix_pages,
                    prefix_len, q_heads, req_begin, req_count, sm_scale, num_ctas, workspace, status, early_start)
    return out
