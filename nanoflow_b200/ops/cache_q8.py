"""A paged KV cache in 8 bits: the write into it, attention over it, and its pages as bf16.

The cache of a layer is a pool ``[num_pages, 2, kv_heads, 16, head_dim]`` of ``float8_e4m3fn`` or ``int8`` numbers and a scale
for every vector, ``[num_pages, 2, kv_heads, 16]`` in fp32; a cached value is number * scale. Pages, page lists and the calls
have the form of the bf16 cache (:func:`nanoflow_b200.ops.rope_append`, :func:`nanoflow_b200.ops.attn_decode`), at half the bytes.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p, Structure, byref
from typing import Optional, Tuple

import torch

from . import _check, _p, lib

PAGE = 16
KINDS = {torch.float8_e4m3fn: 0, torch.int8: 1}


class RopeAppendQ8Params(Structure):
    _fields_ = [("qkv", c_void_p), ("ld_qkv", c_longlong), ("q_off", c_int), ("k_off", c_int), ("v_off", c_int),
                ("q_out", c_void_p), ("kv_pool", c_void_p), ("kv_scale", c_void_p), ("inv_freq", c_void_p),
                ("cos_sin", c_void_p), ("positions", c_void_p), ("token_req", c_void_p), ("kv_indptr", c_void_p),
                ("kv_indices", c_void_p), ("q_norm", c_void_p), ("k_norm", c_void_p), ("eps", c_float), ("T", c_int),
                ("q_heads", c_int), ("kv_heads", c_int), ("head_dim", c_int), ("num_pages", c_int), ("num_reqs", c_int),
                ("num_indices", c_int), ("kind", c_int), ("status", c_void_p)]


class KvReadQ8Params(Structure):
    _fields_ = [("kv_pool", c_void_p), ("kv_scale", c_void_p), ("out", c_void_p), ("page_ids", c_void_p), ("n_pages", c_int),
                ("kv_heads", c_int), ("head_dim", c_int), ("num_pages", c_int), ("kind", c_int), ("status", c_void_p)]


class AttnQ8Params(Structure):
    _fields_ = [("q", c_void_p), ("out", c_void_p), ("kv_pool", c_void_p), ("kv_scale", c_void_p), ("qo_indptr", c_void_p),
                ("kv_indptr", c_void_p), ("kv_indices", c_void_p), ("kv_last_page_len", c_void_p), ("prefix_pages", c_void_p),
                ("q_heads", c_int), ("kv_heads", c_int), ("head_dim", c_int), ("num_pages", c_int), ("num_tokens", c_int),
                ("num_indices", c_int), ("req_begin", c_int), ("req_count", c_int), ("prefix_len", c_int), ("kind", c_int),
                ("sm_scale", c_float), ("num_ctas", c_int), ("workspace", c_void_p), ("workspace_bytes", c_longlong),
                ("status", c_void_p)]


def kv_pool_q8(num_pages: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float8_e4m3fn,
               device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """The pool and the scales of one layer, zeros."""
    if dtype not in KINDS:
        raise RuntimeError(f"kv_pool_q8: numbers are float8_e4m3fn or int8, not {dtype}")
    shape = (num_pages, 2, kv_heads, PAGE)
    pool = torch.zeros((*shape, head_dim), dtype=torch.int8, device=device).view(dtype)
    return pool, torch.zeros(shape, dtype=torch.float32, device=device)


def _pool(what: str, kv_pool: torch.Tensor, kv_scale: torch.Tensor) -> torch.device:
    """Checks a layer's cache; its device."""
    if kv_pool.dtype not in KINDS or kv_pool.dim() != 5 or not kv_pool.is_contiguous() or not kv_pool.is_cuda:
        raise RuntimeError(f"{what}: kv_pool must be a contiguous CUDA float8_e4m3fn or int8 [pages, 2, kv_heads, 16, head_dim]")
    pages, two, _, page_size, head_dim = kv_pool.shape
    if two != 2 or page_size != PAGE or head_dim not in (64, 128):
        raise RuntimeError(f"{what}: pages hold 16 tokens of keys and of values, head_dim is 64 or 128")
    if kv_scale.dtype != torch.float32 or kv_scale.shape != kv_pool.shape[:4] or not kv_scale.is_contiguous():
        raise RuntimeError(f"{what}: kv_scale must be a contiguous float32 [pages, 2, kv_heads, 16]")
    if kv_scale.device != kv_pool.device:
        raise RuntimeError(f"{what}: tensors on more than one device")
    return kv_pool.device


def _tensor(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device) -> None:
    if t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be a contiguous {str(dtype)[6:]} tensor on {device}")


def _status(what: str, status: Optional[torch.Tensor], device: torch.device) -> None:
    if status is not None:
        _tensor(what, "status", status, torch.int32, device)


def _apart(what: str, a: torch.Tensor, b: torch.Tensor) -> None:
    """What a kernel writes must not lie over what other threads of it still read."""
    lo, hi = a.data_ptr(), b.data_ptr()
    span = lambda t: ((t.shape[0] - 1) * t.stride(0) + t[0].numel()) * t.element_size() if t.numel() else 0
    if lo < hi + span(b) and hi < lo + span(a):
        raise RuntimeError(f"{what}: input and output overlap")


def _run(name: str, p: Structure, device: torch.device) -> None:
    """Launch on the current stream of the tensors' device, whichever device is the current one."""
    fn = getattr(lib(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(byref(p), c_void_p(torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            rc = fn(byref(p), c_void_p(torch.cuda.current_stream(device).cuda_stream))
    _check(rc, name)


def rope_append_q8(qkv: torch.Tensor, q_out: torch.Tensor, kv_pool: torch.Tensor, kv_scale: torch.Tensor, inv_freq: torch.Tensor,
                   positions: torch.Tensor, token_req: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor, *,
                   q_heads: int, kv_heads: int, head_dim: int, q_off: int, k_off: int, v_off: int,
                   q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   cos_sin: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """:func:`nanoflow_b200.ops.rope_append` into the 8-bit cache: rotate q and k, write q to ``q_out`` (bf16) and k and v, each
    vector with its own scale (largest magnitude / 448 or / 127), into their page slots.

    ``q_norm`` / ``k_norm`` (bf16 ``[head_dim]``): RMS norm of every query / key head in front of the rotation, with ``eps``.
    ``cos_sin``: the iteration's table from ``rope_table``; without it angles are computed here, in 64 bits.
    Two tokens of a call must not have the same request and position. A vector with an infinity or NaN is cached as NaN, one
    whose largest magnitude is below 2^-80 as zeros. A token whose page does not exist is not cached and reported in ``status``."""
    what = "rope_append_q8"
    device = _pool(what, kv_pool, kv_scale)
    T = qkv.shape[0]
    if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.device != device or (qkv.shape[1] > 1 and qkv.stride(1) != 1):
        raise RuntimeError(f"{what}: qkv must be a bf16 [T, columns] with unit inner stride on {device}")
    if kv_pool.shape[2] != kv_heads or kv_pool.shape[4] != head_dim or q_heads < 1:
        raise RuntimeError(f"{what}: kv_pool does not have these heads")
    for off, n in ((q_off, q_heads), (k_off, kv_heads), (v_off, kv_heads)):
        if off < 0 or off + n * head_dim > qkv.shape[1]:
            raise RuntimeError(f"{what}: heads lie outside qkv's columns")
    _tensor(what, "q_out", q_out, torch.bfloat16, device)
    if q_out.numel() != T * q_heads * head_dim:
        raise RuntimeError(f"{what}: q_out must be [T, q_heads * head_dim]")
    for t, name in ((positions, "positions"), (token_req, "token_req"), (kv_indptr, "kv_indptr"), (kv_indices, "kv_indices")):
        _tensor(what, name, t, torch.int32, device)
    if positions.numel() != T or token_req.numel() != T or kv_indptr.numel() < 2:
        raise RuntimeError(f"{what}: positions and token_req have an entry per token, kv_indptr one per request and one more")
    _tensor(what, "inv_freq", inv_freq, torch.float32, device)
    if inv_freq.numel() != head_dim // 2:
        raise RuntimeError(f"{what}: inv_freq must be fp32 [head_dim/2]")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _tensor(what, name, t, torch.bfloat16, device)
            if t.numel() != head_dim:
                raise RuntimeError(f"{what}: {name} must be [head_dim]")
    if cos_sin is not None:
        _tensor(what, "cos_sin", cos_sin, torch.float32, device)
        if cos_sin.numel() < T * head_dim:
            raise RuntimeError(f"{what}: cos_sin must be [T, head_dim/2, 2]")
    _status(what, status, device)
    if T:
        _apart(what, qkv, q_out.view(T, -1))
    p = RopeAppendQ8Params(_p(qkv), qkv.stride(0), q_off, k_off, v_off, _p(q_out), _p(kv_pool), _p(kv_scale), _p(inv_freq),
                           _p(cos_sin), _p(positions), _p(token_req), _p(kv_indptr), _p(kv_indices), _p(q_norm), _p(k_norm), eps, T,
                           q_heads, kv_heads, head_dim, kv_pool.shape[0], kv_indptr.numel() - 1, kv_indices.numel(),
                           KINDS[kv_pool.dtype], _p(status))
    _run("nfk_rope_append_q8", p, device)


def kv_read_q8(kv_pool: torch.Tensor, kv_scale: torch.Tensor, page_ids: torch.Tensor, *, out: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[i]`` = the bf16 values of page ``page_ids[i]``: a pool that ``attn_prefill`` reads with the page list 0, 1, 2, ...
    Pages that do not exist are reported in ``status`` and leave their place in ``out`` as it was."""
    what = "kv_read_q8"
    device = _pool(what, kv_pool, kv_scale)
    _tensor(what, "page_ids", page_ids, torch.int32, device)
    n, shape = page_ids.numel(), kv_pool.shape
    if out is None:
        out = torch.empty((n, *shape[1:]), dtype=torch.bfloat16, device=device)
    _tensor(what, "out", out, torch.bfloat16, device)
    if out.shape != (n, *shape[1:]):
        raise RuntimeError(f"{what}: out must be [pages, 2, kv_heads, 16, head_dim]")
    _status(what, status, device)
    p = KvReadQ8Params(_p(kv_pool), _p(kv_scale), _p(out), _p(page_ids), n, shape[2], shape[4], shape[0], KINDS[kv_pool.dtype],
                       _p(status))
    _run("nfk_kv_read_q8", p, device)
    return out


def decode_workspace_q8(*, requests: int, q_heads: int, kv_heads: int, head_dim: int, prefix_len: int = 0,
                        device="cuda") -> torch.Tensor:
    """Workspace of ``attn_decode_q8`` and ``attn_decode_shared_q8`` calls of up to these sizes: zeros, which calls leave ready
    for the next one. Calls that may run at the same time (two streams, two captured graphs) each need their own."""
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
        raise RuntimeError("decode_workspace_q8: unsupported configuration (head_dim 64 or 128, up to 16 query heads per KV head)")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def _decode(what, q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, prefix_pages, prefix_len, q_heads,
            req_begin, req_count, sm_scale, num_ctas, workspace, status):
    device = _pool(what, kv_pool, kv_scale)
    pages, _, kv_heads, _, head_dim = kv_pool.shape
    _tensor(what, "q", q, torch.bfloat16, device)
    _tensor(what, "out", out, torch.bfloat16, device)
    if q_heads < 1 or q_heads % kv_heads or q_heads // kv_heads > 16:
        raise RuntimeError(f"{what}: up to 16 query heads share a KV head, all KV heads the same number")
    if q.dim() < 2 or q.shape[0] * q_heads * head_dim != q.numel() or out.shape != q.shape:
        raise RuntimeError(f"{what}: q and out must be [tokens, q_heads * head_dim]")
    for t, name in ((qo_indptr, "qo_indptr"), (kv_indptr, "kv_indptr"), (kv_indices, "kv_indices"),
                    (kv_last_page_len, "kv_last_page_len")):
        _tensor(what, name, t, torch.int32, device)
    end = req_begin + req_count
    if req_begin < 0 or req_count < 0 or qo_indptr.numel() < end or kv_indptr.numel() < end + 1 or kv_last_page_len.numel() < end:
        raise RuntimeError(f"{what}: requests {req_begin} to {end} are not all listed")
    if prefix_len > 0:
        _tensor(what, "prefix_pages", prefix_pages, torch.int32, device)
        if prefix_pages.numel() < (prefix_len + PAGE - 1) // PAGE:
            raise RuntimeError(f"{what}: prefix_pages lists fewer pages than prefix_len needs")
    if workspace is None:
        raise RuntimeError(f"{what}: needs a workspace (decode_workspace_q8)")
    _tensor(what, "workspace", workspace, torch.uint8, device)
    _status(what, status, device)
    if q.numel():
        _apart(what, q, out)
    p = AttnQ8Params(_p(q), _p(out), _p(kv_pool), _p(kv_scale), _p(qo_indptr), _p(kv_indptr), _p(kv_indices), _p(kv_last_page_len),
                     _p(prefix_pages if prefix_len > 0 else None), q_heads, kv_heads, head_dim, pages, q.shape[0], kv_indices.numel(),
                     req_begin, req_count, prefix_len, KINDS[kv_pool.dtype], head_dim ** -0.5 if sm_scale is None else sm_scale,
                     num_ctas, _p(workspace), workspace.numel(), _p(status))
    _run("nfk_attn_decode_q8", p, device)
    return out


def attn_decode_q8(q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, *, q_heads: int, req_begin: int,
                   req_count: int, workspace: torch.Tensor, sm_scale: Optional[float] = None, num_ctas: int = 0,
                   status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`nanoflow_b200.ops.attn_decode` over the 8-bit cache: single-query attention for requests [req_begin, req_begin +
    req_count). Contexts are cut over the CTAs by their pages, whatever their lengths. Requests without pages get zeros; rows of
    other requests are left as they were. ``workspace``: :func:`decode_workspace_q8`. ``num_ctas``: CTA budget, 0 = all that fit."""
    return _decode("attn_decode_q8", q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, None, 0, q_heads,
                   req_begin, req_count, sm_scale, num_ctas, workspace, status)


def attn_decode_shared_q8(q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, prefix_pages: torch.Tensor,
                          prefix_len: int, *, q_heads: int, req_begin: int, req_count: int, workspace: torch.Tensor,
                          sm_scale: Optional[float] = None, num_ctas: int = 0,
                          status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`attn_decode_q8` for requests that all see the same first ``prefix_len`` tokens, those of ``prefix_pages``; their own
    page lists hold what comes after (or nothing). The prefix is read once for all of them."""
    if prefix_len < 0:
        raise RuntimeError("attn_decode_shared_q8: prefix_len is not negative")
    return _decode("attn_decode_shared_q8", q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len,
                   prefix_pages, prefix_len, q_heads, req_begin, req_count, sm_scale, num_ctas, workspace, status)
