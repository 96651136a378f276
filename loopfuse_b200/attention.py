"""PyTorch-facing attention ops over the sm_100a C ABI.

Tensors must be CUDA, bf16 and contiguous; the ops launch on
``torch.cuda.current_stream()`` and return without synchronising.  There is no
CPU or eager fallback: a missing library, a wrong device or dtype raises.

* ``prefill_attention_fwd(q, k, v, causal)`` -- drop-in for the reference's
  ``kernels/triton/prefill_attn.py:127-168`` (``[B,H,S,D]`` layout), extended to
  grouped-query heads (``k, v`` may have fewer heads) and to ``Sq < Sk``
  (queries appended after a cached prefix, bottom-right causal mask).
* ``paged_decode(q, k_pages, v_pages, block_table, seq_lens, ...)`` -- split-KV
  decode over a paged pool, optional shared prefix.
* ``decode_attention_fwd(q, k, v)`` -- drop-in for
  ``kernels/triton/decode_attn.py:133-171`` (contiguous ``[B,H,S,D]`` cache):
  the cache is laid out as pages and handed to ``paged_decode``.

K/V may also be held in 4 bits (4.5 with their scales; format in ``include/loopfuse_b200.h``):

* ``append_qkv_q4(...)`` -- split, rotate and quantise a QKV projection's rows into the pages.
* ``paged_decode_q4(...)`` -- ``paged_decode`` over 4-bit pages.
* ``expand_pages_q4(...)`` -- a batch's pages as bf16, for ``prefill_paged``.
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from ._launch import launch, sm_count
from ._lib import LF_PAGE_SIZE, LoopfuseError

SM_COUNT = 148          # B200; the split heuristic uses the current device's count when it can


def _sm_count() -> int:
    if torch.cuda.is_available():
        return torch.cuda.get_device_properties(torch.cuda.current_device()).multi_processor_count
    return SM_COUNT


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _require(t: torch.Tensor, name: str, dtype=torch.bfloat16) -> None:
    if not t.is_cuda:
        raise LoopfuseError(_lib.LF_EINVAL, f"{name} must be a CUDA tensor (no CPU path)")
    if t.dtype != dtype:
        raise LoopfuseError(_lib.LF_EINVAL, f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise LoopfuseError(_lib.LF_EINVAL, f"{name} must be contiguous")


def prefill_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
                          scale: Optional[float] = None, return_lse: bool = False):
    """Causal GQA attention: ``q [B,Hq,Sq,D]``, ``k, v [B,Hkv,Sk,D]`` -> ``o [B,Hq,Sq,D]``, D 64 or 128."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _require(t, n)
    B, Hq, Sq, D = q.shape
    Bk, Hkv, Sk, Dk = k.shape
    if Bk != B or Dk != D or v.shape != k.shape:
        raise LoopfuseError(_lib.LF_EINVAL, f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} "
                                            f"v{tuple(v.shape)}")
    scale = D ** -0.5 if scale is None else float(scale)
    o = torch.empty_like(q)
    lse = torch.empty((B, Hq, Sq), dtype=torch.float32, device=q.device) if return_lse else None
    _lib.call("lf_prefill_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
              lse.data_ptr() if lse is not None else None, B, Hq, Hkv, Sq, Sk, D, scale,
              int(bool(causal)), _stream())
    return (o, lse) if return_lse else o


def prefill_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                  block_table: torch.Tensor, cu_seqlens_q: torch.Tensor, seqlens_k: torch.Tensor,
                  max_seqlen_q: int, causal: bool = True, scale: Optional[float] = None,
                  return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of newly appended tokens over each session's cached paged K/V.

    ``q [T, Hq, D]``: the new tokens of N sessions back to back, session ``n`` owning rows
    ``cu_seqlens_q[n] .. cu_seqlens_q[n+1]``; ``k_pages, v_pages [P, Hkv, 16, D]`` (one layer,
    new tokens already appended); ``block_table [N, max_pages]``; ``seqlens_k [N]`` context
    lengths including the new tokens.  Causal with the queries at the end of their session.
    Returns ``o [T, Hq, D]`` (and ``lse [T, Hq]``); ``out``, when given, is a contiguous
    ``[T, Hq, D]`` bf16 tensor that receives ``o``.
    """
    for t, n in ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages")):
        _require(t, n)
    for t, n in ((block_table, "block_table"), (cu_seqlens_q, "cu_seqlens_q"),
                 (seqlens_k, "seqlens_k")):
        _require(t, n, torch.int32)
    T, Hq, D = q.shape
    P, Hkv, page, Dk = k_pages.shape
    N = block_table.shape[0]
    if page != LF_PAGE_SIZE or Dk != D or cu_seqlens_q.shape != (N + 1,) or seqlens_k.shape != (N,):
        raise LoopfuseError(_lib.LF_EINVAL, "prefill_paged: inconsistent shapes")
    scale = D ** -0.5 if scale is None else float(scale)
    if out is None:
        o = torch.empty_like(q)
    else:
        _require(out, "out")
        if out.shape != q.shape:
            raise LoopfuseError(_lib.LF_EINVAL, "prefill_paged: out must have q's shape")
        o = out
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    _lib.call("lf_prefill_paged_fwd", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
              block_table.data_ptr(), cu_seqlens_q.data_ptr(), seqlens_k.data_ptr(), o.data_ptr(),
              lse.data_ptr() if lse is not None else None, N, T, int(max_seqlen_q), Hq, Hkv, D, P,
              block_table.shape[1], scale, int(bool(causal)), _stream())
    return (o, lse) if return_lse else o


def default_pages_per_split(num_seqs: int, num_kv_heads: int, max_pages: int,
                            num_prefix_pages: int = 0) -> int:
    """Split size for the sessions' own pages (the shared prefix is read separately): enough
    CTAs for several waves on the device's SMs, 32 to 128 pages each.  ``max_pages`` is the
    block-table width, each session's capacity; sessions are taken to be half full on average.
    The floor of 32 keeps small batches from launching many short or empty splits: the grid is
    sized for the table's capacity, and three split CTAs fit on an SM at a time.  The formula
    lives in the library (``lf_decode_default_split``), shared with the no-allocation decode."""
    out = _lib.c_int(0)
    _lib.call("lf_decode_default_split", int(num_seqs), int(num_kv_heads), int(max_pages),
              int(num_prefix_pages), _sm_count(), _lib.ctypes.byref(out))
    return int(out.value)


def decode_workspace_bytes(num_seqs: int, num_q_heads: int, head_dim: int, max_pages: int,
                           pages_per_split: int, num_prefix_pages: int = 0) -> int:
    n = _lib.c_size_t(0)
    _lib.call("lf_decode_workspace_size", num_seqs, num_q_heads, head_dim, max_pages,
              pages_per_split, num_prefix_pages, _lib.ctypes.byref(n))
    return int(n.value)


def paged_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 block_table: torch.Tensor, seq_lens: torch.Tensor, num_prefix_pages: int = 0,
                 scale: Optional[float] = None, pages_per_split: Optional[int] = None,
                 out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                 return_lse: bool = False, k_new: Optional[torch.Tensor] = None,
                 v_new: Optional[torch.Tensor] = None):
    """One-token attention per session over paged K/V.

    ``q [N,Hq,D]``; ``k_pages, v_pages [P,Hkv,16,D]`` (one layer of the pool);
    ``block_table [N,max_pages]`` int32; ``seq_lens [N]`` int32.  With
    ``num_prefix_pages > 0`` the first that many block-table entries must be the
    same pages for all sessions; they are then read once per group of sessions.

    ``k_new, v_new [N,Hkv,D]`` (both or neither): each session's newest token, at position
    ``seq_lens[i] - 1`` in a page already reserved in ``block_table`` past the shared-prefix
    pages, is stored into ``k_pages`` / ``v_pages`` by the decode itself before it is attended
    (``lf_decode_fwd_append``): the pages end up as a separate ``KVPool.write_layer`` would leave
    them, one kernel launch fewer.
    """
    _require(q, "q")
    _require(k_pages, "k_pages")
    _require(v_pages, "v_pages")
    _require(block_table, "block_table", torch.int32)
    _require(seq_lens, "seq_lens", torch.int32)
    N, Hq, D = q.shape
    P, Hkv, page, Dk = k_pages.shape
    if page != LF_PAGE_SIZE or Dk != D or v_pages.shape != k_pages.shape:
        raise LoopfuseError(_lib.LF_EINVAL, f"pages must be [P,Hkv,{LF_PAGE_SIZE},{D}]")
    if block_table.dim() != 2 or block_table.shape[0] != N or seq_lens.shape != (N,):
        raise LoopfuseError(_lib.LF_EINVAL, "block_table must be [N,max_pages], seq_lens [N]")
    max_pages = block_table.shape[1]
    pps = pages_per_split or default_pages_per_split(N, Hkv, max_pages, num_prefix_pages)
    scale = D ** -0.5 if scale is None else float(scale)
    need = decode_workspace_bytes(N, Hq, D, max_pages, pps, num_prefix_pages)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    o = out if out is not None else torch.empty_like(q)
    lse = torch.empty((N, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    if (k_new is None) != (v_new is None):
        raise LoopfuseError(_lib.LF_EINVAL, "paged_decode: give both k_new and v_new, or neither")
    if k_new is not None:
        for t, n in ((k_new, "k_new"), (v_new, "v_new")):
            _require(t, n)
            if tuple(t.shape) != (N, Hkv, D):
                raise LoopfuseError(_lib.LF_EINVAL, f"{n} must be [N,Hkv,D] = {(N, Hkv, D)}")
        _lib.call("lf_decode_fwd_append", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                  block_table.data_ptr(), seq_lens.data_ptr(), int(num_prefix_pages),
                  k_new.data_ptr(), v_new.data_ptr(), o.data_ptr(),
                  lse.data_ptr() if lse is not None else None, workspace.data_ptr(),
                  workspace.numel() * workspace.element_size(), N, Hq, Hkv, D, P, max_pages, pps,
                  scale, _stream())
        return (o, lse) if return_lse else o
    _lib.call("lf_decode_fwd", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
              block_table.data_ptr(), seq_lens.data_ptr(), int(num_prefix_pages), o.data_ptr(),
              lse.data_ptr() if lse is not None else None, workspace.data_ptr(),
              workspace.numel() * workspace.element_size(), N, Hq, Hkv, D, P, max_pages, pps,
              scale, _stream())
    return (o, lse) if return_lse else o


def contiguous_to_pages(k: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``[B,H,S,D]`` cache -> pages ``[B*ceil(S/16), H, 16, D]`` and block table ``[B, S/16]``."""
    B, H, S, D = k.shape
    npg = math.ceil(S / LF_PAGE_SIZE)
    pad = npg * LF_PAGE_SIZE - S
    if pad:
        k = torch.nn.functional.pad(k, (0, 0, 0, pad))
    pages = k.view(B, H, npg, LF_PAGE_SIZE, D).permute(0, 2, 1, 3, 4).reshape(B * npg, H,
                                                                              LF_PAGE_SIZE, D)
    table = torch.arange(B * npg, dtype=torch.int32, device=k.device).view(B, npg)
    return pages.contiguous(), table


def decode_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """Reference-compatible decode: ``q [B,H,1,D]``, ``k, v [B,Hkv,S,D]`` -> ``[B,H,1,D]``."""
    if q.dim() != 4 or q.shape[2] != 1:
        raise LoopfuseError(_lib.LF_EINVAL, f"decode expects seq_q=1, got {tuple(q.shape)}")
    B, H, _, D = q.shape
    S = k.shape[2]
    kp, table = contiguous_to_pages(k)
    vp, _ = contiguous_to_pages(v)
    lens = torch.full((B,), S, dtype=torch.int32, device=q.device)
    o = paged_decode(q.reshape(B, H, D).contiguous(), kp, vp, table, lens, scale=scale)
    return o.view(B, H, 1, D)


# -- K/V held in 4 bits -------------------------------------------------------------------------------
def q4_head_dim(pages: torch.Tensor) -> int:
    """Head dim of 4-bit pages ``[P, Hkv, 18 * D]``: 64 or 128."""
    _require(pages, "pages", torch.uint8)
    if pages.dim() != 3 or pages.shape[2] not in (18 * 64, 18 * 128):
        raise LoopfuseError(_lib.LF_EINVAL, f"4-bit pages must be [P, Hkv, 18 * D] with D 64 or 128, "
                                            f"got {tuple(pages.shape)}")
    return pages.shape[2] // 18


def _one_device(what: str, *tensors: Optional[torch.Tensor]) -> torch.device:
    """The device all the given tensors are on."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise LoopfuseError(_lib.LF_EINVAL, f"{what}: tensors on {dev} and {t.device}")
    return dev


def append_qkv_q4(qkv: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor,
                  start_pos: torch.Tensor, cu_tokens: torch.Tensor, num_q_heads: int,
                  rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                  q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Quantised append of one layer: ``qkv [T, (Hq + 2 Hkv) * D]`` (q heads, then k heads, then v
    heads per row; rows may be strided), the new tokens of N sessions back to back.

    Token ``t`` of session ``i`` (``cu_tokens [N+1]``) goes to position ``start_pos[i] + t -
    cu_tokens[i]`` of ``block_table [N, max_pages]``, into ``pages [P, Hkv, 18 * D]``; q and k are
    first rotated with ``rope = (cos, sin)`` (``[rows, D/2]`` fp32, "rotate half").  Returns the
    rotated q ``[T, Hq, D]`` (``q_out`` when given).  Block-table rows and pages are the caller's to
    reserve; a token without a page, or a row of no session (before ``cu_tokens[0]`` or from
    ``cu_tokens[N]`` on: its q is not written either), is not stored and is reported by
    ``lf_device_status``.
    """
    D = q4_head_dim(pages)
    P, Hkv, _ = pages.shape
    Hq = int(num_q_heads)
    for t, n in ((block_table, "block_table"), (start_pos, "start_pos"), (cu_tokens, "cu_tokens")):
        _require(t, n, torch.int32)
    N = start_pos.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != N or start_pos.dim() != 1 or \
            cu_tokens.shape != (N + 1,):
        raise LoopfuseError(_lib.LF_EINVAL, "append_qkv_q4: block_table must be [N, max_pages], "
                                            "start_pos [N], cu_tokens [N + 1]")
    if not qkv.is_cuda or qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or Hq <= 0 or \
            qkv.shape[1] != (Hq + 2 * Hkv) * D or qkv.stride(1) != 1 or \
            (qkv.shape[0] > 1 and qkv.stride(0) < qkv.shape[1]):
        raise LoopfuseError(_lib.LF_EINVAL, "append_qkv_q4 expects bf16 rows qkv [T, (Hq + 2 Hkv) * D]")
    T = qkv.shape[0]
    if q_out is None:
        q_out = torch.empty(T, Hq, D, dtype=qkv.dtype, device=qkv.device)
    _require(q_out, "q_out")
    if tuple(q_out.shape) != (T, Hq, D):
        raise LoopfuseError(_lib.LF_EINVAL, f"q_out must be [T, Hq, D] = {(T, Hq, D)}")
    cos, sin, rows = _rope(rope, D)
    dev = _one_device("append_qkv_q4", qkv, pages, block_table, start_pos, cu_tokens, q_out, cos, sin)
    if T == 0 or N == 0:
        return q_out
    base, elem, row = qkv.data_ptr(), qkv.element_size(), qkv.stride(0) if T > 1 else qkv.shape[1]
    launch("lf_q4_append", dev, base, base + Hq * D * elem, base + (Hq + Hkv) * D * elem, row, 0,
           row, D, block_table.data_ptr(), N, block_table.shape[1], None, start_pos.data_ptr(),
           cu_tokens.data_ptr(), N, T, cos.data_ptr() if cos is not None else None,
           sin.data_ptr() if sin is not None else None, rows, q_out.data_ptr(), pages.data_ptr(), P,
           1, Hq, Hkv, D, None)
    return q_out


def _rope(rope, D: int):
    """Checked (cos, sin, rows) of rotation tables; (None, None, 0) without any."""
    if rope is None:
        return None, None, 0
    cos, sin = rope
    for t in (cos, sin):
        _require(t, "rope table", torch.float32)
        if t.dim() != 2 or t.shape[1] != D // 2 or t.shape != cos.shape or t.shape[0] == 0:
            raise LoopfuseError(_lib.LF_EINVAL, f"rope tables must be [rows, {D // 2}]")
    return cos, sin, cos.shape[0]


@lru_cache(maxsize=4096)
def decode_q4_workspace_bytes(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                              max_pages: int, num_prefix_pages: int = 0, sms: int = 0) -> int:
    """Workspace of ``paged_decode_q4`` on a device of ``sms`` SMs (0: the current one)."""
    n = _lib.c_size_t(0)
    _lib.call("lf_q4_decode_workspace_size", num_seqs, num_q_heads, num_kv_heads, head_dim, max_pages,
              num_prefix_pages, sms or _sm_count(), _lib.ctypes.byref(n))
    return int(n.value)


def _check_decode_q4(q, pages, block_table, seq_lens, out, workspace) -> None:
    if workspace is not None and not workspace.is_contiguous():
        raise LoopfuseError(_lib.LF_EINVAL, "paged_decode_q4: workspace must be contiguous")
    _require(q, "q")
    D = q4_head_dim(pages)
    _require(block_table, "block_table", torch.int32)
    _require(seq_lens, "seq_lens", torch.int32)
    if q.dim() != 3 or q.shape[2] != D:
        raise LoopfuseError(_lib.LF_EINVAL, f"q must be [N, Hq, {D}], got {tuple(q.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] != q.shape[0] or seq_lens.shape != q.shape[:1]:
        raise LoopfuseError(_lib.LF_EINVAL, "block_table must be [N,max_pages], seq_lens [N]")
    _one_device("paged_decode_q4", q, pages, block_table, seq_lens, out, workspace)
    if out is not None:
        _require(out, "out")
        if out.shape != q.shape:
            raise LoopfuseError(_lib.LF_EINVAL, "paged_decode_q4: out must have q's shape")


def paged_decode_q4(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, num_prefix_pages: int = 0,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None, return_lse: bool = False):
    """``paged_decode`` over K/V held in 4 bits: ``q [N, Hq, D]``, ``pages [P, Hkv, 18 * D]`` uint8
    (one layer), ``block_table [N, max_pages]`` and ``seq_lens [N]`` int32, Hq / Hkv 1, 2, 4 or 8.
    With ``num_prefix_pages > 0`` the first that many block-table entries must be the same pages
    for all sessions.  A session of length 0 gives zeros and an LSE of -inf."""
    dev, i32, ps, qs = q.device, torch.int32, pages.shape, q.shape
    # In one go; what is wrong, if anything is, is named by the checks one by one.
    if not (q.is_cuda and pages.device == dev and block_table.device == dev and seq_lens.device == dev and
            q.dtype is torch.bfloat16 and pages.dtype is torch.uint8 and block_table.dtype is i32 and
            seq_lens.dtype is i32 and q.is_contiguous() and pages.is_contiguous() and
            block_table.is_contiguous() and seq_lens.is_contiguous() and len(qs) == 3 and len(ps) == 3 and
            ps[2] == 18 * qs[2] and (qs[2] == 128 or qs[2] == 64) and block_table.dim() == 2 and
            block_table.shape[0] == qs[0] and seq_lens.shape == qs[:1] and out is None and workspace is None):
        _check_decode_q4(q, pages, block_table, seq_lens, out, workspace)
    N, Hq, D = qs
    P, Hkv, _ = ps
    o = torch.empty_like(q) if out is None else out
    lse = torch.empty(N, Hq, dtype=torch.float32, device=dev) if return_lse else None
    if N == 0:
        return (o, lse) if return_lse else o
    max_pages, npre = block_table.shape[1], int(num_prefix_pages)
    scale = D ** -0.5 if scale is None else float(scale)
    sms = sm_count(dev.index)
    need = decode_q4_workspace_bytes(N, Hq, Hkv, D, max_pages, npre, sms)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    launch("lf_q4_decode_fwd", dev, q.data_ptr(), pages.data_ptr(), block_table.data_ptr(),
           seq_lens.data_ptr(), npre, o.data_ptr(), lse.data_ptr() if lse is not None else None,
           workspace.data_ptr() if need else None, need, N, Hq, Hkv, D, P, max_pages, scale, sms)
    return (o, lse) if return_lse else o


def expand_pages_q4(pages: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    total_pages: int, num_prefix_pages: int = 0,
                    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A batch's 4-bit pages as bf16 pages for ``prefill_paged``: ``(k_pages, v_pages [total_pages,
    Hkv, 16, D], block_table [N, max_pages])``.

    The shared prefix's pages come first, then each session's own; ``total_pages`` is their number
    (``num_prefix_pages + sum(max(0, ceil(len / 16) - num_prefix_pages))``; more is allowed, the
    rest stays unwritten, fewer is an error that ``lf_device_status`` reports).  Rows at or past a
    session's length are zeros.  ``out`` gives the two page tensors to write."""
    D = q4_head_dim(pages)
    _require(block_table, "block_table", torch.int32)
    _require(seq_lens, "seq_lens", torch.int32)
    P, Hkv, _ = pages.shape
    if block_table.dim() != 2 or seq_lens.shape != (block_table.shape[0],):
        raise LoopfuseError(_lib.LF_EINVAL, "block_table must be [N,max_pages], seq_lens [N]")
    N, max_pages = block_table.shape
    shape = (int(total_pages), Hkv, LF_PAGE_SIZE, D)
    k, v = out if out is not None else (
        torch.empty(shape, dtype=torch.bfloat16, device=pages.device) for _ in range(2))
    for t in (k, v):
        _require(t, "out")
        if tuple(t.shape) != shape:
            raise LoopfuseError(_lib.LF_EINVAL, f"expand_pages_q4: out must be two tensors {shape}")
    dev = _one_device("expand_pages_q4", pages, block_table, seq_lens, k, v)
    table = torch.empty_like(block_table)
    launch("lf_q4_expand", dev, pages.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
           int(num_prefix_pages), k.data_ptr(), v.data_ptr(), table.data_ptr(), N, Hkv, D, P, max_pages,
           shape[0])
    return k, v, table
