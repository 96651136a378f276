"""Decoder ops on the sm_100a library: residual add + RMSNorm, the SwiGLU gate, a
weight-streaming tcgen05 GEMM for decode batches (``gemm_skinny``), low-rank adapters of many
sessions beside a shared projection (``lora_plan`` / ``lora_add``), and the log probabilities of
given tokens with entropy and top alternatives (``token_logprobs``).

Each is one bandwidth-bound kernel in place of the chain of torch elementwise passes a model
would otherwise run around its GEMMs (``lf_add_rmsnorm`` / ``lf_swiglu`` in
``include/loopfuse_b200.h``).  Rounding follows the eager torch sequence: the residual sum is
rounded to bf16, the normalised value is rounded to bf16 before the weight multiply, the SiLU
output is rounded to bf16 before the gate multiply.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._launch import launch, sm_count
from ._lib import LoopfuseError


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _check(t: torch.Tensor, name: str) -> None:
    if t.device.type != "cuda" or t.dtype != torch.bfloat16 or not t.is_contiguous():
        raise LoopfuseError(_lib.LF_EINVAL, f"{name} must be a contiguous CUDA bf16 tensor")


def add_rmsnorm(x: torch.Tensor, delta: Optional[torch.Tensor], w: Optional[torch.Tensor],
                eps: float, out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """``x += delta`` (in place, when given), then ``rmsnorm(x) * w`` (when ``w`` is given).
    ``x, delta, out [rows, dim]``, ``w [dim]``."""
    _check(x, "x")
    rows, dim = x.shape[0], x.shape[-1]
    if delta is not None:
        _check(delta, "delta")
        if delta.shape != x.shape:
            raise LoopfuseError(_lib.LF_EINVAL, "add_rmsnorm: delta must match x")
    if w is not None:
        _check(w, "w")
        if out is None:
            out = torch.empty_like(x)
        _check(out, "out")
    _lib.call("lf_add_rmsnorm", x.data_ptr(), delta.data_ptr() if delta is not None else None,
              w.data_ptr() if w is not None else None, out.data_ptr() if out is not None else None,
              rows, dim, float(eps), _stream())
    return out


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    """``silu(gu[:, :F]) * gu[:, F:]`` for a fused ``[rows, 2F]`` gate|up projection."""
    _check(gu, "gu")
    rows, two_f = gu.shape
    out = torch.empty((rows, two_f // 2), dtype=gu.dtype, device=gu.device)
    _lib.call("lf_swiglu", gu.data_ptr(), out.data_ptr(), rows, two_f // 2, _stream())
    return out


_SKINNY_MAX_M = 128
_skinny_ws: dict = {}


def _sm_count(device: torch.device) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count


def skinny_workspace_bytes(m: int, n: int, k: int, sm_count: int) -> int:
    out = _lib.c_size_t(0)
    _lib.call("lf_gemm_skinny_workspace_size", int(m), int(n), int(k), int(sm_count),
              _lib.ctypes.byref(out))
    return int(out.value)


def gemm_skinny(x: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor] = None,
                workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w`` for a decode batch: ``x [M, K]`` (1 <= M <= 128), ``w [K, N]``, bf16, on the
    weight-streaming tcgen05 GEMM (``lf_gemm_skinny``).  Without ``workspace`` the partial-sum
    buffer is a per-device cache grown on demand (pass one explicitly inside a CUDA graph that
    must not allocate)."""
    _check(x, "x")
    _check(w, "w")
    m, k = x.shape
    k2, n = w.shape
    if k2 != k:
        raise LoopfuseError(_lib.LF_EINVAL, f"gemm_skinny: x is [{m}, {k}] but w is [{k2}, {n}]")
    if not 1 <= m <= _SKINNY_MAX_M:
        raise LoopfuseError(_lib.LF_EINVAL, f"gemm_skinny: M = {m} outside 1..{_SKINNY_MAX_M}")
    sms = _sm_count(x.device)
    need = skinny_workspace_bytes(m, n, k, sms)
    if workspace is None:
        key = x.device.index
        workspace = _skinny_ws.get(key)
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(max(need, 1 << 20), dtype=torch.uint8, device=x.device)
            _skinny_ws[key] = workspace
    if workspace.numel() < need:
        raise LoopfuseError(_lib.LF_EINVAL, f"gemm_skinny: workspace of {workspace.numel()} bytes, "
                                            f"need {need}")
    if out is None:
        out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    _check(out, "out")
    _lib.call("lf_gemm_skinny", x.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k,
              workspace.data_ptr(), workspace.numel(), sms, _stream())
    return out


# -- log probabilities --------------------------------------------------------------------------------
class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor          # [T] fp32: ln p of the given token
    entropy: torch.Tensor          # [T] fp32: -sum p ln p
    top_ids: torch.Tensor          # [T, k] int64: the k most likely tokens, ties to the lowest id
    top_logprobs: torch.Tensor     # [T, k] fp32


_LOGIT_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_TOP_LOGPROBS = 32


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Log probability of ``tokens [T]`` (int64 or int32) under ``softmax(logits [T, V])``, each
    row's entropy and its ``top_k`` (at most 32) most likely tokens, in one pass over the logits.

    ``logits`` is bf16, fp16 or fp32, rows contiguous (their stride is free).  A negative token
    means none was given: its logprob is 0.  A token >= V gives NaN and is reported by
    ``lf_device_status``.  -inf logits have no probability; a row of nothing else has logprob -inf and
    entropy 0; a row with a NaN or +inf has NaN probabilities and entropy."""
    dev, k = logits.device, int(top_k)
    code = _LOGIT_TYPES.get(logits.dtype)
    if not logits.is_cuda or tokens.device != dev:
        raise LoopfuseError(_lib.LF_EINVAL, "token_logprobs: logits and tokens must be on one CUDA device")
    if code is None or logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise LoopfuseError(_lib.LF_EINVAL, "token_logprobs: logits must be bf16, fp16 or fp32 [T, V] "
                                            "with contiguous rows")
    T, V = logits.shape
    wide = tokens.dtype is torch.int64
    if not (wide or tokens.dtype is torch.int32) or tokens.shape != (T,) or not tokens.is_contiguous():
        raise LoopfuseError(_lib.LF_EINVAL, f"token_logprobs: tokens must be contiguous int64 or int32 [{T}]")
    if not 0 <= k <= min(MAX_TOP_LOGPROBS, V):
        raise LoopfuseError(_lib.LF_EINVAL, f"token_logprobs: top_k = {k} outside 0..{min(MAX_TOP_LOGPROBS, V)}")
    logprob = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    top_ids = torch.empty(T, k, dtype=torch.int64, device=dev)
    top = torch.empty(T, k, dtype=torch.float32, device=dev)
    if T:
        launch("lf_token_logprobs", dev, logits.data_ptr(), code, logits.stride(0), tokens.data_ptr(), wide,
               T, V, k, logprob.data_ptr(), entropy.data_ptr(), top_ids.data_ptr(), top.data_ptr())
    return TokenLogprobs(logprob, entropy, top_ids, top)


# -- low-rank adapters ----------------------------------------------------------------------------
LORA_RANKS = (16, 32, 64, 128)
MAX_ADAPTERS = 4096


@dataclass
class LoraPlan:
    """A batch's rows sorted by adapter (``lora_plan``); used by every ``lora_add`` of the batch."""
    buffer: torch.Tensor
    sessions: int
    total_tokens: int
    num_adapters: int


def lora_plan(adapter_ids: torch.Tensor, cu_tokens: torch.Tensor, total_tokens: int,
              num_adapters: int) -> LoraPlan:
    """Sort a batch's rows by adapter on the device, once for all its projections.

    ``adapter_ids [N]`` int32 on the GPU: the adapter of each session (-1: none); ``cu_tokens
    [N + 1]``: session ``i`` owns rows ``cu_tokens[i] .. cu_tokens[i + 1]``, ``total_tokens`` in
    all.  Ids outside ``[-1, num_adapters)`` count as none; they, and offsets that are not rising
    from 0 to ``total_tokens`` (nothing is written then), are reported by ``lf_device_status``."""
    i32, dev = torch.int32, adapter_ids.device
    if not (adapter_ids.is_cuda and adapter_ids.dtype is i32 and cu_tokens.dtype is i32 and
            cu_tokens.device == dev and adapter_ids.is_contiguous() and cu_tokens.is_contiguous()):
        raise LoopfuseError(_lib.LF_EINVAL, "lora_plan: adapter_ids and cu_tokens must be contiguous int32 "
                                            "tensors on one CUDA device")
    n = adapter_ids.numel()
    if adapter_ids.shape != (n,) or cu_tokens.shape != (n + 1,):
        raise LoopfuseError(_lib.LF_EINVAL, "lora_plan: adapter_ids must be [N], cu_tokens [N + 1]")
    total, adapters = int(total_tokens), int(num_adapters)
    size = _plan_bytes(n, total, adapters)
    buf = torch.empty(size, dtype=torch.uint8, device=dev)
    launch("lf_lora_plan", dev, adapter_ids.data_ptr(), cu_tokens.data_ptr(), n, total, adapters,
           buf.data_ptr(), size)
    return LoraPlan(buf, n, total, adapters)


@lru_cache(maxsize=4096)
def _plan_bytes(n: int, total: int, adapters: int) -> int:
    size = _lib.c_size_t(0)
    _lib.call("lf_lora_plan_size", n, total, adapters, _lib.ctypes.byref(size))
    return int(size.value)


@lru_cache(maxsize=4096)
def _lora_workspace_bytes(n: int, total: int, adapters: int, inputs: int, outputs: int, rank: int, sms: int) -> int:
    need = _lib.c_size_t(0)
    _lib.call("lf_lora_workspace_size", n, total, adapters, inputs, outputs, rank, sms, _lib.ctypes.byref(need))
    return int(need.value)


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: LoraPlan,
             scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] + scale[i] * (x[t] @ a[i]) @ b[i]``, ``i`` the adapter of token ``t``'s session.

    ``y [T, N]`` and ``x [T, K]`` bf16 rows (contiguous, row stride a multiple of 8), ``a
    [adapters, K, R]``, ``b [adapters, R, N]`` bf16, ``scale [adapters]`` fp32 (None: 1); R is 16,
    32, 64 or 128 (pad with zeros), K and N multiples of 8.  In place on ``y`` unless ``out`` is
    given; rows without an adapter keep (or, with ``out``, are) ``y``'s."""
    res = y if out is None else out
    dev, bf16 = plan.buffer.device, torch.bfloat16
    if not (y.is_cuda and y.dtype is bf16 and x.dtype is bf16 and res.dtype is bf16 and a.dtype is bf16 and
            b.dtype is bf16 and y.device == dev and x.device == dev and res.device == dev and a.device == dev and
            b.device == dev and y.dim() == 2 and x.dim() == 2 and a.dim() == 3 and b.dim() == 3):
        raise LoopfuseError(_lib.LF_EINVAL, "lora_add: y, x, out [T, .], a and b [adapters, ., .] must be bf16 "
                                            "tensors on the plan's CUDA device")
    T, K = x.shape
    N, R, adapters = y.shape[1], a.shape[2], plan.num_adapters
    if T != plan.total_tokens or y.shape[0] != T or res.shape != y.shape or a.shape != (adapters, K, R) or \
            b.shape != (adapters, R, N):
        raise LoopfuseError(_lib.LF_EINVAL, f"lora_add: y {tuple(y.shape)}, x {tuple(x.shape)}, "
                                            f"a {tuple(a.shape)}, b {tuple(b.shape)} and a plan of "
                                            f"{plan.total_tokens} tokens, {adapters} adapters do not match")
    if not (a.is_contiguous() and b.is_contiguous()):
        raise LoopfuseError(_lib.LF_EINVAL, "lora_add: a and b must be contiguous")
    sy, sx, so = y.stride(0), x.stride(0), res.stride(0)
    if T <= 1:
        sy, sx, so = N, K, N
    if y.stride(1) != 1 or x.stride(1) != 1 or res.stride(1) != 1 or (sy | sx | so) % 8 or sy < N or sx < K or so < N:
        raise LoopfuseError(_lib.LF_EINVAL, "lora_add: rows must be contiguous, their stride a multiple of 8")
    if R not in LORA_RANKS:
        raise LoopfuseError(_lib.LF_EINVAL, f"lora_add: rank {R} is not one of {LORA_RANKS} (pad with zeros)")
    if scale is not None and (scale.device != dev or scale.dtype is not torch.float32 or
                              scale.shape != (adapters,) or not scale.is_contiguous()):
        raise LoopfuseError(_lib.LF_EINVAL, "lora_add: scale must be fp32 [adapters] on y's device")
    if T == 0:
        return res
    sms = sm_count(dev.index)
    need = _lora_workspace_bytes(plan.sessions, T, adapters, K, N, R, sms)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    launch("lf_lora_add", dev, y.data_ptr(), sy, x.data_ptr(), sx, a.data_ptr(), b.data_ptr(),
           scale.data_ptr() if scale is not None else None, plan.buffer.data_ptr(), plan.sessions, T,
           adapters, K, N, R, res.data_ptr(), so, ws.data_ptr() if need else None, need, sms)
    return res
