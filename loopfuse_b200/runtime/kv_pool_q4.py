"""The paged KV pool with its K/V held in 4 bits (4.5 with their scales).

``QuantKVPool`` has the API of :class:`KVPool` and its page bookkeeping (allocation, fork, free,
dedup, block tables are the same device kernels on the same metadata); only the data differ.  New
K/V come in as bf16 and are quantised as they are stored; ``read`` gives the values the codes stand
for, rounded to bf16.  A page of one KV head is one block of ``18 * D`` bytes (format in
``include/loopfuse_b200.h``), so that the same memory holds 3.55 times the tokens.  ``attend_decode``
reads the 4-bit pages as they are; ``attend_prefill`` expands the batch's pages to bf16 first, into
a buffer that lives as long as the forward that asked for it.

The reference's pool (``runtime/kv_pool.py:28-235``) holds 16-bit tensors only.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from .. import _lib
from .. import attention as att
from .._lib import LF_PAGE_SIZE, LoopfuseError
from .kv_pool import KVPool, KVState


class QuantKVPool(KVPool):
    def __init__(self, num_layers: int, num_heads: int, head_dim: int, max_seq_len: int,
                 max_slots: int = 8, dtype: torch.dtype = torch.bfloat16, device: str = "cuda",
                 num_kv_heads: Optional[int] = None, num_pages: Optional[int] = None):
        if dtype != torch.bfloat16:
            raise LoopfuseError(_lib.LF_EINVAL, f"QuantKVPool takes bf16 K/V, got {dtype}")
        if head_dim not in (64, 128):
            raise LoopfuseError(_lib.LF_EINVAL, f"QuantKVPool needs head_dim 64 or 128, got {head_dim}")
        super().__init__(num_layers, num_heads, head_dim, max_seq_len, max_slots=max_slots,
                         dtype=dtype, device=device, num_kv_heads=num_kv_heads, num_pages=num_pages)

    @classmethod
    def from_config(cls, kv_config: dict, device: str = "cuda", max_slots: int = 8,
                    num_pages: Optional[int] = None) -> "QuantKVPool":
        dtype = kv_config.get("dtype", "bf16")
        if dtype != "bf16":
            raise LoopfuseError(_lib.LF_EINVAL, f"QuantKVPool takes bf16 K/V, got {dtype}")
        return cls(num_layers=kv_config["num_layers"], num_heads=kv_config["num_heads"],
                   head_dim=kv_config["head_dim"], max_seq_len=kv_config["max_seq_len"],
                   device=device, max_slots=max_slots, num_kv_heads=kv_config.get("num_kv_heads"),
                   num_pages=num_pages)

    # -- storage ----------------------------------------------------------------------------------
    def _alloc_storage(self) -> None:
        self.pages = torch.zeros((self.num_layers, self.num_pages, self.num_kv_heads,
                                  18 * self.head_dim), dtype=torch.uint8, device=self.device)

    def _storage_bytes(self) -> int:
        return self.pages.numel()

    def layer_pages(self, layer: int):
        raise LoopfuseError(_lib.LF_EINVAL, "a 4-bit pool has no bf16 pages: use layer_pages_q4 with "
                                            "paged_decode_q4, or attend_decode / attend_prefill")

    def layer_pages_q4(self, layer: int) -> torch.Tensor:
        """``[P, Hkv, 18 * D]`` view of one layer's pages (K and V together)."""
        return self.pages[layer]

    # -- writing ----------------------------------------------------------------------------------
    def _quantise(self, q_ptr, k_ptr, v_ptr, q_token, s_layer, s_token, s_head, ids, start, cu, n,
                  total, layer, layers, rope, q_out, stream) -> None:
        cos, sin = rope if rope is not None else (None, None)
        with torch.cuda.device(self.device):
            self._call("lf_q4_append", q_ptr, k_ptr, v_ptr, q_token, s_layer, s_token, s_head,
                       self._table.data_ptr(), self.max_slots, self.max_pages_per_seq,
                       ids.data_ptr(), start.data_ptr(), cu.data_ptr(), n, total,
                       cos.data_ptr() if cos is not None else None,
                       sin.data_ptr() if sin is not None else None,
                       cos.shape[0] if cos is not None else 0,
                       q_out.data_ptr() if q_out is not None else None,
                       self.pages[layer].data_ptr(), self.num_pages, layers,
                       q_out.shape[1] if q_out is not None else 0, self.num_kv_heads, self.head_dim,
                       self._ctrl.data_ptr() + 4 * _lib.LF_CTRL_STATUS, self._stream(stream))
        self._bytes_written += layers * total * self.num_kv_heads * self.head_dim * 9 // 8

    def _write_kv(self, ids, start, cu, n, total, keys, values, s_layer, s_token, s_head, layer,
                  layers, stream) -> None:
        self._quantise(None, keys.data_ptr(), values.data_ptr(), 0, s_layer, s_token, s_head, ids,
                       start, cu, n, total, layer, layers, None, None, stream)

    def _write_qkv(self, ids, start, cu, total, layer, qkv, q_out, rope, stream) -> None:
        Hq, D, elem = q_out.shape[1], self.head_dim, qkv.element_size()
        row = qkv.stride(0) if total > 1 else qkv.shape[1]
        base = qkv.data_ptr()
        self._quantise(base, base + Hq * D * elem, base + (Hq + self.num_kv_heads) * D * elem, row, 0,
                       row, D, ids, start, cu, ids.numel(), total, layer, 1, rope, q_out, stream)

    def _fork_data(self, src: int, ids: torch.Tensor, n: int, prefix_len: int) -> None:
        self._call("lf_q4_fork", self._meta_ref(), src, ids.data_ptr(), n, prefix_len,
                   self.pages.data_ptr(), self.num_layers, self.num_kv_heads, self.head_dim,
                   self._stream())

    # -- reading ----------------------------------------------------------------------------------
    def read(self, state: KVState, layer: int, seq_start: int = 0,
             seq_end: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One layer's values, ``[Hkv, seq_range, D]`` bf16; zeros past the session's length."""
        seq_end = seq_end or state.current_len
        count = max(0, seq_end - seq_start)
        if seq_start < 0 or seq_start + count > self.max_pages_per_seq * LF_PAGE_SIZE or \
                not 0 <= layer < self.num_layers:
            raise LoopfuseError(_lib.LF_EINVAL, "read: bad range")
        table, lens = self.block_table([state])
        held = -(-state.current_len // LF_PAGE_SIZE)
        kp, vp, _ = att.expand_pages_q4(self.pages[layer], table, lens, held)
        out = []
        for pages in (kp, vp):
            x = pages.transpose(0, 1).reshape(self.num_kv_heads, -1, self.head_dim)
            got = torch.zeros((self.num_kv_heads, count, self.head_dim), dtype=self.dtype,
                              device=self.device)
            part = x[:, seq_start:seq_start + count]
            got[:, :part.shape[1]] = part
            out.append(got)
        return out[0], out[1]

    # -- attention --------------------------------------------------------------------------------
    def decode_workspace(self, n: int, num_q_heads: int, width: int,
                         num_prefix_pages: int = 0) -> Tuple[int, int]:
        return 0, att.decode_q4_workspace_bytes(n, num_q_heads, self.num_kv_heads, self.head_dim, width,
                                                num_prefix_pages)

    def attend_decode(self, q: torch.Tensor, layer: int, table: torch.Tensor, lens: torch.Tensor,
                      num_prefix_pages: int = 0, pages_per_split: Optional[int] = None,
                      workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        # the decode cuts the pages itself: no split size
        return att.paged_decode_q4(q, self.pages[layer], table, lens,
                                   num_prefix_pages=num_prefix_pages, workspace=workspace)

    def prefill_buffers(self, lengths: Sequence[int], num_prefix_pages: int = 0):
        total = num_prefix_pages + sum(max(0, -(-int(n) // LF_PAGE_SIZE) - num_prefix_pages)
                                       for n in lengths)
        shape = (total, self.num_kv_heads, LF_PAGE_SIZE, self.head_dim)
        return (torch.empty(shape, dtype=self.dtype, device=self.device),
                torch.empty(shape, dtype=self.dtype, device=self.device), num_prefix_pages)

    def attend_prefill(self, q: torch.Tensor, layer: int, table: torch.Tensor, cu: torch.Tensor,
                       lens: torch.Tensor, max_new: int, buffers) -> torch.Tensor:
        k, v, n_prefix = buffers
        k, v, dense = att.expand_pages_q4(self.pages[layer], table, lens, k.shape[0],
                                          num_prefix_pages=n_prefix, out=(k, v))
        return att.prefill_paged(q, k, v, dense, cu, lens, max_new)
