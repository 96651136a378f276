"""What the 4-bit cache's calls refuse, on the host and before any launch."""
import ctypes

import pytest
import torch

from loopfuse_b200 import _lib
from loopfuse_b200 import attention as att
from loopfuse_b200._lib import LoopfuseError
from loopfuse_b200.runtime import QuantKVPool
from oracle import q4

P = 1 << 20                                   # an aligned stand-in address, never touched


def test_oracle_round_trip_is_within_half_a_step():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(2, 128, generator=gen).bfloat16()
    pages = torch.zeros(1, 1, 18 * 128, dtype=torch.uint8)
    q4.write_token(pages, 0, 0, 3, x[0], x[1])
    k, v, _ = q4.unpack(pages)
    for got, want in ((k[0, 0, 3], x[0]), (v[0, 0, 3], x[1])):
        n, s, low = q4.quantise(want)
        assert torch.equal(got, q4.value(n, s, low))
        # half a step, and at the top the scale's rounding (2^-8 relative) times 15 steps
        assert ((got - want.double()).abs() <= s.repeat_interleave(64) * (0.5 + 15 * 2 ** -8)).all()


def test_every_code_has_its_own_place():
    for D in (64, 128):
        (ka, ku), (va, vu) = q4.places(D)
        seen = {(int(a), int(u)) for at, up in ((ka, ku), (va, vu)) for a, u in zip(at.flatten(), up.flatten())}
        assert len(seen) == 2 * 16 * D and max(a for a, _ in seen) == 16 * D - 1


def test_tensors_off_the_gpu_and_of_other_types_are_refused():
    pages = torch.zeros(2, 1, 18 * 64, dtype=torch.uint8)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(LoopfuseError, match="CUDA"):
        att.paged_decode_q4(torch.zeros(1, 1, 64).bfloat16(), pages, i32[None], i32)
    with pytest.raises(LoopfuseError, match="CUDA"):
        att.append_qkv_q4(torch.zeros(1, 192).bfloat16(), pages, i32[None], i32, torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(LoopfuseError, match="CUDA"):
        att.expand_pages_q4(pages, i32[None], i32, 1)


def test_a_workspace_with_gaps_is_refused():
    """Its bytes are counted as if they followed one another: the partials would go past its end."""
    pages, i32 = torch.zeros(2, 1, 18 * 64, dtype=torch.uint8), torch.zeros(1, dtype=torch.int32)
    for ws in (torch.zeros(1 << 16, dtype=torch.uint8)[::2], torch.zeros(64, 64)[:, :32]):
        with pytest.raises(LoopfuseError, match="workspace"):
            att.paged_decode_q4(torch.zeros(1, 1, 64).bfloat16(), pages, i32[None], i32, workspace=ws)


@pytest.mark.parametrize("change,words", [
    (dict(head_dim=96), b"head_dim"), (dict(num_q_heads=6), b"1, 2, 4 or 8"), (dict(num_q_heads=5), b"multiple"),
    (dict(q=P + 2), b"aligned"), (dict(pages=P + 8), b"aligned"), (dict(q=None), b"null"),
    (dict(num_prefix_pages=5), b"num_prefix_pages"), (dict(num_prefix_pages=-1), b"num_prefix_pages"),
    (dict(workspace_bytes=16, max_pages=600), b"workspace"), (dict(workspace=None, max_pages=600), b"null"), (dict(max_pages=1 << 27), b"max_pages"),
    (dict(num_seqs=1 << 29), b"too many"),
    (dict(num_seqs=-1), b"negative"), (dict(max_pages=0), b"max_pages"),
])
def test_decode_arguments(change, words):
    a = dict(q=P, pages=P, block_table=P, seq_lens=P, num_prefix_pages=0, o=P, lse=None, workspace=P,
             workspace_bytes=1 << 30, num_seqs=2, num_q_heads=4, num_kv_heads=2, head_dim=128, num_pages=8,
             max_pages=4, scale=1.0, sm_count=148, stream=None)
    a.update(change)
    lib = _lib.lib()
    assert lib.lf_q4_decode_fwd(*a.values()) == _lib.LF_EINVAL
    assert words in lib.lf_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(head_dim=32), b"head_dim"), (dict(k=None), b"null"), (dict(k=P + 2), b"aligned"),
    (dict(stride_token=100), b"aligned"), (dict(num_q_heads=2, q=None), b"q_out"), (dict(rope_cos=P), b"cos and sin"),
    (dict(rope_cos=P, rope_sin=P), b"rope"), (dict(n=9), b"rows"), (dict(total_tokens=-1), b"negative"),
    (dict(num_layers=0), b"shape"),
])
def test_append_arguments(change, words):
    a = dict(q=None, k=P, v=P, q_stride_token=0, stride_layer=0, stride_token=256, stride_head=128, block_table=P,
             table_rows=4, max_pages=4, seq_ids=None, start_pos=P, cu_tokens=P, n=2, total_tokens=2, rope_cos=None,
             rope_sin=None, rope_rows=0, q_out=None, pages=P, num_pages=8, num_layers=1, num_q_heads=0,
             num_kv_heads=2, head_dim=128, status=None, stream=None)
    a.update(change)
    lib = _lib.lib()
    assert lib.lf_q4_append(*a.values()) == _lib.LF_EINVAL
    assert words in lib.lf_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(head_dim=32), b"head_dim"), (dict(k_out=None), b"null"), (dict(k_out=P + 16), b"32-byte"),
    (dict(num_prefix_pages=9), b"shape"), (dict(num_seqs=-1), b"negative"), (dict(out_pages=-1), b"null"),
])
def test_expand_arguments(change, words):
    a = dict(pages=P, block_table=P, seq_lens=P, num_prefix_pages=0, k_out=P, v_out=P, out_table=P, num_seqs=2,
             num_kv_heads=2, head_dim=128, num_pages=8, max_pages=4, out_pages=8, stream=None)
    a.update(change)
    lib = _lib.lib()
    assert lib.lf_q4_expand(*a.values()) == _lib.LF_EINVAL
    assert words in lib.lf_last_error()


def test_empty_calls_do_nothing():
    lib = _lib.lib()
    assert lib.lf_q4_expand(None, None, None, 0, None, None, None, 0, 1, 64, 1, 1, 0, None) == _lib.LF_OK
    assert lib.lf_q4_decode_fwd(None, None, None, None, 0, None, None, None, 0, 0, 4, 2, 128, 1, 1, 1.0, 148,
                                None) == _lib.LF_OK


def test_fork_and_pool_arguments():
    lib = _lib.lib()
    m = _lib.PoolMeta()
    assert lib.lf_q4_fork(ctypes.byref(m), 0, None, 1, 5, P, 1, 1, 96, None) == _lib.LF_EINVAL
    assert lib.lf_q4_fork(ctypes.byref(m), 0, None, 1, 5, P + 4, 1, 1, 64, None) == _lib.LF_EINVAL
    with pytest.raises(LoopfuseError, match="bf16"):
        QuantKVPool(1, 1, 64, 64, dtype=torch.float16)
    with pytest.raises(LoopfuseError, match="head_dim"):
        QuantKVPool(1, 1, 96, 64)
    with pytest.raises(LoopfuseError, match="GPU memory"):
        QuantKVPool(1, 1, 64, 64, device="cpu")


def test_a_config_of_another_type_is_refused_as_by_the_constructor(monkeypatch):
    cfg = {"num_layers": 1, "num_heads": 2, "head_dim": 64, "max_seq_len": 64}
    for dtype in ("fp16", "fp32", "int8"):
        with pytest.raises(LoopfuseError, match="bf16"):
            QuantKVPool.from_config(dict(cfg, dtype=dtype))
    made = []
    monkeypatch.setattr(QuantKVPool, "__init__", lambda self, *a, **kw: made.append(kw.get("dtype", torch.bfloat16)))
    for more in ({}, {"dtype": "bf16"}):
        QuantKVPool.from_config(dict(cfg, **more))
    assert made == [torch.bfloat16] * 2


def test_workspace():
    """(148 x 12 ranges (16 of 64 dims) + N Hkv items) x G partials, prefix chunks x N Hq partials, a
    span per item."""
    assert att.decode_q4_workspace_bytes(3, 4, 2, 64, 513, 0, 148) == (2368 + 6) * 2 * (256 + 8) + 6 * 8
    assert att.decode_q4_workspace_bytes(3, 4, 2, 128, 513, 0, 148) == (1776 + 6) * 2 * (512 + 8) + 6 * 8
    # few items whose table allows 64 pages a CTA of their cluster (8, 4 or 2 of the 444 resident): none
    assert att.decode_q4_workspace_bytes(3, 4, 2, 128, 512, 0, 148) == 0
    assert att.decode_q4_workspace_bytes(50, 4, 2, 128, 256, 0, 148) == 0 != att.decode_q4_workspace_bytes(50, 4, 2, 128, 257, 0, 148)
    assert att.decode_q4_workspace_bytes(111, 4, 2, 128, 128, 0, 148) == 0 != att.decode_q4_workspace_bytes(112, 4, 2, 128, 128, 0, 148)
    # a prefix of 16 pages or less is one chunk; no own pages, no ranges
    assert att.decode_q4_workspace_bytes(3, 4, 2, 128, 10, 10, 148) == 3 * 4 * (512 + 8) + 6 * 8
