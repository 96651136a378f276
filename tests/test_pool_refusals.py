"""What both pools refuse, before their sessions grow or a kernel is launched."""
import pytest
import torch

from loopfuse_b200._lib import LoopfuseError
from loopfuse_b200.runtime import KVPool, QuantKVPool


def bare(kind):
    """A pool without storage, on the CPU, which records what it would store."""
    p = kind.__new__(kind)
    p.num_layers, p.num_heads, p.num_kv_heads, p.head_dim = 1, 2, 1, 64
    p.dtype, p.device, p.max_seq_len = torch.bfloat16, torch.device("cpu"), 64
    p.stored = []
    p._write_qkv = lambda *a: p.stored.append(a)
    return p


@pytest.mark.parametrize("kind", [KVPool, QuantKVPool])
def test_write_qkv_takes_rotation_tables_of_one_shape_only(kind):
    """Positions are checked against the rows of cos: with fewer rows of sin they would be read past its end."""
    p = bare(kind)
    index = (torch.zeros(1, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32), 3)
    qkv, q = torch.zeros(3, 4 * 64).bfloat16(), torch.zeros(3, 2, 64).bfloat16()
    cos = torch.zeros(10, 32)
    for rope in ((cos, cos[:4]), (cos[:4], cos), (cos,), (cos, cos, cos), (cos[:0], cos[:0])):
        with pytest.raises(LoopfuseError, match="rope"):
            p.write_qkv(None, None, 0, qkv, q, None, rope=rope, index=index)
    assert p.stored == []
    p.write_qkv(None, None, 0, qkv, q, None, rope=(cos, cos.clone()), index=index)
    assert len(p.stored) == 1


def state():
    from loopfuse_b200.runtime.kv_pool import KVState
    return KVState(0, None)


@pytest.mark.parametrize("kind", [KVPool, QuantKVPool])
def test_append_refuses_rows_before_the_session_grows(kind):
    p = bare(kind)
    p._reserve = lambda *a: pytest.fail("reserved")
    good = torch.zeros(1, 3, 1, 64).bfloat16()
    odd = torch.zeros(1, 3, 1, 128).bfloat16()[..., ::2]
    wide = torch.zeros(1, 3, 2, 64).bfloat16()
    for k, v in ((good.float(), good), (good, good.float()), (odd, odd), (wide, wide), (good, good[:, :2]),
                 (good.expand(2, 3, 1, 64), good.expand(2, 3, 1, 64))):
        with pytest.raises(LoopfuseError):
            p.append([state()], [k], [v])


def test_a_4bit_append_refuses_unaligned_rows_before_the_session_grows():
    p = bare(QuantKVPool)
    p._reserve = lambda *a: pytest.fail("reserved")
    k = torch.zeros(1, 3, 1, 68).bfloat16()[..., :64]           # 136 bytes from row to row
    with pytest.raises(LoopfuseError, match="aligned"):
        p.append([state()], [k], [k])
    k = torch.zeros(1, 3, 1, 72).bfloat16()[..., 4:68]          # begins 8 bytes off
    with pytest.raises(LoopfuseError, match="aligned"):
        p.append([state()], [k], [k])
