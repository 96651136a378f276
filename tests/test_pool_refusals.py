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
