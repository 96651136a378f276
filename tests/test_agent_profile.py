"""Bytes that the agent loop's per-kernel profile counts for the K/V cache."""
import types

import pytest

from loopfuse_b200.agent_loop import AgentLoop
from loopfuse_b200.llama import LlamaConfig

CFG = LlamaConfig(d_model=64, layers=3, q_heads=4, kv_heads=2, head_dim=64, ffn=96, vocab=40)
VALUES = 2 * 2 * 64 * 3                                        # K and V of a token, all layers


def loop(bits):
    return types.SimpleNamespace(cfg=types.SimpleNamespace(kv_bits=bits), model=types.SimpleNamespace(cfg=CFG))


@pytest.mark.parametrize("bits,phase,per_value", [
    (16, "decode", 2), (16, "prefill", 2), (4, "decode", 9 / 16),
    (4, "prefill", 9 / 16 + 2 + 2),                            # codes read, bf16 pages written and read again
])
def test_cache_bytes_of_a_token_attended_to(bits, phase, per_value):
    assert AgentLoop._kv_bytes(loop(bits), phase) == VALUES * per_value


@pytest.mark.parametrize("bits,per_value", [(16, 2), (4, 9 / 16)])
def test_bytes_of_the_append(bits, per_value):
    nq, nkv, T = 4 * 64, 2 * 64, 7
    want = 3 * T * ((nq + 2 * nkv) * 2 + nq * 2 + 2 * nkv * per_value)
    assert AgentLoop._op_work(loop(bits), T, 1, 0.0, 0.0)["qkv_rope_append"] == (0.0, want)
