"""What the log-probability and adapter calls refuse, before any launch."""
import ctypes

import pytest
import torch

from loopfuse_b200 import _lib
from loopfuse_b200 import model_ops as mo
from loopfuse_b200._lib import LoopfuseError

P = 1 << 20                                   # an aligned stand-in address, never touched


@pytest.mark.parametrize("change,words", [
    (dict(dtype=3), b"dtype"), (dict(top_k=33), b"top_k"), (dict(top_k=-1), b"top_k"), (dict(vocab=4, top_k=5), b"top_k"),
    (dict(vocab=0), b"vocab"), (dict(rows=-1), b"rows"), (dict(row_stride=9), b"overlap"), (dict(logits=None), b"null"),
    (dict(logits=P + 1), b"unaligned"), (dict(top_ids=None), b"null"), (dict(entropy=None), b"null"),
])
def test_logprobs_arguments(change, words):
    a = dict(logits=P, dtype=0, row_stride=100, tokens=P, tokens_64bit=1, rows=4, vocab=100, top_k=5, logprob=P,
             entropy=P, top_ids=P, top_logprobs=P, stream=None)
    a.update(change)
    lib = _lib.lib()
    assert lib.lf_token_logprobs(*a.values()) == _lib.LF_EINVAL
    assert words in lib.lf_last_error()


@pytest.mark.parametrize("change,words", [
    (dict(rank=8), b"rank"), (dict(rank=48), b"rank"), (dict(inputs=60), b"multiples of 8"), (dict(outputs=0), b"multiples of 8"),
    (dict(y=P + 2), b"aligned"), (dict(x_stride=65), b"aligned"), (dict(y_stride=64), b"overlap"), (dict(plan=None), b"null"),
    (dict(workspace_bytes=8, rank=64), b"workspace"), (dict(workspace=None, rank=64), b"null"), (dict(num_adapters=0), b"adapters"), (dict(num_adapters=4097), b"adapters"),
    (dict(total_tokens=-1), b"negative"), (dict(out=P, out_stride=136), b"in place"), (dict(total_tokens=1 << 30), b"too many"),
])
def test_lora_arguments(change, words):
    a = dict(y=P, y_stride=128, x=P, x_stride=64, a=P, b=P, scale=None, plan=P, n=2, total_tokens=4, num_adapters=2,
             inputs=64, outputs=128, rank=16, out=P + 4096, out_stride=128, workspace=P, workspace_bytes=1 << 30,
             sm_count=148, stream=None)
    a.update(change)
    lib = _lib.lib()
    assert lib.lf_lora_add(*a.values()) == _lib.LF_EINVAL
    assert words in lib.lf_last_error()


def test_plan_arguments_and_sizes():
    lib = _lib.lib()
    n = ctypes.c_size_t(0)
    _lib.call("lf_lora_plan_size", 3, 130, 5, ctypes.byref(n))
    assert n.value == 4 * (4 + 4 * (3 + 3) + 130 + 3)              # ceil(130 / 64) + min(3, 6) tiles
    assert lib.lf_lora_plan_size(0, 5, 1, ctypes.byref(n)) == _lib.LF_EINVAL
    assert lib.lf_lora_plan(P, P, 3, 130, 5, P, 16, None) == _lib.LF_EINVAL
    assert lib.lf_lora_plan(P, P, 3, 130, 5, P + 4, 1 << 20, None) == _lib.LF_EINVAL
    assert lib.lf_lora_plan(None, P, 3, 130, 5, P, 1 << 20, None) == _lib.LF_EINVAL
    _lib.call("lf_lora_workspace_size", 1, 1, 1, 4096, 6144, 16, 148, ctypes.byref(n))
    assert n.value == 0                                             # one launch of clusters
    _lib.call("lf_lora_workspace_size", 1, 1, 1, 4096, 28672, 16, 148, ctypes.byref(n))
    assert n.value % (16 * 4) == 0 and n.value >= 16 * 4


def test_tensors_off_the_gpu_or_of_other_types():
    x = torch.zeros(2, 8)
    with pytest.raises(LoopfuseError, match="CUDA"):
        mo.token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(LoopfuseError, match="CUDA"):
        mo.lora_plan(torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), 2, 1)
    plan = mo.LoraPlan(torch.zeros(8, dtype=torch.uint8), 1, 2, 1)
    with pytest.raises(LoopfuseError, match="lora_add"):
        mo.lora_add(x.bfloat16(), x.bfloat16(), torch.zeros(1, 8, 16).bfloat16(), torch.zeros(1, 16, 8).bfloat16(), plan)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x = torch.zeros(4, 64, device="cuda")
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (dict(tokens=tok[:3]), dict(tokens=tok.short()), dict(top_k=33), dict(top_k=65), dict(logits=x.double()),
                dict(logits=x[0]), dict(logits=x.t()[:4]), dict(tokens=tok.cpu())):
        a = dict(logits=x, tokens=tok, top_k=2)
        a.update(bad)
        with pytest.raises(LoopfuseError):
            mo.token_logprobs(**a)
    y, xb = x.bfloat16(), torch.zeros(4, 32, device="cuda").bfloat16()
    a, b = torch.zeros(2, 32, 16, device="cuda").bfloat16(), torch.zeros(2, 16, 64, device="cuda").bfloat16()
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    plan = mo.lora_plan(ids, cu, 4, 2)
    mo.lora_add(y, xb, a, b, plan)
    for bad in (dict(x=xb[:3]), dict(y=y.float()), dict(a=a[:1]), dict(b=b[:, :8]), dict(a=a.transpose(1, 2)),
                dict(scale=torch.ones(3, device="cuda")), dict(scale=torch.ones(2, device="cuda").bfloat16()),
                dict(out=y[:2]), dict(a=torch.zeros(2, 32, 24, device="cuda").bfloat16(),
                                      b=torch.zeros(2, 24, 64, device="cuda").bfloat16()),
                dict(y=torch.zeros(4, 65, device="cuda").bfloat16()[:, :64])):
        args = dict(y=y, x=xb, a=a, b=b, plan=plan)
        args.update(bad)
        with pytest.raises(LoopfuseError):
            mo.lora_add(**args)
    for bad in ((ids.long(), cu), (ids, cu[:1]), (ids, cu.long())):
        with pytest.raises(LoopfuseError):
            mo.lora_plan(*bad, 4, 2)
