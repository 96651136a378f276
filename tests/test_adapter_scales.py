"""The scale of a low-rank adapter belongs to the projection it was set with."""
import pytest
import torch

from loopfuse_b200 import llama
from loopfuse_b200 import model_ops as mo
from loopfuse_b200.llama import LlamaConfig, LoraAdapters

TINY = LlamaConfig(d_model=64, layers=2, q_heads=2, kv_heads=1, head_dim=64, ffn=96, vocab=40)


def parts(name, rank, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    i, o = LoraAdapters.shapes_of(TINY)[name]
    return ((torch.randn(i, rank, generator=g) / 8).bfloat16().to(device),
            torch.randn(rank, o, generator=g).bfloat16().to(device))


def loaded(device="cpu"):
    ad = LoraAdapters(TINY, 3, 16, device=device)
    ad.set(1, 0, "qkv", *parts("qkv", 8, 1, device), scale=0.25)
    ad.set(1, 0, "o", *parts("o", 16, 2, device))
    ad.set(1, 1, "qkv", *parts("qkv", 4, 3, device), scale=3.0)
    ad.set(2, 0, "qkv", *parts("qkv", 16, 4, device), scale=0.5)
    return ad


def test_each_projection_keeps_its_scale(monkeypatch):
    used = []
    monkeypatch.setattr(mo, "lora_plan", lambda *a: None)
    monkeypatch.setattr(mo, "lora_add", lambda y, x, a, b, plan, scale: used.append(scale.tolist()) or y)
    ad = loaded()
    ad.scale[2] = 2.0                                  # of the whole adapter, besides
    batch = llama._Adapted(ad, None, None, 0)
    for layer, name in ((0, "qkv"), (0, "o"), (1, "qkv"), (1, "down")):
        batch.add(torch.zeros(1), torch.zeros(1), layer, name)
    assert used == [[1.0, 0.25, 1.0], [1.0, 1.0, 2.0], [1.0, 3.0, 2.0], [1.0, 1.0, 2.0]]


@pytest.mark.gpu
def test_each_projection_adds_its_own_scale():
    ad = loaded("cuda")
    ids = torch.tensor([1, -1, 2], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 3, 4, 9], dtype=torch.int32, device="cuda")
    which = [1, 1, 1, -1, 2, 2, 2, 2, 2]
    batch = llama._Adapted(ad, ids, cu, 9)
    for layer, name, scale in ((0, "qkv", {1: 0.25, 2: 0.5}), (0, "o", {1: 1.0, 2: 1.0}), (1, "qkv", {1: 3.0, 2: 1.0})):
        i, o = ad.shapes[name]
        g = torch.Generator().manual_seed(layer + i)
        x, y = torch.randn(9, i, generator=g).bfloat16().cuda(), torch.randn(9, o, generator=g).bfloat16().cuda()
        got = batch.add(y.clone(), x, layer, name)
        a, b = ad.weights[layer][name]
        for t, w in enumerate(which):
            if w < 0:
                assert torch.equal(got[t], y[t])
                continue
            low = scale[w] * (x[t].double() @ a[w].double())
            want = y[t].double() + low @ b[w].double()
            # h rounded once to bf16, the sum once: half a step (2^-8) of each; fp32 sums of 64 to 128 terms
            tol = 2.0 ** -8 * (low.abs() @ b[w].double().abs()) + 2.0 ** -8 * want.abs() + 1e-4
            assert bool(((got[t].double() - want).abs() <= tol).all()), (layer, name, t)
