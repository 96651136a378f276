"""What the Llama-shaped model's serving calls refuse, before the pool is touched: a batch that is refused
leaves its sessions as they were."""
import pytest
import torch

from loopfuse_b200 import model_ops as mo
from loopfuse_b200._lib import LoopfuseError
from loopfuse_b200.llama import GraphedDecode, LlamaConfig, LlamaShaped, LoraAdapters
from loopfuse_b200.runtime.kv_pool import KVState

TINY = LlamaConfig(d_model=32, layers=2, q_heads=2, kv_heads=1, head_dim=64, ffn=48, vocab=40)
OTHER = LlamaConfig(d_model=32, layers=1, q_heads=2, kv_heads=1, head_dim=64, ffn=48, vocab=40)


class Touched(Exception):
    pass


class Pool:
    """Stands in for a pool: the first call a batch makes of it ends the test."""
    max_pages_per_seq = 4

    def reserve(self, *args):
        raise Touched


@pytest.fixture(scope="module")
def model():
    return LlamaShaped(TINY, device="cpu")


def batch(pool):
    return [KVState(0, pool), KVState(1, pool)], torch.tensor([3, 4, 5])


GOOD = LoraAdapters(TINY, 3, 16, device="cpu")
WRONG = LoraAdapters(OTHER, 3, 16, device="cpu")
BOTH = [dict(adapters=GOOD), dict(adapters=GOOD, adapter_ids=[0]), dict(adapters=GOOD, adapter_ids=[0, 1, 2]),
        dict(adapter_ids=[0, 1]), dict(adapters=GOOD, adapter_ids=[0, 3]), dict(adapters=GOOD, adapter_ids=[-2, 0]),
        dict(adapters=WRONG, adapter_ids=[0, 1]), dict(n_prefix_pages=5), dict(n_prefix_pages=-1),
        dict(tokens=torch.tensor([1, 2])), dict(counts=[3]), dict(counts=[4, -1])]


@pytest.mark.parametrize("change", BOTH + [dict(top_logprobs=k) for k in (-1, 33, 41)])
def test_forward_refuses_before_it_advances_a_session(model, change):
    pool = Pool()
    states, toks = batch(pool)
    a = dict(tokens=toks, pool=pool, states=states, counts=[2, 1])
    a.update(change)
    with pytest.raises(LoopfuseError):
        model.forward(**a)
    assert [s.current_len for s in states] == [0, 0]


@pytest.mark.parametrize("change", BOTH + [dict(top_k=-1), dict(top_k=33), dict(rows=0), dict(rows=-5)])
def test_score_refuses_before_it_advances_a_session(model, change):
    pool = Pool()
    states, toks = batch(pool)
    a = dict(tokens=toks, pool=pool, states=states, counts=[2, 1])
    a.update(change)
    with pytest.raises(LoopfuseError):
        model.score(**a)
    assert [s.current_len for s in states] == [0, 0]


def test_what_is_right_reaches_the_pool(model):
    pool = Pool()
    states, toks = batch(pool)
    for kw in ({}, dict(adapters=GOOD, adapter_ids=[-1, 2]), dict(n_prefix_pages=4)):
        for call in (lambda: model.forward(toks, pool, states, [2, 1], top_logprobs=32, **kw),
                     lambda: model.score(toks, pool, states, [2, 1], top_k=5, rows=1, **kw)):
            with pytest.raises(Touched):
                call()


def test_adapters_that_no_plan_can_hold_are_refused_when_made():
    for n in (0, -1, mo.MAX_ADAPTERS + 1):
        with pytest.raises(LoopfuseError):
            LoraAdapters(TINY, n, 16, device="cpu")


def test_graphed_decode_refuses_adapters_of_another_model_and_unknown_ids(model, monkeypatch):
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, pin_memory=False, **kw: zeros(*a, **kw))
    with pytest.raises(LoopfuseError):
        GraphedDecode(model, Pool(), None, adapters=WRONG)
    gd = GraphedDecode(model, Pool(), None, adapters=GOOD)
    states, _ = batch(gd.pool)
    for ids in ([0, 3], [-2, 0], [0]):
        with pytest.raises(LoopfuseError):
            gd.step(states, [1, 2], adapter_ids=ids)
    with pytest.raises(LoopfuseError):
        gd.step(states, [1])


@pytest.mark.gpu
def test_a_refused_batch_leaves_the_pool_as_it_was():
    from loopfuse_b200.runtime import QuantKVPool
    m = LlamaShaped(TINY)
    pool = QuantKVPool(num_layers=2, num_heads=2, num_kv_heads=1, head_dim=64, max_seq_len=64, max_slots=3)
    states = [pool.alloc(), pool.alloc()]
    toks = torch.tensor([3, 4, 5], device="cuda")
    good = LoraAdapters(TINY, 3, 16)
    first = m.forward(toks, pool, states, [2, 1], adapters=good, adapter_ids=[-1, 2])
    before, pages = pool.snapshot(), pool.pages.clone()
    for kw in (dict(adapters=good), dict(adapter_ids=[0, 0]), dict(top_logprobs=33), dict(n_prefix_pages=5)):
        with pytest.raises(LoopfuseError):
            m.forward(toks, pool, states, [2, 1], **kw)
    assert pool.snapshot() == before and torch.equal(pool.pages, pages)
    assert [s.current_len for s in states] == [2, 1] and first.shape == (2,)


def test_logits_and_alternatives_can_be_asked_for_together(model, monkeypatch):
    x = torch.randn(3, TINY.d_model, generator=torch.Generator().manual_seed(0)).bfloat16()
    monkeypatch.setattr(model, "fused_ops", False)
    monkeypatch.setattr(model, "_trunk", lambda *a: x.clone())
    monkeypatch.setattr(mo, "token_logprobs", lambda logits, tokens, top_k: ("logprobs", tokens, top_k))
    pool = Pool()
    states, toks = batch(pool)
    logits = model.forward(toks, pool, states, [2, 1], return_logits=True)
    chosen, lp = model.forward(toks, pool, states, [2, 1], top_logprobs=4)
    both = model.forward(toks, pool, states, [2, 1], return_logits=True, top_logprobs=4)
    assert torch.equal(both[0], logits) and torch.equal(chosen, logits.argmax(-1))
    assert both[1][0] == "logprobs" and torch.equal(both[1][1], chosen) and both[1][2] == 4
