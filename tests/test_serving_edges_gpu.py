"""Empty and smallest calls of the serving operators, two calls at once, and a step of all of them
captured into one graph and replayed on changed inputs."""
import pytest
import torch

from loopfuse_b200 import attention as att
from loopfuse_b200 import model_ops as mo
from loopfuse_b200._lib import LoopfuseError
from oracle import q4
from test_q4_gpu import drain_status, random_pages, table_for

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(*x):
    return torch.tensor(x, dtype=I32, device="cuda")


def test_calls_without_sessions_or_tokens():
    pages = torch.zeros(4, 2, 18 * 128, dtype=torch.uint8, device="cuda")
    none = torch.empty(0, dtype=I32, device="cuda")
    for width in (0, 3):
        table = torch.empty(0, width, dtype=I32, device="cuda")
        o, lse = att.paged_decode_q4(torch.empty(0, 8, 128, dtype=torch.bfloat16, device="cuda"), pages, table, none,
                                     return_lse=True)
        assert o.shape == (0, 8, 128) and lse.shape == (0, 8)
    qkv = torch.empty(0, 12 * 128, dtype=torch.bfloat16, device="cuda")
    q = att.append_qkv_q4(qkv, pages, torch.empty(0, 3, dtype=I32, device="cuda"), none, ints(0), 8)
    assert q.shape == (0, 8, 128)
    k, v, t = att.expand_pages_q4(pages, torch.empty(0, 3, dtype=I32, device="cuda"), none, 0)
    assert k.shape == v.shape == (0, 2, 16, 128) and t.shape == (0, 3)
    out = mo.token_logprobs(torch.empty(0, 9, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top_k=2)
    assert out.logprob.shape == out.entropy.shape == (0,) and out.top_ids.shape == (0, 2)
    plan = mo.lora_plan(none, ints(0), 0, 3)
    y = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    a = torch.zeros(3, 32, 16, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(3, 16, 64, dtype=torch.bfloat16, device="cuda")
    assert mo.lora_add(y, torch.empty(0, 32, dtype=torch.bfloat16, device="cuda"), a, b, plan) is y
    assert (pages == 0).all() and drain_status() == []


def test_a_session_without_pages_in_the_table():
    """Sessions, but none of them holds a token."""
    pages = torch.full((2, 2, 18 * 64), 255, dtype=torch.uint8, device="cuda")    # scales are NaN
    table = torch.full((3, 2), -1, dtype=I32, device="cuda")
    o, lse = att.paged_decode_q4(torch.randn(3, 4, 64, device="cuda").bfloat16(), pages, table, ints(0, 0, 0), return_lse=True)
    assert (o == 0).all() and torch.isneginf(lse).all()
    k, v, t = att.expand_pages_q4(pages, table, ints(0, 0, 0), 1)
    assert (t == -1).all() and drain_status() == []


def test_one_value_rows_of_log_probabilities():
    x = torch.tensor([[3.0], [float("-inf")]], device="cuda")
    out = mo.token_logprobs(x, torch.tensor([0, -1], device="cuda"), top_k=1)
    assert out.logprob.tolist() == [0.0, 0.0] and out.entropy.tolist() == [0.0, 0.0]
    assert out.top_ids.tolist() == [[0], [0]] and out.top_logprobs.tolist() == [[0.0], [float("-inf")]]


def batch(seed, N=5, Hq=8, Hkv=2, D=128, V=1000, n_adapters=3):
    gen = torch.Generator().manual_seed(seed)
    lens = [1 + int(torch.randint(0, 300, (1,), generator=gen)) for _ in range(N)]
    table, P = table_for(lens, 0, gen, width=20)
    d = {"pages": random_pages(gen, P, Hkv, D), "table": table, "lens": torch.tensor(lens, dtype=I32),
         "start": torch.tensor(lens, dtype=I32) - 1, "cu": torch.arange(N + 1, dtype=I32),
         "x": torch.randn(N, 256, generator=gen).bfloat16(), "qkv": torch.randn(N, (Hq + 2 * Hkv) * D, generator=gen).bfloat16(),
         "ids": torch.randint(-1, n_adapters, (N,), generator=gen).to(I32),
         "a": (torch.randn(n_adapters, 256, 16, generator=gen) / 16).bfloat16(),
         "b": torch.randn(n_adapters, 16, (Hq + 2 * Hkv) * D, generator=gen).bfloat16(),
         "w": (torch.randn(Hq * D, V, generator=gen) / 32).bfloat16(),
         "tok": torch.randint(0, V, (N,), generator=gen)}
    return {k: v.cuda() for k, v in d.items()}


def step(d, Hq=8):
    """Adapters on the projection, quantised append, attention, log probabilities."""
    plan = mo.lora_plan(d["ids"], d["cu"], d["x"].shape[0], d["a"].shape[0])
    y = mo.lora_add(d["qkv"], d["x"], d["a"], d["b"], plan, out=torch.empty_like(d["qkv"]))
    q = att.append_qkv_q4(y, d["pages"], d["table"], d["start"], d["cu"], Hq)
    o = att.paged_decode_q4(q, d["pages"], d["table"], d["lens"])
    lp = mo.token_logprobs(o.flatten(1) @ d["w"], d["tok"], top_k=3)
    return y, q, o, lp


def check_step(d, got):
    """Each operator against its 64-bit form, from the operands that the one before it gave."""
    y, q, o, lp = got
    want = d["qkv"].double()
    own = [int(i) for i in d["ids"]]
    for t, i in enumerate(own):
        if i >= 0:
            low = d["x"][t].double() @ d["a"][i].double()
            want[t] += low @ d["b"][i].double()
            # h rounded once to bf16, the sum once: half a step (2^-8) of each, and fp32 sums
            tol = 2.0 ** -8 * (low.abs() @ d["b"][i].double().abs()) + 2.0 ** -8 * want[t].abs() + 1e-4
            assert bool(((y[t].double() - want[t]).abs() <= tol).all())
        else:
            assert torch.equal(y[t], d["qkv"][t])
    ro, _, to, _ = q4.decode(q.cpu(), d["pages"].cpu(), d["table"].cpu(), d["lens"].tolist(), q.shape[2] ** -0.5)
    assert bool(((o.double().cpu() - ro).abs() <= to).all())
    logits = (o.flatten(1) @ d["w"]).double()
    p = torch.log_softmax(logits, -1)
    assert torch.allclose(lp.logprob.double(), p.gather(1, d["tok"][:, None])[:, 0], rtol=0, atol=1e-5)
    assert torch.equal(lp.top_ids[:, 0], logits.argmax(-1))


def test_a_step_of_all_operators_and_its_graph():
    d = batch(1)
    check_step(d, step(d))                                 # (appended: the pages now hold the new token)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(d)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(d)
    for seed in (2, 3):
        other = batch(seed)
        other["pages"] = other["pages"][:d["pages"].shape[0]]
        for k in ("qkv", "x", "ids", "a", "b", "w", "tok"):
            d[k].copy_(other[k])
        g.replay()
        torch.cuda.synchronize()
        check_step(d, got)
    assert drain_status() == []


def test_two_steps_at_once_on_two_streams():
    ds = [batch(11), batch(12)]
    alone = [step({k: v.clone() for k, v in d.items()}) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    for _ in range(20):
        got = []
        for s, d in zip(streams, ds):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(d))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
            assert torch.equal(a[3].top_ids, b[3].top_ids) and torch.equal(a[3].logprob, b[3].logprob)
    assert drain_status() == []


def test_score_refuses_a_batch_without_tokens():
    from loopfuse_b200.llama import LlamaConfig, LlamaShaped
    from loopfuse_b200.runtime import QuantKVPool
    cfg = LlamaConfig(layers=1, d_model=256, q_heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=128)
    model = LlamaShaped(cfg)
    pool = QuantKVPool(num_layers=1, num_heads=4, num_kv_heads=2, head_dim=64, max_seq_len=64, max_slots=2,
                       dtype=torch.bfloat16, device="cuda")
    state = pool.alloc()
    for states, counts in (([], []), ([state], [0])):
        with pytest.raises(LoopfuseError):
            model.score(torch.empty(0, dtype=torch.int64), pool, states, counts)
    out = model.score(torch.tensor([5]), pool, [state], [1], top_k=1)
    assert out.logprob.tolist() == [0.0] and out.top_ids.shape == (1, 1) and state.current_len == 1
