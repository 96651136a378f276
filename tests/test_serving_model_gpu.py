"""The 4-bit cache, the adapters and the log probabilities together, as the models use them."""
import pytest
import torch
import torch.nn.functional as F

from loopfuse_b200.agent_loop import AgentLoop, AgentLoopConfig
from loopfuse_b200.gpt2 import GPT2Config, GPT2Model
from loopfuse_b200.llama import GraphedDecode, LlamaConfig, LlamaShaped, LoraAdapters
from loopfuse_b200.runtime import KVPool, QuantKVPool
from oracle import attention as ora
from oracle import q4

pytestmark = pytest.mark.gpu

SMALL = LlamaConfig(d_model=256, layers=2, q_heads=4, kv_heads=2, head_dim=128, ffn=512, vocab=1000)


def new_pool(kind=QuantKVPool, slots=24, cfg=SMALL):
    return kind(num_layers=cfg.layers, num_heads=cfg.q_heads, num_kv_heads=cfg.kv_heads,
                head_dim=cfg.head_dim, max_seq_len=512, max_slots=slots, dtype=torch.bfloat16)


def reference_logits(m, tokens, held, ad=None, which=-1):
    """fp32 over one whole sequence, attending to the K/V values that the pool holds; the residual
    stream, the queries and everything dense are this function's own.  Also the K and V that it would
    have stored, per layer."""
    c, T = m.cfg, tokens.numel()
    x = m.embed[tokens.cuda()].float().cpu()
    ang = torch.arange(T).float()[:, None] * m.inv_freq.cpu()[None, :]
    cos, sin = ang.cos()[:, None, :], ang.sin()[:, None, :]

    def rms(v, w):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + c.eps) * w.float().cpu()

    def rope(v):
        h = v.shape[-1] // 2
        return torch.cat([v[..., :h] * cos - v[..., h:] * sin, v[..., h:] * cos + v[..., :h] * sin], -1)

    def proj(v, w, l, name):
        y = v @ w.float().cpu()
        if ad is not None and which >= 0:
            a, b = (t[which].float().cpu() for t in ad.weights[l][name])
            y = y + float(ad.scale[which]) * (v @ a) @ b
        return y

    nq, nk = c.q_heads * c.head_dim, c.kv_heads * c.head_dim
    stored = []
    for l in range(c.layers):
        qkv = proj(rms(x, m.attn_norm[l]), m.wqkv[l], l, "qkv")
        q = rope(qkv[:, :nq].view(T, c.q_heads, c.head_dim))
        stored.append((rope(qkv[:, nq:nq + nk].view(T, c.kv_heads, c.head_dim)),
                       qkv[:, nq + nk:].view(T, c.kv_heads, c.head_dim)))
        k, v = held[l]
        o, _ = ora.prefill(q.permute(1, 0, 2)[None], k[None, :, :T].float().cpu(), v[None, :, :T].float().cpu())
        x = x + proj(o[0].permute(1, 0, 2).reshape(T, nq), m.wo[l], l, "o")
        gu = proj(rms(x, m.ffn_norm[l]), m.w13[l], l, "gate_up")
        x = x + proj(F.silu(gu[:, :c.ffn]) * gu[:, c.ffn:], m.w2[l], l, "down")
    return rms(x, m.final_norm) @ m.lm_head.float().cpu(), stored


def test_model_with_4bit_cache_adapters_and_scores_matches_fp32():
    m = LlamaShaped(SMALL, seed=1, std=0.05)
    ad = LoraAdapters(SMALL, 3, 16, seed=2, std=0.05)
    ad.scale.copy_(torch.tensor([1.0, 0.5, 2.0]))
    pool = new_pool()
    g = torch.Generator().manual_seed(0)
    ids, lens = [1, -1, 0], [40, 23, 17]
    toks = [torch.randint(0, SMALL.vocab, (n + 2,), generator=g) for n in lens]
    ss = [pool.allocate_slot() for _ in lens]
    sc = m.score(torch.cat([t[:n] for t, n in zip(toks, lens)]).cuda(), pool, ss, lens, adapters=ad,
                 adapter_ids=ids, top_k=5, rows=32)
    steps = []
    for i in range(2):                                        # teacher-forced decode, sessions together
        steps.append(m.forward(torch.stack([t[n + i] for t, n in zip(toks, lens)]).cuda(), pool, ss, [1, 1, 1],
                               return_logits=True, adapters=ad, adapter_ids=ids).cpu())
    at = 0
    for s, t, n, a in zip(ss, toks, lens, ids):
        held = [pool.read(s, l) for l in range(SMALL.layers)]
        ref, stored = reference_logits(m, t, held, ad, a)
        for l, (k, v) in enumerate(stored):
            for x, got in ((k, held[l][0]), (v, held[l][1])):
                _, step, _ = q4.quantise(x)
                err = (got.float().cpu().transpose(0, 1) - x).abs()
                # half a step of the held code, and the model's own bf16 roundings upstream of it
                assert bool((err <= step.repeat_interleave(64, -1) * 0.6 + 0.05 * x.abs().amax()).all())
        for i in range(2):
            got, want = steps[i][ss.index(s)], ref[n + i]
            assert F.cosine_similarity(got, want, dim=0).item() > 0.999
            assert (got - want).abs().max().item() < 0.1 * want.abs().max().item()
        logp = torch.log_softmax(ref[:n].double(), -1)
        lp = sc.logprob[at:at + n].double().cpu()
        want = logp[:-1].gather(1, t[1:n, None])[:, 0]
        # both sides' logits differ by the model's bf16 roundings: the tolerance of the logits above
        tol = 0.1 * ref.abs().max().item()
        assert (lp[:-1] - want).abs().max().item() < tol and lp[-1].item() == 0.0
        ent = -(logp.exp() * logp).sum(-1)
        assert (sc.entropy[at:at + n].double().cpu() - ent).abs().max().item() < tol
        top = sc.top_logprobs[at:at + n].double().cpu()
        assert (top - logp.topk(5)[0]).abs().max().item() < tol
        at += n


def test_scores_of_a_batch_are_the_logits_of_its_positions():
    """score() against log_softmax of the same hidden states' logits: only the LM head's chunking and
    the kernel's fp32 arithmetic lie between."""
    m = LlamaShaped(SMALL, seed=3)
    g = torch.Generator().manual_seed(1)
    toks = torch.randint(0, SMALL.vocab, (50,), generator=g).cuda()
    a, b = new_pool(), new_pool()
    sc = m.score(toks, a, [a.alloc(), a.alloc()], [30, 20], top_k=3, rows=16)
    x = m._trunk(toks, b, [b.alloc(), b.alloc()], [30, 20], 0, None, None, None)
    logits = (m._norm_in(x, None, m.final_norm) @ m.lm_head).double()
    logp = torch.log_softmax(logits, -1)
    nxt = toks[1:]
    want = logp[:-1].gather(1, nxt[:, None])[:, 0]
    tol = 2 * 2 ** -8 * logits.abs().max().item() + 1e-5    # one bf16 rounding of the logits on each side
    got = sc.logprob[:-1].double()
    keep = torch.ones(49, dtype=torch.bool, device="cuda")
    keep[29] = False                                        # the first session's last token
    assert (got - want)[keep].abs().max().item() <= tol
    assert sc.logprob[29].item() == 0.0 and sc.logprob[49].item() == 0.0
    tok, lp = m.forward(toks[:1], a, [a.alloc()], [1], top_logprobs=4)
    assert lp.top_ids[0, 0].item() == tok[0].item() and lp.logprob[0].item() == lp.top_logprobs[0, 0].item()


def test_graphed_decode_with_4bit_cache_and_adapters_matches_eager():
    m = LlamaShaped(SMALL, seed=4)
    ad = LoraAdapters(SMALL, 2, 32, seed=5, std=0.05)
    runs = []
    for graphed in (False, True):
        pool = new_pool()
        root = pool.alloc()
        g = torch.Generator().manual_seed(5)
        m.forward(torch.randint(0, SMALL.vocab, (64,), generator=g).cuda(), pool, [root], [64])
        ss = pool.fork(root, 64, n=12)
        lens = [int(x) for x in torch.randint(1, 40, (12,), generator=g)]
        m.forward(torch.randint(0, SMALL.vocab, (sum(lens),), generator=g).cuda(), pool, ss, lens, n_prefix_pages=4)
        pad = pool.pad_session(root, 64)
        gd = GraphedDecode(m, pool, pad, n_prefix_pages=4, adapters=ad) if graphed else None
        outs = []
        for it in range(5):
            batch = ss[:12 - 2 * it]
            ids = [(i + it) % 3 - 1 for i in range(len(batch))]     # changes from step to step
            tb = [int(x) for x in torch.randint(0, SMALL.vocab, (len(batch),), generator=g)]
            if graphed:
                outs.append(gd.step(batch, tb, adapter_ids=ids)[:len(batch)].tolist())
                gd.raise_if_failed()
            else:
                outs.append(m.forward(torch.tensor(tb, device="cuda"), pool, batch, [1] * len(batch),
                                      n_prefix_pages=4, adapters=ad, adapter_ids=ids).tolist())
        runs.append((outs, pool.snapshot(), [pool.read(s, 1)[0].float() for s in ss]))
    (oe, se, ke), (og, sg, kg) = runs
    assert se == sg
    fe, fg = [t for o in oe for t in o], [t for o in og for t in o]
    assert sum(a == b for a, b in zip(fe, fg)) >= 0.9 * len(fe)
    for a, b in zip(ke, kg):          # GEMMs of another batch size may move a value across one step
        assert (a - b).abs().max().item() <= 0.75 * max(1e-3, a.abs().max().item())
        assert (a - b).abs().mean().item() <= 0.02 * a.abs().max().item()


def test_an_adapter_changes_its_own_sessions_only():
    m = LlamaShaped(SMALL, seed=6)
    ad = LoraAdapters(SMALL, 2, 16, seed=7, std=0.2)
    g = torch.Generator().manual_seed(2)
    toks = torch.randint(0, SMALL.vocab, (40,), generator=g).cuda()
    out = []
    for ids in ([-1, -1], [-1, 1], None):
        pool = new_pool(KVPool)
        kw = {} if ids is None else dict(adapters=ad, adapter_ids=ids)
        out.append(m.forward(toks, pool, [pool.alloc(), pool.alloc()], [20, 20], return_logits=True, **kw))
    assert torch.equal(out[0], out[2]) and torch.equal(out[1][0], out[0][0])
    assert not torch.equal(out[1][1], out[0][1])
    ad.set(0, 0, "down", torch.ones(SMALL.ffn, 4), torch.ones(4, SMALL.d_model), scale=0.25)
    wa, wb = ad.weights[0]["down"]
    assert (wa[0, :, :4] == 1).all() and not wa[0, :, 4:].any() and (wb[0, :4] == 1).all() and not wb[0, 4:].any()


def test_agent_loop_and_gpt2_run_over_a_4bit_cache():
    m = LlamaShaped(SMALL, seed=2)
    cfg = AgentLoopConfig(sessions=6, steps=2, prefix_tokens=64, question_tokens=16, decode_tokens=3, tool_ms=5.0,
                          tool_len_mean=10, tool_len_cap=20, spec_tokens=4, seed=3, kv_bits=4)
    loop = AgentLoop(m, cfg)
    st = loop.run(profile_ops=True)
    assert isinstance(loop.pool, QuantKVPool) and st.steps_done == cfg.sessions * cfg.steps
    snap = loop.pool.snapshot()
    assert len(snap["free_queue"]) == loop.pool.num_pages - cfg.prefix_tokens // 16 - 1
    model = GPT2Model(GPT2Config(layers=2, vocab=500), seed=1)
    g = torch.Generator().manual_seed(3)
    toks = torch.randint(0, 500, (70,), generator=g)
    logits = []
    for bits in (16, 4):
        pool = model.new_pool(16, 2, kv_bits=bits)
        s = pool.allocate_slot()
        model.prefill(toks[:66], s)
        logits.append(torch.stack([model.decode(toks[66 + i:67 + i], s)[0] for i in range(4)]))
        assert pool.status() == 0
    assert F.cosine_similarity(logits[0], logits[1], dim=-1).min().item() > 0.99
