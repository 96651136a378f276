"""What is measured of the serving operators: attention over a cache held in 4 bits, log
probabilities of given tokens, and low-rank adapters of many requests.

``run`` computes an operator in its plain form (elementary torch operations in fp32), or, where
``own`` is true, makes the calls a user of the package makes.  The packed page format below is the
package's documented one: a page of one KV head holds 16 tokens as

  K codes   [token 16][c 4][group][word 2] 32-bit words of 8 dims,
  V codes   [token / 8][g 8][c 4][group][word 2][token % 2] 16-bit pieces of 4 dims,
  params    [token 16][K, V][group][scale, bias] bf16,

for ``head_dim / 64`` groups of 64 dims; a value is ``code * scale + bias``.
"""
import math

import torch

own = False

PAGE = 16
GROUP = 64


# -- the cases --------------------------------------------------------------------------------------
def listed():
    return [
        # One session's next token over a short context: launch latency is what counts.
        _decode("decode one session", 1, 777, 777, 0, 32, 8, 128),
        # The agent loop's batch: 64 sessions that share a 4096-token system prompt.
        _decode("decode shared prefix", 64, 4111, 5200, 4096, 32, 8, 128),
        # Sessions of every length, an empty one and a one-token one among them.
        _decode("decode ragged", 47, 0, 6007, 0, 32, 8, 128),
        # The long end: long contexts of many sessions, far larger than the caches on the chip.
        _decode("decode long", 64, 4096, 16384, 0, 32, 8, 128),
        # GPT-2-shaped heads (12 of 64, no sharing) over its position range.
        _decode("decode 64-wide heads", 96, 1, 1280, 0, 12, 12, 64),
        # One decode step's cache work: every session appends its token, then attends.
        dict(_decode("step", 256, 1, 1900, 0, 32, 8, 128), kind="step"),
        # A prefill batch's cache work: tool outputs appended, the context read back for prefill.
        _chunk("chunk", 32, 120, 2000, 32, 8, 128),
        # Per-step log probabilities of a decode batch over a Llama-3-sized vocabulary.
        _logprobs("logprobs decode", 64, 128256, 20, "bf16", 0.0),
        # One row with the most likely tokens, some of the vocabulary banned.
        _logprobs("logprobs one row", 1, 50257, 5, "fp32", 0.1),
        # Scoring a prompt: many positions, no alternatives asked for.
        _logprobs("logprobs scoring", 1501, 128256, 0, "bf16", 0.0),
        # A decode batch of sessions with their own adapters beside the QKV projection.
        _lora("adapters decode", 96, 1, 16, 4096, 6144, 16),
        # A prefill batch beside the gate|up projection, larger rank, uneven requests.
        _lora("adapters prefill", 24, 333, 7, 4096, 28672, 64),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["decode", "decode", "step", "chunk", "logprobs", "logprobs", "lora", "lora"])
    if kind in ("decode", "step", "chunk"):
        hq, hkv, d = rng.choice([(32, 8, 128), (12, 12, 64), (8, 8, 128), (16, 2, 128), (16, 8, 64),
                                 (32, 4, 64)])
        if kind == "chunk":
            return _nameless(_chunk("", log(1, 40), log(1, 200), log(16, 2500), hq, hkv, d))
        n, hi = log(1, 100), log(8, 12000)
        while n * hi > 600000:
            n = max(1, n // 2)
        prefix = 0
        if kind == "decode" and rng.random() < 0.3 and hi > 64:
            prefix = PAGE * rng.randint(1, hi // 32)
        lo = max(prefix, rng.choice([0, 1, hi // 2, hi]))
        return _nameless(dict(_decode("", n, lo, max(hi, lo), prefix, hq, hkv, d), kind=kind))
    if kind == "logprobs":
        v = rng.choice([128256, 50257, log(40, 130000), log(40, 130000)])
        t = min(log(1, 1400), 160000000 // v)
        return _nameless(_logprobs("", t, v, rng.choice([0, 1, 5, 20, 32]), rng.choice(["bf16", "fp32", "fp16"]),
                                   rng.choice([0.0, 0.0, 0.2])))
    per = rng.choice([1, 1, log(1, 300)])
    n = min(log(1, 256), max(1, 6000 // per))
    return _nameless(_lora("", n, per, log(1, 64), 8 * log(8, 1024), 8 * log(8, 2000), rng.choice([16, 32, 64])))


def _nameless(case):
    return {k: v for k, v in case.items() if k != "name"}


def _decode(name, n, lo, hi, prefix, hq, hkv, d):
    return {"name": name, "kind": "decode", "sessions": n, "shortest": lo, "longest": hi,
            "prefix": prefix, "q_heads": hq, "kv_heads": hkv, "head_dim": d}


def _chunk(name, n, new, context, hq, hkv, d):
    return {"name": name, "kind": "chunk", "sessions": n, "new": new, "context": context,
            "q_heads": hq, "kv_heads": hkv, "head_dim": d}


def _logprobs(name, t, v, k, dtype, banned):
    return {"name": name, "kind": "logprobs", "rows": t, "vocab": v, "top": k, "dtype": dtype,
            "banned": banned}


def _lora(name, n, per, adapters, k, nout, r):
    return {"name": name, "kind": "lora", "sessions": n, "tokens": per, "adapters": adapters,
            "inputs": k, "outputs": nout, "rank": r}


# -- sizes that prepare and work agree on: spread evenly, so that they need no seed ------------------
def _lengths(case):
    """Context length of every session, the newest token included."""
    n, lo, hi = case["sessions"], case["shortest"], case["longest"]
    least = 1 if case["kind"] == "step" else 0
    lens = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
    return [max(least, lens[(i * 37) % n] if math.gcd(37, n) == 1 else lens[i]) for i in range(n)]


def _chunk_sizes(case):
    """(tokens already held, new tokens) of every session: uneven around the case's figures."""
    n = case["sessions"]
    old = [case["context"] * (i % 5) // 2 for i in range(n)]
    new = [max(1, case["new"] * (1 + i % 3) // 2 + i % 2) for i in range(n)]
    return old, new


def _session_tokens(case):
    n, per = case["sessions"], case["tokens"]
    return [per if per == 1 else max(1, per * (2 + i % 5) // 4 + i % 3) for i in range(n)]


def _adapter_of(case):
    """Adapter of every session; every ninth session has none."""
    n = case["adapters"]
    return [-1 if i % 9 == 8 else (i * 7 + i // 5) % n for i in range(case["sessions"])]


# -- inputs -----------------------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _codes(x):
    """Codes, scales and biases of ``x [..., D]`` (fp32): groups of 64 dims."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    low = g.amin(-1, keepdim=True)
    span = g.amax(-1, keepdim=True) - low
    scale = (span / torch.full_like(span, 15.0)).bfloat16().float()
    n = ((g - low) / torch.where(scale > 0, scale, torch.ones_like(scale))).round().clamp(0, 15)
    n = torch.where(scale > 0, n, torch.zeros_like(n))
    return n, scale, low


def _pack(k, v):
    """``k, v [pages, heads, 16, D]`` fp32 -> packed pages ``[pages, heads, 18 * D]`` uint8."""
    p, h, _, d = k.shape
    ng = d // GROUP
    kn, ks, kb = _codes(k)
    vn, vs, vb = _codes(v)
    # dims of a K group: c 4, word 2, byte % 2, nibble, byte / 2
    kn = kn.to(torch.uint8).view(p, h, 16, ng, 4, 2, 2, 2, 2).permute(0, 1, 2, 4, 3, 5, 8, 6, 7)
    kb8 = (kn[..., 0] | (kn[..., 1] << 4)).reshape(p, h, 8 * d)
    # tokens of a page: half 2, c 4, parity 2; dims of a V group: g 8, word 2, byte 2, nibble 2
    vn = vn.to(torch.uint8).view(p, h, 2, 4, 2, ng, 8, 2, 2, 2).permute(0, 1, 2, 6, 3, 5, 7, 4, 8, 9)
    vb8 = (vn[..., 0] | (vn[..., 1] << 4)).reshape(p, h, 8 * d)
    par = torch.stack([torch.cat([ks, kb], -1), torch.cat([vs, vb], -1)], dim=3)   # [p,h,16,2,ng,2]
    par8 = par.bfloat16().contiguous().view(torch.uint8).reshape(p, h, 2 * d)
    return torch.cat([kb8, vb8, par8], dim=-1)


def _pages(gen, num, heads, d):
    """Pages of keys and values as a model writes them: keys with a few strong channels."""
    strong = 1.0 + 3.0 * (torch.rand(1, heads, 1, d, generator=gen, device="cuda") > 0.95).float()
    out = torch.empty((num, heads, 18 * d), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (heads * PAGE * d))
    for s in range(0, num, step):
        e = min(num, s + step)
        k = (_randn(gen, e - s, heads, PAGE, d) * strong).bfloat16().float()
        v = _randn(gen, e - s, heads, PAGE, d).bfloat16().float()
        out[s:e] = _pack(k, v)
    return out


def _table(gen, lens, prefix):
    """Block table over shuffled page ids; the first ``prefix`` tokens' pages are shared."""
    width = max(1, -(-max(lens) // PAGE))
    pre = prefix // PAGE
    held = [max(0, -(-x // PAGE) - pre) for x in lens]
    num = max(1, pre + sum(held))
    ids = torch.randperm(num, generator=gen, device="cuda").to(torch.int32)
    col = torch.arange(width, device="cuda")[None, :]
    first = torch.tensor([0] + held[:-1], device="cuda").cumsum(0)[:, None]
    at = torch.where(col < pre, col, pre + first + col - pre)
    used = col < torch.tensor([-(-x // PAGE) for x in lens], device="cuda")[:, None]
    table = torch.where(used, ids[at.clamp(0, num - 1)], torch.full_like(ids[:1], -1))
    if pre:                               # a shorter session still lists the shared pages
        table[:, :pre] = ids[:pre]
    return table.contiguous(), num


def _i32(xs):
    return torch.tensor(xs, dtype=torch.int32, device="cuda")


def _cu(counts):
    return _i32([0] + torch.tensor(counts).cumsum(0).tolist())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind in ("decode", "step", "chunk"):
        hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        if kind == "chunk":
            old, new = _chunk_sizes(case)
            lens, prefix = [a + b for a, b in zip(old, new)], 0
        else:
            lens, prefix = _lengths(case), case["prefix"]
            old, new = [x - 1 for x in lens], [1] * len(lens)
        s["table"], num = _table(gen, lens, prefix)
        s["pages"] = _pages(gen, num, hkv, d)
        s["lens"] = _i32(lens)
        if kind == "decode":
            s["q"] = _randn(gen, len(lens), hq, d).bfloat16()
        else:
            s["qkv"] = _randn(gen, sum(new), (hq + 2 * hkv) * d).bfloat16()
            s["start"], s["cu"] = _i32(old), _cu(new)
            s["total_pages"] = sum(-(-x // PAGE) for x in lens)
            pos = torch.arange(max(lens) + 1, device="cuda", dtype=torch.float64)[:, None]
            ang = pos * 500000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    elif kind == "logprobs":
        t, v = case["rows"], case["vocab"]
        dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
        x = _randn(gen, t, v).mul_(2.5)
        s["tokens"] = torch.randint(0, v, (t,), generator=gen, device="cuda")
        x.scatter_add_(1, s["tokens"][:, None], torch.full((t, 1), 9.0, device="cuda"))
        if case["banned"]:
            ban = torch.rand(t, v, generator=gen, device="cuda") < case["banned"]
            ban.scatter_(1, s["tokens"][:, None], False)
            x.masked_fill_(ban, -math.inf)
        s["logits"] = x.to(dtype)
    else:
        counts = _session_tokens(case)
        t, k, n, r, a = sum(counts), case["inputs"], case["outputs"], case["rank"], case["adapters"]
        s["x"] = _randn(gen, t, k).bfloat16()
        s["y"] = _randn(gen, t, n).bfloat16()
        s["a"] = (_randn(gen, a, k, r) * k ** -0.5).bfloat16()
        s["b"] = (_randn(gen, a, r, n) * r ** -0.5).bfloat16()
        s["scale"] = 0.5 + torch.rand(a, generator=gen, device="cuda")
        s["ids"], s["cu"], s["out"] = _i32(_adapter_of(case)), _cu(counts), torch.empty_like(s["y"])
    return s


# -- one pass -------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    if kind == "decode":
        k, v = _unpack(s["pages"][s["table"].long().clamp(min=0)])
        return _attend(s["q"], k, v, s["lens"])
    if kind in ("step", "chunk"):
        return _appended(s, kind)
    if kind == "logprobs":
        return _scored(s["logits"], s["tokens"], s["case"]["top"])
    return _adapted(s)


def _run_own(s, kind):
    from loopfuse_b200 import attention as att
    from loopfuse_b200 import model_ops as mo
    case = s["case"]
    if kind == "decode":
        return att.paged_decode_q4(s["q"], s["pages"], s["table"], s["lens"],
                                   num_prefix_pages=case["prefix"] // PAGE, return_lse=True)
    if kind in ("step", "chunk"):
        q = att.append_qkv_q4(s["qkv"], s["pages"], s["table"], s["start"], s["cu"],
                              case["q_heads"], rope=(s["cos"], s["sin"]))
        if kind == "step":
            return att.paged_decode_q4(q, s["pages"], s["table"], s["lens"], return_lse=True)
        k, v, _ = att.expand_pages_q4(s["pages"], s["table"], s["lens"], s["total_pages"])
        return q, k, v
    if kind == "logprobs":
        return tuple(mo.token_logprobs(s["logits"], s["tokens"], top_k=case["top"]))
    plan = mo.lora_plan(s["ids"], s["cu"], s["x"].shape[0], case["adapters"])
    return mo.lora_add(s["y"], s["x"], s["a"], s["b"], plan, scale=s["scale"], out=s["out"])


def _unpack(pages):
    """Packed pages ``[..., heads, 18 * D]`` -> fp32 values ``k, v [..., heads, 16, D]``."""
    lead, d = pages.shape[:-1], pages.shape[-1] // 18
    ng = d // GROUP
    flat = pages.reshape(-1, 18 * d)
    m = flat.shape[0]
    k8 = flat[:, :8 * d]
    kn = torch.stack([k8 & 15, k8 >> 4], -1).view(m, 16, 4, ng, 2, 2, 2, 2)
    kn = kn.permute(0, 1, 3, 2, 4, 6, 7, 5).reshape(m, 16, ng, GROUP).float()
    v8 = flat[:, 8 * d:16 * d]
    vn = torch.stack([v8 & 15, v8 >> 4], -1).view(m, 2, 8, 4, ng, 2, 2, 2, 2)
    vn = vn.permute(0, 1, 3, 6, 4, 2, 5, 7, 8).reshape(m, 16, ng, GROUP).float()
    par = flat[:, 16 * d:].contiguous().view(torch.bfloat16).view(m, 16, 2, ng, 2).float()
    k = kn * par[:, :, 0, :, 0:1] + par[:, :, 0, :, 1:2]
    v = vn * par[:, :, 1, :, 0:1] + par[:, :, 1, :, 1:2]
    return k.reshape(*lead, 16, d), v.reshape(*lead, 16, d)


def _attend(q, k, v, lens):
    """``k, v [N, W, heads, 16, D]``: softmax attention of ``q [N, Hq, D]`` over the first tokens."""
    n, hq, d = q.shape
    hkv = k.shape[2]
    k = k.transpose(1, 2).reshape(n, hkv, -1, d)
    v = v.transpose(1, 2).reshape(n, hkv, -1, d)
    seen = torch.arange(k.shape[2], device=q.device)[None, :] < lens[:, None]
    sc = torch.matmul(q.float().view(n, hkv, hq // hkv, d), k.transpose(2, 3)) * d ** -0.5
    sc = sc.masked_fill(~seen[:, None, None, :], -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = torch.log(total) + top
    return o.view(n, hq, d).bfloat16(), lse.view(n, hq)


def _rotated(x, cos, sin):
    half = x.shape[-1] // 2
    x1, x2 = x[..., :half], x[..., half:]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def _token_places(s):
    """Session, position and page of every new token."""
    t = torch.arange(s["qkv"].shape[0], device="cuda")
    sess = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    pos = s["start"].long()[sess] + t - s["cu"].long()[sess]
    return sess, pos


def _appended(s, kind):
    case = s["case"]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    sess, pos = _token_places(s)
    x = s["qkv"].float().view(-1, hq + 2 * hkv, d)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotated(x[:, :hq], cos, sin).bfloat16()
    kn, ks, kb = _codes(_rotated(x[:, hq:hq + hkv], cos, sin).bfloat16().float())
    vn, vs, vb = _codes(x[:, hq + hkv:])
    if kind == "step":
        k, v = _unpack(s["pages"][s["table"].long().clamp(min=0)])          # [N, W, heads, 16, D]
        k[sess, pos // PAGE, :, pos % PAGE] = (kn * ks + kb).view(-1, hkv, d)
        v[sess, pos // PAGE, :, pos % PAGE] = (vn * vs + vb).view(-1, hkv, d)
        return _attend(q, k, v, s["lens"])
    held = (s["lens"].long() + PAGE - 1) // PAGE
    first = held.cumsum(0) - held
    at = torch.arange(s["total_pages"], device="cuda")
    of = torch.searchsorted(held.cumsum(0), at, right=True)
    k, v = _unpack(s["pages"][s["table"].long()[of, at - first[of]]])       # [pages, heads, 16, D]
    k[first[sess] + pos // PAGE, :, pos % PAGE] = (kn * ks + kb).view(-1, hkv, d)
    v[first[sess] + pos // PAGE, :, pos % PAGE] = (vn * vs + vb).view(-1, hkv, d)
    row = (at - first[of])[:, None] * PAGE + torch.arange(PAGE, device="cuda")[None, :]
    keep = (row < s["lens"].long()[of][:, None])[:, None, :, None]
    return q, (k * keep).bfloat16(), (v * keep).bfloat16()


def _scored(logits, tokens, top):
    x = logits.float()
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    logp = d - torch.log(total)
    entropy = torch.log(total)[:, 0] - torch.where(e > 0, e * d, e).sum(-1) / total[:, 0]
    of_token = logp.gather(1, tokens[:, None])[:, 0]
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top] if top else \
        tokens.new_empty((x.shape[0], 0))
    return of_token, entropy, ids, logp.gather(1, ids)


def _adapted(s):
    case = s["case"]
    a, r = case["adapters"], case["rank"]
    t = torch.arange(s["x"].shape[0], device="cuda")
    of = s["ids"].long()[torch.searchsorted(s["cu"][1:].long(), t, right=True)]
    down = s["x"].float() @ s["a"].float().transpose(0, 1).reshape(-1, a * r)
    mine = (of[:, None] == torch.arange(a, device="cuda")[None, :]).float() * s["scale"][None, :]
    down = (down.view(-1, a, r) * mine[:, :, None]).view(-1, a * r)
    return (s["y"].float() + down @ s["b"].float().view(a * r, -1)).bfloat16()


# -- what one pass cannot do without --------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("decode", "step", "chunk"):
        hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        packed = hkv * d * 9 // 8                        # bytes of one token's keys and values
        if kind == "chunk":
            old, new = _chunk_sizes(case)
            t, held = sum(new), sum(old) + sum(new)
            return {"bytes": t * (2 * hq + 2 * hkv) * d * 2 + t * packed + sum(old) * packed +
                    held * hkv * d * 4, "flops": 6 * t * (hq + hkv) * d}
        lens, n, pre = _lengths(case), case["sessions"], case["prefix"]
        own_tokens = sum(max(0, x - pre) for x in lens) + min(pre, max(lens))
        moved = own_tokens * packed + n * hq * d * 4 + n * hq * 4
        if kind == "step":
            moved += n * 2 * hkv * d * 2                     # the new keys and values
        return {"bytes": moved, "flops": 4 * hq * d * sum(lens)}
    if kind == "logprobs":
        t, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": t * v * (4 if case["dtype"] == "fp32" else 2) + t * (16 + 12 * k),
                "flops": 4 * t * v}
    counts, of = _session_tokens(case), _adapter_of(case)
    t, k, n, r = sum(counts), case["inputs"], case["outputs"], case["rank"]
    mine = sum(c for c, a in zip(counts, of) if a >= 0)
    used = len({a for a in of if a >= 0})
    return {"bytes": mine * k * 2 + t * n * 4 + used * (k + n) * r * 2, "flops": 2 * mine * r * (k + n)}


# -- the same from the definitions, in 64 bits ----------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        return _exact_logprobs(s)
    if kind == "lora":
        out = s["y"].double()
        for i, a in enumerate(_adapter_of(case)):
            lo, hi = int(s["cu"][i]), int(s["cu"][i + 1])
            if a >= 0:
                low = s["x"][lo:hi].double() @ s["a"][a].double()
                out[lo:hi] += float(s["scale"][a]) * (low @ s["b"][a].double())
        return out
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    lens = s["lens"].tolist()
    q = s["q"].double() if kind == "decode" else torch.empty((s["qkv"].shape[0], hq, d),
                                                             dtype=torch.float64, device="cuda")
    outs, lses, ks, vs = [], [], [], []
    for i, length in enumerate(lens):
        pages = -(-length // PAGE)
        k, v = _exact_values(s["pages"][s["table"][i, :pages].long()], d)      # [tokens, heads, D]
        if kind != "decode":
            lo, hi = int(s["cu"][i]), int(s["cu"][i + 1])
            at = int(s["start"][i]) + torch.arange(hi - lo, device="cuda")
            x = s["qkv"][lo:hi].double().view(hi - lo, hq + 2 * hkv, d)
            turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None, :]
            z = torch.complex(x[:, :hq + hkv, :d // 2], x[:, :hq + hkv, d // 2:]) * turn
            x[:, :hq + hkv] = torch.cat([z.real, z.imag], -1)
            q[lo:hi] = x[:, :hq]
            k[at] = _exact_held(x[:, hq:hq + hkv].bfloat16())
            v[at] = _exact_held(x[:, hq + hkv:].bfloat16())
        if kind == "chunk":
            for held, got in ((ks, k), (vs, v)):
                got[length:] = 0.0
                held.append(got.view(pages, PAGE, hkv, d).transpose(1, 2))
            continue
        row = q[i].bfloat16().double().view(hkv, hq // hkv, d)
        sc = torch.einsum("hgd,thd->hgt", row, k[:length]) / math.sqrt(d)
        lse = torch.logsumexp(sc, -1)
        p = torch.exp(sc - lse[..., None])
        outs.append(torch.einsum("hgt,thd->hgd", p, v[:length]).reshape(hq, d))
        lses.append(lse.reshape(hq))
    if kind == "chunk":
        return q, torch.cat(ks), torch.cat(vs)
    return torch.stack(outs), torch.stack(lses)


def _exact_values(pages, d):
    """Values of packed pages ``[P, heads, 18 * D]`` as ``k, v [P * 16, heads, D]`` in 64 bits, each
    value's byte and nibble found by the format's formula."""
    p, heads = pages.shape[:2]
    ng = d // GROUP
    t = torch.arange(PAGE, device=pages.device)[:, None]
    x = torch.arange(d, device=pages.device)[None, :]
    grp, e = x // GROUP, x % 8
    bit = 4 * (e // 2) + 16 * (e % 2)
    k_at = t * (32 * ng) + (x % GROUP) // 16 * (8 * ng) + grp * 8 + (x % 16) // 8 * 4 + bit // 8
    k_up = (bit % 8).expand(PAGE, d)
    lane = (x % GROUP) // 8 * 4 + t % 8 // 2
    v_at = 8 * d + t // 8 * (256 * ng) + lane * (8 * ng) + grp * 8 + e // 4 * 4 + t % 2 * 2 + e % 4 // 2
    v_up = (4 * (e % 2)).expand(PAGE, d)
    par = pages[..., 16 * d:].contiguous().view(torch.bfloat16).double()      # [P, heads, 16*2*ng*2]
    out = []
    for which, (at, up) in enumerate(((k_at, k_up), (v_at, v_up))):
        n = (pages[..., at] >> up) & 15
        where = (t * 2 + which) * ng * 2 + grp * 2
        val = n.double() * par[..., where] + par[..., where + 1]
        out.append(val.permute(0, 2, 1, 3).reshape(p * PAGE, heads, d))
    return out


def _exact_held(x):
    """What 4 bits hold of ``x [tokens, heads, D]``, in 64 bits."""
    g = x.double().unflatten(-1, (-1, GROUP))
    low = g.min(-1, keepdim=True).values
    scale = ((g.max(-1, keepdim=True).values - low) / 15).bfloat16().double()
    n = torch.where(scale > 0, ((g - low) / scale).round().clamp(0, 15), torch.zeros_like(g))
    return (n * scale + low).flatten(-2)


def _exact_logprobs(s):
    top = s["case"]["top"]
    got = []
    for x, tok in zip(s["logits"].split(256), s["tokens"].split(256)):
        x = x.double()
        logp = torch.log_softmax(x, -1)
        entropy = -torch.special.xlogy(logp.exp(), logp.exp()).sum(-1)
        ids = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :top]
        got.append((logp.gather(1, tok[:, None])[:, 0], entropy, ids, logp.gather(1, ids)))
    return tuple(torch.cat(g) for g in zip(*got))
