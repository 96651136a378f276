"""The serving kernels begin while the stream's last kernel still runs and wait for it themselves: what
comes before them is read whole, what comes after them does not overtake them, and they can be
captured behind copies and joined streams."""
import pytest
import torch

from loopfuse_b200 import attention as att
from loopfuse_b200 import model_ops as mo

pytestmark = pytest.mark.gpu
HQ, HKV, D, N = 8, 2, 128, 12


class Step:
    """One of everything on fixed buffers: append, decode (with and without a shared prefix), expansion,
    adapters, log probabilities."""

    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens = torch.tensor([200 + 31 * i for i in range(N)], dtype=torch.int32, device="cuda")
        width = 40
        table = 4 + torch.arange(N * (width - 4), device="cuda").view(N, width - 4)
        self.table = torch.cat([torch.arange(4, device="cuda").expand(N, 4), table], 1).int().contiguous()
        self.pages = torch.randint(0, 256, (4 + N * (width - 4), HKV, 18 * D), generator=g, device="cuda").to(torch.uint8)
        s = 0.2 + 0.3 * torch.rand(self.pages.shape[:2] + (16, 2, 2), generator=g, device="cuda")
        self.pages[..., 16 * D:] = torch.stack([s, -7.5 * s], -1).bfloat16().view(torch.uint8).flatten(2)
        self.src = torch.randn(N, (HQ + 2 * HKV) * D, generator=g, device="cuda").bfloat16()
        self.qkv = torch.zeros_like(self.src)
        self.start, self.cu = self.lens - 1, torch.arange(N + 1, dtype=torch.int32, device="cuda")
        self.a = torch.randn(3, HQ * D, 16, generator=g, device="cuda").bfloat16() * 0.05
        self.b = torch.randn(3, 16, 4096, generator=g, device="cuda").bfloat16() * 0.05
        self.ids = torch.arange(N, dtype=torch.int32, device="cuda") % 4 - 1
        self.w = torch.randn(HQ * D, 4096, generator=g, device="cuda").bfloat16() * 0.05
        self.total = int(((self.lens + 15) // 16).sum())

    def tail(self):
        q = att.append_qkv_q4(self.qkv, self.pages, self.table, self.start, self.cu, HQ)
        o = att.paged_decode_q4(q, self.pages, self.table, self.lens)
        p = att.paged_decode_q4(q, self.pages, self.table, self.lens, num_prefix_pages=4)
        k, v, _ = att.expand_pages_q4(self.pages, self.table, self.lens, self.total)
        x = o.view(N, -1)
        y = x @ self.w
        plan = mo.lora_plan(self.ids, self.cu, N, 3)
        mo.lora_add(y, x, self.a, self.b, plan)
        mo.lora_add(y, p.view(N, -1), self.a, self.b, plan)
        lp = mo.token_logprobs(y, self.ids.long() + 5, top_k=8)
        return (q, o, p, k, v, y) + tuple(lp)

    def run(self):
        self.qkv.copy_(self.src)
        return self.tail()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def settled(step):
    """The same with the device idle between any two launches."""
    out = []
    torch.cuda.synchronize()
    step.qkv.copy_(step.src)
    torch.cuda.synchronize()
    real = mo.launch
    def slow(*args):
        real(*args)
        torch.cuda.synchronize()
    try:
        mo.launch = att.launch = slow
        out = step.tail()
    finally:
        mo.launch = att.launch = real
    torch.cuda.synchronize()
    return out


def test_back_to_back_equals_one_at_a_time():
    step = Step()
    want = [t.clone() for t in settled(step)]
    for i in range(30):
        step.qkv.zero_()
        if i % 3 == 0:
            torch.cuda._sleep(200_000)                     # a producer that takes its time
        got = step.run()
        step.qkv.fill_(7.0)                                # what follows does not overtake its readers
        assert same(got, want), i


def test_captured_behind_a_copy():
    step = Step(1)
    want = [t.clone() for t in settled(step)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step.run()                                   # the first node is the copy
    for _ in range(5):
        step.qkv.zero_()
        g.replay()
        assert same(out, want)


def test_captured_behind_joined_streams():
    step = Step(2)
    want = [t.clone() for t in settled(step)]
    side = torch.cuda.Stream()
    half = N // 2
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            step.qkv[half:].copy_(step.src[half:] * 1)
        step.qkv[:half] = step.src[:half] * 1
        main.wait_stream(side)                             # two kernels precede the append
        out = step.tail()
    for _ in range(5):
        step.qkv.zero_()
        g.replay()
        assert same(out, want)


def test_two_streams_at_once():
    a, b = Step(3), Step(4)
    wa, wb = ([t.clone() for t in settled(s)] for s in (a, b))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s1):
            ga = a.run()
        with torch.cuda.stream(s2):
            gb = b.run()
        torch.cuda.synchronize()
        assert same(ga, wa) and same(gb, wb)
