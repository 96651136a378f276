"""Token log probabilities, entropy and top alternatives against float64.

Tolerances per row, from the kernel's arithmetic: an exponential's argument x - m is rounded twice
(2^-23 of it) and ex2 is good to 2^-22; a lane adds at most ceil(V / 256) + 64 terms one after
another (2^-24 each of the sum); the results are rounded to fp32.  With W = sum p |x - m|:
  rel(s) <= (W + 2) 2^-22 + (V / 256 + 80) 2^-24,
  |log p| off by rel(s) + 2^-22 (|x - m| + ln s),   entropy by rel(s) (1 + 2 W) + 2^-22 (ln s + W).
Top ids are compared exactly.
"""
import ctypes
import math

import pytest
import torch

from loopfuse_b200 import _lib
from loopfuse_b200 import model_ops as mo

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def drain_status():
    out, seen = ctypes.c_int(0), []
    for _ in range(64):
        _lib.call("lf_device_status", ctypes.byref(out))
        if out.value == 0:
            return seen
        seen.append(out.value)
    return seen


def check(x, tokens, k):
    """``x`` on the GPU in its own type; rows must have a finite maximum."""
    got = mo.token_logprobs(x, tokens, top_k=k)
    xd = x.double()
    V = x.shape[1]
    m = xd.amax(-1, keepdim=True)
    d = xd - m
    p = torch.softmax(xd, -1)
    ln_s = torch.log(torch.exp(d).sum(-1))
    W = torch.where(p > 0, p * d.abs(), p).sum(-1)
    rel = (W + 2) * 2 ** -22 + (V / 256 + 80) * 2 ** -24
    logp = d - ln_s[:, None]
    ent = ln_s + W                                    # d <= 0
    tok = tokens.long()

    def close(g, w, tol):
        inf = torch.isinf(w)
        assert torch.equal(torch.isinf(g) & (g < 0), inf)
        assert bool(((g.double() - w).abs()[~inf] <= tol[~inf]).all()), ((g.double() - w).abs() / tol).max()

    dt = d.gather(1, tok[:, None])[:, 0]
    close(got.logprob, logp.gather(1, tok[:, None])[:, 0], rel + 2 ** -22 * (torch.nan_to_num(dt.abs(), posinf=0) + ln_s) + 1e-12)
    close(got.entropy, ent, rel * (1 + 2 * W) + 2 ** -22 * (ln_s + W) + 1e-12)
    assert got.top_ids.shape == (x.shape[0], k) and got.top_ids.dtype == torch.int64
    if k:
        ids = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :k]
        assert torch.equal(got.top_ids, ids)
        close(got.top_logprobs, logp.gather(1, ids),
              rel[:, None] + 2 ** -22 * (torch.nan_to_num(d.gather(1, ids).abs(), posinf=0) + ln_s[:, None]) + 1e-12)
    assert drain_status() == []
    return got


def inputs(T, V, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + T + V)
    x = (torch.randn(T, V, generator=g, device="cuda") * scale).to(dtype)
    return x, torch.randint(0, V, (T,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (3, 5, 5), (2, 33, 32), (1, 2047, 20), (5, 2048, 1), (2, 2049, 0),
                                   (1, 50257, 5), (37, 50257, 20), (1, 128256, 32), (3, 300001, 7), (700, 1000, 20)])
def test_matches_float64(dtype, T, V, k):
    check(*inputs(T, V, dtype), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 3, 7])
def test_rows_of_any_alignment_and_stride(dtype, offset):
    x, _ = inputs(6, 5003, dtype)
    view = x[:, offset:offset + 4990]                 # rows start anywhere, stride 5003
    check(view, torch.arange(6, device="cuda") * 700, 20)
    check(view[::2], torch.tensor([0, 4989, 17], device="cuda", dtype=torch.int32), 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_go_to_the_lowest_index(dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-3, 4, (9, 20000), generator=g, device="cuda").to(dtype)
    x[1] = 0.5                                        # all equal
    x[2] = -0.0
    x[2, ::3] = 0.0                                   # zeros of both signs are equal
    check(x, torch.randint(0, 20000, (9,), generator=g, device="cuda"), 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 20, 32])
def test_sorted_rows_and_largest_at_the_ends(dtype, k):
    V = 9000
    up = torch.linspace(-20, 20, V, device="cuda")
    x = torch.stack([up, up.flip(0), torch.cat([up[::2], up[1::2].flip(0)]), torch.zeros_like(up)])
    x[3, -40:] = torch.arange(40, device="cuda").float()
    check(x.to(dtype), torch.tensor([0, 1, V - 1, 77], device="cuda"), k)


@pytest.mark.parametrize("dtype", TYPES)
def test_banned_tokens(dtype):
    x, tok = inputs(5, 50257, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    ban = torch.rand(x.shape, generator=g, device="cuda") < 0.5
    ban[1] = True
    ban[1, 40000:40003] = False                       # fewer left than alternatives asked for
    ban[2] = True
    ban[2, 0] = False
    ban[3, :49000] = True                             # whole slices banned
    x = x.masked_fill(ban, -math.inf)
    got = check(x, tok, 20)
    assert got.entropy[2].item() == 0.0               # one token is certain


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_a_distribution(dtype):
    x, tok = inputs(7, 6001, dtype)
    x[0] = -math.inf                                  # nothing left
    x[1, 3000] = math.nan
    x[2, 5999] = math.inf
    x[3] = torch.finfo(dtype).min                     # the type's lowest value everywhere: uniform
    x[4, :] = torch.finfo(dtype).min
    x[4, 10] = 1.0
    x[5] = math.nan
    got = mo.token_logprobs(x, tok, top_k=4)
    assert got.logprob[0].item() == -math.inf and got.entropy[0].item() == 0.0
    assert got.top_ids[0].tolist() == [0, 1, 2, 3] and (got.top_logprobs[0] == -math.inf).all()
    for r, first in ((1, 3000), (2, 5999), (5, 0)):
        assert got.logprob[r].isnan() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all()
        assert got.top_ids[r, 0].item() == first
    assert got.top_ids[5].tolist() == [0, 1, 2, 3]
    # ln 6001 = 8.7: sums of 6001 ones are exact, logf is good to 2^-22 of it
    assert abs(got.logprob[3].item() + math.log(6001)) < 8.7 * 2 ** -21
    assert abs(got.entropy[3].item() - math.log(6001)) < 8.7 * 2 ** -21
    assert got.top_ids[4].tolist() == [10, 0, 1, 2] and got.entropy[4].item() == 0.0
    check(x[6:], tok[6:], 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_huge_magnitudes_and_peaked_rows(dtype):
    x, tok = inputs(4, 3001, dtype)
    x[0] *= 1e36
    x[1, 77] = 60.0
    x[2] = torch.finfo(dtype).max
    x[2, 5] = torch.finfo(dtype).min
    check(x, tok, 8)


def test_tokens_that_are_none_or_outside_the_vocabulary():
    x, _ = inputs(4, 100, torch.float32)
    got = mo.token_logprobs(x, torch.tensor([-1, 100, 5, -(1 << 40)], device="cuda"), top_k=2)
    assert got.logprob[0].item() == 0.0 and got.logprob[1].isnan() and got.logprob[3].item() == 0.0
    assert drain_status() == [231]
    assert torch.equal(got.top_ids, torch.sort(x, descending=True, stable=True)[1][:, :2])


def test_rows_past_2_31_elements():
    T, V = 16800, 128256                              # 4.3 GB of bf16
    x = torch.zeros((T, V), dtype=torch.bfloat16, device="cuda")
    part, tok = inputs(3, V, torch.bfloat16, seed=5)
    x[-3:] = part
    got = mo.token_logprobs(x, torch.cat([tok.new_zeros(T - 3), tok]), top_k=3)
    want = mo.token_logprobs(part, tok, top_k=3)
    # a row alone is split over more CTAs: sums in another order, ids the same
    assert torch.equal(got.top_ids[-3:], want.top_ids)
    assert (got.logprob[-3:] - want.logprob).abs().max().item() < 1e-5
    assert (got.top_ids[0] == torch.arange(3, device="cuda")).all()
    assert (got.logprob[:-3] + math.log(V)).abs().max().item() < 12 * 2 ** -21


def test_captured_repeated_and_on_another_stream():
    x, tok = inputs(9, 50257, torch.bfloat16)
    want = mo.token_logprobs(x, tok, top_k=20)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(mo.token_logprobs(x, tok, top_k=20), want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mo.token_logprobs(x, tok, top_k=20)
    x.copy_(inputs(9, 50257, torch.bfloat16, seed=3)[0])
    g.replay()
    want = mo.token_logprobs(x, tok, top_k=20)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mo.token_logprobs(x, tok, top_k=20)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = mo.token_logprobs(x[:0], tok[:0], top_k=2)
    assert empty.logprob.shape == (0,) and empty.top_ids.shape == (0, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [16385, 32800, 65537, 70001])
def test_parts_of_a_row_that_end_early(V, dtype):
    """A row cut over 2, 4 or 8 CTAs whose last ones have little or nothing to read: they hand over their
    lists while the first is still at work."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    for T in (1, 3, 70):
        x = (3 * torch.randn(T, V, generator=gen, device="cuda")).to(dtype)
        tok = torch.randint(0, V, (T,), generator=gen, device="cuda")
        x[0, V - 1] = 30.0                                 # the best of a row in its last, short part
        for k in (0, 1, 32):
            first = check(x, tok, k)
            for _ in range(5):
                assert all(torch.equal(a, b) for a, b in zip(first, mo.token_logprobs(x, tok, top_k=k)))
    assert drain_status() == []
