"""Low-rank adapters of many sessions against float64.

Tolerance per element: the result's rounding (2^-8 of it), the rounding of scale * (x A) to bf16
(2^-8 of sum |h| |B|), and the fp32 sums of both products (2^-22 of the sums of magnitudes, once per
16 products added).
"""
import ctypes
import math

import pytest
import torch

from loopfuse_b200 import _lib
from loopfuse_b200 import model_ops as mo

pytestmark = pytest.mark.gpu


def drain_status():
    out, seen = ctypes.c_int(0), []
    for _ in range(64):
        _lib.call("lf_device_status", ctypes.byref(out))
        if out.value == 0:
            return seen
        seen.append(out.value)
    return seen


def batch(ids, counts, K, N, R, adapters, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(counts) + K + N + R)
    T = sum(counts)

    def n(*s):
        return torch.randn(*s, generator=g, device="cuda")
    return dict(x=n(T, K).bfloat16(), y=n(T, N).bfloat16(), a=(n(adapters, K, R) * K ** -0.5).bfloat16(),
                b=(n(adapters, R, N) * R ** -0.5).bfloat16(), scale=n(adapters).abs() + 0.25,
                ids=torch.tensor(ids, dtype=torch.int32, device="cuda"),
                cu=torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda"))


def expected(s, ids, counts, scale):
    out, tol = s["y"].double(), torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    K, R = s["a"].shape[1:]
    at = 0
    for i, c in zip(ids, counts):
        if c and i >= 0:
            sl = slice(at, at + c)
            sc = float(s["scale"][i]) if scale else 1.0
            x, a, b = s["x"][sl].double(), s["a"][i].double(), s["b"][i].double()
            h = sc * (x @ a)
            out[sl] += h @ b
            eh = abs(sc) * (x.abs() @ a.abs()) * 2 ** -22 * (K / 16 + 34)
            tol[sl] = (2 ** -8 * h.abs() + eh) @ b.abs() * (1 + 2 ** -6) + (h.abs() @ b.abs()) * 2 ** -22 * (R / 16 + 2)
        at += c
    return out, tol + 2 ** -8 * out.abs() + 1e-30


def check(ids, counts, K, N, R, adapters, scale=True, in_place=False):
    s = batch(ids, counts, K, N, R, adapters)
    want, tol = expected(s, ids, counts, scale)
    before = s["y"].clone()
    plan = mo.lora_plan(s["ids"], s["cu"], sum(counts), adapters)
    out = None if in_place else torch.full_like(s["y"], math.nan)
    got = mo.lora_add(s["y"], s["x"], s["a"], s["b"], plan, scale=s["scale"] if scale else None, out=out)
    assert got.data_ptr() == (s["y"] if in_place else out).data_ptr()
    assert bool(((got.double() - want).abs() <= tol).all()), ((got.double() - want).abs() / tol).max()
    at = 0
    for i, c in zip(ids, counts):
        if i < 0:                                     # rows without an adapter are y's, bit for bit
            assert torch.equal(got[at:at + c], before[at:at + c])
        at += c
    if not in_place:
        assert torch.equal(s["y"], before)
    assert drain_status() == []
    return got


@pytest.mark.parametrize("R", [16, 32, 64, 128])
@pytest.mark.parametrize("in_place", [False, True])
def test_ranks(R, in_place):
    check([0, 2, -1, 1, 2, 0], [1, 70, 3, 17, 64, 2], 320, 264, R, 3, in_place=in_place)


@pytest.mark.parametrize("K,N", [(8, 8), (24, 136), (72, 1000), (4096, 128), (1000, 6144), (2056, 120)])
@pytest.mark.parametrize("counts", [[1], [1, 1, 1, 1, 1, 1, 1], [0, 33, 0, 5], [130]])
def test_sizes(K, N, counts):
    check([(3 * i) % 4 for i in range(len(counts))], counts, K, N, 16, 4)


def test_many_sessions_and_long_ones():
    ids = [(i * 7) % 13 - 1 for i in range(200)]
    check(ids, [1] * 200, 512, 256, 16, 12)
    check([1, 0, 1, -1], [1500, 2100, 3, 1030], 256, 256, 32, 2)          # sessions copied by the whole CTA
    check([5], [1], 4096, 6144, 64, 6)
    check([i % 1500 for i in range(2000)], [1] * 2000, 64, 64, 16, 1500)  # more adapters than threads
    check([-1] * 5, [3, 0, 70, 1, 2], 64, 64, 16, 2)                      # nobody has one
    check([3, 3], [40, 41], 64, 64, 16, 4096, scale=False)


@pytest.mark.parametrize("R", [16, 32])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("K,N", [(8, 8), (72, 264), (136, 2056), (1032, 512), (4096, 6144)])
def test_decode_batches_of_many_adapters(R, in_place, K, N):
    """14 to 37 tiles, and fewer of a few rows each: a cluster a tile."""
    check([(5 * i) % 17 - 1 for i in range(40)], [(1, 1, 2, 0, 1, 40, 1, 17)[i % 8] for i in range(40)], K, N, R, 16,
          in_place=in_place)
    check([i % 14 for i in range(30)], [1] * 30, K, N, R, 14, scale=False, in_place=in_place)
    check([2, -1, 0, 2, 1], [1, 3, 1, 0, 20], K, N, R, 3, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_strided_rows(in_place):
    s = batch([0, -1, 1], [5, 2, 30], 64, 128, 16, 2)
    wide_y = torch.full((37, 400), 7.0, dtype=torch.bfloat16, device="cuda")
    wide_x = torch.full((37, 80), math.nan, dtype=torch.bfloat16, device="cuda")
    wide_y[:, 104:232], wide_x[:, 8:72] = s["y"], s["x"]
    y, x = wide_y[:, 104:232], wide_x[:, 8:72]
    wide_o = wide_y if in_place else torch.full((37, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    out = y if in_place else wide_o[:, 64:192]
    want, tol = expected(s, [0, -1, 1], [5, 2, 30], True)
    plan = mo.lora_plan(s["ids"], s["cu"], 37, 2)
    got = mo.lora_add(y, x, s["a"], s["b"], plan, scale=s["scale"], out=None if in_place else out)
    assert bool(((got.double() - want).abs() <= tol).all())
    lo = 104 if in_place else 64
    assert (wide_o[:, :lo] == 7.0).all() and (wide_o[:, lo + 128:] == 7.0).all()


def test_other_sessions_nan_and_other_adapters_nan_stay_theirs():
    ids, counts = [0, 1, 0, 2], [3, 2, 4, 1]
    s = batch(ids, counts, 128, 128, 16, 3)
    clean, _ = expected(s, ids, counts, True)
    s["a"][1] = math.nan
    s["b"][2] = math.inf
    s["x"][0] = math.nan
    plan = mo.lora_plan(s["ids"], s["cu"], 10, 3)
    got = mo.lora_add(s["y"], s["x"], s["a"], s["b"], plan, scale=s["scale"])
    keep = [1, 2, 5, 6, 7, 8]
    assert got[0].isnan().all() and got[3:5].isnan().all()
    assert (got[keep].double() - clean[keep]).abs().max().item() < 0.1 and not got[keep].isnan().any()


def test_same_row_alone_and_in_a_batch():
    """A session's result does not depend on the adapters of others (the split of the sums may differ
    with the batch's size, so within the tolerance, not by bits)."""
    ids, counts = [1, 0, 1, 2], [4, 9, 1, 70]
    s = batch(ids, counts, 1024, 256, 16, 3)
    plan = mo.lora_plan(s["ids"], s["cu"], 84, 3)
    got = mo.lora_add(s["y"], s["x"], s["a"], s["b"], plan, out=torch.empty_like(s["y"]))
    for i, (at, c) in enumerate(zip([0, 4, 13, 14], counts)):
        one = mo.lora_plan(s["ids"][i:i + 1].clone(), torch.tensor([0, c], dtype=torch.int32, device="cuda"), c, 3)
        alone = mo.lora_add(s["y"][at:at + c], s["x"][at:at + c], s["a"], s["b"], one,
                            out=torch.empty(c, 256, dtype=torch.bfloat16, device="cuda"))
        d = (alone.float() - got[at:at + c].float()).abs()
        # h differs by fp32 sums only, which can move it across one bf16 rounding (2^-8, both sides)
        assert bool((d <= 2 ** -6 * got[at:at + c].float().abs() + 0.03).all())


def test_bad_ids_and_offsets_are_reported():
    s = batch([0, 7, -5, 1], [2, 2, 2, 2], 64, 64, 16, 2)
    plan = mo.lora_plan(s["ids"], s["cu"], 8, 2)
    got = mo.lora_add(s["y"], s["x"], s["a"], s["b"], plan, out=torch.empty_like(s["y"]))
    assert drain_status() == [241]
    assert torch.equal(got[2:6], s["y"][2:6]) and not torch.equal(got[:2], s["y"][:2])
    s["ids"].zero_()
    for cu in ([0, 2, 4, 6, 7], [1, 2, 4, 6, 8], [0, 5, 3, 6, 8], [0, 2, 4, 6, 9], [-2, 2, 4, 6, 8]):
        plan = mo.lora_plan(s["ids"], torch.tensor(cu, dtype=torch.int32, device="cuda"), 8, 2)
        out = torch.full_like(s["y"], 3.0)
        mo.lora_add(s["y"], s["x"], s["a"], s["b"], plan, out=out)
        assert drain_status() == [242] and (out == 3.0).all(), cu


def test_captured_with_new_ids_repeated_and_on_another_stream():
    counts = [1] * 9
    s = batch([0] * 9, counts, 512, 256, 32, 4)

    def step():
        plan = mo.lora_plan(s["ids"], s["cu"], 9, 4)
        return mo.lora_add(s["y"], s["x"], s["a"], s["b"], plan, s["scale"], out=torch.empty_like(s["y"]))
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for ids in ([3, 2, 1, 0, -1, 3, 2, 1, 0], [-1] * 9, [2] * 9):
        s["ids"].copy_(torch.tensor(ids, dtype=torch.int32))
        g.replay()
        want, tol = expected(s, ids, counts, True)
        assert bool(((out.double() - want).abs() <= tol).all())
        for _ in range(2):
            assert torch.equal(step(), out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, out)


def test_row_offsets_past_2_31_elements():
    T, N = 20000, 114688                              # 4.6 GB of y
    y = torch.zeros((T, N), dtype=torch.bfloat16, device="cuda")
    s = batch([1], [3], 64, N, 16, 2)
    x = torch.zeros((T, 64), dtype=torch.bfloat16, device="cuda")
    x[-3:], y[-3:] = s["x"], s["y"]
    want, tol = expected(s, [1], [3], False)
    cu = torch.tensor([0, T - 3, T], dtype=torch.int32, device="cuda")
    plan = mo.lora_plan(torch.tensor([-1, 1], dtype=torch.int32, device="cuda"), cu, T, 2)
    mo.lora_add(y, x, s["a"], s["b"], plan)
    assert bool(((y[-3:].double() - want).abs() <= tol).all()) and not y[:-3].any()
