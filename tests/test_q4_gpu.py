"""The 4-bit K/V cache against its 64-bit oracle: quantised append, expansion, decode, the pool.

The append is compared byte for byte, the expansion bit for bit (a value is ``n * s + low`` rounded
once).  Decode tolerances are per element, from ``oracle.q4.decode``: they count the output's rounding,
the rounding of the probabilities, and the fp32 sums, and nothing else.
"""
import ctypes
import math

import pytest
import torch

from loopfuse_b200 import _lib
from loopfuse_b200 import attention as att
from loopfuse_b200._lib import LoopfuseError
from loopfuse_b200.runtime import KVPool, QuantKVPool
from oracle import q4

pytestmark = pytest.mark.gpu


def drain_status():
    out, seen = ctypes.c_int(0), []
    for _ in range(64):
        _lib.call("lf_device_status", ctypes.byref(out))
        if out.value == 0:
            return seen
        seen.append(out.value)
    return seen


def random_pages(gen, P, Hkv, D):
    """Random codes; scales and lows as of unit-variance groups."""
    pages = torch.randint(0, 256, (P, Hkv, 18 * D), generator=gen).to(torch.uint8)
    ng = D // 64
    s = (0.2 + 0.3 * torch.rand(P, Hkv, 16, 2, ng, generator=gen))
    par = torch.stack([s, -7.5 * s + 0.5 * torch.randn(s.shape, generator=gen)], -1).bfloat16()
    pages[..., 16 * D:] = par.contiguous().view(torch.uint8).flatten(2)
    return pages


def table_for(lens, npre=0, gen=None, width=None):
    """Block table over permuted page ids (-1 past a session), shared prefix pages first."""
    held = [-(-x // 16) for x in lens]
    n_ids = npre + sum(max(0, h - npre) for h in held)
    ids = torch.randperm(max(1, n_ids), generator=gen).to(torch.int32)
    table = torch.full((len(lens), width or max(1, max(held))), -1, dtype=torch.int32)
    at = npre
    for i, h in enumerate(held):
        table[i, :min(h, npre)] = ids[:min(h, npre)]
        own = max(0, h - npre)
        table[i, npre:npre + own] = ids[at:at + own]
        at += own
    return table, max(1, n_ids)


def check_decode(lens, Hq, Hkv, D, npre=0, scale=None, width=None, seed=0, spoil=False):
    gen = torch.Generator().manual_seed(seed + sum(lens) + Hq)
    table, P = table_for(lens, npre, gen, width)
    pages = random_pages(gen, P, Hkv, D)
    if spoil:                             # NaN scales in every row that no session holds
        par = pages[..., 16 * D:].clone().contiguous().view(torch.bfloat16).view(P, Hkv, 16, -1)
        for i, L in enumerate(lens):
            if L % 16 and L // 16 >= npre:
                par[int(table[i, L // 16]), :, L % 16:] = math.nan
        pages[..., 16 * D:] = par.contiguous().view(torch.uint8).flatten(2)
    q = torch.randn(len(lens), Hq, D, generator=gen).bfloat16()
    o, lse = att.paged_decode_q4(q.cuda(), pages.cuda(), table.cuda(),
                                 torch.tensor(lens, dtype=torch.int32).cuda(), num_prefix_pages=npre,
                                 scale=scale, return_lse=True)
    ro, rl, to, tl = q4.decode(q, pages, table, lens, scale if scale is not None else D ** -0.5)
    err = (o.double().cpu() - ro).abs()
    assert bool((err <= to).all()), (err / to.clamp_min(1e-30)).max()
    dead = torch.isinf(rl)
    assert torch.equal(torch.isinf(lse.cpu()), dead)
    assert bool(((lse.double().cpu() - rl).abs()[~dead] <= tl[~dead]).all())
    assert drain_status() == []
    return o


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 128), (16, 2, 128), (4, 2, 64), (3, 3, 64), (8, 1, 64)])
def test_decode_matches_the_oracle(Hq, Hkv, D):
    check_decode([0, 1, 15, 16, 17, 333, 64], Hq, Hkv, D, spoil=True)


@pytest.mark.parametrize("lens", [[513, 1, 0, 1000], [0, 0, 0], [0, 0, 40, 0, 0, 3000, 0, 2, 0], [16] * 300,
                                  [1 + (i * 37) % 700 for i in range(150)], [33] * 129 + [0] * 140 + [5000]])
def test_decode_ranges_over_sessions_of_all_lengths(lens):
    check_decode(lens, 4, 2, 64, spoil=True)
    check_decode(lens[:40], 8, 1, 128)


def test_decode_one_long_session_and_a_wide_table():
    check_decode([5000], 4, 1, 128)
    check_decode([37, 2], 4, 1, 128, width=300)            # capacity far past the lengths


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (2, 2, 64), (8, 1, 128), (4, 2, 64)])
@pytest.mark.parametrize("npre", [1, 5, 40])
def test_decode_shared_prefix(Hq, Hkv, D, npre):
    lens = [npre * 16 + x for x in (0, 1, 16, 130, 33, 7)] * 3 + [npre * 16 - 3, 1, 0]
    check_decode(lens, Hq, Hkv, D, npre=npre, spoil=True)


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (8, 8, 128), (12, 12, 64), (8, 1, 64)])
@pytest.mark.parametrize("lens", [[1], [0], [16], [31], [777], [8192], [0, 4000, 1], [5, 0, 1023, 2048, 64, 1, 700]])
def test_decode_of_few_sessions(Hq, Hkv, D, lens):
    check_decode(lens, Hq, Hkv, D, spoil=True)
    check_decode(lens, Hq, Hkv, D, scale=-0.7)


def test_decode_of_few_sessions_equals_that_of_a_wide_table():
    gen = torch.Generator().manual_seed(2)
    lens = torch.tensor([777, 40], dtype=torch.int32).cuda()
    table, P = table_for([777, 40], 0, gen)
    pages = random_pages(gen, P, 2, 128).cuda()
    q = torch.randn(2, 8, 128, generator=gen).bfloat16().cuda()
    few = att.paged_decode_q4(q, pages, table.cuda(), lens)
    wide = torch.full((2, 2000), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    flat = att.paged_decode_q4(q, pages, wide.cuda(), lens)
    assert ((few - flat).float().abs() <= 2 ** -6 * flat.float().abs().clamp_min(0.25)).all()   # two bf16 steps
    assert torch.equal(few, att.paged_decode_q4(q, pages, table.cuda(), lens))


def test_decode_of_few_long_sessions():
    check_decode([40000, 20001], 8, 2, 128)                # many partials a row
    check_decode([30000], 4, 4, 64, npre=3)


# rows x pages x KV heads x head_dim past 2^25: the prefix goes to tiles of 128 rows
TILED = [(40, 32, 4, 128, 205), (130, 4, 4, 128, 505), (101, 8, 4, 64, 650), (33, 16, 2, 64, 993)]


@pytest.mark.parametrize("N,Hq,Hkv,D,npre", TILED)
def test_decode_long_shared_prefix_of_many_rows(N, Hq, Hkv, D, npre):
    ends = [npre * 16 + x for x in (0, 1, 16, 130, 33, 7)] + [npre * 16 - 3, 1, 0, 8 * npre + 5, 500, 16 * npre - 16]
    lens = [ends[(i * 7) % len(ends)] for i in range(N)]
    check_decode(lens, Hq, Hkv, D, npre=npre, spoil=True)
    check_decode([min(x, npre * 16) for x in lens], Hq, Hkv, D, npre=npre, scale=-0.4)   # peaked, negative


def test_long_shared_prefix_beside_other_work_and_captured():
    """Two decodes and a prefill attention, all with tensor memory, on three streams; then from a graph."""
    N, Hq, Hkv, D, npre = 80, 32, 8, 128, 160
    gen = torch.Generator().manual_seed(9)
    lens = [npre * 16 + 5 + 3 * i for i in range(N)]
    table, P = table_for(lens, npre, gen)
    pages = [random_pages(gen, P, Hkv, D).cuda() for _ in range(2)]
    q = torch.randn(N, Hq, D, generator=gen).bfloat16().cuda()
    table, lens = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    x = torch.randn(2, 8, 1500, 128, generator=gen).bfloat16().cuda()
    k, v = x[:, :4].contiguous(), x[:, 4:].contiguous()

    def decode(i):
        return att.paged_decode_q4(q, pages[i], table, lens, num_prefix_pages=npre)
    alone = [decode(0), decode(1), att.prefill_attention_fwd(x, k, v)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(15):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(decode(i) if i < 2 else att.prefill_attention_fwd(x, k, v))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = decode(0), decode(1)
    for _ in range(3):
        a.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, alone[0]) and torch.equal(b, alone[1])
    assert drain_status() == []


@pytest.mark.parametrize("N,Hq,Hkv,D,npre", [(6, 8, 2, 128, 5), (5, 2, 2, 64, 40), TILED[0], TILED[3]])
def test_nan_in_a_shared_prefix_reaches_the_rows_that_hold_it(N, Hq, Hkv, D, npre):
    gen = torch.Generator().manual_seed(3)
    at = npre * 8 + 3                                      # the token with NaN
    lens = [npre * 16 + 20 if i % 2 else at - i % 3 for i in range(N)]
    table, P = table_for(lens, npre, gen)
    lead = next(i for i in range(N) if i % 2)
    pages = random_pages(gen, P, Hkv, D)
    q = torch.randn(N, Hq, D, generator=gen).bfloat16()
    q[lead, 1] = math.nan

    def run(kv):
        x = pages.clone()
        if kv is not None:
            par = x[..., 16 * D:].clone().contiguous().view(torch.bfloat16).view(P, Hkv, 16, 2, D // 64, 2)
            par[int(table[lead, at // 16]), 0, at % 16, kv, 0] = math.nan
            x[..., 16 * D:] = par.contiguous().view(torch.uint8).flatten(2)
        return att.paged_decode_q4(q.cuda(), x.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                   num_prefix_pages=npre).cpu()
    clean, k_nan, v_nan = run(None), run(0), run(1)
    assert torch.equal(clean.isnan().nonzero(), torch.cartesian_prod(
        torch.tensor([lead]), torch.tensor([1]), torch.arange(D)))
    G = Hq // Hkv
    for i in range(N):
        want = clean[i].clone()
        if i % 2:
            want[:G] = math.nan
        assert torch.allclose(k_nan[i], want, rtol=0, atol=0, equal_nan=True)
        want = clean[i].clone()
        if i % 2:
            want[:G, :64] = math.nan
        assert torch.allclose(v_nan[i], want, rtol=0, atol=0, equal_nan=True)


def test_decode_prefix_only_and_equal_to_unshared():
    lens = [96, 96, 96]
    check_decode(lens, 8, 2, 128, npre=6)
    gen = torch.Generator().manual_seed(1)
    table, P = table_for([200, 180], 4, gen)
    pages = random_pages(gen, P, 2, 128).cuda()
    q = torch.randn(2, 8, 128, generator=gen).bfloat16().cuda()
    lens = torch.tensor([200, 180], dtype=torch.int32).cuda()
    a = att.paged_decode_q4(q, pages, table.cuda(), lens, num_prefix_pages=4)
    b = att.paged_decode_q4(q, pages, table.cuda(), lens)
    assert ((a - b).float().abs() <= 2 ** -6 * b.float().abs().clamp_min(0.25)).all()   # two bf16 steps


@pytest.mark.parametrize("scale", [0.0, 1.5, -0.1])
def test_decode_scales(scale):
    check_decode([100, 5], 4, 2, 128, scale=scale)


def test_decode_page_offsets_past_2_31():
    P, Hkv, D = 120000, 8, 128                              # 2.2 GB of pages
    gen = torch.Generator().manual_seed(3)
    small = random_pages(gen, 4, Hkv, D)
    pages = torch.zeros((P, Hkv, 18 * D), dtype=torch.uint8, device="cuda")
    pages[-4:] = small.cuda()
    table = torch.arange(P - 4, P, dtype=torch.int32)[None]
    q = torch.randn(1, 16, D, generator=gen).bfloat16()
    lens = torch.tensor([61], dtype=torch.int32).cuda()
    o = att.paged_decode_q4(q.cuda(), pages, table.cuda(), lens)
    ro, _, to, _ = q4.decode(q, small, torch.arange(4)[None], [61], D ** -0.5)
    assert bool(((o.double().cpu() - ro).abs() <= to).all())
    k, v, _ = att.expand_pages_q4(pages, table.cuda(), lens, 4)
    ke, ve, _ = q4.unpack(small)
    assert torch.equal(k.cpu().transpose(1, 2).reshape(-1, Hkv, D)[:61],
                       ke.transpose(1, 2).reshape(-1, Hkv, D)[:61].bfloat16())
    qkv = torch.randn(1, (16 + 16) * D, generator=gen).bfloat16().cuda()
    att.append_qkv_q4(qkv, pages, table.cuda(), torch.tensor([60], dtype=torch.int32).cuda(),
                      torch.tensor([0, 1], dtype=torch.int32).cuda(), 16)
    want = small.clone()
    for h in range(Hkv):
        row = qkv.cpu()[0].view(-1, D)
        q4.write_token(want, 3, h, 12, row[16 + h], row[16 + Hkv + h])
    assert torch.equal(pages[-4:].cpu(), want)


def test_decode_bad_page_id_is_reported_and_reads_page_zero():
    gen = torch.Generator().manual_seed(5)
    pages = random_pages(gen, 3, 1, 64).cuda()
    q = torch.randn(1, 1, 64, generator=gen).bfloat16().cuda()
    lens = torch.tensor([20], dtype=torch.int32).cuda()
    bad = torch.tensor([[1, 7]], dtype=torch.int32).cuda()
    good = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    a = att.paged_decode_q4(q, pages, bad, lens)
    assert drain_status() == [200]
    assert torch.equal(a, att.paged_decode_q4(q, pages, good, lens))
    assert drain_status() == []


# -- append -----------------------------------------------------------------------------------------
def rope_tables(rows, D):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, D, 2).double() / D)
    return ang.cos().float(), ang.sin().float()


def rotated(x, cos, sin):
    """fp32, every product and sum rounded separately, then bf16."""
    h = x.shape[-1] // 2
    a, b = x[..., :h].float(), x[..., h:].float()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).bfloat16()


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 4, 2), (64, 3, 3), (128, 1, 1), (64, 8, 1)])
@pytest.mark.parametrize("turn", [False, True])
def test_append_writes_the_oracles_bytes(D, Hq, Hkv, turn):
    gen = torch.Generator().manual_seed(D + Hq)
    old, new = [0, 13, 31, 5], [3, 0, 7, 1]
    table, P = table_for([a + b for a, b in zip(old, new)], gen=gen)
    pages = random_pages(gen, P, Hkv, D)
    wide = torch.randn(sum(new), (Hq + 2 * Hkv) * D + 16, generator=gen).bfloat16()
    wide[0, Hq * D:Hq * D + 64] = 3.0                       # a constant group: scale 0
    wide[1, Hq * D:Hq * D + 64] *= 1e-38
    wide[2, -16 - 64:-16] = 1e38 * torch.linspace(-3, 3, 64)
    wide[3, -16 - 7] = math.inf
    wide[4, -16 - 9] = math.nan
    qkv = wide.cuda()[:, :(Hq + 2 * Hkv) * D]               # strided rows
    rope = rope_tables(64, D) if turn else None
    dev = pages.cuda()
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
    got_q = att.append_qkv_q4(qkv, dev, table.cuda(), torch.tensor(old, dtype=torch.int32).cuda(),
                              cu.cuda(), Hq, rope=tuple(t.cuda() for t in rope) if rope else None)
    want, t = pages.clone(), 0
    for i, n in enumerate(new):
        for j in range(n):
            row = qkv[t].cpu().view(-1, D)
            pos = old[i] + j
            qk = row[:Hq + Hkv] if not turn else rotated(row[:Hq + Hkv], rope[0][pos], rope[1][pos])
            assert torch.equal(got_q[t].cpu(), qk[:Hq])
            for h in range(Hkv):
                q4.write_token(want, int(table[i, pos // 16]), h, pos % 16, qk[Hq + h], row[Hq + Hkv + h])
            t += 1
    got = dev.cpu()
    # one bit pattern for NaN on each side: compare params as values there, bytes everywhere else
    gp, wp = (x[..., 16 * D:].contiguous().view(torch.bfloat16).float() for x in (got, want))
    assert torch.equal(got[..., :16 * D], want[..., :16 * D])
    assert torch.equal(torch.nan_to_num(gp, 77.0), torch.nan_to_num(wp, 77.0))
    assert drain_status() == []


def test_append_without_a_page_stores_nothing_and_is_reported():
    gen = torch.Generator().manual_seed(9)
    pages = random_pages(gen, 2, 1, 64)
    table = torch.tensor([[0, -1], [1, 5]], dtype=torch.int32).cuda()
    dev = pages.cuda()
    qkv = torch.randn(3, 3 * 64, generator=gen).bfloat16().cuda()
    for start in ([16, 16], [32, 1 << 20], [-1, -16]):       # no page, bad id, past the table, negative
        att.append_qkv_q4(qkv, dev, table, torch.tensor(start, dtype=torch.int32).cuda(),
                          torch.tensor([0, 1, 1], dtype=torch.int32).cuda(), 1)
        assert drain_status() == [252]
    assert torch.equal(dev.cpu(), pages)
    cos, sin = (t.cuda() for t in rope_tables(4, 64))
    att.append_qkv_q4(qkv[:1], dev, table[:1], torch.tensor([4], dtype=torch.int32).cuda(),
                      torch.tensor([0, 1], dtype=torch.int32).cuda(), 1, rope=(cos, sin))
    assert drain_status() == [252] and torch.equal(dev.cpu(), pages)


@pytest.mark.parametrize("power", [-100, -88, -20, 0, 40])
def test_append_of_groups_whose_scale_is_rounded_down_most(power):
    """Span / 15 halfway between two bf16 values: the largest code is that of 15 (1 + 2^-8) steps."""
    gen = torch.Generator().manual_seed(1)
    D, unit = 64, 2.0 ** power
    rows = (torch.rand(4, 3, D, generator=gen) * 15).bfloat16().float()
    rows[..., 0], rows[..., 1] = -15 / 256, 15.0
    rows[1::2] = -rows[1::2]
    rows = (rows * unit).bfloat16()
    for x in rows[:, 1:].reshape(-1, D):                     # (the case is what it claims to be)
        n, s, low = q4.quantise(x)
        assert float(s) == unit and int(n.max()) == 15
        assert float(((x.double() - low) / s).max()) == 15 + 15 / 256
    pages = torch.zeros(1, 1, 18 * D, dtype=torch.uint8)
    dev = pages.cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    att.append_qkv_q4(rows.reshape(4, -1).cuda(), dev, torch.zeros(1, 1, **i32), torch.zeros(1, **i32),
                      torch.tensor([0, 4], **i32), 1)
    for t in range(4):
        q4.write_token(pages, 0, 0, t, rows[t, 1], rows[t, 2])
    assert torch.equal(dev.cpu(), pages) and drain_status() == []


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 4, 2), (64, 3, 3)])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("cu,T", [([2, 5], 5), ([0, 3], 7), ([3, 3, 4, 9], 11), ([0, 0], 2), ([6, 6, 6], 9)])
def test_append_leaves_rows_of_no_session_alone(D, Hq, Hkv, turn, cu, T):
    """Rows before cu[0] and from cu[n] on, as of a padded batch: no page, no q, one report."""
    gen = torch.Generator().manual_seed(T + D)
    N = len(cu) - 1
    start = [20 + 3 * i for i in range(N)]
    table, P = table_for([64] * N, gen=gen)
    pages = random_pages(gen, P, Hkv, D)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen).bfloat16().cuda()
    rope = tuple(t.cuda() for t in rope_tables(64, D)) if turn else None
    i32 = dict(dtype=torch.int32, device="cuda")
    runs = []
    for rows, offsets in ((qkv, cu), (qkv[cu[0]:cu[-1]], [c - cu[0] for c in cu])):
        dev, q = pages.cuda(), torch.full((rows.shape[0], Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
        att.append_qkv_q4(rows, dev, table.cuda(), torch.tensor(start, **i32), torch.tensor(offsets, **i32), Hq,
                          rope=rope, q_out=q)
        runs.append((dev, q, drain_status()))
    (dev, q, status), (dev2, q2, status2) = runs
    assert torch.equal(dev, dev2) and torch.equal(q[cu[0]:cu[-1]], q2)
    assert (q[:cu[0]] == 7).all() and (q[cu[-1]:] == 7).all()
    assert status == [252] and status2 == []
    # with a pool's status: that instead of the device's word
    st = torch.zeros(1, **i32)
    dev = pages.cuda()
    base, row = qkv.data_ptr(), qkv.shape[1]
    tb, sp, ct = table.cuda(), torch.tensor(start, **i32), torch.tensor(cu, **i32)
    _lib.call("lf_q4_append", None, base + Hq * D * 2, base + (Hq + Hkv) * D * 2, 0, 0, row, D, tb.data_ptr(), N,
              table.shape[1], None, sp.data_ptr(), ct.data_ptr(), N, T, None, None, 0, None, dev.data_ptr(), P, 1, 0,
              Hkv, D, st.data_ptr(), None)
    torch.cuda.synchronize()
    assert st.item() == _lib.LF_EINVAL and drain_status() == []


# -- expansion --------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,Hkv", [(128, 2), (64, 3)])
@pytest.mark.parametrize("npre", [0, 2])
def test_expansion_is_the_values_rounded_once(D, Hkv, npre):
    gen = torch.Generator().manual_seed(D + npre)
    lens = [70, 0, 33, 16, 1, 48]
    table, P = table_for(lens, npre, gen)
    pages = random_pages(gen, P, Hkv, D)
    held = [-(-x // 16) for x in lens]
    total = npre + sum(max(0, h - npre) for h in held)
    k, v, out = att.expand_pages_q4(pages.cuda(), table.cuda(),
                                    torch.tensor(lens, dtype=torch.int32).cuda(), total, npre)
    ke, ve, _ = q4.unpack(pages)
    at = npre
    for i, L in enumerate(lens):
        for j in range(held[i]):
            o = j if j < npre else at + j - npre
            assert int(out[i, j]) == o
            rows = min(16, max(0, L - 16 * j))
            if j < npre and L < max(lens):
                rows = min(16, max(0, max(lens) - 16 * j))  # shared pages: the longest session's rows
            for got, want in ((k, ke), (v, ve)):
                page = want[int(table[i, j])].bfloat16().clone()
                page[:, rows:] = 0
                assert torch.equal(got[o].cpu(), page)
        at += max(0, held[i] - npre)
        assert (out[i, max(held[i], npre):] == -1).all()
    assert drain_status() == []


def test_expansion_reports_too_few_output_pages_and_bad_ids():
    gen = torch.Generator().manual_seed(2)
    pages = random_pages(gen, 4, 1, 64).cuda()
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    lens = torch.tensor([32, 20], dtype=torch.int32).cuda()
    k, v, out = att.expand_pages_q4(pages, table, lens, 3)
    assert out.tolist() == [[0, 1], [2, -1]] and drain_status() == [253]
    full, _, _ = att.expand_pages_q4(pages, table, lens, 4)
    assert torch.equal(k, full[:3]) and drain_status() == []
    table[1, 1] = 9
    att.expand_pages_q4(pages, table, lens, 4)
    assert drain_status() == [254]


# -- streams, graphs, workspaces ---------------------------------------------------------------------
def test_decode_and_append_captured_and_on_another_stream():
    gen = torch.Generator().manual_seed(4)
    lens = [40, 700, 3]
    table, P = table_for(lens, gen=gen)
    Hq, Hkv, D = 8, 2, 128
    pages = random_pages(gen, P, Hkv, D).cuda()
    eager_pages = pages.clone()
    table, lens_d = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    start, cu = lens_d - 1, torch.arange(4, dtype=torch.int32).cuda()
    qkv = torch.randn(3, (Hq + 2 * Hkv) * D, generator=gen).bfloat16().cuda()

    def step(pg):
        q = att.append_qkv_q4(qkv, pg, table, start, cu, Hq)
        return att.paged_decode_q4(q, pg, table, lens_d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pages)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(pages)
    for seed in range(3):
        qkv.copy_(torch.randn(qkv.shape, generator=gen).bfloat16())
        g.replay()
        want = step(eager_pages)
        assert torch.equal(out, want) and torch.equal(pages, eager_pages)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        again = step(pages)
    side.synchronize()
    assert torch.equal(again, out)


def test_decode_repeats_bit_for_bit_and_takes_a_given_workspace():
    gen = torch.Generator().manual_seed(8)
    lens = [900, 20, 0, 333]
    table, P = table_for(lens, 1, gen)
    pages, q = random_pages(gen, P, 2, 128).cuda(), torch.randn(4, 8, 128, generator=gen).bfloat16().cuda()
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    need = att.decode_q4_workspace_bytes(4, 8, 2, 128, table.shape[1], 1)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")       # NaN bits
    out = torch.full_like(q, math.nan)
    a = att.paged_decode_q4(q, pages, table.cuda(), lens_d, 1, workspace=ws, out=out)
    assert a.data_ptr() == out.data_ptr()
    for _ in range(3):
        assert torch.equal(a, att.paged_decode_q4(q, pages, table.cuda(), lens_d, 1))


# -- the pool ---------------------------------------------------------------------------------------
def both_pools(**kw):
    args = dict(num_layers=2, num_heads=4, num_kv_heads=2, head_dim=128, max_seq_len=256, max_slots=6,
                dtype=torch.bfloat16)
    args.update(kw)
    return KVPool(**args), QuantKVPool(**args)


def test_pool_write_read_fork_release_matches_the_bf16_pools_bookkeeping():
    gen = torch.Generator().manual_seed(0)
    pools = both_pools()
    k = torch.randn(2, 2, 45, 128, generator=gen).bfloat16()
    v = torch.randn(2, 2, 45, 128, generator=gen).bfloat16()
    snaps, reads = [], []
    for pool in pools:
        a = pool.allocate_slot()
        assert pool.write(a, k[:, :, :37].cuda(), v[:, :, :37].cuda()) == 37
        b, c = pool.fork(a, 35, n=2)
        pool.append([b, c], [k[:, :, 37:41].transpose(1, 2).contiguous().cuda(),
                             k[:, :, 41:45].transpose(1, 2).contiguous().cuda()],
                    [v[:, :, 37:41].transpose(1, 2).contiguous().cuda(),
                     v[:, :, 41:45].transpose(1, 2).contiguous().cuda()])
        reads.append([pool.read(s, layer) for s in (a, b, c) for layer in (0, 1)])
        snaps.append([pool.snapshot()])
        pool.release(a)
        snaps[-1].append(pool.snapshot())
        pool.release_all([b, c])
        snaps[-1].append(pool.snapshot())
    assert snaps[0] == snaps[1]
    for (ka, va), (kb, vb) in zip(*reads):
        for x, y in ((ka, kb), (va, vb)):
            want = q4.value(*q4.quantise(x.cpu())).bfloat16()
            assert torch.equal(y.cpu(), want)
    assert pools[1].hbm_usage_bytes() < pools[0].hbm_usage_bytes() / 3
    # past the session's length a read gives zeros
    s = pools[1].allocate_slot()
    pools[1].write(s, k[:, :, :3].cuda(), v[:, :, :3].cuda())
    kz, _ = pools[1].read(s, 0, 1, 20)
    assert kz.shape == (2, 19, 128) and (kz[:, 2:] == 0).all() and (kz[:, :2] != 0).any()


def test_pool_overflow_bad_rows_and_refusals():
    _, pool = both_pools(max_seq_len=32, num_pages=3)
    a, b = pool.allocate_slot(), pool.allocate_slot()
    k = torch.randn(2, 2, 33, 128).bfloat16().cuda()
    with pytest.raises(RuntimeError, match="overflow"):
        pool.write(a, k, k)
    pool.write(a, k[:, :, :32].contiguous(), k[:, :, :32].contiguous())
    with pytest.raises(RuntimeError, match="exhausted"):
        pool.write(b, k[:, :, :32].contiguous(), k[:, :, :32].contiguous())
    with pytest.raises(LoopfuseError):
        pool.layer_pages(0)
    with pytest.raises(LoopfuseError):
        pool.write(b, k[:, :, :2].float(), k[:, :, :2].float())
    # a row whose session holds no page: the pool's sticky status, nothing stored
    before = pool.pages.clone()
    start = torch.tensor([0], dtype=torch.int32, device="cuda")
    c = pool.allocate_slot()
    pool.write_layer([c], start, 0, k[0, :, :1].transpose(0, 1).contiguous(),
                     k[0, :, :1].transpose(0, 1).contiguous(), [1])
    assert pool.status() == _lib.LF_EINVAL and torch.equal(pool.pages, before)
