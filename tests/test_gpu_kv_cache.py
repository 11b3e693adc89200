"""The paged cache's kernels against plain 64-bit forms: one token to long contexts, every page size, head dims, shared
key heads, cut and uncut keys, masked places that hold infinities and NaN, graphs and streams.  (Tolerances:
paged_check.attention_bound.)"""

import math

import pytest
import torch

import paged_check as pc
from abacus_amd.kv_cache import E4M3, BatchRows, PagedKVCache

pytestmark = pytest.mark.gpu

KINDS = [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, E4M3), (torch.float32, E4M3)]


def _filled(plan, H, K, page, dtype, held, seed=0, fill=None, max_new=None, spread=1.0):
    """Pages that hold random keys and values of the plan's whole sequences, and those rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, n = pc.rows_of(plan, page, "cuda", seed=seed, max_new=max_new)
    pages = pc.pages_of(n, H, page, K, held, "cuda", fill=fill)
    whole = BatchRows(rows.page_table_SP, torch.tensor([0] + [length for _, length in plan]).cumsum(0).to(torch.int32).cuda(),
                      rows.lengths)
    total = sum(length for _, length in plan)
    k, v = (spread * torch.randn(total, H, K, device="cuda", generator=g).to(dtype) for _ in range(2))
    pages.write(k, v, whole)
    return pages, rows, k, v, g


def _check(pages, plan, rows, k, v, q, o, held, scale=None):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    at = first = 0
    for n, length in plan:
        if n:
            qs = q[first:first + n]
            ks, vs = pc.held(k[at:at + length], held), pc.held(v[at:at + length], held)
            want, weight = pc.attention(qs, ks, vs, scale)
            got = o[first:first + n].double()
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (n, length)
            off, most = (got - want).abs(), pc.attention_bound(qs, ks, want, weight, scale)
            worst = float((off / most.clamp(min=1e-300)).nan_to_num(0.0).max())
            assert worst <= 1.0, (n, length, worst)
        at, first = at + length, first + n


@pytest.mark.parametrize("dtype,held", KINDS)
@pytest.mark.parametrize("K,page", [(16, 16), (64, 32), (80, 64), (128, 256)])
def test_write_and_read(dtype, held, K, page):
    """Whole groups, groups begun and ended inside, single rows: bit for bit what the cache should hold, and no other
    slot is touched."""
    H = 3
    plan = [(1, 1), (40, 40), (0, 5), (17, 50), (1, 16), (1, 33), (300, 333), (2, 1)]
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, n = pc.rows_of(plan, page, "cuda")
    fill = 0x55 if held == E4M3 else 3.0
    pages = pc.pages_of(n, H, page, K, held, "cuda", fill=fill)
    T = sum(n for n, _ in plan)
    k, v = (torch.randn(T, H, K, device="cuda", generator=g).to(dtype) for _ in range(2))
    k[3] = 0.0
    k[5] *= 1e-30  # exponents at their least, and large
    v[6] *= 1e30
    pages.write(k, v, rows)
    kr, vr = pages.read(rows, 340, torch.float32 if held == E4M3 else None)
    untouched = 1.625 * 2.0 ** (3 + 0x55 - 127) if held == E4M3 else 3.0  # code 0x55: exponent 10 - 7, 1 + 5 / 8
    first = 0
    for s, (new, length) in enumerate(plan):
        for got, x in ((kr, k), (vr, v)):
            there = min(new, length)
            assert torch.equal(got[s, length - there:length].double(), pc.held(x[first + new - there:first + new], held))
            assert (got[s, :length - there] == untouched).all() and not got[s, length:].any()
        first += new
    taken = sum(min(new, length) for new, length in plan) * H * K
    for t in (pages.k, pages.v):
        other = (t.view(torch.uint8) == 0x55 if held == E4M3 else t == 3.0).sum()
        assert int(other) >= t.numel() - taken


@pytest.mark.parametrize("dtype,held", KINDS)
@pytest.mark.parametrize("H,K,page,L", [(2, 16, 16, 333), (3, 80, 64, 290), (1, 128, 256, 705)])
def test_read_of_many_sequences(dtype, held, H, K, page, L):
    """Blocks of four groups (2048 of them and more): ragged sequences, empty ones, some longer than what is read, a last
    block that is not full, pages outside the pool and a length past its table."""
    S = 220
    plan = [(n, n) for n in ((s * 53) % (L + 40) if s % 9 else 0 for s in range(S))]
    assert (-(-L // 64)) * H * S >= 2048 and L % 64
    pages, rows, k, v, _ = _filled(plan, H, K, page, dtype, held, fill=0x55 if held == E4M3 else 3.0)
    rows.page_table_SP[7, 2], rows.page_table_SP[8, 0] = -1, len(pages.k)
    width = rows.page_table_SP.shape[1]
    rows.lengths[12] = width * page + 1
    kr, vr = pages.read(rows, L, torch.float32 if held == E4M3 else None)
    at = 0
    for s, (_, length) in enumerate(plan):
        n = min(length, L)
        bad = torch.zeros(L, dtype=torch.bool, device="cuda")
        if s == 7:
            bad[2 * page:3 * page] = True
        if s in (8, 12):
            bad[:page if s == 8 else min(width * page, L)] = True
        there = torch.arange(L, device="cuda") < (L if s == 12 else n)
        for got, x in ((kr[s], k), (vr[s], v)):
            assert torch.equal(torch.isnan(got).all(-1).all(-1), bad & there)
            fine = ~bad & (torch.arange(L, device="cuda") < n)
            assert torch.equal(got[fine].double(), pc.held(x[at:at + n], held)[fine[:n]])
            assert not got[~there].any()
        at += length


@pytest.mark.parametrize("dtype,held", KINDS)
@pytest.mark.parametrize("H,G,K,page,plan", [
    (2, 1, 64, 16, [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 700)]),
    (1, 4, 128, 64, [(1, 1500), (1, 40), (0, 9)]),
    (2, 3, 80, 32, [(5, 5), (4, 130), (6, 1100)]),
    (4, 8, 16, 128, [(3, 200), (9, 9)]),
    (1, 16, 96, 16, [(1, 77), (2, 640)]),
    (2, 2, 128, 16, [(40, 40), (1, 900), (130, 520), (1, 3)]),
    (1, 1, 64, 256, [(257, 800)]),
    (2, 5, 32, 64, [(70, 70), (3, 2)]),
    (2, 4, 32, 16, [(1, 3000), (4, 1100), (1, 1)]),
    (3, 1, 16, 256, [(20, 1700), (1, 31)]),
])
def test_attention(dtype, held, H, G, K, page, plan):
    pages, rows, k, v, g = _filled(plan, H, K, page, dtype, held)
    T = sum(n for n, _ in plan)
    q = torch.randn(T, H * G, K, device="cuda", generator=g).to(dtype)
    o = pages.attend(q, rows)
    _check(pages, plan, rows, k, v, q, o, held)
    known = BatchRows(rows.page_table_SP, rows.query_start, rows.lengths, max_new=max(n for n, _ in plan))
    _check(pages, plan, known, k, v, q, pages.attend(q, known, scale=0.3), held, 0.3)


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("H,G,K,page,plan", [
    (1, 1, 64, 16, [(200, 2500), (1, 700), (17, 17)]),
    (1, 3, 128, 64, [(150, 3000), (2, 90)]),
    (2, 1, 128, 256, [(129, 129), (300, 1400), (0, 60), (1, 1)]),
    (2, 8, 64, 32, [(31, 2100), (128, 128)]),
    (1, 2, 96, 16, [(150, 2000), (3, 3)]),
    (2, 1, 16, 64, [(260, 700), (1, 50)]),
    (1, 1, 112, 128, [(90, 90)]),
    (1, 5, 48, 32, [(40, 1500)]),
])
def test_chunks(held, H, G, K, page, plan):
    """Chunks over what was cached before: units that are cut and units that are not, partly filled ones, and a
    decode step beside them; padded rows behind."""
    pages, rows, k, v, g = _filled(plan, H, K, page, torch.bfloat16, held)
    T = sum(n for n, _ in plan)
    q = torch.randn(T + 5, H * G, K, device="cuda", generator=g).bfloat16()
    o = pages.attend(q, rows)
    assert not o[T:].any()
    _check(pages, plan, rows, k, v, q[:T], o[:T], held)
    kept = torch.full_like(q, 7.0)
    pages.attend(q, rows, out=kept)
    assert torch.equal(kept[:T], o[:T]) and (kept[T:] == 7.0).all()


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("K", [16, 64, 80, 128])
def test_chunk_units_of_at_most_64_rows(held, K):
    """Two waves have the same rows and half of each tile: rows of one wave and of two, pieces that end inside a half,
    sequences shorter than one, what no row sees, and a page that is missing."""
    plan = [(33, 2100), (64, 64), (40, 1000), (50, 97), (36, 40), (1, 300), (192, 500)]
    pages, rows, k, v, g = _filled(plan, 1, K, 32, torch.bfloat16, held, fill=0x7f if held == E4M3 else math.nan)
    T = sum(n for n, _ in plan)
    q = torch.randn(T, 1, K, device="cuda", generator=g).bfloat16()
    o = pages.attend(q, rows)
    _check(pages, plan, rows, k, v, q, o, held)
    v[2099, 0, 5], k[2099 + 64, 0, 3] = math.inf, math.nan  # the last positions of the first two sequences
    whole = BatchRows(rows.page_table_SP, torch.tensor([0] + [n for _, n in plan]).cumsum(0).to(torch.int32).cuda(), rows.lengths)
    pages.write(k, v, whole)
    got = pages.attend(q, rows)
    same = torch.ones(T, dtype=torch.bool, device="cuda")
    same[[32, 96]] = False
    assert torch.isfinite(got[same]).all() and not torch.isfinite(got[32, 0, 5]) and not torch.isfinite(got[96]).any()
    rows.page_table_SP[2, 30] = -1  # positions 960 to 991: all 40 rows see the first of them
    rows.page_table_SP[3, 2] = -1   # positions 64 to 95: rows 17 on
    got = pages.attend(q, rows)
    assert torch.isnan(got[97:137]).all() and torch.isfinite(got[137:154]).all() and torch.isnan(got[154:187]).all()


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
def test_a_wrong_hint_changes_no_result(held):
    """max_new says one row and there are many: other kernels, the same attention."""
    plan = [(1, 40), (70, 900), (3, 2000)]
    pages, rows, k, v, g = _filled(plan, 2, 64, 16, torch.bfloat16, held, max_new=1)
    q = torch.randn(74, 4, 64, device="cuda", generator=g).bfloat16()
    _check(pages, plan, rows, k, v, q, pages.attend(q, rows), held)


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
def test_a_chunk_with_pages_outside_the_pool(held):
    """Rows that see a position in no page are NaN, the others are not touched by it."""
    plan = [(200, 600)]
    pages, rows, k, v, g = _filled(plan, 1, 128, 32, torch.bfloat16, held)
    q = torch.randn(200, 2, 128, device="cuda", generator=g).bfloat16()
    whole = pages.attend(q, rows)
    rows.page_table_SP[0, 16] = -1  # positions 512 to 543: rows 112 on see them
    o = pages.attend(q, rows)
    assert torch.equal(o[:112], whole[:112]) and torch.isnan(o[112:]).all()
    rows.page_table_SP[0, 3] = 1 << 30
    assert torch.isnan(pages.attend(q, rows)).all()


@pytest.mark.parametrize("dtype,held", KINDS)
def test_long_context_is_cut_and_joined(dtype, held):
    plan = [(1, 9000), (2, 33), (1, 20001)]
    pages, rows, k, v, g = _filled(plan, 1, 64, 64, dtype, held, max_new=2)
    q = 3 * torch.randn(4, 2, 64, device="cuda", generator=g).to(dtype)
    o = pages.attend(q, rows)
    _check(pages, plan, rows, k, v, q, o, held)
    assert torch.equal(o, pages.attend(q, rows))  # the same bits again


def test_many_sequences():
    """More sequences than a wave scans at once, some without rows."""
    plan = [((s * 7) % 3, 1 + (s * 37) % 90) for s in range(200)]
    pages, rows, k, v, g = _filled(plan, 2, 64, 16, torch.bfloat16, torch.bfloat16)
    T = sum(n for n, _ in plan)
    q = torch.randn(T, 2, 64, device="cuda", generator=g).bfloat16()
    _check(pages, plan, rows, k, v, q, pages.attend(q, rows), torch.bfloat16)


@pytest.mark.parametrize("dtype,held", KINDS)
@pytest.mark.parametrize("plan,K", [([(1, 5), (3, 70), (1, 130)], 64), ([(100, 300)], 64), ([(2, 9), (140, 140)], 128), ([(100, 300)], 80),
                                    ([(1, 5), (3, 70), (1, 130)], 32), ([(20, 300), (2, 40)], 16)])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, held, plan, K):
    """Pages full of NaN and infinities before the sequences are written; then a NaN and an infinity in the keys and
    values of the last token: only the rows that see it have them, dim by dim as the formula has."""
    H = 2
    for fill in ((0x7f, 0xff) if held == E4M3 else (math.nan, math.inf)):
        pages, rows, k, v, g = _filled(plan, H, K, 32, dtype, held, fill=fill)
        T = sum(n for n, _ in plan)
        q = torch.randn(T, H, K, device="cuda", generator=g).to(dtype)
        _check(pages, plan, rows, k, v, q, pages.attend(q, rows), held)
    at = first = 0
    for s, (n, length) in enumerate(plan):
        last = at + length - 1
        k[last, 0, 3] = math.nan
        v[last, 1, 7] = math.inf
        at += length
    whole = BatchRows(rows.page_table_SP, torch.tensor([0] + [l for _, l in plan]).cumsum(0).to(torch.int32).cuda(), rows.lengths)
    pages.write(k, v, whole)
    o = pages.attend(q, rows)
    at = first = 0
    for n, length in plan:
        for j in range(n):
            row = o[first + j]
            if j < n - 1:
                assert torch.isfinite(row).all()
            else:
                assert torch.isnan(row[0]).all()
                if held == E4M3:
                    assert torch.isnan(row[1]).all()
                else:
                    assert row[1, 7] == math.inf and torch.isfinite(row[1, :7]).all() and torch.isfinite(row[1, 8:]).all()
        if n > 1:  # the others as if it were not there
            kk, vv = k[at:at + length].clone(), v[at:at + length].clone()
            kk[-1], vv[-1] = 0.0, 0.0
            want, weight = pc.attention(q[first:first + n], pc.held(kk, held), pc.held(vv, held), K ** -0.5)
            most = pc.attention_bound(q[first:first + n], pc.held(kk, held), want, weight, K ** -0.5)
            assert ((o[first:first + n].double() - want).abs() <= most)[:-1].all()
        at, first = at + length, first + n


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
def test_large_scores(held):
    """Scores far beyond what exp holds without its running maximum, and a maximum that grows late."""
    plan = [(2, 600)]
    pages, rows, k, v, g = _filled(plan, 1, 64, 16, torch.bfloat16, held, spread=8.0)
    q = 20 * torch.randn(2, 1, 64, device="cuda", generator=g).bfloat16()
    _check(pages, plan, rows, k, v, q, pages.attend(q, rows), held)


@pytest.mark.parametrize("dtype,held", KINDS)
@pytest.mark.parametrize("exponent", [-100, 107])
@pytest.mark.parametrize("plan", [[(2, 600), (1, 9)], [(70, 500)]])
def test_small_and_large_values(dtype, held, exponent, plan):
    """Values up to the documented limit (7 * 2^107 < 2^110, and 2^110 * 2^8 * 600 < 2^128) under scores that grow late,
    and ones whose products with small probabilities are still normal numbers."""
    pages, rows, k, v, g = _filled(plan, 2, 64, 16, dtype, held)
    at = torch.arange(k.shape[0], device="cuda") / k.shape[0]
    k = (k.float() * (0.5 + at[:, None, None])).to(dtype)
    v = (v.float().clamp(-7, 7) * 2.0 ** exponent).to(dtype)
    lengths = [length for _, length in plan]
    whole = BatchRows(rows.page_table_SP, torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda(), rows.lengths)
    pages.write(k, v, whole)
    q = 3 * torch.randn(sum(n for n, _ in plan), 4, 64, device="cuda", generator=g).to(dtype)
    _check(pages, plan, rows, k, v, q, pages.attend(q, rows), held)


def test_refused_by_the_pages_on_the_device():
    """Page ids outside the pool, lengths past the table, ranges of rows outside the batch: NaN or nothing, as on the
    CPU (test_kv_cache.py)."""
    for held in (torch.float32, E4M3):
        rows, n = pc.rows_of([(1, 20), (1, 20), (1, 20), (1, 20)], 16, "cuda")
        rows.page_table_SP[1, 1] = n
        rows.lengths[2] = 33
        rows.query_start[4] = 9  # past the batch: no rows
        pages = pc.pages_of(n, 1, 16, 16, held, "cuda")
        x = torch.ones(4, 1, 16, device="cuda")
        pages.write(x, x, rows)
        k, _ = pages.read(rows, 20, torch.float32)
        assert torch.isnan(k[1, 16:]).all() and not torch.isnan(k[1, :16]).any() and torch.isnan(k[2]).all()
        assert torch.equal(k[0, 19], x[0]) and not k[3].any()
        out = torch.full_like(x, 7.0)
        pages.attend(x, rows, out=out)
        assert torch.isfinite(out[0]).all() and torch.isnan(out[1:3]).all() and (out[3] == 7.0).all()


@pytest.mark.parametrize("S", [3, 201])
@pytest.mark.parametrize("dtype,T", [(torch.float32, 40), (torch.bfloat16, 300)])
def test_no_rows_after_a_range_that_runs_backwards(dtype, T, S):
    """Ranges 0..T, T..0, 0..T, ...: only the first counts, and the others' pieces have no room in the workspace."""
    context = 2000
    rows, n = pc.rows_of([(T, context)] + [(0, context)] * (S - 1), 64, "cuda", n_pages=-(-context // 64) * S)
    pages = pc.pages_of(n, 2, 64, 64, dtype, "cuda")
    g = torch.Generator("cuda").manual_seed(3)
    for held in (pages.k, pages.v):
        held.copy_(torch.randn(held.shape, device="cuda", generator=g))
    new = torch.randn(2, T, 2, 64, device="cuda", generator=g).to(dtype)
    q = torch.randn(T, 4, 64, device="cuda", generator=g).to(dtype)
    pages.write(*new, rows)
    want, held = pages.attend(q, rows), (pages.k.clone(), pages.v.clone())
    rows.query_start[2::2] = 0
    pages.write(*new, rows)
    assert torch.equal(pages.k, held[0]) and torch.equal(pages.v, held[1])
    assert torch.equal(pages.attend(q, rows), want)


# Ranges of rows and the rows of the call: (query_start, T, how many sequences count).
CUT_SHORT = [([0, 2, 0], 2, 1), ([0, 1, 2, 0], 3, 2), ([0, 5, 20], 10, 1), ([0, 5, 3, 10], 10, 1), ([0, 1, 2, 3, 9], 4, 3),
             ([2, 5, 5, 4, 8], 8, 2), ([-1, 3, 6], 6, 0), ([4, 2, 6], 6, 0), ([9, 9, 9], 6, 0), ([3, 3, 3], 6, 2),
             ([0, 6, *[6] * 70, 7, *[0] * 60], 9, 72)]


@pytest.mark.parametrize("dtype,held", KINDS)
@pytest.mark.parametrize("G", [1, 8])  # (8 heads a key head: the launch that has chunks as well)
@pytest.mark.parametrize("start,T,good", CUT_SHORT, ids=[str(i) for i in range(len(CUT_SHORT))])
def test_every_row_of_no_sequence_is_cleared_and_no_other(dtype, held, G, start, T, good):
    """From the first bad range on sequences have no rows, whatever the last entry says: the rows before it are those of
    a call in which the others have none, bit for bit, and all the others are 0."""
    S, H, K, page = len(start) - 1, 2, 64, 32
    g = torch.Generator("cuda").manual_seed(1)
    table = torch.randperm(2 * S, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(S, 2).cuda()
    pages = pc.pages_of(2 * S, H, page, K, held, "cuda")
    lengths = torch.tensor([30 + s % 35 for s in range(S)], dtype=torch.int32, device="cuda")
    new = torch.randn(2, int(lengths.sum()), H, K, device="cuda", generator=g).to(dtype)
    as_start = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    pages.write(*new, BatchRows(table, as_start([0] + lengths.cumsum(0).tolist()), lengths))
    q = torch.randn(T, H * G, K, device="cuda", generator=g).to(dtype)
    end = start[good] if good else 0
    clean = BatchRows(table, as_start(start[:good + 1] + [end] * (S - good) if good else [0] * (S + 1)), lengths)
    want = torch.zeros_like(q)
    pages.attend(q, clean, out=want)
    for _ in range(3):
        dirty = torch.full_like(q, 7.0)  # what the next allocation of this size holds
        del dirty
        got = pages.attend(q, BatchRows(table, as_start(start), lengths))
        assert torch.equal(got, want)
    first = start[0] if good else 0
    assert not want[:first].any() and not want[end:].any() and (end == first or want[first:end].abs().sum(-1).min() > 0)


def test_rows_of_nothing():
    rows, n = pc.rows_of([(2, 1), (1, 0)], 16, "cuda")
    pages = pc.pages_of(n, 1, 16, 16, torch.float32, "cuda")
    k = torch.ones(3, 1, 16, device="cuda")
    pages.write(k, 2 * k, rows)
    out = torch.full((5, 1, 16), 7.0, device="cuda")
    q = torch.ones(5, 1, 16, device="cuda")
    assert pages.attend(q, rows, out=out)[:, 0, 0].tolist() == [0.0, 2.0, 0.0, 7.0, 7.0]
    assert pages.attend(q, rows)[:, 0, 0].tolist() == [0.0, 2.0, 0.0, 0.0, 0.0]
    rows.query_start += 1  # a row before the first sequence
    assert pages.attend(q, rows)[:, 0, 0].tolist() == [0.0, 0.0, 2.0, 0.0, 0.0]
    assert pages.attend(q[:0], rows).shape == (0, 1, 16)


def test_operands_of_any_stride():
    plan = [(5, 90), (1, 33)]
    pages, rows, k, v, g = _filled(plan, 2, 64, 16, torch.bfloat16, torch.bfloat16)
    wide = torch.randn(6, 3, 4, 64, device="cuda", generator=g).bfloat16()
    q = wide[:, 1]
    assert not q.is_contiguous()
    assert torch.equal(pages.attend(q, rows), pages.attend(q.contiguous(), rows))
    flat = torch.empty(q.numel() + 1, device="cuda", dtype=q.dtype)
    off = flat[1:].view(q.shape).copy_(q)
    assert off.data_ptr() % 16 and torch.equal(pages.attend(off, rows), pages.attend(q.contiguous(), rows))
    kn, vn = wide[:, 0, :2], wide[:, 2, 2:]
    pages.write(kn, vn, rows)
    kr, vr = pages.read(rows, 90)
    assert torch.equal(kr[0, 85:], kn[:5]) and torch.equal(vr[0, 85:], vn[:5])
    assert torch.equal(kr[1, 32], kn[5]) and torch.equal(vr[1, 32], vn[5])


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
def test_captured_step_follows_its_rows(held):
    """A write and an attention captured once: each replay writes and reads where the index tensors then say, and
    eager work between the replays changes nothing."""
    H, K, page, S = 2, 64, 16, 3
    cache = PagedKVCache(1, 160, page, H, K, dtype=held, device="cuda")
    pages = cache.layer(0)
    twin = PagedKVCache(1, 160, page, H, K, dtype=held, device="cuda").layer(0)
    seqs = [cache.add() for _ in range(S)]
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda T, heads: torch.randn(T, heads, K, device="cuda", generator=g).bfloat16()
    rows = cache.extend({s: 30 + 600 * s for s in seqs})
    k, v = rand(int(rows.query_start[-1]), H), rand(int(rows.query_start[-1]), H)
    pages.write(k, v, rows)
    twin.write(k, v, rows)
    static = BatchRows(torch.zeros(S, 100, dtype=torch.int32, device="cuda"), torch.zeros(S + 1, dtype=torch.int32, device="cuda"),
                       torch.zeros(S, dtype=torch.int32, device="cuda"))
    T = 9
    q, k, v = rand(T, 2 * H), rand(T, H), rand(T, H)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pages.attend(q, static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.write(k, v, static)
        out = pages.attend(q, static)
    for step in ({seqs[0]: 1, seqs[1]: 3, seqs[2]: 2}, {seqs[0]: 2, seqs[1]: 1, seqs[2]: 1}, {seqs[0]: 5, seqs[1]: 0, seqs[2]: 4}):
        rows = cache.extend(step)
        static.page_table_SP[:, :rows.page_table_SP.shape[1]] = rows.page_table_SP
        static.query_start.copy_(rows.query_start)
        static.lengths.copy_(rows.lengths)
        for t, heads in ((q, 2 * H), (k, H), (v, H)):
            t.copy_(rand(T, heads))
        graph.replay()
        twin.write(k, v, rows)
        want = twin.attend(q, static)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(pages.read(rows, 1300), twin.read(rows, 1300)))


def test_calls_on_two_streams():
    plan = [(1, 5000), (1, 3000)]
    pages, rows, k, v, g = _filled(plan, 2, 64, 64, torch.bfloat16, torch.bfloat16, max_new=1)
    qs = [torch.randn(2, 2, 64, device="cuda", generator=g).bfloat16() for _ in range(2)]
    want = [pages.attend(q, rows) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for q, stream in zip(qs, streams):
            with torch.cuda.stream(stream):
                got.append(pages.attend(q, rows))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes (and 2^31 elements): its last pages are written and read."""
    H, K, page = 8, 128, 256
    n = (1 << 31) // (H * K * page) + 3  # 8195 pages of 2^18 elements
    pages = pc.pages_of(n, H, page, K, torch.bfloat16, "cuda")
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    rows = BatchRows(as_int([[n - 2, n - 1], [0, 1]]), as_int([0, 300, 310]), as_int([300, 10]))
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(310, H, K, device="cuda", generator=g).bfloat16() for _ in range(2))
    pages.write(k, v, rows)
    assert torch.equal(pages.k[n - 2].transpose(0, 1), k[:256])
    assert torch.equal(pages.v[n - 1, :, :, :44].permute(2, 0, 1), v[256:300])
    kr, vr = pages.read(rows, 300)
    assert torch.equal(kr[0], k[:300]) and torch.equal(vr[0], v[:300]) and torch.equal(kr[1, :10], k[300:])
    q = torch.randn(310, H, K, device="cuda", generator=g).bfloat16()
    _check(pages, [(300, 300), (10, 10)], rows, k, v, q, pages.attend(q, rows), torch.bfloat16)
