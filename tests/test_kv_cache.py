"""The paged cache on the CPU: what it holds, what its attention gives, and what it refuses.  (The same calls on the
GPU: test_gpu_kv_cache.py.)"""

import math

import pytest
import torch

import paged_check as pc
from abacus_amd import _lib
from abacus_amd.kv_cache import E4M3, BatchRows, KVPages, PagedKVCache

PLANS = [[(1, 1)], [(3, 3), (1, 40), (0, 17), (5, 21)], [(2, 0 + 2), (0, 0), (33, 50)]]


@pytest.mark.parametrize("held", [torch.float32, torch.bfloat16, E4M3])
@pytest.mark.parametrize("plan", PLANS)
def test_write_read_and_attend_match_the_formulas(plan, held):
    H, K, page, G = 2, 32, 16, 2
    dtype = torch.bfloat16 if held == torch.bfloat16 else torch.float32
    g = torch.Generator().manual_seed(3)
    rows, n = pc.rows_of(plan, page, "cpu")
    whole, _ = pc.rows_of([(length, length) for _, length in plan], page, "cpu")
    pages = pc.pages_of(n, H, page, K, held, "cpu", fill=0xff if held == E4M3 else math.nan)
    total, new = sum(length for _, length in plan), sum(n for n, _ in plan)
    k, v = (torch.randn(total, H, K, generator=g).to(dtype) for _ in range(2))
    k[0, 0] = 0.0
    pages.write(k, v, whole)
    q = torch.randn(new, H * G, K, generator=g).to(dtype)
    longest = max(length for _, length in plan)
    kr, vr = pages.read(rows, longest, torch.float32 if held == E4M3 else None)
    o = pages.attend(q, rows)
    at = first = 0
    for s, (n_new, length) in enumerate(plan):
        ks, vs = pc.held(k[at:at + length], held), pc.held(v[at:at + length], held)
        assert torch.equal(kr[s, :length].double(), ks) and torch.equal(vr[s, :length].double(), vs)
        assert not kr[s, length:].any() and not vr[s, length:].any()
        if n_new:
            qs = q[first:first + n_new]
            want, weight = pc.attention(qs, ks, vs, 1 / math.sqrt(K))
            off = (o[first:first + n_new].double() - want).abs()
            assert (off <= pc.attention_bound(qs, ks, want, weight, 1 / math.sqrt(K))).all()
        at, first = at + length, first + n_new


def test_positions():
    rows, _ = pc.rows_of([(2, 9), (0, 4), (1, 1), (3, 2)], 16, "cpu")
    assert rows.positions(7).tolist() == [7, 8, 0, 0, 0, 1, 0]  # a row before position 0, and one of no sequence: 0


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("start,lengths,T,want", [
    ([0, 1, 0, 0], [5, 9, 9], 1, [4]),
    ([0, 2, 0, 3], [7, 8, 9], 3, [5, 6, 0]),
    ([0, 2, 2, 5], [7, 8, 9], 4, [5, 6, 0, 0]),
    ([-1, 2, 3], [4, 4], 3, [0, 0, 0]),
    ([9, 9, 9], [4, 4], 3, [0, 0, 0]),
    ([2, 1, 3], [4, 4], 3, [0, 0, 0]),
    ([1, 1, 3, 3], [4, 6, 8], 4, [0, 4, 5, 0]),
    ([0, 3], [2], 3, [0, 0, 1]),
    ([0, 2], [2**31 - 1], 2, [2**31 - 3, 2**31 - 2]),
    ([0, 2], [-(2**31)], 2, [0, 0]),
    ([0, *range(300, 600, 2), 7, *range(598, 700, 2)], [1000 + s for s in range(202)], 700,
     [*range(700, 1000), *(998 + s + j for s in range(1, 150) for j in (0, 1)), *[0] * 102])])
def test_positions_end_where_the_ranges_do(device, start, lengths, T, want):
    """From the first range that runs backwards or past the rows on sequences have none."""
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    rows = BatchRows(torch.zeros(len(lengths), 1, dtype=torch.int32, device=device), as_int(start), as_int(lengths))
    got = rows.positions(T)
    assert got.dtype == torch.int64 and got.tolist() == want and rows.positions(0).shape == (0,)


def test_rows_of_nothing():
    """Rows of no sequence are 0, or left alone in `out`; rows that see nothing are 0."""
    rows, n = pc.rows_of([(2, 1), (1, 0)], 16, "cpu")
    pages = pc.pages_of(n, 1, 16, 16, torch.float32, "cpu")
    k = torch.ones(3, 1, 16)
    pages.write(k, 2 * k, rows)
    out = torch.full((5, 1, 16), 7.0)
    got = pages.attend(torch.ones(5, 1, 16), rows, out=out)
    assert got is out
    assert got[:, 0, 0].tolist() == [0.0, 2.0, 0.0, 7.0, 7.0]
    assert pages.attend(torch.ones(5, 1, 16), rows)[:, 0, 0].tolist() == [0.0, 2.0, 0.0, 0.0, 0.0]


@pytest.mark.parametrize("held", [torch.float32, E4M3])
def test_pages_outside_the_pool_and_lengths_past_the_table(held):
    rows, n = pc.rows_of([(1, 20), (1, 20), (1, 20)], 16, "cpu")
    rows.page_table_SP[1, 1] = n
    rows.lengths[2] = 33
    pages = pc.pages_of(n, 1, 16, 16, held, "cpu")
    x = torch.ones(3, 1, 16)
    pages.write(x, x, rows)
    k, _ = pages.read(rows, 20, torch.float32)
    assert torch.isnan(k[1, 16:]).all() and not torch.isnan(k[1, :16]).any() and torch.isnan(k[2]).all()
    assert torch.equal(k[0, 19], x[0])
    o = pages.attend(x, rows)
    assert torch.isfinite(o[0]).all() and torch.isnan(o[1:]).all()


def test_rows_are_not_copied():
    """A call reads what the caller's tensors hold then, so a strided view, which would be copied, is refused."""
    table, start, lengths = torch.zeros(2, 8, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    assert BatchRows(table, start, lengths).page_table_SP.data_ptr() == table.data_ptr()
    for bad in ((table[:, :4], start, lengths), (table, torch.zeros(6, dtype=torch.int32)[::2], lengths),
                (table, start, torch.ones(4, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError, match="contiguous"):
            BatchRows(*bad)


def test_no_gradient():
    """Rows that ask for a gradient are refused, not cut off from it silently."""
    rows, n = pc.rows_of([(2, 5)], 16, "cpu")
    pages = pc.pages_of(n, 2, 16, 16, torch.float32, "cpu")
    x = torch.ones(2, 2, 16)
    leaf = x.clone().requires_grad_()
    for call in (lambda: pages.attend(leaf, rows), lambda: pages.write(leaf, x, rows), lambda: pages.write(x, leaf, rows)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_no_gradient_of_pages_outputs_and_forward_mode(device):
    """What a call would drop silently is refused: the gradient of pages and of `out`, and tangents, which no_grad keeps."""
    forward_ad = torch.autograd.forward_ad
    rows, n = pc.rows_of([(2, 5)], 16, device)
    pages = pc.pages_of(n, 2, 16, 16, torch.float32, device)
    x = torch.ones(2, 2, 16, device=device)
    leaves = [KVPages(pages.k.clone().requires_grad_(), pages.v), KVPages(pages.k, pages.v.clone().requires_grad_())]
    out = torch.empty_like(x).requires_grad_()
    for call in (*(lambda p=p: p.attend(x, rows) for p in leaves), *(lambda p=p: p.read(rows, 5) for p in leaves),
                 *(lambda p=p: p.write(x, x, rows) for p in leaves), lambda: pages.attend(x, rows, out=out)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad():
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        held = KVPages(pages.k, forward_ad.make_dual(pages.v, pages.v))
        for call in (lambda: pages.attend(dual, rows), lambda: pages.write(dual, x, rows), lambda: pages.write(x, dual, rows),
                     lambda: held.attend(x, rows), lambda: held.read(rows, 5), lambda: held.write(x, x, rows)):
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()
        pages.attend(x, rows)


def test_no_rows_after_a_range_that_runs_backwards():
    """Overlapping ranges would be more rows than the call has: what comes after the bad range has none."""
    rows, n = pc.rows_of([(2, 2), (0, 0), (2, 2)], 16, "cpu")
    rows.query_start.copy_(torch.tensor([0, 2, 0, 2]))
    pages = pc.pages_of(n, 1, 16, 16, torch.float32, "cpu")
    x = torch.ones(2, 1, 16)
    pages.write(x, 3 * x, rows)
    _, v = pages.read(rows, 2)
    assert (v[0] == 3.0).all() and not v[2].any()
    assert (pages.attend(x, rows) == 3.0).all()


@pytest.mark.parametrize("start,T,valid", [([0, 2, 0], 2, (0, 2)), ([0, 5, 20], 10, (0, 5)), ([0, 5, 3, 10], 10, (0, 5)),
                                           ([2, 5, 5, 4, 8], 8, (2, 5)), ([-1, 3, 6], 6, (0, 0)), ([4, 2, 6], 6, (0, 0))])
def test_rows_of_no_sequence_are_cleared_and_no_others(start, T, valid):
    S = len(start) - 1
    table = torch.arange(S, dtype=torch.int32)[:, None]
    pages = pc.pages_of(S, 1, 16, 16, torch.float32, "cpu", fill=1.0)
    rows = BatchRows(table, torch.tensor(start, dtype=torch.int32), torch.full((S,), 16, dtype=torch.int32))
    got = pages.attend(torch.ones(T, 1, 16), rows)
    want = torch.zeros(T, 1, 16)
    want[valid[0]:valid[1]] = 1.0
    assert torch.allclose(got, want, rtol=0, atol=17 * 2.0 ** -24)  # a mean of 16 ones


def test_nonfinite_rows_of_a_quantised_cache():
    rows, n = pc.rows_of([(3, 3)], 16, "cpu")
    pages = pc.pages_of(n, 2, 16, 16, E4M3, "cpu")
    k, v = torch.ones(3, 2, 16), torch.ones(3, 2, 16)
    k[1, 0, 3] = math.inf
    v[2, 1, 0] = math.nan
    pages.write(k, v, rows)
    kr, vr = pages.read(rows, 3)
    bad = torch.tensor([[False, False], [True, False], [False, True]])
    for x in (kr, vr):
        assert torch.equal(torch.isnan(x[0]).all(-1), bad) and torch.equal(torch.isnan(x[0]).any(-1), bad)
    o = pages.attend(torch.ones(3, 2, 16), rows)
    assert torch.equal(torch.isnan(o).all(-1), torch.tensor([[False, False], [True, False], [True, True]]))


def test_refusals():
    k = torch.zeros(4, 2, 16, 32)
    v = torch.zeros(4, 2, 32, 16)
    pages = KVPages(k, v)
    rows, _ = pc.rows_of([(2, 5)], 16, "cpu", n_pages=4)
    x = torch.zeros(2, 2, 32)
    with pytest.raises(ValueError):
        KVPages(k, k)
    with pytest.raises(ValueError, match="page_size"):
        KVPages(torch.zeros(4, 2, 24, 32), torch.zeros(4, 2, 32, 24))
    with pytest.raises(ValueError, match="head_dim"):
        KVPages(torch.zeros(4, 2, 16, 40), torch.zeros(4, 2, 40, 16))
    with pytest.raises(ValueError, match="head_dim"):
        KVPages(torch.zeros(4, 2, 16, 144), torch.zeros(4, 2, 144, 16))
    with pytest.raises(TypeError):
        KVPages(k.half(), v.half())
    with pytest.raises(ValueError, match="scale"):
        KVPages(k.to(E4M3), v.to(E4M3))
    with pytest.raises(ValueError, match="contiguous"):
        KVPages(k.transpose(0, 1).contiguous().transpose(0, 1), v)
    with pytest.raises(ValueError):
        pages.write(x[:, :1], x[:, :1], rows)
    with pytest.raises(ValueError):
        pages.write(x, x[:1], rows)
    with pytest.raises(TypeError):
        pages.write(x.bfloat16(), x.bfloat16(), rows)
    with pytest.raises(TypeError):
        pages.read(rows, 5, torch.bfloat16)
    with pytest.raises(ValueError):
        pages.read(rows, -1)
    with pytest.raises(ValueError, match="multiple"):
        pages.attend(torch.zeros(2, 3, 32), rows)
    with pytest.raises(ValueError, match="scale"):
        pages.attend(x, rows, scale=0.0)
    with pytest.raises(ValueError, match="scale"):
        pages.attend(x, rows, scale=math.nan)
    with pytest.raises(ValueError, match="out"):
        pages.attend(x, rows, out=torch.zeros(2, 2, 64)[..., :32])
    with pytest.raises(ValueError, match="int32"):
        BatchRows(rows.page_table_SP.long(), rows.query_start, rows.lengths)
    with pytest.raises(ValueError, match="shape"):
        BatchRows(rows.page_table_SP, rows.query_start[:1], rows.lengths)
    with pytest.raises(ValueError, match="max_new"):
        BatchRows(rows.page_table_SP, rows.query_start, rows.lengths, max_new=0)


@pytest.mark.parametrize("held", [torch.float32, E4M3])
def test_pages_that_were_given_other_memory_are_refused(held):
    """Calls take the addresses that the pages had when they were checked."""
    rows, n = pc.rows_of([(2, 5)], 16, "cpu")
    x = torch.ones(2, 2, 16)
    for name in ("k", "v", *(("k_scale", "v_scale") if held == E4M3 else ())):
        pages = pc.pages_of(n, 2, 16, 16, held, "cpu")
        pages.write(x, x, rows)
        tensor = getattr(pages, name)
        before, tensor.data = tensor.data, tensor.data.view(torch.uint8).clone().view(tensor.dtype)
        for call in (lambda: pages.attend(x, rows), lambda: pages.write(x, x, rows), lambda: pages.read(rows, 5)):
            with pytest.raises(RuntimeError, match="no longer"):
                call()
        tensor.data = before
        pages.read(rows, 5)


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.BF16])
def test_more_blocks_than_a_launch_holds_are_refused(dtype):
    """2^30 (row, head) pairs of single tokens, 256 threads each: a launch has at most 2^32 threads."""
    T = S = 1 << 20
    assert _lib.query("abacus_paged_attention_ws_bytes", T, 1024, 1024, 64, dtype, dtype, S, 1, 16, 1) == 0
    with pytest.raises(RuntimeError, match="too many"):
        _lib.call("abacus_paged_attention", 16, T, 1024, 1024, 64, dtype, 16, 16, 16, S, 1, 16, 1, dtype, 16, 16, None, None, 0.125,
                  1, 1, 16, None, 0, None)


def test_bookkeeping():
    cache = PagedKVCache(2, 5, 16, 1, 16, dtype=torch.float32)
    a, b = cache.add(), cache.add()
    rows = cache.extend({a: 17, b: 16})
    assert rows.query_start.tolist() == [0, 17, 33] and rows.lengths.tolist() == [17, 16] and rows.max_new == 17
    assert cache.free_pages == 2 and len({*rows.page_table_SP.flatten().tolist()}) >= 3
    with pytest.raises(RuntimeError, match="free pages"):
        cache.extend({a: 60})  # 77 tokens: 5 pages, 3 more than it has
    assert cache.length(a) == 17 and cache.free_pages == 2  # nothing was taken
    cache.truncate(a, 16)
    assert cache.free_pages == 3 and cache.length(a) == 16
    with pytest.raises(ValueError):
        cache.truncate(a, 17)
    cache.free(b)
    assert cache.free_pages == 4
    x = torch.randn(20, 1, 16)
    rows = cache.extend({a: 20})
    cache.layer(1).write(x, -x, rows)
    k, v = cache.layer(1).read(rows, 36)
    assert torch.equal(k[0, 16:], x) and torch.equal(v[0, 16:], -x)
    assert not cache.layer(0).read(rows, 36)[0].any()
