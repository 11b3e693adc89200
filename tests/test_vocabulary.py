"""linear_cross_entropy and embedding (abacus_amd.vocabulary): refusals and the CPU's steps, and on the GPU the kernels
against 64-bit sums.

Tolerances count roundings, each half a step of its type (u = eps / 2: bf16 2^-8, fp32 2^-24), times what is summed:
a sum of n products by matrix instructions adds n / 16 (bf16) or n / 2 (fp32) times in fp32, and 64 more for its slices
and the instructions' own order.  A logit is off by that of its row (delta); the loss by twice that and what the
exponentials of numbers up to the largest logit lose in fp32; P by its rounding, the same share of the probability, and
in bf16 half a step of the 10-bit exponentials (2^-11); a gradient by its rounding, its products' P and its sum.
"""

import ctypes

import pytest
import torch
import torch.nn.functional as F
import torch.utils.checkpoint

from abacus_amd import vocabulary
from abacus_amd.vocabulary import embedding, linear_cross_entropy

DTYPES = [torch.bfloat16, torch.float32]
IDS = ["bf16", "fp32"]


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _adds(n, dtype):
    return (n / (16 if dtype == torch.bfloat16 else 2) + 64) * 2.0 ** -24


def _loss_case(T, D, V, dtype, ignored=0.0, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed + T + 7 * D + 13 * V)
    x = torch.randn(T, D, device=device, generator=g).to(dtype)
    w = (torch.randn(D, V, device=device, generator=g) * 2.5 / D ** 0.5).to(dtype)
    t = torch.randint(0, V, (T,), device=device, generator=g)
    t[torch.rand(T, device=device, generator=g) < ignored] = -100
    return x, w, t


def _check_loss(x, w, t, reduction, got, grads, row_grad=None):
    """got and grads (dx, dw, None: not looked at) against 64 bits, value by value."""
    dtype, V = x.dtype, w.shape[1]
    xd, wd = x.detach().double(), w.detach().double()
    kept = t != -100
    n = int(kept.sum())
    l = xd @ wd
    delta = _adds(xd.shape[1], dtype) * (xd.abs() @ wd.abs()).amax(-1)
    far = 2 * delta + 2.0 ** -22 * (4 + l.abs().amax(-1))
    lse = torch.logsumexp(l, -1)
    at = torch.where(kept, t, 0)[:, None]
    rows = torch.where(kept, lse - l.gather(1, at)[:, 0], 0.0)
    far = torch.where(kept, far, 0.0)
    if reduction == "none":
        assert got.shape == t.shape and torch.all((got.double() - rows).abs() <= far + 2.0 ** -24 * rows.abs())
        s = torch.where(kept, row_grad.double(), 0.0) if row_grad is not None else kept.double()
    else:
        s = kept.double() / (n if reduction == "mean" else 1)
        want = rows.sum() / (n if reduction == "mean" else 1)
        if n == 0 and reduction == "mean":
            assert torch.isnan(got)
            s = torch.zeros_like(s)
        else:
            assert abs(float(got) - float(want)) <= float((far * s).sum()) + 2.0 ** -22 * abs(float(want))
    if grads is None:
        return
    p = torch.exp(l - lse[:, None])
    P = (p - torch.zeros_like(p).scatter_(1, at, 1.0)) * s[:, None]
    off = _u(dtype) * P.abs() + p * (far + (2.0 ** -11 if dtype == torch.bfloat16 else 0.0))[:, None] * s.abs()[:, None]
    for d, a, b, summed in ((grads[0], None, wd.t(), V), (grads[1], xd.t(), None, max(n, 1))):
        if d is None:
            continue
        assert d.dtype == dtype
        of = lambda m: m @ b.abs() if a is None else a.abs() @ m
        want = P @ b if a is None else a @ P
        bound = 1.01 * (_u(dtype) * want.abs() + of(off) + (_adds(summed, dtype) + 2.0 ** -22) * of(P.abs()))
        err = (d.double() - want).abs() - bound
        assert torch.all(err <= 0), f"off by {float((d.double() - want).abs().max()):.3g}, {float(err.max()):.3g} too much"


# ---------------------------------------------------------------- refusals and the CPU


def test_linear_cross_entropy_refusals():
    x, w, t = _loss_case(4, 8, 11, torch.float32, device="cpu")
    for args, error in (((x, w[:7], t), ValueError), ((x, w.bfloat16(), t), TypeError), ((x, w, t[:3]), ValueError),
                        ((x, w, t.int()), ValueError), ((x, w[0], t), ValueError), ((x[0, 0], w, t), ValueError),
                        ((x, w[:, :0], t), ValueError)):
        with pytest.raises(error):
            linear_cross_entropy(*args)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="max")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy_on_cpu_is_torchs(reduction):
    x, w, t = _loss_case(6, 8, 11, torch.float64, 0.3, device="cpu")
    x, w = x.view(2, 3, 8).requires_grad_(), w.requires_grad_()
    got = linear_cross_entropy(x, w, t.view(2, 3), reduction=reduction)
    want = F.cross_entropy((x @ w).view(6, 11), t, reduction=reduction)
    assert torch.allclose(got.reshape(-1), want.reshape(-1), rtol=1e-12)
    assert torch.autograd.gradcheck(lambda x, w: linear_cross_entropy(x, w, t.view(2, 3), reduction=reduction), (x, w))


def test_embedding_refusals_and_cpu():
    w = torch.randn(5, 3, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([[0, 4], [-1, 0]])
    assert torch.equal(embedding(t, w), w[t]) and torch.equal(embedding(t, w, 2.0), w[t] * 2.0)
    assert torch.autograd.gradcheck(lambda w: embedding(t, w, 0.5), (w,))
    for args in ((t.int(), w), (t, w[0]), (t, w[:0])):
        with pytest.raises(ValueError):
            embedding(*args)


# ---------------------------------------------------------------- the loss on the GPU

# rows of each path: one, a few (at most 32, 64), thin tiles, tiles and a ragged end; D and V of any size and alignment
SHAPES = [(1, 8, 5), (1, 512, 2000), (3, 64, 64), (7, 9, 65), (24, 100, 1000), (31, 1000, 5003), (32, 2048, 800), (33, 16, 100),
          (50, 520, 3200), (64, 136, 3001), (65, 64, 50), (128, 72, 257), (129, 65, 255), (300, 512, 1003), (513, 1000, 2049),
          (700, 260, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,D,V", SHAPES)
def test_linear_cross_entropy_matches_64_bits(T, D, V, dtype):
    for ignored, reduction in ((0.0, "mean"), (0.4, "mean"), (0.4, "sum"), (0.3, "none"), (1.0, "mean")):
        x, w, t = _loss_case(T, D, V, dtype, ignored)
        x, w = x.requires_grad_(), w.requires_grad_()
        got = linear_cross_entropy(x, w, t, reduction=reduction)
        assert got.dtype == torch.float32
        g = torch.rand(T, device="cuda") - 0.3 if reduction == "none" else None
        grads = torch.autograd.grad(got, (x, w), g)
        _check_loss(x, w, t, reduction, got.detach(), grads, g)
        assert torch.all(grads[0][t == -100] == 0)
        with torch.no_grad():
            again = linear_cross_entropy(x, w, t, reduction=reduction)
        assert torch.equal(again, got.detach()) or torch.isnan(got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_cross_entropy_of_many_rows_and_few_classes(dtype):
    x, w, t = _loss_case(20011, 12, 3, dtype, 0.1)
    x, w = x.requires_grad_(), w.requires_grad_()
    got = linear_cross_entropy(x, w, t)
    _check_loss(x, w, t, "mean", got.detach(), torch.autograd.grad(got, (x, w)))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 150])
def test_linear_cross_entropy_ignores_any_index(T):
    """A class as the ignored one, and a number outside int32: the bits of the same rows ignored by -100."""
    x, w, t = _loss_case(T, 64, 300, torch.bfloat16, 0.3)
    x, w = x.requires_grad_(), w.requires_grad_()
    for index in (0, 299, -(1 << 40)):
        kept = torch.where(t == index, -100, t)
        want = linear_cross_entropy(x, w, kept)
        got = linear_cross_entropy(x, w, torch.where(kept == -100, index, kept), ignore_index=index)
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, (x, w)), torch.autograd.grad(want, (x, w))))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 40001), (torch.float32, 20000)], ids=IDS)
@pytest.mark.parametrize("ignored", [0.0, 0.3, 1.0])
def test_linear_cross_entropy_over_chunks(dtype, V, ignored):
    """P past its chunk (1 GiB): two chunks of rows, or rows for the first alone."""
    x, w, t = _loss_case(15000, 64, V, dtype, ignored)
    x, w = x.requires_grad_(), w.requires_grad_()
    got = linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(got, (x, w))
    some = torch.arange(0, 15000, 97, device="cuda")
    n = max(1, int((t != -100).sum()))
    # a part of the rows' dx, and dw by columns, as 64-bit logits of all would not fit beside
    _check_loss(x.detach()[some], w, t[some], "none", linear_cross_entropy(x[some].detach(), w.detach(), t[some], reduction="none"),
                (dx[some], None), torch.full((len(some),), 1.0 / n, device="cuda"))
    xd, wd = x.detach().double(), w.detach().double()
    kept = (t != -100).double() / n
    dw_want, size, off = (torch.zeros(64, V, dtype=torch.float64, device="cuda") for _ in range(3))
    for a in range(0, 15000, 3000):
        l = xd[a:a + 3000] @ wd
        p = torch.softmax(l, -1) * kept[a:a + 3000, None]
        P = p.clone().scatter_add_(1, t[a:a + 3000].clamp(min=0)[:, None], -kept[a:a + 3000, None])
        far = 2 * _adds(64, dtype) * (xd[a:a + 3000].abs() @ wd.abs()).amax() + 2.0 ** -22 * (4 + l.abs().amax())
        dw_want += xd[a:a + 3000].t() @ P
        size += xd[a:a + 3000].abs().t() @ P.abs()
        off += xd[a:a + 3000].abs().t() @ (_u(dtype) * P.abs() + p * (far + (2.0 ** -11 if dtype == torch.bfloat16 else 0.0)))
    bound = 1.01 * (_u(dtype) * dw_want.abs() + off + (_adds(15000, dtype) + 2.0 ** -22) * size)
    assert torch.all((dw.double() - dw_want).abs() <= bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T", [20, 300])
def test_linear_cross_entropy_layouts_and_incoming_gradient(T, dtype):
    """Rows and weights that are parts of larger tensors, turned ones, leading dimensions, one gradient alone, a loss
    that is scaled, and a graph whose gradients are taken twice."""
    x, w, t = _loss_case(T, 96, 700, dtype, 0.2)
    want = linear_cross_entropy(x.requires_grad_(), w.requires_grad_(), t)
    dx, dw = torch.autograd.grad(want, (x, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, (x, w)), (dx, dw)))
    wide = torch.full((T, 101), float("nan"), device="cuda", dtype=dtype)
    wide[:, 3:99] = x.detach()
    views = [wide[:, 3:99], x.detach().t().contiguous().t(), x.detach().view(4, T // 4, 96)]
    flat = torch.zeros(96 * 700 + 1, device="cuda", dtype=dtype)
    flat[1:] = w.detach().reshape(-1)
    weights = [flat[1:].view(96, 700), w.detach().t().contiguous().t()]
    for xv in views:
        for wv in weights:
            a, b = xv.detach().requires_grad_(), wv.detach().requires_grad_()
            got = linear_cross_entropy(a, b, t.view(a.shape[:-1]))
            da, db = torch.autograd.grad(got, (a, b))
            assert torch.equal(got, want) and torch.equal(da.reshape(T, 96), dx) and torch.equal(db, dw)
    one, = torch.autograd.grad(linear_cross_entropy(x, w.detach(), t), x)
    other, = torch.autograd.grad(linear_cross_entropy(x.detach(), w, t), w)
    assert torch.equal(one, dx) and torch.equal(other, dw)
    # the backward's product with 0.37: one rounding more
    got = torch.autograd.grad(linear_cross_entropy(x, w, t) * 0.37, (x, w))
    for a, b in zip(got, (dx, dw)):
        assert torch.all((a.double() - 0.37 * b.double()).abs() <= (_u(dtype) + 2.0 ** -23) * 0.37 * b.double().abs() + 1e-38)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T", [12, 200])
def test_linear_cross_entropy_of_odd_values(T, dtype):
    """What ignored rows hold reaches nothing; a target outside the vocabulary and a NaN spoil their row alone; logits of -inf
    over whole strips are no probability; large logits."""
    x, w, t = _loss_case(T, 64, 600, dtype, 0.3)
    clean = linear_cross_entropy(x.requires_grad_(), w.requires_grad_(), t)
    grads = torch.autograd.grad(clean, (x, w))
    dirty = x.detach().clone()
    dirty[t == -100] = torch.tensor([float("nan"), float("inf")] * 32, device="cuda", dtype=dtype)
    dirty.requires_grad_()
    got = linear_cross_entropy(dirty, w, t)
    assert torch.equal(got, clean) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, (dirty, w)), grads))

    rows = linear_cross_entropy(x.detach(), w.detach(), t, reduction="none")
    t2, x2 = t.clone(), x.detach().clone()
    t2[:4] = torch.tensor([600, -1, -101, 1 << 40], device="cuda")
    x2[5] = float("nan")
    t2[5] = 3
    odd = linear_cross_entropy(x2, w.detach(), t2, reduction="none")
    assert torch.isnan(odd[:4]).all() and torch.isnan(odd[5]) and torch.equal(odd[6:], rows[6:]) and torch.equal(odd[4], rows[4])
    assert torch.isnan(linear_cross_entropy(x2, w.detach(), t2))

    x3 = x.detach().abs() + 0.1
    w3 = w.detach().clone()
    w3[:, :300] = -float("inf")
    t3 = torch.full((T,), 450, device="cuda")
    w4 = w.detach()[:, 300:].contiguous()
    a = linear_cross_entropy(x3, w3, t3, reduction="none")
    l = x3.double() @ w4.double()
    far = 2 * _adds(64, dtype) * (x3.double().abs() @ w4.double().abs()).amax(-1) + 2.0 ** -22 * (4 + l.abs().amax(-1))
    assert torch.all((a.double() - (torch.logsumexp(l, -1) - l[:, 150])).abs() <= far)

    big = (w.detach().double() * 200).to(dtype)  # logits of hundreds: probabilities of 0 and 1
    _check_loss(x.detach(), big, t, "none", linear_cross_entropy(x.detach(), big, t, reduction="none"), None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T", [30, 60, 200])
def test_linear_cross_entropy_of_the_largest_logits(T, dtype):
    """Logits of up to 10^8, 2^18 and more apart: probabilities are 0 and 1, every product and sum below is exact, and the gradients
    are 64 bits' rounded once."""
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randint(-2, 3, (T, 8), device="cuda", generator=g).to(dtype)
    x[:, 0] = torch.tensor([-2, -1, 1, 2], device="cuda").repeat(T // 4 + 1)[:T].to(dtype)
    w = torch.randint(-4, 5, (8, 200), device="cuda", generator=g).to(dtype)
    w[0] = (torch.randperm(200, device="cuda", generator=g) * 2.0 ** 18).to(dtype)
    t = torch.randint(0, 200, (T,), device="cuda", generator=g)
    x, w = x.requires_grad_(), w.requires_grad_()
    got = torch.autograd.grad(linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
    a, b = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want = torch.autograd.grad(F.cross_entropy(a @ b, t, reduction="sum"), (a, b))
    assert all(torch.equal(v, d.to(dtype)) for v, d in zip(got, want))


@pytest.mark.gpu
def test_linear_cross_entropy_of_no_rows():
    w = torch.randn(8, 16, device="cuda", requires_grad=True)
    x = torch.randn(0, 8, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert torch.isnan(linear_cross_entropy(x, w, t)) and linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
    assert dx.shape == (0, 8) and torch.all(dw == 0)
    with pytest.raises(TypeError):
        linear_cross_entropy(torch.randn(2, 8, device="cuda").half(), w.half(), torch.zeros(2, dtype=torch.int64, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [10, 70])
def test_linear_cross_entropy_past_32_bits(T):
    """w and its gradient of more than 2^31 values (and 2^32 bytes): the last columns against 64 bits."""
    D, V = 2048, 1_050_000
    x, _, t = _loss_case(T, D, 8, torch.bfloat16)
    w = torch.empty(D, V, dtype=torch.bfloat16, device="cuda").normal_(0.0, 0.04, generator=torch.Generator(device="cuda").manual_seed(3))
    t = V - 1 - t
    xs, ws = x.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(xs, ws, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (xs, ws))
    lse = torch.full((T,), -float("inf"), dtype=torch.float64, device="cuda")
    xd = x.detach().double()
    for a in range(0, V, 50_000):
        lse = torch.logaddexp(lse, torch.logsumexp(xd @ w.detach()[:, a:a + 50_000].double(), -1))
    tail = w.detach()[:, -64:].double()
    l = xd @ tail
    want = (lse - l.gather(1, (t - (V - 64))[:, None])[:, 0]).sum()
    far = 2 * _adds(D, torch.bfloat16) * (xd.abs() @ tail.abs()).amax() + 2.0 ** -22 * (4 + 12)
    assert abs(float(loss.detach()) - float(want)) <= T * float(far)
    p = torch.exp(l - lse[:, None])
    P = p.clone().scatter_add_(1, (t - (V - 64))[:, None], -torch.ones(T, 1, dtype=torch.float64, device="cuda"))
    off = 2.0 ** -8 * P.abs() + p * (float(far) + 2.0 ** -11)
    want = xd.t() @ P
    bound = 1.01 * (2.0 ** -8 * want.abs() + xd.abs().t() @ off + _adds(T, torch.bfloat16) * (xd.abs().t() @ P.abs()))
    assert torch.all((dw[:, -64:].double() - want).abs() <= bound)
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_linear_cross_entropy_second_derivatives(reduction):
    """Of gradients that are recorded: torch's, in 64 bits of the same operands.

    What comes of a scalar g is the sum of f cos(f) / g over all first gradients f, of both signs: each f is off by some 100
    steps of 2^-24 of its own size (sums of at most 40 products and the rows' sums), so the sum is by 1e-5 of the sum of
    magnitudes, however small the signs leave the sum itself."""
    x, w, t = _loss_case(9, 16, 40, torch.float32, 0.2)
    g = torch.rand(9, device="cuda") if reduction == "none" else torch.tensor(1.5, device="cuda")

    def second(loss, x, w, g):
        x, w, g = (v.detach().clone().requires_grad_() for v in (x, w, g))
        first = torch.autograd.grad(loss(x, w), (x, w), g, create_graph=True)
        return [*first, *torch.autograd.grad(sum((f * f.detach().cos()).sum() for f in first), (x, w, g))]

    got = second(lambda x, w: linear_cross_entropy(x, w, t, reduction=reduction), x, w, g)
    want = second(lambda x, w: F.cross_entropy(x @ w, t, reduction=reduction), x.double(), w.double(), g.double())
    for a, b in zip(got, want):
        size = b.norm() if b.dim() else sum((f * f.cos()).abs().sum() for f in want[:2]) / g
        assert float((a.double() - b).detach().norm()) <= 1e-5 * float(size)


# ---------------------------------------------------------------- the embedding on the GPU


def _check_embedding(t, w, scale, out, d_out, dw):
    dtype, V = w.dtype, w.shape[0]
    rows = w.detach().double()[t] * scale
    if scale == 1.0:
        assert torch.equal(out, w.detach()[t])
    else:  # the scale in fp32, the product, the rounding
        assert torch.all((out.double() - rows).abs() <= (_u(dtype) + 2.0 ** -23) * rows.abs())
    flat = torch.where(t < 0, t + V, t).reshape(-1)
    d = d_out.reshape(-1, w.shape[1]).double()
    want, size = (torch.zeros(w.shape, dtype=torch.float64, device="cuda").index_add_(0, flat, v) for v in (d, d.abs()))
    most = int(torch.bincount(flat, minlength=V).max()) if flat.numel() else 0
    bound = _u(dtype) * (want * scale).abs() + 1.01 * (most + 2) * 2.0 ** -24 * size * abs(scale)
    assert dw.dtype == dtype and torch.all((dw.double() - want * scale).abs() <= bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (5, 7, 3), (64, 50, 8), (33, 2, 40), (200, 3, 520), (1000, 1, 64), (3000, 1000, 264),
                                   (70, 300000, 17), (9000, 50257, 128), (20000, 96, 7)])
def test_embedding_matches_64_bits(T, V, D, dtype):
    """Ids of none, one and thousands of tokens, at most 32 of them and more, at the ends of pieces; odd rows."""
    g = torch.Generator(device="cuda").manual_seed(T + V)
    w = torch.randn(V, D, device="cuda", generator=g).to(dtype).requires_grad_()
    for kind, scale in (("uniform", 1.0), ("padded", 1.0), ("skewed", 3.3), ("one", 0.7)):
        t = torch.randint(-V, V, (T,), device="cuda", generator=g)
        if kind == "padded":
            t[T // 2:] = 0
        elif kind == "skewed":
            t = (torch.rand(T, device="cuda", generator=g) ** 8 * V).long().clamp(max=V - 1)
        elif kind == "one":
            t[:] = V - 1
        out = embedding(t, w, scale)
        d_out = torch.randn(T, D, device="cuda", generator=g).to(dtype)
        dw, = torch.autograd.grad(out, w, d_out)
        _check_embedding(t, w, scale, out.detach(), d_out, dw)
        again, = torch.autograd.grad(embedding(t, w, scale), w, d_out)
        assert torch.equal(again, dw)
        with torch.no_grad():
            assert torch.equal(embedding(t, w, scale), out)


@pytest.mark.gpu
def test_embedding_layouts_bad_tokens_and_second_derivatives():
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(40, 24, device="cuda", generator=g).requires_grad_()
    t = torch.randint(0, 40, (6, 10), device="cuda", generator=g)
    d = torch.randn(6, 10, 24, device="cuda", generator=g)
    dw, = torch.autograd.grad(embedding(t, w), w, d)
    flat = torch.zeros(40 * 24 + 1, device="cuda")
    flat[1:] = w.detach().reshape(-1)
    for wv in (flat[1:].view(40, 24), w.detach().t().contiguous().t()):
        wv = wv.detach().requires_grad_()
        for tv, dv in ((t, d), (t.t().contiguous().t(), d.transpose(0, 1).contiguous().transpose(0, 1))):
            out = embedding(tv, wv)
            assert torch.equal(out, w.detach()[t]) and torch.equal(torch.autograd.grad(out, wv, dv)[0], dw)
    # tokens outside the table: rows of NaN, no gradient
    bad = t.clone()
    bad[0, :3] = torch.tensor([40, -41, 1 << 40], device="cuda")
    out = embedding(bad, w)
    assert torch.isnan(out[0, :3]).all() and torch.equal(out[0, 3:], w.detach()[t][0, 3:])
    keep = d.clone()
    keep[0, :3] = 0.0
    assert torch.equal(torch.autograd.grad(out, w, d)[0], torch.autograd.grad(embedding(t, w), w, keep)[0])
    # none at all
    assert embedding(t[:0], w).shape == (0, 10, 24)
    assert torch.all(torch.autograd.grad(embedding(t[:0], w).sum(), w)[0] == 0)
    # the gradient is linear in what comes in
    d2 = d.clone().requires_grad_()
    first, = torch.autograd.grad(embedding(t, w, 2.0), w, d2, create_graph=True)
    u = torch.randn_like(first)
    assert torch.equal(torch.autograd.grad(first, d2, u)[0], embedding(t, u, 2.0))


@pytest.mark.gpu
def test_embedding_past_32_bits():
    V, D = 1_050_000, 2048
    w = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    w[-3:] = torch.randn(3, D, device="cuda").bfloat16()
    w.requires_grad_()
    t = torch.tensor([V - 1, 0, V - 3, V - 1], device="cuda")
    d = torch.randn(4, D, device="cuda").bfloat16()
    out = embedding(t, w)
    assert torch.equal(out, w.detach()[t])
    dw, = torch.autograd.grad(out, w, d)
    assert torch.equal(dw[-3], d[2]) and torch.equal(dw[-2], torch.zeros_like(d[0])) and torch.equal(dw[0], d[1])
    assert torch.equal(dw[-1], (d[0].float() + d[3].float()).bfloat16())
    assert int((dw[::4096] != 0).sum()) == D  # row 0 alone of these


# ---------------------------------------------------------------- both, as a program has them


@pytest.mark.gpu
@pytest.mark.parametrize("T", [16, 200])
def test_captured_and_replayed(T):
    """A step of both ends in a graph: every replay on new inputs has the eager call's bits."""
    g = torch.Generator(device="cuda").manual_seed(8)
    V, D = 333, 64
    table, w = (torch.randn(s, device="cuda", generator=g).bfloat16().requires_grad_() for s in ((V, D), (D, V)))
    tokens, targets = (torch.randint(0, V, (T,), device="cuda", generator=g) for _ in range(2))

    def step(table, w):
        loss = linear_cross_entropy(embedding(tokens, table, 1.5), w, targets)
        return [loss.detach(), *torch.autograd.grad(loss, (table, w))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(table, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(table, w)
    twin = [t.detach().clone().requires_grad_() for t in (table, w)]
    for k in range(4):
        tokens.copy_(torch.randint(0, V, (T,), device="cuda", generator=g))
        tokens[T // 2:] = k
        targets.copy_(torch.randint(0, V, (T,), device="cuda", generator=g))
        targets[:k * T // 4] = -100
        graph.replay()
        want = step(*twin)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [16, 200])
def test_forward_and_backward_in_graphs_of_their_own(T):
    """Either of the two in a graph without the other, and each in its own: any number of replays of either."""
    g = torch.Generator(device="cuda").manual_seed(8)
    x, w, t = _loss_case(T, 64, 333, torch.bfloat16, 0.2)
    up = torch.full((), 0.5, device="cuda")

    def want(k):
        up.fill_(k)
        a, b = (v.detach().clone().requires_grad_() for v in (x, w))
        return torch.autograd.grad(linear_cross_entropy(a, b, t), (a, b), up)

    side = torch.cuda.Stream()  # of the forward, the backward and their graphs: none of them waits for another's stream

    def recorded(f):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = f()
        return graph, out

    leaves = [v.detach().requires_grad_() for v in (x, w)]
    want(1.0)
    for forward_in, backward_in in ((False, True), (True, True), (True, False)):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            forward = lambda: linear_cross_entropy(*leaves, t)
            backward = lambda: torch.autograd.grad(loss, leaves, up, retain_graph=True)
            first, loss = recorded(forward) if forward_in else (None, forward())
            if forward_in:
                first.replay()
            side.synchronize()
            second, grads = recorded(backward) if backward_in else (None, None)
            for k in (0.5, 3.0, 0.25):
                expected = want(k)
                for _ in range(2):
                    if backward_in:
                        second.replay()
                    else:
                        grads = backward()
                    side.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(grads, expected))
                if forward_in:
                    first.replay()


@pytest.mark.gpu
def test_two_streams_at_once():
    cases = [_loss_case(T, 128, 3001, torch.bfloat16, 0.2, seed) for seed, T in ((0, 40), (1, 500))]

    def run(x, w, t):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(x, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w))]

    want = [run(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for case, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                got.append(run(*case))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T", [20, 64, 150])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf"), 0.0])
def test_weights_of_rows_that_are_no_numbers_or_zero(T, odd, dtype):
    """One spoils its own row's dx, and dw, wherever the row stands; a weight of 0 is a row without a gradient."""
    x, w, t = _loss_case(T, 64, 300, dtype, 0.2)
    rows = linear_cross_entropy(x, w, t, reduction="none")
    x, w = x.requires_grad_(), w.requires_grad_()
    g = torch.rand(T, device="cuda") + 0.2
    kept = (t != -100).nonzero()[:, 0]
    for at in (kept[:1], kept[len(kept) // 2:][:1], kept[-1:], kept[1::3], kept):
        weights = g.clone()
        weights[at] = odd
        dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, t, reduction="none"), (x, w), weights)
        others = torch.ones(T, dtype=torch.bool, device="cuda")
        others[at] = False
        _check_loss(x.detach()[others], w, t[others], "none", rows[others], (dx[others], None), weights[others])
        assert torch.all(dx[t == -100] == 0)
        if odd == 0.0:
            assert torch.all(dx[at] == 0)
            _check_loss(x.detach(), w, t, "none", rows, (None, dw), weights)
        else:
            assert not torch.isfinite(dx[at]).any() and not torch.isfinite(dw).any()


def _with_unknown_targets(x, w, t, reduction):
    """The loss that the kernels' gradients are of: of the rows not ignored alone, without a target where it is outside the
    vocabulary."""
    kept = t != -100
    l = x[kept] @ w
    known = (t[kept] >= 0) & (t[kept] < w.shape[1])
    rows = torch.logsumexp(l, -1) - torch.where(known, l.gather(1, torch.where(known, t[kept], 0)[:, None])[:, 0], 0.0)
    return rows.mean() if reduction == "mean" else torch.zeros(len(t), dtype=l.dtype, device=l.device).index_put((kept.nonzero()[:, 0],), rows)


def _odd_rows(device):
    x, w, t = _loss_case(9, 16, 40, torch.float32, device=device)
    t[1], t[4], t[6], t[7] = -100, 40, -1, -100
    x[1], x[7, 3] = float("nan"), float("inf")
    return x, w, t


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_second_derivatives_are_of_the_kernels_gradient(reduction):
    """Rows that are ignored reach nothing, whatever they hold, and a target outside the vocabulary is none."""
    x, w, t = _odd_rows("cpu")
    g = torch.rand(9) if reduction == "none" else torch.tensor(1.5)
    grads = []
    for f in (vocabulary._loss_op, lambda x, w, t, _, reduction: _with_unknown_targets(x, w, t, reduction)):
        a, b = (v.double().requires_grad_() for v in (x, w))
        grads.append(torch.autograd.grad(f(a, b, t, -100, reduction), (a, b), g.double()))
    assert all(torch.allclose(a, b, rtol=1e-12, atol=1e-15) for a, b in zip(*grads))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_second_derivatives_beside_odd_rows(reduction):
    """As test_linear_cross_entropy_second_derivatives, with NaN and infinities in ignored rows and targets outside the vocabulary."""
    x, w, t = _odd_rows("cuda")
    g = torch.rand(9, device="cuda") if reduction == "none" else torch.tensor(1.5, device="cuda")

    def second(loss, x, w, g):
        x, w, g = (v.detach().clone().requires_grad_() for v in (x, w, g))
        first = torch.autograd.grad(loss(x, w), (x, w), g, create_graph=True)
        return [*first, *torch.autograd.grad(sum((f * f.detach().cos()).sum() for f in first), (x, w, g))]

    got = second(lambda x, w: linear_cross_entropy(x, w, t, reduction=reduction), x, w, g)
    want = second(lambda x, w: _with_unknown_targets(x, w, t, reduction), x.double(), w.double(), g.double())
    for a, b in zip(got, want):
        size = b.norm() if b.dim() else sum((f * f.cos()).abs().sum() for f in want[:2]) / g
        assert float((a.double() - b).detach().norm()) <= 1e-5 * float(size)


def test_the_graph_of_another_device_is_asked_for(monkeypatch):
    """A call on a device that is not the current one is in the graph that its own device's stream records."""
    def call(device, name, address):
        assert name == "abacus_capture_id" and device.index == 1
        ctypes.c_int64.from_address(address).value = 7

    monkeypatch.setattr(vocabulary, "_call", call)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    assert vocabulary._capture(torch.device("cuda", 0)) == 0
    assert vocabulary._capture(torch.device("cuda", 1)) == 7


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_gradients_between_forward_and_backward_are_saved_tensors(reduction):
    """Hooks on saved tensors see the gradients that the forward has formed, may move them, and checkpointing drops them; a
    backward that is made again has them too."""
    x, w, t = _loss_case(150, 512, 4000, torch.bfloat16, 0.2)
    leaves = x.requires_grad_(), w.requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(x, w, t, reduction=reduction) * 0.5, leaves)
    shapes = []

    def pack(v):
        shapes.append(tuple(v.shape))
        return v.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v.cuda()):
        loss = linear_cross_entropy(x, w, t, reduction=reduction) * 0.5
    assert shapes.count((150, 512)) == 2 and shapes.count((512, 4000)) == 2
    plain = linear_cross_entropy(x, w, t, reduction=reduction) * 0.5
    for again in (loss, plain):
        for _ in range(2):
            got = torch.autograd.grad(again, leaves, retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            for d in got:
                d.zero_()
    del again, plain, got
    del loss
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = torch.utils.checkpoint.checkpoint(lambda x, w: linear_cross_entropy(x, w, t, reduction=reduction), x, w, use_reentrant=False) * 0.5
    assert torch.cuda.memory_allocated() - before < 512 * 4000
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_one_row_of_any_stride(dtype):
    """A single row has no stride to speak of: a column that is turned to one, and one that is expanded."""
    w = torch.randn(24, 90, device="cuda").to(dtype).requires_grad_()
    t = torch.tensor([7], device="cuda")
    column = torch.randn(24, 1, device="cuda").to(dtype)
    row = column.reshape(1, 24).clone().requires_grad_()
    want = linear_cross_entropy(row, w, t)
    for x in (column.t(), column[:, 0].as_strided((1, 24), (0, 1)), column.t().expand(1, 24)):
        assert x.stride(0) < 24
        x = x.detach().requires_grad_()
        got = linear_cross_entropy(x, w, t)
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, (x, w)), torch.autograd.grad(want, (row, w), retain_graph=True)))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [10, 70])
def test_gradient_of_rows_past_32_bits(T):
    """dx of a w of more than 2^31 values, against 64 bits: targets and the likeliest columns lie past the 2^31st value."""
    D, V, piece = 2048, 1_050_000, 50_000
    x, _, t = _loss_case(T, D, 8, torch.bfloat16)
    w = torch.empty(D, V, dtype=torch.bfloat16, device="cuda").normal_(0.0, 0.04, generator=torch.Generator(device="cuda").manual_seed(5))
    t = V - 1 - t * 1000
    dx, = torch.autograd.grad(linear_cross_entropy(x.requires_grad_(), w, t, reduction="sum"), x)
    xd = x.detach().double()
    lse, top, most = torch.full((T,), -float("inf"), dtype=torch.float64, device="cuda"), 0.0, 0.0
    for a in range(0, V, piece):
        l = xd @ w[:, a:a + piece].double()
        lse = torch.logaddexp(lse, torch.logsumexp(l, -1))
        top = max(top, float(l.abs().max()))
        most = max(most, float((xd.abs() @ w[:, a:a + piece].double().abs()).max()))
    far = 2 * _adds(D, torch.bfloat16) * most + 2.0 ** -22 * (4 + top)
    want, size, off = (torch.zeros(T, D, dtype=torch.float64, device="cuda") for _ in range(3))
    for a in range(0, V, piece):
        wd = w[:, a:a + piece].double()
        p = torch.exp(xd @ wd - lse[:, None])
        here = (t >= a) & (t < a + piece)
        P = p.clone()
        P[here, t[here] - a] -= 1.0
        turned = wd.t().contiguous()
        want += P @ turned
        size += P.abs() @ turned.abs()
        off += (_u(torch.bfloat16) * P.abs() + p * (far + 2.0 ** -11)) @ turned.abs()
    bound = 1.01 * (_u(torch.bfloat16) * want.abs() + off + (_adds(V, torch.bfloat16) + 2.0 ** -22) * size)
    assert torch.all((dx.double() - want).abs() <= bound)
    # the bound tells the target's column from the one that 32 bits would reach
    assert float(bound.max()) < 0.25 * float(w[:, -1].float().abs().max())
