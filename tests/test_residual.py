"""residual_norm (abacus_amd.residual): refusals and the CPU's steps, and on the GPU the kernels against 64-bit formulas.

Tolerances count roundings of u = eps / 2 (bf16 2^-8, fp32 2^-24).  r has one.  h and the gradients are those of the r that
was returned, so each value has one, and fp32 sums: a row's sums add at most 64 values a lane, 6 times over the lanes and 16
over the waves, so what they are in is off by 100 * 2^-24 of the sum of magnitudes; a sum over n rows by
(n + 100) * 2^-24 of its magnitudes, and that of its terms.
"""

import pytest
import torch

from abacus_amd import _lib
from abacus_amd import transformer as tr
from abacus_amd.residual import residual_norm

DTYPES = [torch.bfloat16, torch.float32]
IDS = ["bf16", "fp32"]
F32 = 2.0 ** -24
EPS = 1e-5


def _leaves(rows, D, dtype, post, gate, device="cuda", seed=0):
    g = torch.Generator(device=device).manual_seed(seed + 1000 * rows + D)
    rand = lambda *s: torch.randn(*s, device=device, generator=g).to(dtype)
    shape = {"none": None, "channel": (D,), "token": (rows, D)}[gate]
    return {"x": rand(rows, D), "y": rand(rows, D), "gamma": rand(D), "post_gamma": rand(D) if post else None,
            "gate": None if shape is None else rand(*shape)}


def _check(leaves, scale, r, h, dr, dh, grads):
    dtype, D, rows = r.dtype, r.shape[-1], r.shape[0]
    u = torch.finfo(dtype).eps / 2
    x, y, gamma, post, gate = (None if t is None else t.detach().double() for t in leaves.values())
    inv = lambda v: torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    off = 100 * F32

    def near(got, want, size, k=off):
        err = (got.double() - want).abs() - (1.01 * u * want.abs() + k * size + 1e-38)
        assert torch.all(err <= 0), f"{float(err.max()):.3g} too much"

    p = inv(y)
    branch = y if post is None else post * y * p
    added = scale * (branch if gate is None else gate * branch)
    near(r, x + added, x.abs() + added.abs())
    rd = r.detach().double()
    q = inv(rd)
    n = rd * q
    near(h, gamma * n, (gamma * n).abs())
    if grads is None:
        return
    dr = torch.zeros_like(rd) if dr is None else dr.double()
    dh = torch.zeros_like(rd) if dh is None else dh.double()
    mean = lambda v: v.mean(-1, keepdim=True)
    g = dh * gamma
    dx = dr + q * (g - n * mean(g * n))
    dx_size = dr.abs() + q * (g.abs() + n.abs() * mean((g * n).abs()))
    near(grads["x"], dx, dx_size)
    over = (rows + 100) * F32
    near(grads["gamma"], (dh * n).sum(0), (dh * n).abs().sum(0), over)
    db, db_size = scale * dx, abs(scale) * dx_size
    if gate is not None:
        if gate.dim() == 1:
            near(grads["gate"], (db * branch).sum(0), (db_size * branch.abs()).sum(0), over + 2 * off)
        else:
            near(grads["gate"], db * branch, db_size * branch.abs(), 2 * off)
        db, db_size = db * gate, db_size * gate.abs()
    if post is not None:
        m = y * p
        near(grads["post_gamma"], (db * m).sum(0), (db_size * m.abs()).sum(0), over + 2 * off)
        t, t_size = db * post, db_size * post.abs()
        db, db_size = p * (t - m * mean(t * m)), p * (t_size + m.abs() * mean(t_size * m.abs()))
    near(grads["y"], db, db_size, 3 * off)


def test_refusals():
    d = _leaves(3, 8, torch.float32, True, "channel", "cpu")
    for bad, error in (({"y": d["y"][:2]}, ValueError), ({"gamma": d["gamma"][:7]}, ValueError),
                       ({"post_gamma": d["x"]}, ValueError), ({"gate": d["x"][:2]}, ValueError),
                       ({"gate": d["gate"].double()}, TypeError), ({"x": d["x"][0, 0], "y": d["y"][0, 0]}, ValueError)):
        with pytest.raises(error):
            residual_norm(**(d | bad))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_on_cpu(gate, post):
    d = {n: None if t is None else t.requires_grad_() for n, t in _leaves(3, 8, torch.float64, post, gate, "cpu").items()}
    r, h = residual_norm(**d, scale=0.5)
    b = d["y"] if not post else tr._norm_op(d["y"], d["post_gamma"], EPS)
    want = d["x"] + 0.5 * (b if d["gate"] is None else d["gate"] * b)
    assert torch.allclose(r, want, rtol=1e-12) and torch.allclose(h, tr._norm_op(want, d["gamma"], EPS), rtol=1e-12)
    there = [n for n, t in d.items() if t is not None]
    f = lambda *a: residual_norm(**dict(zip(there, a)), scale=0.5)
    assert torch.autograd.gradcheck(f, tuple(d[n] for n in there))


# dims of each layout: whole rows over lanes, a wave, waves; odd ones, the least and the most
DIMS = {torch.bfloat16: [8, 64, 512, 1024, 2048, 4096, 9, 100, 1000, 1023, 1025, 2568, 6000, 8192],
        torch.float32: [4, 64, 256, 512, 1024, 2048, 5, 33, 500, 511, 513, 1000, 3001, 4096]}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(t, D) for t in DTYPES for D in DIMS[t]], ids=lambda v: str(v).replace("torch.", ""))
def test_matches_64_bits(dtype, D):
    for rows in (1, 7, 260):
        for post, gate, scale in ((False, "none", 1.0), (False, "none", 0.3), (True, "none", 1.0), (False, "channel", 1.0),
                                  (True, "channel", 0.5), (True, "token", 1.0), (False, "token", -2.0)):
            d = {n: None if t is None else t.requires_grad_() for n, t in _leaves(rows, D, dtype, post, gate).items()}
            there = {n: t for n, t in d.items() if t is not None}
            r, h = residual_norm(**d, scale=scale)
            dr, dh = torch.randn_like(r), torch.randn_like(h)
            grads = dict(zip(there, torch.autograd.grad((r, h), tuple(there.values()), (dr, dh))))
            _check(d, scale, r, h, dr, dh, grads)
            with torch.no_grad():
                assert all(torch.equal(a, b) for a, b in zip(residual_norm(**d, scale=scale), (r, h)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_rows_and_one_output_alone(dtype):
    d = {n: None if t is None else t.requires_grad_() for n, t in _leaves(20011, 256, dtype, True, "channel").items()}
    there = {n: t for n, t in d.items() if t is not None}
    r, h = residual_norm(**d, scale=0.5)
    dr, dh = torch.randn_like(r), torch.randn_like(h)
    for a, b in ((dr, dh), (dr, None), (None, dh)):
        r, h = residual_norm(**d, scale=0.5)
        outs = [(o, v) for o, v in ((r, a), (h, b)) if v is not None]
        grads = torch.autograd.grad([o for o, _ in outs], tuple(there.values()), [v for _, v in outs], allow_unused=True)
        _check(d, 0.5, r, h, a, b, dict(zip(there, grads)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("D", [16, 64, 128, 1024, 2048])
def test_bits_of_the_sum_and_the_norm(D, dtype):
    """Without post, gate and scale: x + y and RMSNorm's, bit for bit."""
    d = _leaves(37, D, dtype, False, "none")
    norm = tr.RMSNorm(D).cuda().to(dtype)
    with torch.no_grad():
        norm.w_gamma_D.copy_(d["gamma"])
        r, h = residual_norm(d["x"], d["y"], norm.w_gamma_D)
        assert tr._fused_norm_ok(r, norm.w_gamma_D)
        assert torch.equal(r, d["x"] + d["y"]) and torch.equal(h, norm(d["x"] + d["y"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layouts_and_odd_values(dtype):
    """Views that start at any element, leading dimensions, turned gradients, rows of infinities and NaN beside others."""
    d = _leaves(30, 72, dtype, True, "token")
    want = residual_norm(**d, scale=0.5)
    flat = {n: torch.zeros(t.numel() + 1, device="cuda", dtype=dtype) for n, t in d.items()}
    views = {}
    for n, t in d.items():
        flat[n][1:] = t.reshape(-1)
        views[n] = flat[n][1:].view(t.shape)
    assert all(torch.equal(a, b) for a, b in zip(residual_norm(**views, scale=0.5), want))
    turned = {n: t.t().contiguous().t() if t.dim() == 2 else t for n, t in d.items()}
    assert all(torch.equal(a, b) for a, b in zip(residual_norm(**turned, scale=0.5), want))
    more = {n: t.view(5, 6, 72) if t.dim() == 2 else t for n, t in d.items()}
    leaves = [more["x"].detach().requires_grad_(), more["y"].detach().requires_grad_()]
    r, h = residual_norm(*leaves, *(more[n] for n in ("gamma", "post_gamma", "gate")), scale=0.5)
    assert torch.equal(r.view(30, 72), want[0]) and r.shape == (5, 6, 72)
    g = torch.randn(6, 5, 72, device="cuda").to(dtype).transpose(0, 1)
    dx, dy = torch.autograd.grad((r, h), leaves, (g, g))
    r, h = residual_norm(*leaves, *(more[n] for n in ("gamma", "post_gamma", "gate")), scale=0.5)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad((r, h), leaves, (g.contiguous(),) * 2), (dx, dy)))

    odd = {n: t.clone() for n, t in d.items()}
    odd["x"][3, 5], odd["y"][4, 0], odd["x"][29, 71] = float("inf"), float("nan"), -float("inf")
    got = residual_norm(**odd, scale=0.5)
    rest = [i for i in range(30) if i not in (3, 4, 29)]
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got, want))
    assert torch.isnan(got[1][4]).all() and torch.isnan(got[1][3]).any()


@pytest.mark.gpu
def test_a_scale_that_rounds_to_one():
    """1 + 2^-30 is 1 in fp32: the bits of no scale, both ways."""
    d = _leaves(9, 40, torch.float32, False, "none")
    leaves = [d[n].requires_grad_() for n in ("x", "y", "gamma")]
    dr, dh = torch.randn_like(d["x"]), torch.randn_like(d["x"])
    got, want = (torch.autograd.grad(residual_norm(*leaves, scale=s), leaves, (dr, dh)) for s in (1 + 2.0 ** -30, 1.0))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_no_rows_and_refusals_on_gpu():
    d = _leaves(0, 16, torch.float32, False, "channel")
    r, h = residual_norm(**d)
    assert r.shape == h.shape == (0, 16)
    with pytest.raises(ValueError):
        residual_norm(*(torch.zeros(s, device="cuda") for s in ((2, 4097), (2, 4097), (4097,))))
    with pytest.raises(ValueError):
        residual_norm(*(torch.zeros(s, device="cuda") for s in ((2, 3), (2, 3), (3,))))
    with pytest.raises(TypeError):
        residual_norm(*(torch.zeros(s, device="cuda", dtype=torch.float16) for s in ((2, 8), (2, 8), (8,))))


@pytest.mark.gpu
@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "token"), (True, "channel")])
def test_second_derivatives(post, gate):
    """Of gradients that are recorded: torch's of the formula in 64 bits (sums of at most 16 x 5 terms in fp32)."""
    d = _leaves(5, 16, torch.float32, post, gate)
    names = [n for n, t in d.items() if t is not None]
    dr, dh = (torch.randn(5, 16, device="cuda") for _ in range(2))

    def second(f, wide):
        a = [d[n].to(wide).requires_grad_() for n in names] + [dr.to(wide).requires_grad_(), dh.to(wide).requires_grad_()]
        first = torch.autograd.grad(f(**dict(zip(names, a))), a[:-2], a[-2:], create_graph=True)
        return [*first, *torch.autograd.grad(sum((v * v.detach().cos()).sum() for v in first), a)]

    def plain(x, y, gamma, post_gamma=None, gate=None):
        b = y if post_gamma is None else tr._norm_op(y, post_gamma, EPS)
        r = x + 0.5 * (b if gate is None else gate * b)
        return r, tr._norm_op(r, gamma, EPS)

    for a, b in zip(second(lambda **k: residual_norm(**k, scale=0.5), torch.float32), second(plain, torch.float64)):
        assert float((a.double() - b).detach().norm()) <= 2e-5 * float(b.norm())


@pytest.mark.gpu
def test_captured_and_on_two_streams():
    d = [{n: t.requires_grad_() for n, t in _leaves(rows, D, torch.bfloat16, True, "channel").items()}
         for rows, D in ((300, 1000), (50, 4096))]

    def run(leaves):
        r, h = residual_norm(**leaves, scale=0.5)
        return [r.detach(), h.detach(), *torch.autograd.grad((r, h), tuple(leaves.values()), (r.detach().cos(), h.detach().cos()))]

    twins = [{n: t.detach().clone().requires_grad_() for n, t in leaves.items()} for leaves in d]
    streams = [torch.cuda.Stream() for _ in d]
    want = [run(t) for t in twins]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for leaves, stream in zip(twins, streams):
            with torch.cuda.stream(stream):
                got.append(run(leaves))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    leaves = d[0]
    streams[0].wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams[0]):
        run(leaves)
    torch.cuda.current_stream().wait_stream(streams[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(leaves)
    g = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(4):
        with torch.no_grad():
            for n, t in leaves.items():
                t.copy_(torch.randn(t.shape, device="cuda", generator=g))
                twins[0][n].copy_(t)
        graph.replay()
        want = run(twins[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_frozen_operands_have_no_gradient_formed(gate):
    """The norms' weights and the gate that ask for none: the others' gradients are the same bits, and nothing of a frozen gate's size
    is allocated."""
    rows, D = 2048, 1024
    d = _leaves(rows, D, torch.float32, True, gate)
    dr, dh = torch.randn_like(d["x"]), torch.randn_like(d["x"])
    there = [n for n, t in d.items() if t is not None]

    def run(asked):
        leaves = {n: None if t is None else t.detach().requires_grad_(n in asked) for n, t in d.items()}
        r, h = residual_norm(**leaves, scale=0.5)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        torch.autograd.backward((r, h), (dr, dh))
        peak = torch.cuda.max_memory_allocated() - before
        assert all(leaves[n].grad is None for n in there if n not in asked)
        return {n: leaves[n].grad for n in asked}, peak

    whole, _ = run(there)
    for asked in (["x", "y"], ["x", "y", "gamma"], ["x", "y", "post_gamma"], [n for n in there if n != "post_gamma"],
                  [n for n in there if n != "gate"]):
        got, peak = run(asked)
        assert all(torch.equal(got[n], whole[n]) for n in asked)
        big = 2 + (gate == "token" and "gate" in asked)
        sums = _lib.query("abacus_residual_norm_bwd_ws_bytes", rows, D, 1, int(gate == "channel"))
        # (each large allocation may hold up to 1 MiB more of its block, and the small ones are some KiB; one tensor more is 8 MiB)
        assert peak < big * rows * D * 4 + sums + (big + 2 << 20)


def test_workspaces_of_few_rows_are_small():
    """Partial sums of as many work-groups as there are rows at most."""
    for rows in (1, 5, 200):
        for gate_kind, sums in ((0, 2), (1, 3), (2, 2)):
            assert 0 < _lib.query("abacus_residual_norm_bwd_ws_bytes", rows, 4096, 1, gate_kind) <= rows * sums * 4096 * 4


@pytest.mark.gpu
def test_second_derivatives_beside_frozen_operands():
    """Of gradients that are recorded, with the post norm's weight and the gate frozen."""
    d = _leaves(5, 16, torch.float32, True, "channel")
    dr, dh = (torch.randn(5, 16, device="cuda") for _ in range(2))

    def second(f, wide):
        x, y, gamma = (d[n].detach().to(wide).requires_grad_() for n in ("x", "y", "gamma"))
        first = torch.autograd.grad(f(x, y, gamma, d["post_gamma"].to(wide), d["gate"].to(wide)), (x, y, gamma),
                                    (dr.to(wide), dh.to(wide)), create_graph=True)
        return [*first, *torch.autograd.grad(sum((v * v.detach().cos()).sum() for v in first), (x, y, gamma))]

    def plain(x, y, gamma, post, gate):
        r = x + 0.5 * gate * tr._norm_op(y, post, EPS)
        return r, tr._norm_op(r, gamma, EPS)

    for a, b in zip(second(lambda *a: residual_norm(*a, scale=0.5), torch.float32), second(plain, torch.float64)):
        assert float((a.double() - b).detach().norm()) <= 2e-5 * float(b.norm())
