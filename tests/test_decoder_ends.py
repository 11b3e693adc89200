"""The decoder with its embedding, its sums and norms and its head's loss by the kernels (train_step's fused_loss, hidden,
forward_cached), against the steps one by one; and the three operators' gradients against differences.

The same bits are asked for where both take the same roundings; elsewhere the criterion of test_gpu_transformer.py: the
normwise error against 64 bits is within twice that of the CPU in the same type, or below the type's tolerance.
"""

import copy

import pytest
import torch

from abacus_amd import _lib
from abacus_amd import transformer as tr
from abacus_amd.kv_cache import PagedKVCache
from abacus_amd.residual import residual_norm
from abacus_amd.train import Trainer, head_loss, make_optimizer, next_token_loss, train_step
from abacus_amd.vocabulary import embedding, linear_cross_entropy

from test_gpu_transformer import CFG, RTOL, _OracleMoE, _rel


def _model(dtype=torch.bfloat16, device="cuda", **changes):
    torch.manual_seed(4)
    return tr.TransformerMoe(**(CFG | changes)).to(dtype).to(device)


def _tokens(device="cuda", vocab=97, shape=(3, 24)):
    tokens = torch.randint(0, vocab, shape, generator=torch.Generator().manual_seed(2))
    tokens[1, 5:9] = tokens[2, 17:] = -100
    return tokens.to(device)


# ---------------------------------------------------------------- CPU


def test_head_loss_is_next_token_loss_on_cpu():
    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((3, 24, 8), (8, 97)))
    tokens = _tokens("cpu")
    loss, want = head_loss(x, w, tokens), next_token_loss(x @ w, tokens)
    assert torch.allclose(loss, want, rtol=1e-12)
    for a, b in zip(torch.autograd.grad(loss, (x, w)), torch.autograd.grad(want, (x, w))):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-14)
    with pytest.raises(ValueError):
        head_loss(x, w, tokens[:, 1:])


@pytest.mark.parametrize("name,args,msg", [
    ("abacus_linear_cross_entropy", (16, 8, 16, 16, 4, 8, 10, -100, 5, 2, None, 16, 16, 16, 16, 1 << 20, None), "dtype"),
    ("abacus_linear_cross_entropy", (16, 8, 16, 16, 4, 8, 10, -100, 1, 3, None, 16, 16, 16, 16, 1 << 20, None), "reduction"),
    ("abacus_linear_cross_entropy", (16, 8, 16, 16, 4, 0, 10, -100, 1, 2, None, 16, 16, 16, 16, 1 << 20, None), "dim 0"),
    ("abacus_linear_cross_entropy", (16, 8, 16, 16, 0, 8, 10, -100, 1, 2, None, 16, 16, 16, 16, 1 << 20, None), "no rows"),
    ("abacus_linear_cross_entropy", (16, 7, 16, 16, 4, 8, 10, -100, 1, 2, None, 16, 16, 16, 16, 1 << 20, None), "stride"),
    ("abacus_linear_cross_entropy", (16, 8, 16, 16, 4, 8, 10, -100, 1, 0, None, 16, 16, 16, 16, 1 << 20, None), "weights"),
    ("abacus_linear_cross_entropy", (16, 8, 16, 16, 4, 8, 10, -100, 1, 2, None, 16, 16, 16, 16, 64, None), "workspace"),
    ("abacus_scale_by", (16, 4, 16, 4, 5, 16, None), "dtype"),
    ("abacus_scale_by", (16, -1, 16, 4, 1, 16, None), "values"),
    ("abacus_embedding_fwd", (16, 16, 4, 0, 8, 1.0, 1, 16, None), "table"),
    ("abacus_embedding_fwd", (16, 16, 4, 8, 8, 1.0, 5, 16, None), "dtype"),
    ("abacus_embedding_bwd", (16, 16, 4, 8, 8, 1.0, 1, 16, 16, 0, None), "workspace"),
    ("abacus_residual_norm_fwd", (16, 16, 16, None, None, 1, 4, 64, 1.0, 1e-5, 1, 16, 16, None, None, None), "gate"),
    ("abacus_residual_norm_fwd", (16, 16, 16, None, None, 0, 4, 7, 1.0, 1e-5, 1, 16, 16, None, None, None), "dim 7"),
    ("abacus_residual_norm_bwd", (16, 16, 16, 16, 16, None, None, 0, 16, None, 4, 64, 1.0, 1, 16, 16, 16, 16, None, 16, 1 << 30, None),
     "gradients"),
    ("abacus_residual_norm_bwd", (16, 16, 16, None, 16, None, None, 0, 16, None, 4, 64, 1.0, 1, 16, 32, 16, None, None, 16, 1 << 30, None),
     "dx's memory"),
    ("abacus_residual_norm_bwd", (16, 16, 16, None, 16, None, None, 0, 16, None, 4, 64, 0.5, 1, 16, None, 16, None, None, 16, 1 << 30, None),
     "its own"),
    ("abacus_residual_norm_bwd", (16, 16, 16, 16, 16, 16, None, 0, 16, None, 4, 64, 1.0, 1, 16, 32, 16, 16, None, 16, 1 << 30, None),
     "y_rstd"),
    ("abacus_residual_norm_bwd", (16, 16, 16, None, 16, None, 16, 1, 16, None, 4, 64, 1.0, 1, 16, 32, 16, None, 16, 16, 1 << 30, None),
     "a gate y"),
    ("abacus_residual_norm_bwd", (16, 16, 16, 16, 16, None, None, 0, 16, None, 4, 64, 1.0, 1, 16, 16, 16, None, None, 16, 0, None),
     "workspace"),
])
def test_entry_points_refuse(name, args, msg):
    with pytest.raises(RuntimeError, match=msg):
        _lib.call(name, *args)


def test_workspaces_cover_every_size():
    """Sizes are 0 for calls that are refused, and near the kept rows' copy, a piece of the logits (1 GiB) and the
    operands' sums over pieces: at 2^20 rows of 4096 in 4 bytes 16 GiB, 1 GiB and 1 GiB."""
    of = lambda *a: _lib.query("abacus_linear_cross_entropy_ws_bytes", *a)
    assert of(-1, 8, 8, 1, 1) == of(4, 0, 8, 1, 1) == of(4, 8, 0, 1, 1) == 0
    for dtype in (_lib.F32, _lib.BF16):
        assert 0 < of(1, 8, 8, dtype, 0) <= of(1, 8, 8, dtype, 1)
        assert of(1 << 20, 4096, 65536, dtype, 1) < 20 << 30
    assert _lib.query("abacus_embedding_bwd_ws_bytes", 0, 8, 8) >= 0


# ---------------------------------------------------------------- differences


def _directional(f, leaves, seed):
    """The derivative of f's 64-bit sums along a random direction, by central differences of 2^-13: the third order left
    out is 2^-26 / 6 of the third derivative."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    along = [torch.randn(t.shape, device="cuda", generator=g, dtype=torch.float64) for t in leaves]
    h = 2.0 ** -13
    at = [f(*(t.detach().double() + s * h * a for t, a in zip(leaves, along))) for s in (1, -1)]
    return along, float((at[0] - at[1]) / (2 * h))


def _agrees(f, plain, leaves, seed=0):
    """fp32 gradients of f along a direction: off by 1e-5 of the sum of magnitudes (some 100 steps of 2^-24 each), and
    1e-6 of it for the differences' own third order."""
    leaves = [t.requires_grad_() for t in leaves]
    grads = torch.autograd.grad(f(*leaves), leaves)
    along, want = _directional(plain, leaves, seed)
    terms = torch.cat([(d.double() * a).reshape(-1) for d, a in zip(grads, along)])
    assert abs(float(terms.sum()) - want) <= 1.1e-5 * float(terms.abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 150])
def test_gradients_agree_with_differences(T):
    g = torch.Generator(device="cuda").manual_seed(T)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    t = torch.randint(0, 130, (T,), device="cuda", generator=g)
    t[::5] = -100
    loss = lambda x, w: torch.nn.functional.cross_entropy(x @ w, t)
    _agrees(lambda x, w: linear_cross_entropy(x, w, t), loss, [rand(T, 40), rand(40, 130) / 6])
    kept = t.clamp(min=0)
    d = rand(T, 40)
    _agrees(lambda w: (embedding(kept, w, 1.5) * d).sum(), lambda w: (1.5 * w[kept] * d).sum(), [rand(130, 40)])
    e = rand(T, 40)
    for gate in (None, rand(40), rand(T, 40)):
        def both(x, y, gamma, post, *gate):
            norm = lambda v, w: tr._norm_op(v, w, 1e-5)
            r = x + 0.5 * (gate[0] * norm(y, post) if gate else norm(y, post))
            return (r * d).sum() + (norm(r, gamma) * e).sum()

        def by_kernel(x, y, gamma, post, *gate):
            r, h = residual_norm(x, y, gamma, post, *gate, scale=0.5)
            return (r * d).sum() + (h * e).sum()

        _agrees(by_kernel, both, [rand(T, 40), rand(T, 40), rand(40), rand(40), *(() if gate is None else (gate,))])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 150])
def test_shared_and_broadcast_operands(T):
    """A table that is the head too, and a gate and a weight that are one value a row and one in all: their gradients are the
    sums of what each use has, in fp32 the separate operands' up to the order of those sums."""
    g = torch.Generator(device="cuda").manual_seed(T)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    t = torch.randint(0, 70, (2, T), device="cuda", generator=g)
    table, post, gate, gamma = (v.requires_grad_() for v in (rand(70, 24), rand(24), rand(T, 1), rand(1)))

    def run(first, second, gate, gamma):
        x = embedding(t[0], first)
        r, h = residual_norm(x, x, gamma, post, gate)
        return linear_cross_entropy(h + 0.1 * r, second, t[1])

    shared = torch.autograd.grad(run(table, table.t(), gate.expand(T, 24), gamma.expand(24)), (table, gate, gamma))
    apart = [v.detach().clone().requires_grad_() for v in (table, table.t().contiguous(), gate.expand(T, 24).contiguous(),
                                                           gamma.expand(24).contiguous())]
    one, two, dgate, dgamma = torch.autograd.grad(run(*apart), apart)
    for got, want, terms in ((shared[0], one + two.t(), one.abs() + two.t().abs()), (shared[1], dgate.sum(1, True), dgate.abs().sum(1, True)),
                             (shared[2], dgamma.sum(0, True), dgamma.abs().sum(0, True))):
        assert torch.all((got - want).abs() <= 26 * 2.0 ** -24 * terms)


# ---------------------------------------------------------------- the decoder


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dim", [64, 256])
def test_step_without_logits_matches_64_bits(dtype, dim):
    """Loss and every parameter's gradient of a step with the embedding, the sums with their norms and the head's loss by the
    kernels."""
    base = _model(torch.float32, "cpu", dim=dim, n_heads=dim // 16)
    tokens = _tokens("cpu")

    def run(model, tokens):
        loss = head_loss(model.hidden(tokens.clamp(min=0)), model.w_D_vocab, tokens)
        loss.backward()
        return loss.detach().double().cpu(), {n.replace(".moe.moe.", ".moe."): p.grad.detach().double().cpu()
                                              for n, p in model.named_parameters() if p.grad is not None}

    gpu = copy.deepcopy(base).to(dtype).cuda()
    got, got_grads = run(gpu, tokens.cuda())
    routes = [b.moe.router.last_routing.indices_TK.detach().long().cpu() for b in gpu.blocks]

    def on_cpu(dt):
        m = copy.deepcopy(base).to(dt)
        for b, idx in zip(m.blocks, routes):
            b.moe = _OracleMoE(b.moe, idx)
        return run(m, tokens)

    (ref, ref_grads), (tru, tru_grads) = on_cpu(dtype), on_cpu(torch.float64)
    assert _rel(got, tru) <= max(2 * _rel(ref, tru), RTOL[dtype])
    assert set(got_grads) == set(tru_grads)
    for name in tru_grads:
        assert _rel(got_grads[name], tru_grads[name]) <= max(2 * _rel(ref_grads[name], tru_grads[name]), RTOL[dtype]), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dim", [64, 72, 256])
def test_forward_has_the_bits_of_the_steps(dtype, dim, monkeypatch):
    """hidden, forward and forward_cached with the sums and norms in one pass and the embedding's kernel are the steps one
    by one, bit for bit, whether or not something has to look between them."""
    model = _model(dtype, dim=dim, n_heads=dim // 8, head_dim=16).eval()
    tokens = _tokens().clamp(min=0)

    def cached():
        cache = PagedKVCache(2, 12, 16, dim // 8, 16, dtype=dtype, device="cuda")
        seq = cache.add()
        out = [model.forward_cached(tokens[0, :17], cache, cache.extend({seq: 17}), torch.tensor([3, 16], device="cuda"))]
        out += [model.forward_cached(tokens[0, i:i + 1], cache, cache.extend({seq: 1})) for i in range(17, 20)]
        return torch.cat(out)

    with torch.no_grad():
        seen = []
        got = model(tokens), model.hidden(tokens), cached()
        handle = model.blocks[1].norm_attention.register_forward_hook(lambda m, i, o: seen.append(i[0]))
        hooked = model(tokens), model.hidden(tokens), cached()
        handle.remove()
        assert len(seen) == 2 + 1 + 3 or len(seen) == 2 + 4
        whole = []
        handle = model.blocks[0].register_forward_hook(lambda m, i, o: whole.append(o))
        by_blocks = model(tokens), model.hidden(tokens), cached()
        handle.remove()
        assert len(whole) == 2
        monkeypatch.setattr(tr, "_add_norm", lambda x, y, norm: (x + y, norm(x + y)))
        monkeypatch.setattr(tr, "embedding", lambda t, w: w[t])
        steps = model(tokens), model.hidden(tokens), cached()
    for other in (hooked, by_blocks, steps):
        assert all(torch.equal(a, b) for a, b in zip(got, other))
    assert torch.equal(seen[0], whole[0])


@pytest.mark.gpu
def test_training_runs_with_and_without_logits():
    """train_step and Trainer with fused_loss: the same losses as each other, of the loss with the logits up to bf16's
    rounding of those (half a step of 2^-8 of each).  Every parameter has a gradient, and the table and the head move (a
    norm's weights of 1 need not: their bf16 neighbours are 2^-8 and 2^-7 away, and a step of 2^-10 rounds to none)."""
    model = _model(vocab_size=1003, dim=128, n_heads=2, head_dim=64)
    tokens = _tokens(vocab=1003)
    with torch.no_grad():
        inputs = tokens.clamp(min=0)
        plain = float(next_token_loss(model(inputs), tokens))
        logits = model.hidden(inputs).float() @ model.w_D_vocab.float()
    twin = copy.deepcopy(model)
    before = [p.detach().clone() for p in (model.embedding.w_vocab_D, model.w_D_vocab)]
    trainer, opt = Trainer(model, fused_loss=True), make_optimizer(twin)
    for step in range(2):
        loss, local = trainer.step(tokens.cpu())
        want = train_step(twin, opt, tokens, fused_loss=True)
        assert torch.equal(loss, want) and torch.equal(local, want)
        if step == 0:
            assert abs(float(loss) - plain) <= 2 * 2.0 ** -8 * float(logits.abs().max())
    assert all(p.grad is not None and bool((p.grad != 0).any()) for p in model.parameters())
    assert all(not torch.equal(p, b) for p, b in zip((model.embedding.w_vocab_D, model.w_D_vocab), before))
    # no target at all: NaN, and nothing waits
    nothing = torch.full((2, 5), -100, device="cuda")
    assert torch.isnan(head_loss(model.hidden(nothing.clamp(min=0)), model.w_D_vocab, nothing))


@pytest.mark.gpu
def test_transforms_of_the_embedding_and_refused_tangents():
    """Forward mode and functional transforms go through the module's indexing; the operators refuse a tangent."""
    emb = tr.Embedding(7, 8).cuda()
    t = torch.tensor([1, 6, 1], device="cuda")
    tangent = torch.randn(7, 8, device="cuda")
    call = lambda w: torch.func.functional_call(emb, {"w_vocab_D": w}, (t,))
    out, d = torch.func.jvp(call, (emb.w_vocab_D.detach(),), (tangent,))
    assert torch.equal(out, emb.w_vocab_D[t]) and torch.equal(d, tangent[t])
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), torch.no_grad():
        w = fw.make_dual(emb.w_vocab_D.detach(), tangent)
        x = torch.randn(3, 7, device="cuda")
        for f in (lambda: embedding(t, w), lambda: linear_cross_entropy(x, w, t), lambda: residual_norm(w, w, w[0])):
            with pytest.raises(RuntimeError):
                f()


class _WholeModules(torch.fx.Tracer):
    def __init__(self, *opened):
        super().__init__()
        self.opened = opened

    def is_leaf_module(self, m, name):
        return not isinstance(m, self.opened)


def test_modules_are_traced_and_scripted():
    """torch.fx of the embedding, of a block and of the model around their parts, and torch.jit.script of the embedding."""
    emb = tr.Embedding(7, 8)
    t = torch.tensor([[1, 6, 1]])
    other = torch.tensor([[0, 3], [2, 2]])
    for made in (torch.fx.symbolic_trace(emb), torch.jit.script(emb), torch.jit.trace(emb, t)):
        assert torch.equal(made(other), emb.w_vocab_D[other])
    model = _model(torch.float32, "cpu")
    calls = lambda tracer, m: [n.target for n in tracer.trace(m).nodes if n.op == "call_module"]
    assert calls(_WholeModules(), model) == ["embedding", "blocks.0", "blocks.1", "norm"]
    assert calls(_WholeModules(), model.blocks[0]) == ["norm_attention", "attention", "dropout", "norm_mlp", "moe", "dropout"]
    parts = calls(_WholeModules(tr.TransformerBlockMoe), model)
    assert len(parts) == 2 + 2 * 6 and parts[-1] == "norm"


@pytest.mark.gpu
def test_embedding_is_recorded_on_the_gpu():
    """Programs that record torch's operations record the module's: a trace, a graph of them, fake tensors, a compiled whole."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    emb = tr.Embedding(700, 8).cuda()
    t = torch.randint(0, 700, (40, 30), device="cuda")
    other = torch.randint(0, 700, (40, 30), device="cuda")
    for made in (torch.fx.symbolic_trace(emb), torch.jit.script(emb), torch.jit.trace(emb, t), make_fx(emb)(t),
                 torch.compile(emb, backend="eager", fullgraph=True)):
        assert torch.equal(made(other), emb.w_vocab_D[other])
    with FakeTensorMode(), torch.device("cuda"):
        assert tr.Embedding(700, 8)(torch.zeros(40, 30, dtype=torch.int64)).shape == (40, 30, 8)


def test_what_stands_in_for_a_call_is_seen(monkeypatch):
    """Module.compile's replacement of a module's call, and another forward of the class."""
    norm, block = tr.RMSNorm(8), _model(torch.float32, "cpu").blocks[0]
    assert tr._bare(norm, tr.RMSNorm) and tr._bare(block, tr.TransformerBlockMoe)
    norm.compile(backend="eager")
    block.compile(backend="eager")
    assert not tr._bare(norm, tr.RMSNorm) and not tr._bare(block, tr.TransformerBlockMoe)
    for kind, module in ((tr.RMSNorm, tr.RMSNorm(8)), (tr.TransformerBlockMoe, _model(torch.float32, "cpu").blocks[0])):
        assert tr._bare(module, kind)
        forward = kind.forward
        monkeypatch.setattr(kind, "forward", lambda self, *a: forward(self, *a))
        assert not tr._bare(module, kind)
    assert tr._bare(module, kind, "forward_cached")
    monkeypatch.setattr(kind, "forward_cached", lambda self, *a: None)
    assert not tr._bare(module, kind, "forward_cached")


@pytest.mark.gpu
def test_compiled_parts_are_called():
    """hidden, forward and forward_cached call a block or norm through what Module.compile has put in its place."""
    model = _model().eval()
    tokens = _tokens().clamp(min=0)
    with torch.no_grad():
        want = model(tokens)
        for part, times in ((model.blocks[1], 1), (model.blocks[1].norm_attention, 2), (model.blocks[0].norm_mlp, 2), (model.norm, 2)):
            seen = []

            def call(*a, impl=part._call_impl):
                seen.append(a)
                return impl(*a)

            part._compiled_call_impl = call
            assert torch.equal(model(tokens), want)
            cache = PagedKVCache(2, 12, 16, 4, 16, dtype=torch.bfloat16, device="cuda")
            model.forward_cached(tokens[0], cache, cache.extend({cache.add(): 24}))
            part._compiled_call_impl = None
            assert len(seen) == times


def test_chunks_of_rows_are_what_a_launch_holds():
    """Past 2^26 rows the statistics of a chunk are those of 2^26 (4 numbers of 4 bytes and 8 values of 2 a row beside them)."""
    of = lambda T: _lib.query("abacus_linear_cross_entropy_ws_bytes", T, 8, 8, _lib.BF16, 0)
    assert of(1 << 27) - of(1 << 26) == (1 << 26) * (4 * 4 + 8 * 2)


@pytest.mark.parametrize("name,args,msg", [
    ("abacus_embedding_bwd", (16, 16, 4, 1 << 29, 8, 1.0, 1, 16, 16, 1 << 40, None), "tokens of a table of 536870912 x 8"),
])
def test_entry_points_refuse_what_no_launch_holds(name, args, msg):
    with pytest.raises(RuntimeError, match=msg):
        _lib.call(name, *args)


@pytest.mark.gpu
@pytest.mark.parametrize("V,D", [((1 << 30) + 8, 1), ((1 << 28) + 8, 2), (3, (1 << 22) + 8)])
def test_embedding_of_tables_past_the_kernels(V, D):
    """Rows, columns and tokens past what the kernels hold go by indexing, as all did, both ways."""
    emb = torch.nn.Module.__new__(tr.Embedding)
    torch.nn.Module.__init__(emb)
    emb.w_vocab_D = torch.nn.Parameter(torch.zeros(V, D, device="cuda", dtype=torch.bfloat16))
    with torch.no_grad():
        emb.w_vocab_D[-2:] = torch.arange(1, 3, device="cuda")[:, None].bfloat16()
    t = torch.tensor([[0, V - 1], [V - 1, V - 2]], device="cuda")
    out = emb(t)
    assert torch.equal(out[..., -1].float(), torch.tensor([[0.0, 2.0], [2.0, 1.0]], device="cuda"))
    dw, = torch.autograd.grad(out, emb.w_vocab_D, torch.ones_like(out))
    assert torch.equal(dw[[0, 1, V - 2, V - 1], 0].float().cpu(), torch.tensor([1.0, 1.0 if V == 3 else 0.0, 1.0, 2.0]))


@pytest.mark.gpu
def test_embedding_of_more_tokens_than_the_kernels_hold(monkeypatch):
    emb = tr.Embedding(50, 8).cuda()
    t = torch.randint(0, 50, (9, 4), device="cuda")
    monkeypatch.setattr(tr, "_EMBEDDING_MOST", (50, 8, 36))
    monkeypatch.setattr(tr, "embedding", lambda t, w: torch.zeros(0))
    assert emb(t).numel() == 0 and torch.equal(emb(t.repeat(2, 1)), emb.w_vocab_D[t.repeat(2, 1)])


_LOSS = ("abacus_linear_cross_entropy", (16, 8, 16, 16, 4, 8, 10, -100, 1, 2, None, 16, 16, 16, 16, 1 << 20, None))
_SCALE = ("abacus_scale_by", (16, 4, 16, 4, 1, 16, None))
_EMBED = ("abacus_embedding_fwd", (16, 16, 4, 8, 8, 1.0, 1, 16, None))
_EMBED_BWD = ("abacus_embedding_bwd", (16, 16, 4, 8, 8, 1.0, 1, 16, 16, 1 << 20, None))
_NORM = ("abacus_residual_norm_fwd", (16, 16, 16, None, None, 0, 4, 64, 1.0, 1e-5, 1, 16, 16, None, None, None))
_NORM_BWD = ("abacus_residual_norm_bwd", (16, 16, 16, None, 16, None, None, 0, 16, None, 4, 64, 1.0, 1, 16, None, 16, None, None, 16, 1 << 20, None))


@pytest.mark.parametrize("call,at,value,msg", [
    *((_LOSS, at, None, "null") for at in (0, 2, 3)), *((_LOSS, at, 8, "aligned") for at in (2, 12, 13, 14)),
    *((_SCALE, at, None, "null") for at in (0, 2, 5)), *((_SCALE, at, 24, "aligned") for at in (0, 2)),
    *((_EMBED, at, None, "null") for at in (0, 1, 7)),
    *((_EMBED_BWD, at, None, "null") for at in (0, 1, 7)), (_EMBED_BWD, 8, 20, "aligned"),
    *((_NORM, at, None, "null") for at in (0, 1, 2, 11, 12)),
    *((_NORM_BWD, at, None, "null") for at in (2, 4, 14)), (_NORM_BWD, 19, 24, "aligned"),
], ids=lambda v: v[0] if isinstance(v, tuple) else str(v))
def test_entry_points_refuse_missing_and_unaligned_operands(call, at, value, msg):
    name, args = call
    with pytest.raises(RuntimeError, match=msg):
        _lib.call(name, *args[:at], value, *args[at + 1:])


def _elsewhere(v):
    """v's values at another place: rows with gaps between them, no vector aligned."""
    if v.dim() < 2:
        return torch.zeros(2 * v.numel() + 1, dtype=v.dtype, device=v.device)[1::2].copy_(v)
    return torch.zeros(v.shape[0], v.shape[1] + 3, dtype=v.dtype, device=v.device)[:, 1:-2].copy_(v)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 150])
def test_saved_tensors_of_other_strides(T):
    """Hooks on saved tensors may bring them back at other places, with other strides: the same gradients."""
    g = torch.Generator(device="cuda").manual_seed(T)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16().requires_grad_()
    t = torch.randint(0, 70, (2, T), device="cuda", generator=g)
    table, w, y, gamma, post, gate = rand(70, 40), rand(40, 70), rand(T, 40), rand(40), rand(40), rand(T, 40)
    leaves = table, w, y, gamma, post, gate

    def run(reduction):
        x = embedding(t[0], table)
        r, h = residual_norm(x, y, gamma, post, gate, scale=0.5)
        return linear_cross_entropy(h + r, w, t[1], reduction=reduction).sum()

    for reduction in ("mean", "none"):
        want = torch.autograd.grad(run(reduction), leaves)
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, _elsewhere):
            got = torch.autograd.grad(run(reduction), leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_embedding_of_empty_tables():
    """Nothing to look up, or rows of nothing: indexing's results, as before."""
    assert tr.Embedding(0, 8).cuda()(torch.zeros(0, 3, dtype=torch.int64, device="cuda")).shape == (0, 3, 8)
    emb = tr.Embedding(5, 0).cuda()
    out = emb(torch.tensor([4, 0], device="cuda"))
    assert out.shape == (2, 0) and torch.autograd.grad(out.sum(), emb.w_vocab_D)[0].shape == (5, 0)


@pytest.mark.gpu
def test_step_without_logits_holds_no_more_than_with_them():
    """The most that a step allocates, with gradients (200 MiB) of more than what the head's loss holds (its 16 MiB of probabilities and
    up to 128 MiB of partial sums): the last step's are gone by then."""
    peaks = []
    for fused_loss in (False, True):
        model = _model(vocab_size=8000, dim=256, n_heads=4, head_dim=64, n_experts=16, hidden_dim=4096)
        opt = make_optimizer(model)
        tokens = torch.randint(0, 8000, (4, 256), device="cuda")
        for step in range(3):
            if step == 1:
                torch.cuda.synchronize()
                torch.cuda.reset_peak_memory_stats()
            train_step(model, opt, tokens, fused_loss=fused_loss)
        torch.cuda.synchronize()
        peaks.append(torch.cuda.max_memory_allocated())
        del model, opt
    assert peaks[1] <= peaks[0]
