"""Performance cases of the operators around the decoder's blocks: what a training step calls before, between and after them.

``own`` chooses what ``run`` does: False computes each operator in its plain form (elementary torch operations in 32
bits, or 64 where 32 lose what matters), True calls the framework.  The operator a case measures is in its ``"op"``:

  loss    linear_cross_entropy: the head's product and the cross-entropy of its logits, with the gradients of both
          operands ("grad"), or each row's loss alone
  embed   embedding: rows of the table times a scale, and with "grad" the table's gradient
  norm    residual_norm: a block's output (through a norm of its own, "post", and a gate) added to the residual
          stream, and the next block's norm; with "grad" both ways

A batch is ``rows`` tokens of ``dim`` values over a vocabulary of ``vocab``; ``ignored`` of the loss's targets are the
ignore index (a prompt that is not trained on, padding), ``padded`` of the embedded tokens are one padding id.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp32": 4}
EPS = 1e-5
IGNORE = -100


def _loss(rows, dim, vocab, dtype, ignored=0, grad=True):
    return {"op": "loss", "rows": rows, "dim": dim, "vocab": vocab, "dtype": dtype, "ignored": ignored, "grad": grad}


def _embed(rows, dim, vocab, dtype, padded=0, scaled=False, grad=True):
    return {"op": "embed", "rows": rows, "dim": dim, "vocab": vocab, "dtype": dtype, "padded": padded, "scaled": scaled,
            "grad": grad}


def _norm(rows, dim, dtype, post=False, gate="none", scale=1.0, grad=True):
    return {"op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "post": post, "gate": gate, "scale": scale, "grad": grad}


def listed():
    cases = {
        # the loss of the decoder's own training step: 4 x 2048 tokens, the last of each sequence without a target
        "loss_decoder_bf16": _loss(8192, 1024, 32000, "bf16", ignored=4),
        # a wide model over a large vocabulary: the largest case
        "loss_large_bf16": _loss(16384, 4096, 65536, "bf16"),
        # fine-tuning on answers: over half of the rows are prompt and padding; an odd vocabulary and count of rows
        "loss_answers_bf16": _loss(4093, 2048, 50257, "bf16", ignored=2300),
        # a small model in fp32
        "loss_small_fp32": _loss(1000, 512, 8000, "fp32", ignored=100),
        # the losses of a few given tokens, no gradient: scoring in a serving loop
        "score_rows_bf16": _loss(24, 2048, 50257, "bf16", grad=False),
        # the embedding of a decode step of 64 sequences: latency
        "embed_step_bf16": _embed(64, 2048, 32000, "bf16", grad=False),
        # the embedding of the decoder's own training step, with the table's gradient
        "embed_decoder_bf16": _embed(8192, 1024, 32000, "bf16"),
        # a padded batch, scaled, in fp32 over an odd vocabulary: one id has a third of the tokens
        "embed_padded_fp32": _embed(16384, 2048, 50257, "fp32", padded=5500, scaled=True),
        # between two blocks in a decode step: latency
        "norm_step_bf16": _norm(64, 4096, "bf16", grad=False),
        # between two blocks of a training step, both ways
        "norm_train_bf16": _norm(16384, 4096, "bf16"),
        # norms before and after the block, a gate a channel and a residual scale; odd rows and dim
        "norm_gated_bf16": _norm(4095, 2568, "bf16", post=True, gate="channel", scale=0.5),
        # a gate of each token and channel, fp32
        "norm_token_gate_fp32": _norm(2048, 1000, "fp32", gate="token"),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("loss", "loss", "loss", "embed", "embed", "norm", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if op == "norm":
        dim = rng.choice((64, 256, 1000, 1024, 2048, 2560, 4096, 8 * rng.randint(8, 512), rng.randint(33, 2049)))
        rows = _log(rng, 1, 65536)
        rows = max(1, min(rows, 16384 * 4096 * 2 // (dim * SIZES[dtype])))
        return _norm(rows, dim, dtype, rng.random() < 0.4, rng.choice(("none", "none", "channel", "token")),
                     rng.choice((1.0, 1.0, 0.5, 0.17)), rng.random() < 0.7)
    vocab = rng.choice((1000, 8000, 32000, 32000, 50257, 65536, _log(rng, 50, 65536)))
    if op == "embed":
        dim = rng.choice((64, 512, 1024, 2048, 2560, 4096, 8 * rng.randint(8, 512)))
        rows = _log(rng, 1, 65536)
        rows = max(1, min(rows, 65536 * 2048 // dim))
        return _embed(rows, dim, vocab, dtype, rng.choice((0, 0, rows // 10, rows // 2)), rng.random() < 0.4,
                      rng.random() < 0.7)
    dim = rng.choice((64, 512, 1000, 1024, 2048, 2560, 4096, 8 * rng.randint(8, 512)))
    grad = rng.random() < 0.75
    # no more products than the largest listed cases have
    most = (16384 if dtype == "bf16" else 4096) * 4096.0 * 65536.0
    rows = max(1, min(_log(rng, 1, 16384), int(most / (dim * vocab))))
    return _loss(rows, dim, vocab, dtype, rng.choice((0, 0, rows // 20, rows // 2)), grad)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * (seed + 1) % (1 << 40))


def _normal(gen, shape, std, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _tokens(gen, rows, vocab):
    """Token ids as text has them: a few of them most of the time, at ids in no order."""
    order = torch.randperm(vocab, device="cuda", generator=gen)
    # the id at rank k with a probability near 1 / (k + 2.7), by the inverse of its sum
    share = torch.rand(rows, device="cuda", generator=gen, dtype=torch.float64)
    rank = 2.7 * ((vocab + 2.7) / 2.7) ** share - 2.7
    return order[rank.long().clamp(0, vocab - 1)]


def prepare(case, seed):
    gen, dtype, rows, D = _generator(seed), DTYPES[case["dtype"]], case["rows"], case["dim"]
    state = {"case": case}
    if case["op"] == "loss":
        V = case["vocab"]
        # logits as a trained model's: a deviation of 2.5, and the target's well above the others in most rows
        w = _normal(gen, (D, V), 2.5 / math.sqrt(D), dtype)
        targets = _tokens(gen, rows, V)
        x = _normal(gen, (rows, D), 1.0, torch.float32)
        x += torch.rand(rows, 1, device="cuda", generator=gen) * 1.5 * w[:, targets].t().float()
        x = (x / x.square().mean(dim=-1, keepdim=True).sqrt()).to(dtype)  # as the norm before the head leaves it
        # the ignored rows: prompts of all lengths, so runs of rows and single ones
        targets[torch.randperm(rows, device="cuda", generator=gen)[:case["ignored"] // 2]] = IGNORE
        left = case["ignored"] - case["ignored"] // 2
        at = (targets != IGNORE).nonzero()[:left, 0]
        targets[at] = IGNORE
        return state | {"x": x.requires_grad_(case["grad"]), "w": w.requires_grad_(case["grad"]), "targets": targets}
    if case["op"] == "embed":
        tokens = _tokens(gen, rows, case["vocab"])
        tokens[rows - case["padded"]:] = 0  # padding at the end
        state |= {"w": _normal(gen, (case["vocab"], D), 1.0, dtype).requires_grad_(case["grad"]), "tokens": tokens,
                  "scale": math.sqrt(D) if case["scaled"] else 1.0}
        return state | ({"d_out": _normal(gen, (rows, D), 1e-3, dtype)} if case["grad"] else {})
    # the stream has grown over the blocks before; a block's output is smaller; norm weights around 1
    names = {"x": _normal(gen, (rows, D), 2.0, dtype), "y": _normal(gen, (rows, D), 0.5, dtype),
             "gamma": (1.0 + 0.1 * _normal(gen, (D,), 1.0, torch.float32)).to(dtype)}
    if case["post"]:
        names["post_gamma"] = (0.7 + 0.1 * _normal(gen, (D,), 1.0, torch.float32)).to(dtype)
    if case["gate"] != "none":
        shape = (D,) if case["gate"] == "channel" else (rows, D)
        names["gate"] = torch.sigmoid(_normal(gen, shape, 1.0, torch.float32)).to(dtype)
    state |= {"leaves": {n: t.requires_grad_(case["grad"]) for n, t in names.items()}}
    if case["grad"]:
        state |= {"dr": _normal(gen, (rows, D), 1e-3, dtype), "dh": _normal(gen, (rows, D), 1e-3, dtype)}
    return state


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"loss": _plain_loss, "embed": _plain_embed, "norm": _plain_norm}[state["case"]["op"]](state)


def _own(state):
    from abacus_amd.residual import residual_norm
    from abacus_amd.vocabulary import embedding, linear_cross_entropy

    case = state["case"]
    with torch.set_grad_enabled(case["grad"]):
        if case["op"] == "loss":
            x, w = state["x"], state["w"]
            loss = linear_cross_entropy(x, w, state["targets"], ignore_index=IGNORE,
                                        reduction="mean" if case["grad"] else "none")
            return [loss.detach(), *torch.autograd.grad(loss, (x, w))] if case["grad"] else [loss]
        if case["op"] == "embed":
            out = embedding(state["tokens"], state["w"], scale=state["scale"])
            return [out.detach(), *torch.autograd.grad(out, state["w"], state["d_out"])] if case["grad"] else [out]
        leaves = state["leaves"]
        r, h = residual_norm(**leaves, scale=case["scale"], eps=EPS)
        if not case["grad"]:
            return {"r": r, "h": h}
        grads = torch.autograd.grad((r, h), tuple(leaves.values()), (state["dr"], state["dh"]))
        return {"r": r.detach(), "h": h.detach(), **{f"d_{n}": g for n, g in zip(leaves, grads)}}


# ---------------------------------------------------------------- the plain forms


def _plain_loss(state):
    x, w, targets = state["x"].float(), state["w"].float(), state["targets"]
    kept = targets != IGNORE
    at = torch.where(kept, targets, 0)[:, None]
    logits = x @ w
    top = logits.amax(-1, keepdim=True)
    picked = logits.gather(1, at) - top
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    losses = torch.where(kept, (total.log() - picked)[:, 0], 0.0)
    if not state["case"]["grad"]:
        return [losses]
    count = kept.sum()
    loss = losses.sum(dtype=torch.float64) / count
    p = p.div_(total).scatter_add_(1, at, -torch.ones_like(picked)).mul_((kept / count)[:, None])
    return [loss.float(), (p @ w.t()).to(state["x"].dtype), (x.t() @ p).to(state["w"].dtype)]


def _plain_embed(state):
    w, tokens, scale = state["w"], state["tokens"], state["scale"]
    out = [(w[tokens].float() * scale).to(w.dtype)]
    if state["case"]["grad"]:
        # an id may have tens of thousands of tokens: its sum in 64 bits where the result has 32
        wide = torch.float64 if w.dtype == torch.float32 else torch.float32
        sums = torch.zeros(w.shape, dtype=wide, device="cuda").index_add_(0, tokens, state["d_out"].to(wide))
        out.append((sums * scale).to(w.dtype))
    return out


def _plain_norm(state):
    case, scale = state["case"], state["case"]["scale"]
    x, y, gamma, post, gate = (t if t is None else t.float() for t in
                               (state["leaves"].get(n) for n in ("x", "y", "gamma", "post_gamma", "gate")))
    branch = y
    if post is not None:
        y_inv = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
        normed = y * y_inv
        branch = post * normed
    added = branch if gate is None else gate * branch
    r = (x + scale * added).to(state["leaves"]["x"].dtype)
    # h is the norm of r as it is returned
    inv = (r.float().square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = r.float() * inv
    out = {"r": r, "h": (gamma * n).to(r.dtype)}
    if not case["grad"]:
        return out
    dh = state["dh"].float()
    g = dh * gamma
    dr = state["dr"].float() + inv * (g - n * (g * n).mean(-1, keepdim=True))
    grads = {"x": dr, "gamma": (dh * n).sum(0)}
    d_branch = scale * dr
    if gate is not None:
        d_gate = d_branch * branch
        grads["gate"] = d_gate.sum(0) if case["gate"] == "channel" else d_gate
        d_branch = d_branch * gate
    if post is not None:
        grads["post_gamma"] = (d_branch * normed).sum(0)
        g = d_branch * post
        d_branch = y_inv * (g - normed * (g * normed).mean(-1, keepdim=True))
    grads["y"] = d_branch
    return out | {f"d_{name}": grads[name].to(r.dtype) for name in state["leaves"]}


# ---------------------------------------------------------------- work and 64-bit results


def work(case):
    rows, D, size = case["rows"], case["dim"], SIZES[case["dtype"]]
    ways = 2 if case["grad"] else 1
    if case["op"] == "loss":
        V, kept = case["vocab"], case["rows"] - case["ignored"]
        given = ways * (kept * D + D * V) * size  # x and w, and their gradients
        return {"bytes": given + (ways - 1) * case["ignored"] * D * size + rows * 8 + (4 if case["grad"] else 4 * rows),
                "flops": (6 if case["grad"] else 2) * kept * D * V}
    if case["op"] == "embed":
        moved = 2 * rows * D + (rows * D + case["vocab"] * D if case["grad"] else 0)
        return {"bytes": moved * size + ways * rows * 8, "flops": rows * D * ways}
    token_gate = case["gate"] == "token"
    tensors = 4 + token_gate  # x, y, the gate in; r, h out
    if case["grad"]:
        # r, dr, dh in and dx out; dy out where it is another than dx; y and the gate in again where they are needed
        changed = case["post"] or case["gate"] != "none" or case["scale"] != 1.0
        tensors += 4 + changed + (case["post"] or case["gate"] != "none") + 2 * token_gate
    vectors = (1 + case["post"] + (case["gate"] == "channel")) * ways * D
    return {"bytes": (tensors * rows * D + vectors) * size, "flops": (8 if case["grad"] else 4) * rows * D}


def exact(case, seed):
    state = prepare(case, seed)
    return {"loss": _exact_loss, "embed": _exact_embed, "norm": _exact_norm}[case["op"]](state)


def _exact_loss(state):
    """torch's cross-entropy and its derivatives in 64 bits, a few rows at a time."""
    case, targets = state["case"], state["targets"]
    w = state["w"].detach().double().requires_grad_(case["grad"])
    count = int((targets != IGNORE).sum())
    losses, dx = [], []
    for at in range(0, case["rows"], 2048):
        x = state["x"].detach()[at:at + 2048].double().requires_grad_(case["grad"])
        with torch.set_grad_enabled(case["grad"]):
            each = torch.nn.functional.cross_entropy(x @ w, targets[at:at + 2048], ignore_index=IGNORE, reduction="none")
        losses.append(each.detach())
        if case["grad"]:
            (each.sum() / count).backward()  # w's gradient adds up over the pieces
            dx.append(x.grad)
    losses = torch.cat(losses)
    return [losses.sum() / count, torch.cat(dx), w.grad] if case["grad"] else [losses]


def _exact_embed(state):
    w = state["w"].detach().double().requires_grad_(state["case"]["grad"])
    out = torch.nn.functional.embedding(state["tokens"], w) * state["scale"]
    if not state["case"]["grad"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, w, state["d_out"].double())]


def _exact_norm(state):
    case = state["case"]
    leaves = {n: t.detach().double().requires_grad_(case["grad"]) for n, t in state["leaves"].items()}
    norm = lambda v, weight: weight * v / torch.sqrt(torch.mean(v * v, dim=-1, keepdim=True) + EPS)
    branch = norm(leaves["y"], leaves["post_gamma"]) if case["post"] else leaves["y"]
    r = leaves["x"] + case["scale"] * branch * leaves.get("gate", 1.0)
    h = norm(r, leaves["gamma"])
    if not case["grad"]:
        return {"r": r, "h": h}
    grads = torch.autograd.grad((r, h), tuple(leaves.values()), (state["dr"].double(), state["dh"].double()))
    return {"r": r.detach(), "h": h.detach(), **{f"d_{n}": g for n, g in zip(leaves, grads)}}
