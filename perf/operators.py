"""Performance cases of the serving operators: what one step of a decoding program calls, layer by layer.

``own`` chooses what ``run`` does: False computes each operator in its plain form (elementary torch operations in 32
bits, or 64 where 32 lose what matters), True calls the framework.  The operator a case measures is in its ``"op"``:

  write   KVPages.write: keys and values of new tokens into the pages of a cache, as they are or quantised to e4m3
  read    KVPages.read: the cached keys and values of some sequences, one row per token
  attend  KVPages.attend: attention of new tokens (one each, a few drafted ones, a chunk of a prompt) over the pages
  verify  verify_drafts: drafted tokens against the target's probabilities, and the next token

A batch is ``seqs`` sequences; ``new`` tokens of each are new in this call ("mixed": the first has that many, the
others one), and each has about ``context`` tokens behind it.  Key pages hold (page, head, slot, dim), value pages
(page, head, dim, slot); a quantised cache has one exponent byte per token and head.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
SIZES = {"bf16": 2, "fp32": 4, "e4m3": 1}


def _cache(op, seqs, new, context, heads, kv_heads, head_dim, page, dtype, held, mixed=False):
    return {"op": op, "seqs": seqs, "new": new, "context": context, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype, "held": held, "mixed": mixed}


def _verify(seqs, drafts, vocab, dtype, drafter, temperature):
    return {"op": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "dtype": dtype, "drafter": drafter,
            "temperature": temperature}


def listed():
    cases = {
        # the cache write of a decode step: one token of each of 64 sequences, quantised
        "write_step_S64_e4m3": _cache("write", 64, 1, 1500, 16, 16, 64, 64, "bf16", "e4m3"),
        # the cache write of a long prompt chunk, off every page boundary
        "write_chunk_bf16": _cache("write", 3, 2730, 701, 32, 8, 128, 16, "bf16", "bf16"),
        # reading a quantised cache back, to move the sequences elsewhere
        "read_e4m3": _cache("read", 16, 1, 4096, 16, 16, 64, 64, "bf16", "e4m3"),
        # reading one short sequence back as it is
        "read_one_bf16": _cache("read", 1, 1, 1000, 16, 8, 128, 16, "bf16", "bf16"),
        # one token of one sequence in the decoder's own head layout: the latency of a decode step
        "attend_one_token_bf16": _cache("attend", 1, 1, 700, 16, 16, 64, 64, "bf16", "bf16"),
        # a decode step of a large batch over a quantised cache with shared key heads
        "attend_step_S64_e4m3": _cache("attend", 64, 1, 8192, 32, 8, 128, 64, "bf16", "e4m3"),
        # one token over a very long context: the axis has to be split
        "attend_long_bf16": _cache("attend", 2, 1, 131072, 32, 8, 128, 256, "bf16", "bf16"),
        # drafted tokens of a small fp32 model, small pages
        "attend_drafts_fp32": _cache("attend", 8, 5, 1300, 16, 16, 64, 16, "fp32", "fp32"),
        # a chunk of two prompts over what was cached before: the largest case
        "attend_chunk_bf16": _cache("attend", 2, 2048, 8192, 32, 8, 128, 128, "bf16", "bf16"),
        # a chunk of a prompt beside a decode step of the other sequences, quantised
        "attend_mixed_e4m3": _cache("attend", 25, 1000, 2100, 16, 16, 64, 32, "bf16", "e4m3", mixed=True),
        # four drafted tokens of each of 64 sequences against the drafter's probabilities
        "verify_S64": _verify(64, 4, 32000, "bf16", True, 0.8),
        # one sequence whose drafts come from a lookup: the latency of a step
        "verify_one_lookup_fp32": _verify(1, 7, 50257, "fp32", False, 1.0),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("write", "write", "read", "read", "attend", "attend", "attend", "attend", "attend", "verify", "verify"))
    if op == "verify":
        drafts = rng.randint(0, 8)
        seqs = _log(rng, 1, min(128, 600 // (drafts + 1)))
        return _verify(seqs, drafts, rng.choice((1000, 8000, 32000, 32000, 50257, 65536)), rng.choice(("bf16", "bf16", "fp32")),
                       rng.random() < 0.6, rng.choice((0.0, 0.5, 0.8, 1.0, 1.3)))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    held = "e4m3" if rng.random() < 0.4 else dtype
    head_dim = rng.choice((64, 64, 64, 128, 128, 128, 16, 32, 80, 96))
    group = rng.choice((1, 1, 1, 2, 4, 4, 8, 3))
    kv_heads = rng.choice((1, 2, 4, 8, 8)) if group > 1 else rng.choice((4, 8, 12, 16))
    heads = group * kv_heads
    page = rng.choice((16, 32, 64, 64, 128, 256))
    if op in ("write", "read"):
        new = _log(rng, 1, 4096) if op == "write" and rng.random() < 0.6 else 1
        seqs = _log(rng, 1, max(1, min(128, 12000 // new)))
        context = _log(rng, 1, max(1, min(8192, 65536 // seqs)))
        return _cache(op, seqs, new, context, heads, kv_heads, head_dim, page, dtype, held)
    kind = rng.random()
    if kind < 0.4:  # a decode step
        new, seqs, mixed = 1, _log(rng, 1, 128), False
    elif kind < 0.65:  # drafted tokens
        new, seqs, mixed = rng.randint(2, 9), _log(rng, 1, 64), False
    else:  # a chunk of a prompt, alone or beside a decode step
        new, mixed = _log(rng, 10, 2048), rng.random() < 0.4
        seqs = rng.randint(2, 24) if mixed else rng.randint(1, 2)
    # no more cached values, scores or products than the largest listed cases have
    rows = seqs * heads
    new = min(new, int(math.sqrt(1.3e9 / rows)))
    flops = 4.0 * (seqs if not mixed else 1) * new * heads * head_dim
    most = min(1.3e9 / (seqs * kv_heads * head_dim), 1.3e9 / (rows * new), (6e11 if dtype == "bf16" else 2e11) / flops)
    context = max(1, min(_log(rng, 1, 131072), int(most) - new))
    return _cache("attend", seqs, new, context, heads, kv_heads, head_dim, page, dtype, held, mixed)


def _plan(case):
    """(new tokens, length) of each sequence: lengths differ, up to the context and the new tokens."""
    plan = []
    for s in range(case["seqs"]):
        new = case["new"] if s == 0 or not case["mixed"] else 1
        # a third of the sequences short, the first as long as the case says
        share = 1.0 if s == 0 else (0.35, 1.0, 0.8)[s % 3] - 0.11 * (s % 5) * (s % 3 == 2)
        plan.append((new, max(0, int(case["context"] * share)) + new))
    return plan


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * (seed + 1) % (1 << 40))


def _normal(gen, shape, std, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _quantise(x):
    """(codes, exponent bytes) of the last dimension's rows: code * 2^(byte - 127), |code| at most 448."""
    x = x.float()
    mantissa, exponent = torch.frexp(x.abs().amax(-1))  # mantissa in [0.5, 1)
    e = exponent - torch.where(mantissa <= 0.875, 9, 8)
    e = torch.where(mantissa == 0, 0, e.clamp(-110, 120))
    return (x * _power(-e)[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _power(e):
    """2^e in fp32, exactly, for -127 < e < 128."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _prepare_verify(case, gen):
    rows, vocab, dtype = case["seqs"] * (case["drafts"] + 1), case["vocab"], DTYPES[case["dtype"]]
    # logits as a trained model's: a few likely tokens over a long tail; the drafter's are near the target's
    target = _normal(gen, (rows, vocab), 2.5, dtype)
    near = (target.float() + _normal(gen, (rows, vocab), 0.7, torch.float32)).to(dtype)
    gumbel = -torch.empty(rows, vocab, device="cuda").exponential_(generator=gen).log_()
    drafted = (near.float() / max(case["temperature"], 0.05) + gumbel).argmax(-1)  # the token drawn after each row
    tokens = torch.cat([drafted.new_zeros(1), drafted[:-1]])
    return {"case": case, "target": target, "draft": near if case["drafter"] else None, "tokens": tokens,
            "query_start": torch.arange(0, rows + 1, case["drafts"] + 1, dtype=torch.int32, device="cuda"),
            "uniforms": torch.rand(rows, 2, device="cuda", generator=gen)}


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, gen)
    plan = _plan(case)
    S, page, H, K = len(plan), case["page"], case["kv_heads"], case["head_dim"]
    dtype, held = DTYPES[case["dtype"]], DTYPES[case["held"]]
    used = [-(-length // page) for _, length in plan]
    pages, width = sum(used) + 2, max(used)
    # pages are handed out in no order, as after some time of serving
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).cpu()
    table, at = torch.zeros(S, width, dtype=torch.int32), 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + [new for new, _ in plan]).cumsum(0)
    state = {"case": case, "page_table": table.cuda(), "query_start": starts.to(torch.int32).cuda(),
             "lengths": torch.tensor([length for _, length in plan], dtype=torch.int32).cuda(),
             "longest": max(length for _, length in plan), "max_new": max(new for new, _ in plan),
             "k_scale": None, "v_scale": None}
    T = int(starts[-1])
    if case["op"] == "write":
        state["k_pages"] = torch.zeros(pages, H, page, K, device="cuda").to(held)
        state["v_pages"] = torch.zeros(pages, H, K, page, device="cuda").to(held)
        if held == torch.float8_e4m3fn:
            state["k_scale"] = torch.full((pages, H, page), 127, dtype=torch.uint8, device="cuda")
            state["v_scale"] = state["k_scale"].clone()
        state["k"], state["v"] = (_normal(gen, (T, H, K), 1.0, dtype) for _ in range(2))
        return state
    # q and k as the norms and the rotary embedding leave them (rms 1 per head), v as a projection does
    k = _normal(gen, (pages, H, page, K), 1.0, dtype)
    if held == torch.float8_e4m3fn:
        k, state["k_scale"] = _quantise(k)
    state["k_pages"] = k.to(held)
    v = _normal(gen, (pages, H, page, K), 1.0, dtype)
    if held == torch.float8_e4m3fn:
        v, state["v_scale"] = _quantise(v)
    state["v_pages"] = v.to(held).transpose(2, 3).contiguous()
    if case["op"] == "attend":
        state["q"] = _normal(gen, (T, case["heads"], K), 1.0, dtype)
    return state


def run(state):
    if own:
        return _own(state)
    return {"write": _write, "read": _read, "attend": _attend, "verify": _verify_plain}[state["case"]["op"]](state)


def _own(state):
    from abacus_amd.kv_cache import BatchRows, KVPages
    from abacus_amd.speculative import verify_drafts

    case = state["case"]
    if case["op"] == "verify":
        return verify_drafts(state["target"], state["tokens"], state["query_start"], state["uniforms"],
                             draft_logits_TV=state["draft"], temperature=case["temperature"])
    pages = KVPages(state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"])
    rows = BatchRows(state["page_table"], state["query_start"], state["lengths"], max_new=state["max_new"])
    if case["op"] == "write":
        pages.write(state["k"], state["v"], rows)
        return [t for t in (pages.k, pages.v, pages.k_scale, pages.v_scale) if t is not None]
    if case["op"] == "read":
        return pages.read(rows, state["longest"], dtype=DTYPES[case["dtype"]])
    return pages.attend(state["q"], rows)


# ---------------------------------------------------------------- the plain forms


def _rows_of(state, T):
    """(sequence, position) of each of the T rows."""
    row = torch.arange(T, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(state["query_start"], row, right=True) - 1
    return seq, state["lengths"][seq] - state["query_start"][seq + 1] + row


def _write(state):
    page = state["case"]["page"]
    seq, pos = _rows_of(state, state["k"].shape[0])
    where, slot = state["page_table"][seq, pos // page].long(), (pos % page).long()
    if state["k_scale"] is None:
        state["k_pages"][where, :, slot] = state["k"]
        state["v_pages"][where, :, :, slot] = state["v"]
        return [state["k_pages"], state["v_pages"]]
    for x, pages, scale in ((state["k"], state["k_pages"], state["k_scale"]),
                            (state["v"], state["v_pages"].transpose(2, 3), state["v_scale"])):
        codes, exponents = _quantise(x)
        pages.view(torch.uint8)[where, :, slot] = codes.view(torch.uint8)
        scale[where, :, slot] = exponents
    return [state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"]]


def _held(state):
    """The cached keys and values of all the table's pages in fp32: (S, kv head, position, dim)."""
    table, out = state["page_table"].long(), []
    S = table.shape[0]
    for pages, scale, swap in ((state["k_pages"], state["k_scale"], False), (state["v_pages"], state["v_scale"], True)):
        x = pages.view(torch.uint8)[table].view(pages.dtype) if scale is not None else pages[table]
        x = x.float().transpose(3, 4) if swap else x.float()  # (S, P, H, page, K)
        if scale is not None:
            x = x * _power(scale[table].int() - 127)[..., None]
        out.append(x.transpose(1, 2).reshape(S, x.shape[2], -1, x.shape[4]))
    return out


def _read(state):
    L = state["longest"]
    there = (torch.arange(L, device="cuda") < state["lengths"][:, None])[:, :, None, None]
    return tuple(torch.where(there, x[:, :, :L].transpose(1, 2), 0.0).to(DTYPES[state["case"]["dtype"]]).contiguous()
                 for x in _held(state))


def _attend(state):
    q, starts, lengths, new = state["q"], state["query_start"].long(), state["lengths"], state["max_new"]
    T, H, K = q.shape
    k, v = _held(state)
    S, Hk, L = k.shape[:3]
    row = torch.arange(new, device="cuda")
    there = row < (starts[1:] - starts[:-1])[:, None]  # (S, new)
    at = torch.where(there, starts[:-1, None] + row, 0)
    rows = q.float()[at].view(S, new, Hk, H // Hk, K).permute(0, 2, 3, 1, 4).reshape(S, Hk, -1, K)
    scores = torch.matmul(rows, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(K))
    pos = torch.where(there, lengths[:, None] - (starts[1:] - starts[:-1])[:, None] + row, L)
    unseen = torch.arange(L, device="cuda") > pos[:, :, None]  # (S, new, L)
    scores = scores.view(S, Hk, H // Hk, new, L).masked_fill_(unseen[:, None, None], float("-inf"))
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = weights.sum(-1, keepdim=True)
    v = torch.where(torch.arange(L, device="cuda")[:, None] < lengths[:, None, None, None], v, 0.0)
    out = torch.matmul(weights.view(S, Hk, -1, L), v).view(S, Hk, H // Hk, new, K) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(S, new, H, K)
    return out[there].to(q.dtype)


def _first(seen, counts):
    """The index of the first true value of each row, `counts` where there is none."""
    n = seen.shape[-1]
    return torch.where(seen, torch.arange(n, device=seen.device), n).amin(-1).clamp(max=counts)


def _verify_plain(state):
    case = state["case"]
    S, D, V = case["seqs"], case["drafts"], case["vocab"]
    target, tokens = state["target"].view(S, D + 1, V), state["tokens"].view(S, D + 1)[:, 1:]
    u = state["uniforms"].view(S, D + 1, 2).double()
    if case["temperature"] == 0.0:
        best = torch.where(target == target.amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1)
        accepted = _first(best[:, :D] != tokens, D) if D else tokens.new_zeros(S)
        return accepted.to(torch.int32), best.gather(1, accepted[:, None])[:, 0]
    # borders between two tokens are as fine as the random numbers, so in 64 bits
    p = _softmax(target.double() / case["temperature"])
    if case["drafter"]:
        q = _softmax(state["draft"].view(S, D + 1, V)[:, :D].double() / case["temperature"])
    else:
        q = torch.zeros(S, D, V, dtype=torch.float64, device="cuda").scatter_(2, tokens[:, :, None], 1.0)
    of = lambda x: x.gather(2, tokens[:, :, None])[:, :, 0]
    accepted = _first(u[:, :D, 0] * of(q) >= of(p[:, :D]), D) if D else tokens.new_zeros(S)
    q = torch.cat([q, q.new_zeros(S, 1, V)], dim=1)
    pick = accepted[:, None, None].expand(S, 1, V)
    p_at, q_at = p.gather(1, pick)[:, 0], q.gather(1, pick)[:, 0]
    mass = (p_at - q_at).clamp_(min=0.0)
    mass = torch.where(mass.sum(-1, keepdim=True) > 0, mass, p_at)
    upto = mass.cumsum(-1)
    border = u[:, :, 1].gather(1, accepted[:, None]) * upto[:, -1:]
    return accepted.to(torch.int32), _first(upto > border, V - 1)


def _softmax(x):
    e = (x - x.amax(-1, keepdim=True)).exp_()
    return e / e.sum(-1, keepdim=True)


# ---------------------------------------------------------------- work and 64-bit results


def work(case):
    if case["op"] == "verify":
        rows, drafted = case["seqs"] * (case["drafts"] + 1), case["seqs"] * case["drafts"] * case["drafter"]
        logits = (rows + drafted) * case["vocab"]
        return {"bytes": logits * SIZES[case["dtype"]] + rows * 16 + case["seqs"] * 12, "flops": 4 * logits}
    plan = _plan(case)
    H, Hk, K = case["heads"], case["kv_heads"], case["head_dim"]
    new, known = sum(n for n, _ in plan), sum(length for _, length in plan)
    row = K * SIZES[case["held"]] + (case["held"] == "e4m3")  # one token's key or value of one head, as it is held
    if case["op"] == "write":
        return {"bytes": 2 * new * Hk * (K * SIZES[case["dtype"]] + row), "flops": 2 * new * Hk * K}
    if case["op"] == "read":
        return {"bytes": 2 * known * Hk * row + 2 * len(plan) * max(n for _, n in plan) * Hk * K * SIZES[case["dtype"]],
                "flops": 0}
    seen = sum(n * length - n * (n - 1) // 2 for n, length in plan)
    return {"bytes": 2 * new * H * K * SIZES[case["dtype"]] + 2 * known * Hk * row, "flops": 4 * K * H * seen}


def exact(case, seed):
    state = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](state)


def _sequences(state):
    """Of each sequence: its rows, its length, and the pool's (page, slot) of its positions."""
    page, starts = state["case"]["page"], state["query_start"].tolist()
    for s, length in enumerate(state["lengths"].tolist()):
        at = torch.arange(length, device="cuda")
        yield slice(starts[s], starts[s + 1]), length, state["page_table"][s].long()[at // page], at % page


def _values(state, where, slot):
    """Cached keys and values of these positions, (positions, kv head, dim), in 64 bits."""
    k, v = state["k_pages"].double()[where, :, slot], state["v_pages"].double()[where, :, :, slot]
    if state["k_scale"] is not None:
        k = k * _exact_power(state["k_scale"][where, :, slot].int() - 127)[..., None]
        v = v * _exact_power(state["v_scale"][where, :, slot].int() - 127)[..., None]
    return k, v


def _exact_power(e):
    """2^e in 64 bits from its bits (a pow() may be off by a step)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest_code(x):
    """The e4m3 value nearest to x (|x| at most 448), halves to even: 3 bits after the leading one, steps of 2^-9 below 2^-6."""
    step = _exact_power(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)  # frexp's exponent is one more than the leading bit's
    return torch.round(x / step) * step


def _exact_write(state):
    k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
    quantised = state["k_scale"] is not None
    scales = [state["k_scale"], state["v_scale"]] if quantised else []
    for rows, length, where, slot in _sequences(state):
        new = rows.stop - rows.start
        where, slot = where[length - new:], slot[length - new:]
        held = []
        for i, x in enumerate((state["k"][rows].double(), state["v"][rows].double())):
            if quantised:
                half, e = torch.frexp(x.abs().amax(-1) / 448.0)  # half in [0.5, 1): the exponent is e, or e - 1 on a border
                e = torch.where(half == 0.0, 0, e - (half == 0.5).int())
                x = _nearest_code(x * _exact_power(-e)[..., None])
                scales[i][where, :, slot] = (e + 127).to(torch.uint8)
            held.append(x)
        k_pages[where, :, slot] = held[0]
        v_pages[where, :, :, slot] = held[1]
    return [k_pages, v_pages, *scales]


def _exact_read(state):
    case = state["case"]
    k, v = (torch.zeros(case["seqs"], state["longest"], case["kv_heads"], case["head_dim"], dtype=torch.float64,
                        device="cuda") for _ in range(2))
    for s, (_, length, where, slot) in enumerate(_sequences(state)):
        k[s, :length], v[s, :length] = _values(state, where, slot)
    return k, v


def _exact_attend(state):
    case, q = state["case"], state["q"]
    if work(case)["flops"] > 4e12:
        return None
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for rows, length, where, slot in _sequences(state):
        k, v = _values(state, where, slot)
        new = rows.stop - rows.start
        later = torch.arange(length, device="cuda") > torch.arange(length - new, length, device="cuda")[:, None]
        for h in range(case["heads"]):
            z = (q[rows, h].double() @ k[:, h // group].t().contiguous()) / math.sqrt(case["head_dim"])
            z[later] = float("-inf")
            out[rows, h] = torch.softmax(z, dim=-1) @ v[:, h // group].contiguous()
    return out


def _exact_verify(state):
    case = state["case"]
    D, temperature = case["drafts"], case["temperature"]
    accepted, following = [], []
    target, tokens, u = state["target"], state["tokens"].tolist(), state["uniforms"].double().tolist()
    for s in range(case["seqs"]):
        first = s * (D + 1)
        for r in range(first, first + D + 1):
            drafted = tokens[r + 1] if r < first + D else None
            if temperature == 0.0:
                token = int((target[r] == target[r].max()).nonzero()[0])
                if token == drafted:
                    continue
                break
            p = torch.softmax(target[r].double() / temperature, dim=0)
            q = torch.zeros_like(p)
            if drafted is not None:
                if case["drafter"]:
                    q = torch.softmax(state["draft"][r].double() / temperature, dim=0)
                else:
                    q[drafted] = 1.0
                if u[r][0] * float(q[drafted]) < float(p[drafted]):
                    continue
            mass = torch.clamp(p - q, min=0.0)
            mass = mass if float(mass.sum()) > 0.0 else p
            upto = torch.cumsum(mass, dim=0)
            token = min(int((upto <= u[r][1] * upto[-1]).sum()), case["vocab"] - 1)
            break
        accepted.append(r - first)
        following.append(token)
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(following)
