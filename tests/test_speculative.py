"""verify_drafts against a restatement by running sums in Python, on the CPU and on the GPU."""

import math

import pytest
import torch

from abacus_amd.speculative import verify_drafts

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _probabilities(row, temperature):
    top = max(row)
    e = [math.exp((x - top) / temperature) for x in row]
    total = math.fsum(e)
    return [x / total for x in e]


def _restated(target, tokens, start, u, draft, temperature):
    accepted, following = [], []
    for a, b in zip(start, start[1:]):
        n, token = 0, -1
        for t in range(a, b):
            x = tokens[t + 1] if t + 1 < b else None
            p = _probabilities(target[t], temperature)
            q = [0.0] * len(p) if x is None else _probabilities(draft[t], temperature) if draft else [
                float(i == x) for i in range(len(p))]
            if x is not None and u[t][0] * q[x] < p[x]:
                n += 1
                continue
            mass = [max(y - z, 0.0) for y, z in zip(p, q)]
            border, run = u[t][1] * math.fsum(mass), 0.0
            for token, m in enumerate(mass):
                run += m
                if run > border:
                    break
            break
        accepted.append(n)
        following.append(token)
    return accepted, following


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,sizes,drafter,temperature", [
    (11, [1, 3, 0, 5], True, 1.0), (4097, [4, 1], True, 0.7), (9001, [2, 3], False, 1.3), (2, [6, 1, 1], False, 0.5),
    (1, [3], True, 1.0)])
def test_matches_the_restatement(device, dtype, V, sizes, drafter, temperature):
    g = torch.Generator().manual_seed(V)
    T = sum(sizes)
    target = (2 * torch.randn(T, V, generator=g)).to(dtype)
    draft = (target.float() + 0.5 * torch.randn(T, V, generator=g)).to(dtype) if drafter else None
    for seed in range(4):
        g.manual_seed(100 + seed)
        tokens = torch.multinomial(torch.softmax(target.float() / temperature, -1), 1, generator=g)[:, 0].roll(1)
        u = torch.rand(T, 2, generator=g)
        start = torch.tensor([0, *sizes]).cumsum(0).to(torch.int32)
        want = _restated(target.tolist(), tokens.tolist(), start.tolist(), u.tolist(), draft.tolist() if drafter else None,
                         temperature)
        got = verify_drafts(target.to(device), tokens.to(device), start.to(device), u.to(device),
                            draft.to(device) if drafter else None, temperature)
        assert got[0].dtype == torch.int32 and got[1].dtype == torch.int64
        for s, n in enumerate(sizes):
            if n == 0:
                want[1][s] = -1
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]


def _restated64(target, tokens, start, u, draft, temperature):
    """The same in torch's 64-bit operations, for large vocabularies; p itself where p - q leaves nothing."""
    V, accepted, following = target.shape[1], [], []
    for a, b in zip(start, start[1:]):
        n, token = 0, -1
        for t in range(a, b):
            x = tokens[t + 1] if t + 1 < b else None
            p = torch.softmax(target[t].double() / temperature, 0)
            q = torch.zeros_like(p)
            if x is not None and draft is not None:
                q = torch.softmax(draft[t].double() / temperature, 0)
            elif x is not None and 0 <= x < V:
                q[x] = 1.0
            if x is not None and 0 <= x < V and u[t][0] * float(q[x]) < float(p[x]):
                n += 1
                continue
            mass = (p - q).clamp(min=0.0)
            upto = (mass if float(mass.sum()) > 0 else p).cumsum(0)
            token = int((upto <= u[t][1] * float(upto[-1])).sum())
            break
        accepted.append(n)
        following.append(token)
    return accepted, following


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,sizes,drafter", [
    (9001, [4] * 40, True),       # blocks enough for 32 logits a thread, a slice that is not full
    (8193, [3] * 100, False),
    (300007, [3, 1], True),       # more than 64 slices of the second launch
    (600011, [2, 2], True),       # and of the first
    (600011, [3], False),
    (5003, [41, 33, 2], True),    # more rows than a block keeps
])
def test_sizes_that_other_launches_serve(device, dtype, V, sizes, drafter):
    g = torch.Generator().manual_seed(V)
    T = sum(sizes)
    start = torch.tensor([0, *sizes]).cumsum(0).to(torch.int32)
    target = (3 * torch.randn(T, V, generator=g)).to(dtype)
    draft = (target.float() + 0.2 * torch.randn(T, V, generator=g)).to(dtype) if drafter else None
    tokens = (draft if drafter else target).float().argmax(-1).roll(1)  # likely ones: long runs are accepted
    accepted = []
    for seed in range(3):
        u = torch.rand(T, 2, generator=g.manual_seed(seed))
        if max(sizes) > 32:
            u[:, 0] *= 0.02 * (seed + 1)  # a rejection late in the long sequences, or none
        if seed == 2:
            tokens[start[1:-1].long() - 1] = V - 1  # an unlikely last draft
        want = _restated64(target, tokens.tolist(), start.tolist(), u.tolist(), draft, 0.8)
        got = verify_drafts(target.to(device), tokens.to(device), start.to(device), u.to(device),
                            draft.to(device) if drafter else None, 0.8)
        assert (got[0].tolist(), got[1].tolist()) == want
        accepted += want[0]
    assert max(sizes) <= 32 or max(accepted) > 32


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3000, 9001, 300007])
def test_no_mass_is_left_of_the_difference(device, dtype, V):
    """A draft outside the vocabulary from a drafter that agrees with the target: the next token is drawn from p."""
    g = torch.Generator().manual_seed(V)
    target = (2 * torch.randn(3, V, generator=g)).to(dtype)
    tokens, start = torch.tensor([0, V, 1]), torch.tensor([0, 2, 3], dtype=torch.int32)
    for u1 in (0.0, 0.3, 0.77, 1.0 - 2.0 ** -24):
        u = torch.tensor([[0.0, u1], [0.0, 0.0], [0.0, u1]])
        want = _restated64(target, tokens.tolist(), start.tolist(), u.tolist(), target, 1.1)
        got = verify_drafts(target.to(device), tokens.to(device), start.to(device), u.to(device), target.to(device), 1.1)
        assert (got[0].tolist(), got[1].tolist()) == want and want[0] == [0, 0]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,T", [(600011, 3), (9001, 300)])
def test_temperature_zero_over_many_slices(device, dtype, V, T):
    """The lowest of the largest logits, wherever its slice is; a NaN in the last slice is found."""
    g = torch.Generator().manual_seed(V)
    target = torch.randn(T, V, generator=g).to(dtype)
    at = torch.randint(0, V, (T, 2), generator=g)
    target.scatter_(1, at, 50.0)
    target[T - 1, V - 1] = math.nan
    best = at.amin(1)
    start = torch.arange(T + 1, dtype=torch.int32)
    got = verify_drafts(target.to(device), torch.zeros(T, dtype=torch.int64, device=device), start.to(device), temperature=0.0)
    assert not got[0].any() and got[1].tolist() == [*best[:-1].tolist(), -1]
    one = torch.tensor([0, T], dtype=torch.int32, device=device)
    got = verify_drafts(target.to(device), best.roll(1).to(device), one, temperature=0.0)
    assert (got[0].item(), got[1].item()) == (T - 1, -1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("temperature", [1e-3, 1e-15, 1e-30, 1e-310, 1e30])
def test_temperatures_far_from_one(device, drafter, temperature):
    """Far below 1 the tokens that share the largest logit share the row, whatever its size; far above all do."""
    V, T = 9001, 6
    g = torch.Generator().manual_seed(7)
    target = torch.randn(T, V, generator=g) + 50.3
    draft = torch.randn(T, V, generator=g) - 77.7 if drafter else None
    tokens = torch.tensor([0, 100, 8500, 3, 100, 100])
    for row in range(T):
        target[row, [100, 8500, 40]] = 61.7
        if drafter:
            draft[row, [100, 8500, 7, 8]] = -60.3
    start = torch.tensor([0, 1, 3, 6], dtype=torch.int32)
    for seed in range(6):
        u = torch.rand(T, 2, generator=g.manual_seed(seed))
        want = _restated(target.tolist(), tokens.tolist(), start.tolist(), u.tolist(), draft.tolist() if drafter else None,
                         temperature)
        got = verify_drafts(target.to(device), tokens.to(device), start.to(device), u.to(device),
                            draft.to(device) if drafter else None, temperature)
        assert (got[0].tolist(), got[1].tolist()) == want


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_temperature_zero_takes_the_lowest_of_equals(device, dtype):
    V = 8200
    target = torch.zeros(4, V, dtype=dtype)
    target[0, [5, 4100]] = 1.0
    target[1, [8199, 8000]] = 2.0
    target[3] = -1.0
    start = torch.tensor([0, 3, 4], dtype=torch.int32)
    for tokens, want in (([9, 5, 8000, 1], ([2, 0], [0, 0])), ([9, 5, 8199, 1], ([1, 0], [8000, 0])),
                         ([9, 4100, 8000, 1], ([0, 0], [5, 0])), ([9, -1, V, 1], ([0, 0], [5, 0]))):
        got = verify_drafts(target.to(device), torch.tensor(tokens).to(device), start.to(device), temperature=0.0)
        assert (got[0].tolist(), got[1].tolist()) == want


@pytest.mark.parametrize("device", DEVICES)
def test_borders(device):
    """Probabilities 1/4, 1/4, 1/2: a random number on a border belongs to the token after it."""
    target = torch.log(torch.tensor([[1.0, 1.0, 2.0]])).repeat(2, 1)
    target[:, 2] = 2 * torch.log(torch.tensor(1.0)) + target[:, 2]
    start = torch.tensor([0, 2], dtype=torch.int32)

    def run(x, u0, u1, draft=None):
        got = verify_drafts(target.to(device), torch.tensor([0, x]).to(device), start.to(device),
                            torch.tensor([[u0, u1], [0.0, 0.0]]).to(device), draft)
        return got[0].item(), got[1].item()

    assert run(0, 0.2, 0.9) == (1, 0)   # 0.2 * 1 < 1/4
    assert run(0, 0.3, 0.0) == (0, 1)   # p without token 0: 1/4, 1/2
    assert run(0, 0.3, 0.34) == (0, 2)
    assert run(2, 0.6, 0.4) == (0, 0) and run(2, 0.6, 0.6) == (0, 1)
    assert run(7, 0.0, 0.2) == (0, 0) and run(-1, 0.0, 0.3) == (0, 1)  # no such token: from p
    same = target.to(device)
    assert run(1, 1.0 - 2.0 ** -24, 0.0, same) == (1, 0)  # p = q is always accepted


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_rows_without_a_distribution(device, temperature):
    inf = math.inf
    target = torch.tensor([[0.0, math.nan], [0.0, inf], [-inf, -inf], [-inf, 0.0]])
    for t, want in ((0, (0, -1)), (1, (0, -1)), (2, (0, -1)), (3, (1, 1))):
        rows = torch.stack([target[t], target[3]]).to(device)
        got = verify_drafts(rows, torch.tensor([0, 1]).to(device), torch.tensor([0, 2], dtype=torch.int32).to(device),
                            torch.full((2, 2), 0.5).to(device), None, temperature)
        assert (got[0].item(), got[1].item()) == want
    if temperature:  # the drafter's row
        rows = torch.zeros(2, 2, device=device)
        got = verify_drafts(rows, torch.tensor([0, 1]).to(device), torch.tensor([0, 2], dtype=torch.int32).to(device),
                            torch.full((2, 2), 0.5).to(device), torch.full((2, 2), math.nan).to(device))
        assert (got[0].item(), got[1].item()) == (0, -1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("temperature,drafter", [(0.9, True), (0.9, False), (0.0, False)])
@pytest.mark.parametrize("start,T,good", [([0, 2, 0, 3], 3, 1), ([0, 5, 3, 8], 8, 1), ([0, 3, 1, 3, 4], 4, 1), ([0, 2, 5, 9, 8], 8, 2),
                                          ([-1, 2, 4], 4, 0), ([0, 4, 4, 8, 0, 0], 8, 3), ([8, 8], 4, 0), ([1, 4, 3, 8], 8, 1),
                                          ([0, *range(2, 301, 2), 6, 300], 300, 150), ([0, *[4] * 1100, 2, 8], 8, 1100)])
def test_no_rows_from_the_first_bad_range_on(device, temperature, drafter, start, T, good):
    """What comes before a range that runs backwards or past the rows is as without the rest, whose ranges share
    its rows; the rest has none.  (What a kernel left out would be what the last call of these sizes wrote.)"""
    V, S = 9001, len(start) - 1
    g = torch.Generator().manual_seed(T)
    target = (2 * torch.randn(T, V, generator=g)).to(device)
    draft = target + 0.3 * torch.randn(T, V, generator=g).to(device) if drafter else None
    tokens = target.argmax(-1).roll(1)
    u = torch.rand(T, 2, generator=g).to(device) * torch.tensor([0.5, 1.0], device=device)
    call = lambda start, draft: [x.tolist() for x in verify_drafts(
        target, tokens, torch.tensor(start, dtype=torch.int32, device=device), u, draft, temperature)]
    want = call(start[:good + 1] + [start[good]] * (S - good) if good else [0] * (S + 1), draft)
    assert want[0][good:] == [0] * (S - good) and want[1][good:] == [-1] * (S - good)
    for other in (draft, None if draft is None else draft.flip(0)):
        call([0] * (S + 1), other)
        assert call(start, draft) == want


@pytest.mark.parametrize("device", DEVICES)
def test_tokens_are_distributed_as_the_target(device):
    """The first token that comes out of a sequence (its draft or what replaces it) has the target's probabilities:
    over n sequences a token's count is within 5 standard deviations, 5 sqrt(n p (1 - p))."""
    n, V = 20000, 5
    g = torch.Generator().manual_seed(0)
    p, q = torch.randn(1, V, generator=g), torch.randn(1, V, generator=g)
    drafts = torch.multinomial(torch.softmax(q[0], -1), n, replacement=True, generator=g)
    first = []
    for part in drafts.split(10000):
        m = part.numel()
        tokens = torch.stack([torch.zeros_like(part), part], dim=1).flatten()
        start = torch.arange(0, 2 * m + 1, 2, dtype=torch.int32)
        accepted, following = verify_drafts(p.repeat(2 * m, 1).to(device), tokens.to(device), start.to(device),
                                            torch.rand(2 * m, 2, generator=g).to(device), q.repeat(2 * m, 1).to(device))
        first.append(torch.where(accepted.cpu() == 1, part, following.cpu()))
    counts = torch.bincount(torch.cat(first), minlength=V).double()
    want = torch.softmax(p[0].double(), -1)
    assert ((counts - n * want).abs() <= 5 * torch.sqrt(n * want * (1 - want))).all()


def test_refusals():
    x = torch.zeros(3, 4)
    tokens, start, u = torch.zeros(3, dtype=torch.int64), torch.tensor([0, 3], dtype=torch.int32), torch.zeros(3, 2)
    with pytest.raises(ValueError, match="temperature"):
        verify_drafts(x, tokens, start, u, None, -1.0)
    with pytest.raises(ValueError, match="uniforms"):
        verify_drafts(x, tokens, start)
    with pytest.raises(ValueError, match="uniforms"):
        verify_drafts(x, tokens, start, u.double())
    with pytest.raises(TypeError):
        verify_drafts(x.double(), tokens, start, u)
    with pytest.raises(ValueError, match="tokens"):
        verify_drafts(x, tokens.int(), start, u)
    with pytest.raises(ValueError, match="query_start"):
        verify_drafts(x, tokens, start.long(), u)
    with pytest.raises(ValueError, match="draft"):
        verify_drafts(x, tokens, start, u, x[:2])
    with pytest.raises(ValueError, match="logits"):
        verify_drafts(x[0], tokens, start, u)
