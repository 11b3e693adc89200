"""Generation from a TransformerMoe over a paged cache, with drafted tokens if a drafter is given.

The reference trains its decoder and does not sample from it.  ``generate`` runs the steps of a decoding program:
prompts go into the cache in chunks, then every step feeds each sequence's last token (and the drafts after it) through
``forward_cached``, and ``verify_drafts`` accepts drafts and draws the next token.
"""

from __future__ import annotations

import torch

from .kv_cache import E4M3, PagedKVCache
from .speculative import verify_drafts
from .transformer import TransformerMoe

__all__ = ["generate"]


class _Side:
    """A model, its cache, and what of each sequence is in it."""

    def __init__(self, model: TransformerMoe, room: list[int], page_size: int, dtype: torch.dtype | None):
        self.model = model
        w = model.w_D_vocab
        self.device = w.device
        pages = sum(-(-n // page_size) for n in room)
        self.cache = PagedKVCache(model.n_blocks, pages, page_size, model.n_heads, model.head_dim,
                                  dtype=w.dtype if dtype is None else dtype, device=w.device)
        self.seqs = [self.cache.add() for _ in room]

    def feed(self, tokens: dict[int, list[int]], wanted: dict[int, int]) -> torch.Tensor:
        """Runs these tokens of each sequence; logits of the last wanted[s] rows of each, one after the other."""
        rows = self.cache.extend({self.seqs[s]: len(t) for s, t in tokens.items()})
        at, out = 0, []
        for s, t in tokens.items():
            at += len(t)
            out.extend(range(at - wanted[s], at))
        flat = torch.tensor([x for t in tokens.values() for x in t], dtype=torch.int64).to(self.device)
        return self.model.forward_cached(flat, self.cache, rows, torch.tensor(out, dtype=torch.int64).to(self.device))

    def prefill(self, known: list[list[int]], chunk: int) -> None:
        """All but each sequence's last token."""
        while True:
            have = [self.cache.length(s) for s in self.seqs]
            parts = {s: t[have[s]:min(have[s] + chunk, len(t) - 1)] for s, t in enumerate(known)}
            parts = {s: t for s, t in parts.items() if t}
            if not parts:
                return
            self.feed(parts, dict.fromkeys(parts, 0))

    def keep(self, s: int, length: int) -> None:
        seq = self.seqs[s]
        self.cache.truncate(seq, min(length, self.cache.length(seq)))


def generate(model: TransformerMoe, prompts: list[list[int]], max_new_tokens: int, *, temperature: float = 0.0,
             draft_model: TransformerMoe | None = None, n_draft: int = 4, stop_token: int | None = None,
             generator: torch.Generator | None = None, page_size: int = 64, cache_dtype: torch.dtype | None = None,
             prefill_chunk: int = 2048) -> list[list[int]]:
    """The tokens that follow each prompt: at most max_new_tokens, up to and with stop_token.

    temperature 0 takes the likeliest token each time; above it tokens are drawn with random numbers of `generator`
    (on the model's device).  draft_model (the same vocabulary; of any dtype that a cache holds, on any device) proposes
    n_draft tokens a step, which changes how many steps it takes and not what the tokens are distributed as: its logits
    take the model's dtype before tokens are drawn from them.  cache_dtype: the model's own, or torch.float8_e4m3fn
    (the drafter's cache then too, otherwise that has its own).  Both models must be in eval mode.
    """
    if not prompts or any(len(p) == 0 for p in prompts):
        raise ValueError("prompts must hold at least one token each")
    if max_new_tokens < 0 or n_draft < 1 or prefill_chunk < 1:
        raise ValueError(f"max_new_tokens {max_new_tokens}, n_draft {n_draft}, prefill_chunk {prefill_chunk}")
    if draft_model is not None and draft_model.vocab_size != model.vocab_size:
        raise ValueError(f"a drafter of {draft_model.vocab_size} tokens for a model of {model.vocab_size}")
    known = [[int(x) for x in p] for p in prompts]
    if any(not 0 <= x < model.vocab_size for p in known for x in p):
        raise ValueError(f"tokens must be in 0..{model.vocab_size - 1}")
    ends = [len(p) + max_new_tokens for p in known]
    n_draft = 0 if draft_model is None else n_draft
    room = [end + n_draft for end in ends]
    target = _Side(model, room, page_size, cache_dtype)
    drafter = None if draft_model is None else _Side(draft_model, room, page_size, E4M3 if cache_dtype == E4M3 else None)
    device, dtype = target.device, model.w_D_vocab.dtype
    target.prefill(known, prefill_chunk)
    if drafter is not None:
        drafter.prefill(known, prefill_chunk)
    active = [s for s in range(len(known)) if len(known[s]) < ends[s]]
    while active:
        drafts, draft_logits = {s: [] for s in active}, []
        for _ in range(n_draft):
            new = {s: (known[s] + drafts[s])[drafter.cache.length(drafter.seqs[s]):] for s in active}
            logits = drafter.feed(new, dict.fromkeys(active, 1)).to(device=device, dtype=dtype)
            # one row a sequence and no drafts: a token drawn from each
            start = torch.arange(len(active) + 1, dtype=torch.int32, device=device)
            _, drawn = verify_drafts(logits, torch.zeros(len(active), dtype=torch.int64, device=device), start,
                                     _uniforms(len(active), temperature, generator, device), None, temperature)
            proposals = drawn.tolist()
            if min(proposals) < 0:  # a row without a distribution proposes token 0, with certainty
                certain = torch.full_like(logits[:1], -torch.inf)
                certain[:, 0] = 0.0
                logits = torch.where(drawn[:, None] < 0, certain, logits)
            draft_logits.append(logits)
            for s, x in zip(active, proposals):
                drafts[s].append(max(x, 0))
        logits = target.feed({s: [known[s][-1], *drafts[s]] for s in active}, dict.fromkeys(active, n_draft + 1))
        T = len(active) * (n_draft + 1)
        tokens = torch.tensor([x for s in active for x in (known[s][-1], *drafts[s])], dtype=torch.int64).to(device)
        start = torch.arange(0, T + 1, n_draft + 1, dtype=torch.int32, device=device)
        proposed = None
        if n_draft and temperature > 0:
            proposed = torch.stack([*draft_logits, draft_logits[-1]], dim=1).reshape(T, -1)
        accepted, following = verify_drafts(logits, tokens, start, _uniforms(T, temperature, generator, device), proposed,
                                            temperature)
        for s, n, x in zip(active, accepted.tolist(), following.tolist()):
            if x < 0:
                raise RuntimeError(f"sequence {s}: the model's logits after {len(known[s]) + n} tokens are no distribution")
            new = [*drafts[s][:n], x][:ends[s] - len(known[s])]
            if stop_token in new:
                new = new[:new.index(stop_token) + 1]
            known[s].extend(new)
            for side in (target, drafter):
                if side is not None:
                    side.keep(s, len(known[s]) - 1)
        active = [s for s in active if len(known[s]) < ends[s] and known[s][-1] != stop_token]
    return [t[len(p):] for t, p in zip(known, prompts)]


def _uniforms(n: int, temperature: float, generator: torch.Generator | None, device: torch.device) -> torch.Tensor | None:
    return None if temperature == 0 else torch.rand(n, 2, generator=generator, device=device)
