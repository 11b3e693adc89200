"""Verification of drafted tokens (speculative decoding) against a target model's probabilities.

The reference has no decoding program; this stands beside ``abacus_amd.kv_cache``, whose ``BatchRows`` lay out the
rows.  On the GPU the logits are read once, by HIP kernels on torch's current stream with no host synchronisation;
CPU tensors take torch's operations.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .kv_cache import _call

__all__ = ["verify_drafts"]


def verify_drafts(target_logits_TV: torch.Tensor, tokens_T: torch.Tensor, query_start: torch.Tensor,
                  uniforms_T2: torch.Tensor | None = None, draft_logits_TV: torch.Tensor | None = None,
                  temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """How many drafts of each sequence are accepted, and the token that follows them.

    The rows of sequence s are query_start[s] .. query_start[s + 1] - 1 (int32, (S + 1,)): its last known token,
    then its drafts (int64 tokens_T).  As in ``BatchRows``, from the first range that runs backwards or past the
    rows on sequences have none.  Row t of target_logits_TV, and of draft_logits_TV, is what the target, and
    the drafter, say about the token after row t; draft_logits_TV of a sequence's last row is not read.  Without
    draft_logits_TV the drafts are taken as certain (a lookup, a greedy drafter).

    With p = softmax(target / temperature) and q = softmax(draft / temperature), draft x after row t is accepted
    where uniforms_T2[t, 0] * q(x) < p(x).  After the first one that is not, row r, the next token is drawn from
    max(p - q, 0) with uniforms_T2[r, 1]: the smallest i whose running sum passes that share of the whole.  With
    all accepted it is drawn from the last row's p.  uniforms_T2: float32 (T, 2) in [0, 1).  So the tokens are
    distributed as if each had been drawn from p.

    temperature 0: a draft is accepted where it is the row's largest logit, the lowest index of equals, and the next
    token is that one; uniforms_T2 and draft_logits_TV are not needed.

    Returns (int32 (S,), int64 (S,)).  A draft outside the vocabulary is not accepted.  A row that is no
    distribution (NaN, +inf, or -inf throughout) accepts nothing and gives -1, a sequence without rows 0 and -1.
    Exponentials and sums are 64-bit, so only a random number within 1e-13 of a border can fall on its other side.
    """
    if target_logits_TV.dim() != 2 or target_logits_TV.shape[1] < 1:
        raise ValueError(f"target logits must be (rows, vocabulary), got {tuple(target_logits_TV.shape)}")
    T, V = target_logits_TV.shape
    dev = target_logits_TV.device
    temperature = float(temperature)
    if not 0.0 <= temperature < math.inf:
        raise ValueError(f"temperature must not be negative, got {temperature}")
    if target_logits_TV.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"logits must be float32 or bfloat16, got {target_logits_TV.dtype}")
    if tokens_T.shape != (T,) or tokens_T.dtype != torch.int64:
        raise ValueError(f"tokens must be int64 of shape {(T,)}, got {tokens_T.dtype} of {tuple(tokens_T.shape)}")
    if query_start.dim() != 1 or query_start.shape[0] < 2 or query_start.dtype != torch.int32:
        raise ValueError("query_start must be int32 of shape (sequences + 1,)")
    if temperature == 0.0:
        uniforms_T2 = draft_logits_TV = None
    elif uniforms_T2 is None or uniforms_T2.shape != (T, 2) or uniforms_T2.dtype != torch.float32:
        raise ValueError(f"uniforms must be float32 of shape {(T, 2)} at a temperature above 0")
    if draft_logits_TV is not None and (draft_logits_TV.shape != (T, V) or draft_logits_TV.dtype != target_logits_TV.dtype):
        raise ValueError(f"draft logits must be {target_logits_TV.dtype} of shape {(T, V)}, got "
                         f"{draft_logits_TV.dtype} of {tuple(draft_logits_TV.shape)}")
    for t in (tokens_T, query_start, uniforms_T2, draft_logits_TV):
        if t is not None and t.device != dev:
            raise ValueError("logits, tokens, query_start and uniforms must be on one device")
    S = query_start.shape[0] - 1
    if not target_logits_TV.is_cuda:
        return _verify_cpu(target_logits_TV, tokens_T, query_start.tolist(), uniforms_T2, draft_logits_TV, temperature)
    if T > 65535 or S > 65535:
        raise ValueError(f"{T} rows of {S} sequences: at most 65535 at once")
    target, tokens, start = target_logits_TV.contiguous(), tokens_T.contiguous(), query_start.contiguous()
    draft = None if draft_logits_TV is None else draft_logits_TV.contiguous()
    uniforms = None if uniforms_T2 is None else uniforms_T2.contiguous()
    nbytes = _lib.query("abacus_verify_drafts_ws_bytes", T, V, S)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    accepted = torch.empty(S, dtype=torch.int32, device=dev)
    following = torch.empty(S, dtype=torch.int64, device=dev)
    at = [None if t is None else t.data_ptr() for t in (target, draft, tokens, start, uniforms)]
    _call(dev, "abacus_verify_drafts", *at, T, V, S, _lib.dtype_code(target.dtype), temperature, accepted.data_ptr(),
          following.data_ptr(), ws.data_ptr(), nbytes)
    return accepted, following


def _softmax(row: torch.Tensor, temperature: float) -> torch.Tensor | None:
    top = row.max()
    if not bool(torch.isfinite(top)):
        return None
    e = torch.exp((row.double() - top.double()) / temperature)
    return e / e.sum()


@torch.no_grad()
def _verify_cpu(target, tokens, start, uniforms, draft, temperature):
    T, V = target.shape
    accepted, following, ended = [], [], False
    for s in range(len(start) - 1):
        first, end = start[s], start[s + 1]
        ended = ended or first < 0 or end < first or end > T
        if ended:
            end = first
        n, token = 0, -1
        for t in range(first, end):
            x = int(tokens[t + 1]) if t + 1 < end else None
            if temperature == 0.0:
                top = target[t].max()
                token = int((target[t] == top).nonzero()[0]) if bool(torch.isfinite(top)) else -1
                if x is None or token < 0 or token != x:
                    break
                n += 1
                continue
            token = -1
            p = _softmax(target[t], temperature)
            if p is None:
                break
            q = torch.zeros_like(p)
            if x is not None and draft is not None:
                q = _softmax(draft[t], temperature)
                if q is None:
                    break
            elif x is not None and 0 <= x < V:
                q[x] = 1.0
            if x is not None and 0 <= x < V and float(uniforms[t, 0]) * float(q[x]) < float(p[x]):
                n += 1
                continue
            mass = torch.clamp(p - q, min=0.0)
            if not bool(mass.sum() > 0):
                mass = p
            upto = torch.cumsum(mass, dim=0)
            passed = (upto > min(float(uniforms[t, 1]), 1.0 - 2.0 ** -53) * float(upto[-1])).nonzero()
            token = int(passed[0]) if len(passed) else int((mass > 0).nonzero()[-1])
            break
        accepted.append(n)
        following.append(token)
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(following, dtype=torch.int64)
