"""Plain 64-bit forms of the paged cache's operators, for its tests: built from the unquantised rows, by sequence."""

import math

import torch

from abacus_amd.kv_cache import E4M3, BatchRows, KVPages


def pages_of(n, H, page, K, dtype, device, fill=None):
    """KVPages; `fill`: what every slot holds before anything is written (bytes for e4m3)."""
    if dtype == E4M3:
        k = torch.full((n, H, page, K), 0 if fill is None else fill, dtype=torch.uint8, device=device)
        v = torch.full((n, H, K, page), 0 if fill is None else fill, dtype=torch.uint8, device=device)
        scales = [torch.full((n, H, page), 127 if fill is None else fill, dtype=torch.uint8, device=device) for _ in "kv"]
        return KVPages(k.view(E4M3), v.view(E4M3), *scales)
    k = torch.full((n, H, page, K), 0.0 if fill is None else fill, dtype=dtype, device=device)
    return KVPages(k, torch.full((n, H, K, page), 0.0 if fill is None else fill, dtype=dtype, device=device))


def rows_of(plan, page, device, n_pages=None, seed=0, width=None, max_new=None):
    """BatchRows of (new, length) pairs over pages in no order, and the number of pages."""
    used = [-(-length // page) for _, length in plan]
    total = sum(used) + 1 if n_pages is None else n_pages
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, max(used)) if width is None else width
    table = [[order.pop() for _ in range(n)] + [-7] * (width - n) for n in used]  # past the length: never looked at
    start = torch.tensor([0] + [new for new, _ in plan]).cumsum(0)
    as_int = lambda x: torch.as_tensor(x, dtype=torch.int32).to(device)
    return BatchRows(as_int(table), as_int(start), as_int([length for _, length in plan]), max_new=max_new), total


def held(x, dtype):
    """What a cache of `dtype` holds of the rows x (..., K), in 64 bits."""
    if dtype != E4M3:
        return x.to(dtype).double()
    x = x.double()
    half, e = torch.frexp(x.abs().amax(-1) / 448.0)
    e = torch.where(half == 0, 0, (e - (half == 0.5).int()).clamp(min=-110))
    scale = ((e.long() + 1023) << 52).view(torch.float64)[..., None]
    y = x / scale
    step = (((torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4).long() + 1023) << 52).view(torch.float64)
    return torch.round(y / step) * step * scale


def attention(q, k, v, scale):
    """q (n, H, K) the last n of the L positions of k, v (L, Hk, K), 64 bits: o, and sum_j p_j |v_j| beside it."""
    n, H, K = q.shape
    L, Hk, _ = k.shape
    k, v = (x.repeat_interleave(H // Hk, dim=1).permute(1, 0, 2).contiguous() for x in (k, v))
    z = q.double().permute(1, 0, 2) @ k.transpose(1, 2).contiguous() * scale  # (H, n, L)
    seen = torch.arange(L, device=q.device) <= torch.arange(L - n, L, device=q.device)[:, None]
    z = z.masked_fill(~seen, -math.inf)
    some = seen.any(-1)[None, :, None]
    p = torch.where(some, torch.softmax(torch.where(some, z, 0.0), -1), 0.0)
    weight = lambda w: torch.stack([(p[:, j][:, :, None] * torch.where(seen[j][None, :, None], w, 0.0)).sum(1)
                                    for j in range(n)])
    if n > 64 and bool(torch.isfinite(v).all()):
        return (p @ v).permute(1, 0, 2), (p @ v.abs()).permute(1, 0, 2)
    return weight(v), weight(v.abs())


def attention_bound(q, k, o, weight, scale):
    """How far the kernels' o may be off.  With bf16 rows: o is rounded once (half a step, 2^-8 of it) and so is each
    probability for its product (2^-8 of sum p |v|).  A score is a sum of K products in fp32 of which each addition rounds
    by 2^-24 of at most sum |q k|, then a product and the exponential (2 more); an error E of the scores is a relative
    error of 2 E of o's terms (numerator and sum).  The sums over L keys, the joins of the pieces and the division
    round L + 16 times by 2^-24.  fp32 rows: the same without the two roundings to bf16, and 2^-24 of o."""
    K, L = q.shape[-1], k.shape[0]
    half = torch.finfo(q.dtype).eps / 2
    products = float((q.abs().double().amax() * k.abs().amax()) * K * scale)
    largest = min(products, float(q.double().norm(dim=-1).max() * k.norm(dim=-1).max() * scale) * math.sqrt(K))
    e = (K + 4) * 2.0 ** -24 * largest
    return half * o.abs() + (2 * e + (L + 16) * 2.0 ** -24 + (half if q.dtype == torch.bfloat16 else 0.0)) * weight
