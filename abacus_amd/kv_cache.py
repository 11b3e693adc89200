"""The paged key/value cache of a decoding program, and attention over it.

The reference's decoder (abacus/transformer_moe.py) runs whole sequences and keeps nothing; a program that
produces tokens from it runs the whole prefix again for each.  Here the keys and values of a layer stay in pages:

  KVPages       one layer's pages: ``write`` (the keys and values of new tokens), ``read`` (back, one row per
                token) and ``attend`` (attention of new tokens over them)
  BatchRows     which rows of a call belong to which sequence, and where that sequence's pages are
  PagedKVCache  the layers' KVPages together with the pages' bookkeeping on the host

``TransformerMoe.forward_cached`` calls them layer by layer, ``abacus_amd.generate`` token by token.

On the GPU each call is one HIP launch (``attend``: two where the keys are cut over several work-groups) on
torch's current stream; nothing is copied to the host, nothing is kept between calls and every workspace is the
call's own, so calls can be captured into a graph and run on several streams.  CPU tensors take the same steps in
torch's operations.
"""

from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .moe import _contig

__all__ = ["BatchRows", "KVPages", "PagedKVCache"]

PAGE_SIZES = (16, 32, 64, 128, 256)
E4M3 = torch.float8_e4m3fn
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_HELD = {**_CODES, E4M3: _lib.E4M3}


@functools.lru_cache(maxsize=4096)
def _attention_ws_bytes(*sizes: int) -> int:
    return _lib.query("abacus_paged_attention_ws_bytes", *sizes)


def _index(name: str, t: torch.Tensor, shape: tuple[int, ...], device: torch.device) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device:
        raise ValueError(f"{name} must be int32 on {device}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if not t.is_contiguous():  # (a copy would not follow what the caller writes there later)
        raise ValueError(f"{name} must be contiguous")
    return t


def _no_gradient(name: str, *tensors: torch.Tensor) -> None:
    """Refuses tensors whose derivative a call would drop: backward's where it is recorded, forward mode's always."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} requires a gradient, and a cache gives none: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has a forward-mode tangent, and a cache carries none")


class BatchRows:
    """The T rows of a call, new tokens of S sequences one after the other.

    page_table_SP: (S, P) int32, page of positions 0 .. page_size - 1 of each sequence, and so on (entries past
    its length are not read).  query_start: (S + 1,) int32, sequence s has the rows query_start[s] ..
    query_start[s + 1] - 1, none among them (from the first range that runs backwards or past the rows on, sequences
    are taken to have none).  lengths: (S,) int32, its tokens in all, the new ones included: its
    last row is position lengths[s] - 1.  max_new: the most rows of one sequence, where the caller knows; it
    chooses the kernels and bounds nothing.

    The three are read on the device when a call runs, so a captured graph follows what they hold at each replay.
    """

    __slots__ = ("page_table_SP", "query_start", "lengths", "max_new", "device", "_sizes")

    def __init__(self, page_table_SP: torch.Tensor, query_start: torch.Tensor, lengths: torch.Tensor,
                 max_new: int | None = None):
        shape = page_table_SP.shape
        if len(shape) != 2 or 0 in shape:
            raise ValueError(f"page_table must be (sequences, pages), got {tuple(shape)}")
        if max_new is not None and max_new < 1:
            raise ValueError(f"max_new must be at least 1, got {max_new}")
        S, P = shape
        device = page_table_SP.device
        self.page_table_SP = _index("page_table", page_table_SP, (S, P), device)
        self.query_start = _index("query_start", query_start, (S + 1,), device)
        self.lengths = _index("lengths", lengths, (S,), device)
        self.max_new, self.device, self._sizes = max_new, device, (S, P)

    def positions(self, n_rows: int) -> torch.Tensor:
        """(n_rows,) int64: each row's position in its sequence (0 for rows of none and rows before position 0)."""
        start, S = self.query_start, self._sizes[0]
        pos = torch.empty(n_rows, dtype=torch.int64, device=self.device)
        if pos.is_cuda:
            _call(self.device, "abacus_batch_positions", start.data_ptr(), self.lengths.data_ptr(), S, n_rows, pos.data_ptr())
            return pos
        pos.zero_()
        good = int(((start[:-1] >= 0) & (start[1:] >= start[:-1]) & (start[1:] <= n_rows)).cumprod(0).sum())
        if good:
            first, ends = int(start[0]), start[1:good + 1].long()
            seq = torch.repeat_interleave(torch.arange(good), ends - start[:good])
            row = first + torch.arange(len(seq))
            pos[first:first + len(seq)] = (self.lengths[seq].long() - ends[seq] + row).clamp(min=0)
        return pos


def _call(device: torch.device, name: str, *args) -> None:
    """_lib.call on torch's current stream of `device`, which is made current where it is not (a launch takes place on
    the current one)."""
    if device.index == torch._C._cuda_getDevice():
        _lib.call(name, *args, _lib.stream_of(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _lib.stream_of(device))


class KVPages:
    """The pages of one layer: keys (pages, heads, page_size, head_dim), values (pages, heads, head_dim, page_size).

    The values lie with their slots together because attention reads them so: a page is turned once, as it is
    written.  bf16 and fp32 pages hold keys and values as they are.  float8_e4m3fn pages hold codes, with one
    exponent byte per token and head in k_scale and v_scale (pages, heads, page_size): the value is
    code * 2^(byte - 127), the byte the least that keeps the row's largest magnitude within 448.  Where a key or a
    value of a token's head holds an infinity or NaN, e4m3 pages give NaN for both.

    page_size is a power of two from 16 to 256, head_dim a multiple of 16 up to 128.  The tensors stay where they are:
    once one has been given other memory (``.data``, ``resize_``), calls are refused.
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "n_pages", "n_heads", "page_size", "head_dim", "dtype", "device",
                 "_args")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dim() != 4:
            raise ValueError("pages must be (pages, heads, page_size, head_dim) and (pages, heads, head_dim, page_size)")
        n, H, page, K = k.shape
        dtype, device = k.dtype, k.device
        if page not in PAGE_SIZES or K % 16 or not 16 <= K <= 128 or n < 1 or not 1 <= H <= 1024:
            raise ValueError(f"{n} pages of {H} heads, {page} slots and head_dim {K}: page_size is one of {PAGE_SIZES}, "
                             "head_dim a multiple of 16 up to 128")
        if dtype not in _HELD:
            raise TypeError(f"a cache holds float32, bfloat16 or float8_e4m3fn, got {dtype}")
        if v.shape != (n, H, K, page) or v.dtype != dtype:
            raise ValueError(f"value pages must be {dtype} of {(n, H, K, page)} beside key pages {tuple(k.shape)}, got "
                             f"{v.dtype} of {tuple(v.shape)}")
        tensors = (k, v)
        if dtype == E4M3:
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.uint8 or s.shape != (n, H, page):
                    raise ValueError(f"float8_e4m3fn pages need uint8 k_scale and v_scale of {(n, H, page)}")
            tensors = (k, v, k_scale, v_scale)
        elif k_scale is not None or v_scale is not None:
            raise ValueError(f"{dtype} pages have no scales")
        at = [t.data_ptr() for t in tensors]
        for t, p in zip(tensors, at):
            if t.device != device:
                raise ValueError("a layer's pages must be on one device")
            if p % 16 or not t.is_contiguous():
                raise ValueError("pages must be contiguous and 16-byte aligned")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_heads, self.page_size, self.head_dim = n, H, page, K
        self.dtype, self.device = dtype, device
        self._args = (page, n, _HELD[dtype], *at, *(None,) * (4 - len(at)))

    def _check(self, name: str, x: torch.Tensor, rows: BatchRows, heads: int | None) -> torch.Size:
        shape, dtype = x.shape, x.dtype
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            want = "heads" if heads is None else heads
            raise ValueError(f"{name} must be (rows, {want}, {self.head_dim}), got {tuple(shape)}")
        if dtype not in _CODES or (self.dtype != dtype and self.dtype != E4M3):
            raise TypeError(f"{name} of {dtype} over a cache of {self.dtype}: the cache holds the rows' dtype "
                            "(float32 or bfloat16) or float8_e4m3fn")
        if x.device != self.device or rows.device != self.device:
            raise ValueError(f"{name}, the rows and the pages must be on one device")
        self._usable(name, x)
        return shape

    def _usable(self, name: str, x: torch.Tensor) -> None:
        """The pages lie where they were checked, and neither they nor x have a derivative to carry."""
        k, v = self.k, self.v
        _, _, _, k_at, v_at, k_scale_at, v_scale_at = self._args
        if k.data_ptr() != k_at or v.data_ptr() != v_at or k_scale_at is not None and (
                self.k_scale.data_ptr() != k_scale_at or self.v_scale.data_ptr() != v_scale_at):
            raise RuntimeError("the pages are no longer where they were: make KVPages of them anew")
        if x.requires_grad or k.requires_grad or v.requires_grad or forward_ad._current_level >= 0:
            _no_gradient(name, x)
            _no_gradient("the cache", k, v)

    def _rows_args(self, rows: BatchRows) -> tuple:
        return (rows.page_table_SP.data_ptr(), rows.query_start.data_ptr(), rows.lengths.data_ptr(), *rows._sizes,
                *self._args)

    def write(self, k_THK: torch.Tensor, v_THK: torch.Tensor, rows: BatchRows) -> None:
        """Keys and values (T, heads, head_dim) of the rows into their slots.

        Rows of no sequence, of a sequence longer than its table, or whose page is not in the pool are not
        written.  Two rows of a call with the same slot leave one or the other (of e4m3 pages possibly codes of
        one and exponents of the other): sequences may share pages that they only read."""
        T, H, K = self._check("k", k_THK, rows, self.n_heads)
        if v_THK.shape != k_THK.shape or v_THK.dtype != k_THK.dtype or v_THK.device != self.device:
            raise ValueError("k and v must have one shape, dtype and device")
        if v_THK.requires_grad or forward_ad._current_level >= 0:
            _no_gradient("v", v_THK)
        if not k_THK.is_cuda:
            return self._write_cpu(k_THK, v_THK, rows)
        k_THK, v_THK = _contig(k_THK), _contig(v_THK)
        _call(self.device, "abacus_kv_write", k_THK.data_ptr(), v_THK.data_ptr(), T, H, K, _CODES[k_THK.dtype],
              *self._rows_args(rows))

    def read(self, rows: BatchRows, length: int, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values (S, length, heads, head_dim): position l of sequence s in row (s, l), 0 past its length.

        dtype: the pages' own, or for e4m3 pages bfloat16 (which holds every value of theirs exactly; the
        default) or float32."""
        if dtype is None:
            dtype = torch.bfloat16 if self.dtype == E4M3 else self.dtype
        if dtype not in _CODES or (self.dtype != dtype and self.dtype != E4M3):
            raise TypeError(f"a cache of {self.dtype} is not read as {dtype}")
        if rows.device != self.device:
            raise ValueError("the rows and the pages must be on one device")
        if length < 0:
            raise ValueError(f"length must not be negative, got {length}")
        self._usable("the cache", self.k)
        S, P = rows._sizes
        shape = (S, length, self.n_heads, self.head_dim)
        if not self.k.is_cuda:
            return self._read_cpu(rows, shape, dtype)
        k, v = torch.empty((2, *shape), dtype=dtype, device=self.device).unbind()
        _call(self.device, "abacus_kv_read", rows.page_table_SP.data_ptr(), rows.lengths.data_ptr(), S, P, *self._args[:2],
              self.n_heads, self.head_dim, *self._args[2:], length, _CODES[dtype], k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, q_THK: torch.Tensor, rows: BatchRows, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale q k^T) v of each row over the cached positions up to its own, which have to be written.

        q_THK: (T, G * heads, head_dim); query head h reads key head h // G.  scale: 1 / sqrt(head_dim) unless
        given, positive.  A row that sees no position gives 0, one whose sequence is longer than its table or has
        a page outside the pool NaN.  Rows of no sequence give 0, or with ``out`` (T, G * heads, head_dim) are
        left as they are there.

        Statistics and sums are fp32, and a sum is divided once it is whole, with weights of up to 2^8: it is finite as
        long as the largest |v| times 2^8 times the positions seen is below 2^128 (|v| to 2^100 at 2^20 positions), and
        the products q . k, which are scaled after they are formed, are below 2^128 too.  With bf16 queries the probabilities are rounded to bf16 for the product
        with the values, as the training kernels do.  No gradient is formed: rows, pages or an ``out`` that ask for one
        are refused, and so are forward-mode tangents."""
        T, H, K = self._check("q", q_THK, rows, None)
        if H % self.n_heads or H < 1 or H > 1024:
            raise ValueError(f"{H} query heads over {self.n_heads} key heads: they must be a multiple (at most 1024)")
        scale = 1.0 / math.sqrt(K) if scale is None else float(scale)
        if not 0.0 < scale < math.inf:
            raise ValueError(f"scale must be positive, got {scale}")
        if out is not None:
            if out.shape != q_THK.shape or out.dtype != q_THK.dtype or out.device != self.device:
                raise ValueError("out must have q's shape, dtype and device")
            if not out.is_contiguous() or out.data_ptr() % 16:
                raise ValueError("out must be contiguous and 16-byte aligned")
            _no_gradient("out", out)
        if not q_THK.is_cuda:
            return self._attend_cpu(q_THK, rows, scale, out)
        q, code = _contig(q_THK), _CODES[q_THK.dtype]
        zero_rest = int(out is None)
        if out is None:
            out = torch.empty_like(q)
        most = max(1, T) if rows.max_new is None else rows.max_new
        nbytes = _attention_ws_bytes(T, H, self.n_heads, K, code, self._args[2], *rows._sizes, self.page_size, most)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        _call(self.device, "abacus_paged_attention", q.data_ptr(), T, H, self.n_heads, K, code, *self._rows_args(rows), scale,
              most, zero_rest, out.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
        return out

    # ------------------------------------------------------------ CPU tensors

    def _sequences(self, rows: BatchRows, n_rows: int):
        """Of each sequence: its number, first row, rows, length, and (page, slot) of its positions; page None
        where the table does not hold the sequence or its pages are not in the pool."""
        P = rows._sizes[1]
        start, lengths = rows.query_start.tolist(), rows.lengths.tolist()
        ended = False
        for s, length in enumerate(lengths):
            first, n = start[s], start[s + 1] - start[s]
            ended = ended or first < 0 or n < 0 or start[s + 1] > n_rows
            if ended:
                first, n = 0, 0
            at = torch.arange(min(max(length, 0), P * self.page_size))
            page = rows.page_table_SP[s].long()[at // self.page_size]
            there = (page >= 0) & (page < self.n_pages) & (length <= P * self.page_size)
            yield s, first, n, max(length, 0), torch.where(there, page, 0), at % self.page_size, there

    def _quantise(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        mantissa, exponent = torch.frexp(x.float().abs().amax(-1))  # mantissa in [0.5, 1)
        e = torch.where(mantissa == 0, 0, (exponent - torch.where(mantissa <= 0.875, 9, 8)).clamp(min=-110))
        return (x.float() * _power(-e)[..., None]).to(E4M3), (e + 127).to(torch.uint8)

    @torch.no_grad()
    def _write_cpu(self, k, v, rows):
        for _, first, n, length, page, slot, there in self._sequences(rows, k.shape[0]):
            new = min(n, length)
            at = slice(length - new, length)
            if new == 0 or length > there.numel():
                continue
            keep = there[at]
            page, slot = page[at][keep], slot[at][keep]
            kn, vn = (x[first + n - new:first + n][keep] for x in (k, v))
            if self.dtype == E4M3:
                fine = (torch.isfinite(kn) & torch.isfinite(vn)).all(-1)
                (kc, ks), (vc, vs) = (self._quantise(torch.where(fine[..., None], x, 0)) for x in (kn, vn))
                kc = torch.where(fine[..., None], kc.view(torch.uint8), 0x7f)
                self.k.view(torch.uint8)[page, :, slot] = kc
                self.v.view(torch.uint8)[page, :, :, slot] = vc.view(torch.uint8)
                self.k_scale[page, :, slot], self.v_scale[page, :, slot] = ks, vs
            else:
                self.k[page, :, slot] = kn
                self.v[page, :, :, slot] = vn

    def _values(self, page, slot, there, dtype=torch.float32):
        """Keys and values (positions, heads, head_dim); NaN where a position is in no page."""
        if self.dtype == E4M3:
            k = self.k.view(torch.uint8)[page, :, slot].view(E4M3).to(dtype) * _power(
                self.k_scale[page, :, slot].int() - 127)[..., None]
            v = self.v.view(torch.uint8)[page, :, :, slot].view(E4M3).to(dtype) * _power(
                self.v_scale[page, :, slot].int() - 127)[..., None]
            v = torch.where(torch.isnan(k[..., :1]), math.nan, v)
        else:
            k, v = self.k[page, :, slot].to(dtype), self.v[page, :, :, slot].to(dtype)
        there = there[:, None, None]
        return torch.where(there, k, math.nan), torch.where(there, v, math.nan)

    @torch.no_grad()
    def _read_cpu(self, rows, shape, dtype):
        k, v = torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)
        for s, _, _, _, page, slot, there in self._sequences(rows, 0):
            n = min(shape[1], page.numel())
            kn, vn = self._values(page[:n], slot[:n], there[:n])
            k[s, :n], v[s, :n] = kn.to(dtype), vn.to(dtype)
        return k, v

    @torch.no_grad()
    def _attend_cpu(self, q, rows, scale, out):
        if out is None:
            out = torch.zeros(q.shape, dtype=q.dtype)
        G = q.shape[1] // self.n_heads
        for _, first, n, length, page, slot, there in self._sequences(rows, q.shape[0]):
            if length > page.numel():
                out[first:first + n] = math.nan
                continue
            k, v = (x.repeat_interleave(G, dim=1) for x in self._values(page, slot, there))
            for j in range(n):
                seen = max(0, length - n + j + 1)
                if seen == 0:
                    out[first + j] = 0
                    continue
                z = (q[first + j].float() * k[:seen]).sum(-1) * scale  # (seen, heads)
                p = torch.softmax(z, dim=0)
                out[first + j] = (p[..., None] * v[:seen]).sum(0).to(q.dtype)
        return out


def _power(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for -127 < e < 128."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


class PagedKVCache:
    """A pool of pages per layer, and which of its sequences has which pages.

    ``layer(i)`` are layer i's KVPages; page numbers mean the same in every layer.  ``add()`` opens a sequence,
    ``extend({sequence: new tokens})`` gives their pages and the call's BatchRows, ``truncate`` takes tokens
    back (drafts that were not accepted), ``free`` closes a sequence.  Pages go to other sequences as they are:
    slots past a sequence's length are never looked at.
    """

    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None):
        if n_layers < 1:
            raise ValueError(f"n_layers must be at least 1, got {n_layers}")
        self.page_size, self.n_pages, self.dtype = page_size, n_pages, dtype
        code = torch.uint8 if dtype == E4M3 else dtype

        def pool(*shape, dtype=code, fill=0):
            return torch.full((n_layers, n_pages, n_heads, *shape), fill, dtype=dtype, device=device)

        k, v = pool(page_size, head_dim), pool(head_dim, page_size)
        if dtype == E4M3:
            scales = [pool(page_size, dtype=torch.uint8, fill=127) for _ in range(2)]
            k, v = k.view(E4M3), v.view(E4M3)
        else:
            scales = [[None] * n_layers] * 2
        self._layers = [KVPages(k[i], v[i], scales[0][i], scales[1][i]) for i in range(n_layers)]
        self.device = k.device
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    def layer(self, i: int) -> KVPages:
        return self._layers[i]

    @property
    def n_layers(self) -> int:
        return len(self._layers)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._lengths[seq]

    def add(self) -> int:
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lengths[seq] = [], 0
        return seq

    def free(self, seq: int) -> None:
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._lengths[seq]

    def truncate(self, seq: int, length: int) -> None:
        """The sequence's first `length` tokens stay."""
        if not 0 <= length <= self._lengths[seq]:
            raise ValueError(f"sequence {seq} has {self._lengths[seq]} tokens, not {length}")
        keep = -(-length // self.page_size)
        pages = self._pages[seq]
        self._free.extend(reversed(pages[keep:]))
        del pages[keep:]
        self._lengths[seq] = length

    def extend(self, new: dict[int, int]) -> BatchRows:
        """Room for new[s] more tokens of each sequence s, whose rows follow each other in the dict's order."""
        if not new:
            raise ValueError("no sequences")
        want = {}
        for s, n in new.items():
            if n < 0:
                raise ValueError(f"sequence {s}: {n} new tokens")
            want[s] = max(0, -(-(self._lengths[s] + n) // self.page_size) - len(self._pages[s]))
        if sum(want.values()) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages of {self.n_pages}, need {sum(want.values())}")
        for s, n in new.items():
            self._pages[s].extend(self._free.pop() for _ in range(want[s]))
            self._lengths[s] += n
        return self.rows(new)

    def rows(self, new: dict[int, int]) -> BatchRows:
        """The BatchRows of sequences whose last new[s] tokens are the call's."""
        width = max(1, max(len(self._pages[s]) for s in new))
        table = [page for s in new for page in self._pages[s] + [0] * (width - len(self._pages[s]))]
        lengths = [self._lengths[s] for s in new]
        start = [0]
        for n in new.values():
            start.append(start[-1] + n)
        S = len(lengths)
        every = torch.tensor(table + start + lengths, dtype=torch.int32).to(self.device)  # one copy
        return BatchRows(every[:S * width].view(S, width), every[S * width:S * width + S + 1], every[S * width + S + 1:],
                         max_new=max(1, max(new.values())))
