"""Paged cache of keys and values in 16 or 8 bits: writing, reading back, and attention of the newest tokens over it.

Kernels: ``csrc/kernels/kv_cache.cu``, ``csrc/kernels/cache_attention.cu`` (up to 16 query rows to a head of the cache) and
``csrc/kernels/cache_attention_sm100.cu`` (more); CPU tensors, and types or head sizes that the kernels do not take, run the same
formulas in PyTorch. The reference has no cache: its generation loop runs the whole context through the model
for every token (``crates/torsh-text/src/generation.rs``).

Layout: ``k_pages`` and ``v_pages`` are ``[num_pages, H, page, D]`` (a page holds ``page`` consecutive tokens of one sequence, a
multiple of 16 for the kernels), ``page_table`` ``[B, pages]`` int32 names the pages of each sequence in order. 8-bit pages have one
fp32 scale per row (one token of one head), ``[num_pages, H, page]``:

* ``int8``: ``scale = max|x| / 127``, codes to the nearest, halves to even
* ``float8_e4m3fn``: ``scale`` is the least power of two with ``max|x| / scale <= 448``

Rows whose largest magnitude is below 2^-100 are held as zeros; a row that has an infinity or a NaN gets the scale NaN.
"""
from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as fwd

from .. import _native as nv

_TINY = 2.0 ** -100
_CODES = (torch.int8, torch.float8_e4m3fn)


# ------------------------------------------------------------------------------------------------ checks
def _check_pages(what, k_pages, v_pages, k_scales, v_scales, page_table, B, device):
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        raise ValueError(f"{what}: k_pages and v_pages are [num_pages, H, page, D] of one shape and type")
    dt = k_pages.dtype
    if dt in _CODES:
        for s in (k_scales, v_scales):
            if s is None or s.shape != k_pages.shape[:3] or s.dtype != torch.float32 or not s.is_contiguous():
                raise ValueError(f"{what}: pages of {dt} need contiguous fp32 scales {tuple(k_pages.shape[:3])}")
    elif not dt.is_floating_point or dt.itemsize == 1:
        raise TypeError(f"{what}: pages of bf16, int8 or float8_e4m3fn (or another 16- to 64-bit floating type on the plain path), got {dt}")
    elif k_scales is not None or v_scales is not None:
        raise ValueError(f"{what}: pages of {dt} have no scales")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError(f"{what}: pages have to be contiguous")
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: page_table is [{B}, pages], int32")
    for t in (k_pages, v_pages, k_scales, v_scales, page_table):
        if t is not None and t.device != device:
            raise ValueError(f"{what}: all tensors are on one device")


def _per_sequence(what, name, t, B, device):
    """A vector of B integers as the kernels read it."""
    if t.shape != (B,) or t.is_floating_point() or t.device != device:
        raise ValueError(f"{what}: {name} is a vector of {B} integers on {device}")
    return _int32(t).contiguous()


def _int32(t):
    """As 32-bit integers; what does not fit becomes the next that does, which no table reaches and no pool has."""
    return t.clamp(-0x80000000, 0x7FFFFFFF).to(torch.int32) if t.dtype == torch.int64 else t.to(torch.int32)


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under no_grad()")


def _no_tangent(what, *tensors):
    if any(fwd.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: what is read back would not carry it")


def _table(page_table):
    return page_table if page_table.dtype is torch.int32 and page_table.stride(1) == 1 else _int32(page_table).contiguous()


def _rows(x):
    """Rows that start on 16 bytes, less than 2^31 elements apart; copied where they are not so."""
    n = 16 // x.element_size()
    return x if max(x.stride()[1:]) < 1 << 31 and x.stride(3) == 1 and not x.data_ptr() % 16 and not any(s % n for s in x.stride()[:3]) else x.clone(memory_format=torch.contiguous_format)


# ------------------------------------------------------------------------------------------------ the formulas in PyTorch
def quantize_rows(x: torch.Tensor, dtype: torch.dtype):
    """``(codes, scales)`` of rows ``[..., D]`` as :func:`kv_cache_write` stores them (scales None where ``dtype`` has none)."""
    if dtype not in _CODES:
        return x.to(dtype), None
    big = x.float().abs().amax(-1)
    if dtype == torch.int8:
        scale = big / torch.full_like(big, 127)     # by a tensor: by a number, a GPU multiplies with the rounded 1 / 127
    else:
        m, e = torch.frexp(big)
        scale = ((e.long() - 9 + (m > 0.875) + 1023) << 52).view(torch.float64).float()   # from the bits: exact on every device
    wild, none = ~torch.isfinite(big), big < _TINY
    scale = torch.where(wild, math.nan, torch.where(none, 0.0, scale))
    live = ~(wild | none)[..., None]
    # 64 bits: a quotient next to a half must not be rounded onto it
    r = torch.where(live, x.double() / torch.where(live, scale[..., None], 1.0).double(), 0.0)
    return (r.round().to(torch.int8) if dtype == torch.int8 else r.float().to(dtype)), scale


def _bits(pages):
    """Pages as a type that every indexing operation takes."""
    return pages.view(torch.int8) if pages.dtype == torch.float8_e4m3fn else pages


def _slots(page_table, num_pages, page, positions):
    """``(pages, rows, there)`` of positions ``[B, n]``: positions that the table does not name, or that it gives a page outside the pool, are not there."""
    width = page_table.shape[1] * page
    there = (positions >= 0) & (positions < width)
    if width == 0:
        return torch.zeros_like(positions), torch.zeros_like(positions), there
    at = positions.clamp(0, width - 1)
    pages = page_table.long().gather(1, at // page)
    there = there & (pages >= 0) & (pages < num_pages)
    return torch.where(there, pages, 0), at % page, there


def _gather(pages, scales, slot, row, there, dtype):
    """Rows ``[B, n, H, D]`` in ``dtype``, zeros where there is none."""
    if pages.shape[0] == 0:
        return torch.zeros(*slot.shape, *pages.shape[1::2], dtype=dtype, device=pages.device)
    x = _bits(pages)[slot, :, row].view(pages.dtype).to(dtype)
    if scales is not None:
        x = x * scales[slot, :, row][..., None].to(dtype)
    return torch.where(there[..., None, None], x, 0)


# ------------------------------------------------------------------------------------------------ write and read
def kv_cache_write(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                   start: torch.Tensor, counts: torch.Tensor | None = None, k_scales: torch.Tensor | None = None,
                   v_scales: torch.Tensor | None = None) -> None:
    """Writes the keys and values of ``T`` new tokens per sequence into their pages, quantised to the pages' type.

    ``k`` and ``v`` are ``[B, T, H, D]``; token ``t`` of sequence ``b`` goes to position ``start[b] + t``, tokens from ``counts[b]`` on are
    left out, and so are sequences whose ``start`` is negative. Positions that the table does not reach, or to which it gives a page
    outside the pool, are skipped (and reported where the device-side index checks are on, but for pages -1 of a sequence whose first page is -1: a
    place of the batch without a sequence). Two sequences may share pages, but not the positions that one call writes.
    No derivatives, of either mode: such inputs are refused.
    """
    if k.is_cuda and (nv._decode or nv.decode_calls()).kv_write(k, v, k_pages, v_pages, page_table, start, counts, k_scales, v_scales):
        return
    # not as the kernel takes it: refused, converted, or computed here
    if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or not k.is_floating_point():
        raise ValueError("kv_cache_write: k and v are [B, T, H, D] of one floating type")
    B, T, H, D = k.shape
    _check_pages("kv_cache_write", k_pages, v_pages, k_scales, v_scales, page_table, B, k.device)
    if k_pages.shape[1] != H or k_pages.shape[3] != D or v.device != k.device:
        raise ValueError(f"kv_cache_write: pages of {k_pages.shape[1]} heads of {k_pages.shape[3]}, rows of {H} of {D}")
    _no_grad("kv_cache_write", k, v)
    _no_tangent("kv_cache_write", k, v)
    start = _per_sequence("kv_cache_write", "start", start, B, k.device)
    if counts is not None:
        counts = _per_sequence("kv_cache_write", "counts", counts, B, k.device)
    if k.numel() == 0:
        return
    num_pages, _, page, _ = k_pages.shape
    if k.is_cuda:
        with torch.cuda.device(k.device):
            if nv.decode_calls().kv_write(_rows(k), _rows(v), k_pages, v_pages, _table(page_table), start, counts, k_scales, v_scales):
                return
    at = torch.arange(T, device=k.device)
    slot, row, there = _slots(page_table, num_pages, page, start.long()[:, None] + at)
    there = there & (start >= 0)[:, None]
    if counts is not None:
        there = there & (at < counts[:, None])
    slot, row = slot[there], row[there]
    for x, pages, scales in ((k, k_pages, k_scales), (v, v_pages, v_scales)):
        codes, scale = quantize_rows(x[there], pages.dtype)
        bits = _bits(pages)
        bits[slot, :, row] = codes.view(bits.dtype)
        if scales is not None:
            scales[slot, :, row] = scale


def kv_cache_read(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, max_len: int,
                  begin: torch.Tensor | None = None, k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """Reads ``lengths[b]`` tokens of each sequence back, from position ``begin[b]`` (0) on: keys and values ``[B, max_len, H, D]`` in
    ``dtype``. Rows from ``lengths[b]`` on, and rows that no page of the pool holds, are zeros."""
    fast = k_pages.is_cuda and dtype in (torch.bfloat16, torch.float32)
    if fast:
        out = (nv._decode or nv.decode_calls()).kv_read(k_pages, v_pages, page_table, lengths, max_len, begin, k_scales, v_scales, dtype is torch.float32)
        if out is not None:
            return out
    # not as the kernel takes it: refused, converted, or computed here
    B = page_table.shape[0] if page_table.dim() == 2 else -1
    dev = k_pages.device
    _check_pages("kv_cache_read", k_pages, v_pages, k_scales, v_scales, page_table, B, dev)
    if max_len < 0:
        raise ValueError("kv_cache_read: max_len is not negative")
    if not dtype.is_floating_point or dtype.itemsize < 2:
        raise TypeError(f"kv_cache_read: rows are read in a floating type of 16 bits or more, got {dtype}")
    num_pages, H, page, D = k_pages.shape
    lengths = _per_sequence("kv_cache_read", "lengths", lengths, B, dev)
    if begin is not None:
        begin = _per_sequence("kv_cache_read", "begin", begin, B, dev)
    if fast:
        with torch.cuda.device(dev):
            out = nv.decode_calls().kv_read(k_pages, v_pages, _table(page_table), lengths, int(max_len), begin, k_scales, v_scales, dtype is torch.float32)
        if out is not None:
            return out
    at = torch.arange(max_len, device=dev)[None].expand(B, -1)
    slot, row, there = _slots(page_table, num_pages, page, at if begin is None else at + begin.long()[:, None])
    there = there & (at < lengths[:, None])
    if begin is not None:
        there = there & (begin >= 0)[:, None]
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    return tuple(_gather(p, s, slot, row, there, wide).to(dtype) for p, s in ((k_pages, k_scales), (v_pages, v_scales)))


# ------------------------------------------------------------------------------------------------ attention
def _attention_plain(q, k_pages, v_pages, page_table, start, tree_mask, counts, k_scales, v_scales, scale, limit):
    """fp32 (fp64 for fp64) maths; the CPU path and the test oracle. What a row does not see is never multiplied: an infinity there stays there."""
    B, T, Hq, D = q.shape
    num_pages, H, page, _ = k_pages.shape
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    dev = q.device
    start = start.long().clamp(min=0)
    live = torch.full((B,), T, device=dev) if counts is None else counts.long().clamp(0, T)
    n = min(limit, page_table.shape[1] * page)
    if n and B:
        n = min(n, int((start + live).max()))
    at = torch.arange(n, device=dev)
    slot, row, there = _slots(page_table, num_pages, page, at[None].expand(B, -1))
    k, v = (_gather(p, s, slot, row, there, wide).permute(0, 2, 1, 3) for p, s in ((k_pages, k_scales), (v_pages, v_scales)))   # [B, H, n, D]
    new = at[None] - start[:, None]                                       # [B, n]: which of the new tokens
    j = new.clamp(0, max(T - 1, 0))
    t = torch.arange(T, device=dev)
    if tree_mask is None:
        among = j[:, None] <= t[:, None]
    else:
        m = tree_mask if tree_mask.dim() == 3 else tree_mask[None].expand(B, -1, -1)
        among = m.gather(2, j[:, None].expand(-1, T, -1))
    seen = ((new < 0)[:, None] | ((new < live[:, None])[:, None] & among)) & (t < live[:, None])[..., None]   # [B, T, n]
    qf = q.to(wide).view(B, T, H, Hq // H, D).permute(0, 2, 3, 1, 4)     # [B, H, G, T, D]
    # a key that no row may see must not reach the product, one that some rows see only theirs: -inf in its place either way
    s = torch.matmul(qf, k[:, :, None].transpose(-1, -2)) * scale
    s = torch.where(seen[:, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True) if n else s.new_zeros(s.shape[:-1] + (1,))
    p = torch.exp(s - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    finite = torch.isfinite(v)
    o = torch.matmul(p, torch.where(finite, v, 0)[:, :, None])
    if not bool(finite.all()):
        for b, h, i in (~finite).any(-1).nonzero().tolist():             # rows of V with something odd, one by one
            odd = torch.where(finite[b, h, i], 0, v[b, h, i])
            w = p[b, h, :, :, i, None]
            o[b, h] += torch.where(w != 0, w * odd, 0)
    o = o / torch.where(total == 0, 1, total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(q.dtype)


def kv_cache_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor,
                       tree_mask: torch.Tensor | None = None, counts: torch.Tensor | None = None, k_scales: torch.Tensor | None = None,
                       v_scales: torch.Tensor | None = None, scale: float | None = None, max_len: int | None = None) -> torch.Tensor:
    """Attention of the newest tokens over the cache: ``q [B, T, Hq, D]`` -> ``[B, T, Hq, D]``, ``Hq`` a multiple of the cache's heads.

    Sequence ``b`` has ``start[b]`` tokens of context, and its ``T`` (``counts[b]``) new tokens, whose keys and values are in the cache
    already, follow at positions ``start[b] ..``. A new token sees all of the context, and the new tokens ``j`` with
    ``tree_mask[t, j]`` (bool, ``[T, T]`` or ``[B, T, T]``; :func:`tree_mask_of`) - without a mask those up to itself. ``T = 1`` is an
    ordinary decoding step. Rows from ``counts[b]`` on, and rows that see nothing, come out as zeros; infinities and NaN in
    places that a row does not see do not reach it (a value scale that is no finite number leaves none among its token's values). ``scale`` is ``1 / sqrt(D)`` unless given; positions from ``max_len`` on, if given, are
    not read. Pages outside the pool read as zeros. No backward pass; forward-mode derivatives are computed in PyTorch.

    Probabilities are rounded to bf16 over bf16 pages. Over 8-bit pages queries are multiplied as halves relative to a power of two near the
    row's largest column (columns below 2^-16 of it lose bits, below 2^-25 they count as zero), and probabilities are rounded to halves, times the scale of their value and relative to
    the largest such product that the row sees: a scale that a row does not see, or hardly attends to, takes nothing from the others. Scales of
    ``v_scales`` from 2^122 on count as infinite, those below 2^-92 as zero.
    """
    if q.is_cuda:
        out = (nv._decode or nv.decode_calls()).kv_attention(q, k_pages, v_pages, page_table, start, tree_mask, counts, k_scales, v_scales, scale, max_len,
                                                             nv.status_ptr(q.device))
        if out is not None:
            return out
    # not as the kernels take it: refused, converted, or computed here
    if q.dim() != 4 or not q.is_floating_point():
        raise ValueError("kv_cache_attention: q is [B, T, Hq, D]")
    B, T, Hq, D = q.shape
    _check_pages("kv_cache_attention", k_pages, v_pages, k_scales, v_scales, page_table, B, q.device)
    num_pages, H, page, Dk = k_pages.shape
    if Dk != D or H == 0 or Hq % H:
        raise ValueError(f"kv_cache_attention: {Hq} query heads of {D} over {H} heads of {Dk}")
    if tree_mask is not None and (tree_mask.shape not in ((T, T), (B, T, T)) or tree_mask.dtype != torch.bool or tree_mask.device != q.device):
        raise ValueError(f"kv_cache_attention: tree_mask is bool [{T}, {T}] or [{B}, {T}, {T}] on {q.device}")
    if max_len is not None and max_len < 0:
        raise ValueError("kv_cache_attention: max_len is not negative")
    _no_grad("kv_cache_attention", q)
    start = _per_sequence("kv_cache_attention", "start", start, B, q.device)
    if counts is not None:
        counts = _per_sequence("kv_cache_attention", "counts", counts, B, q.device)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0 <= scale < math.inf:
        raise ValueError(f"kv_cache_attention: scale is a number that is not negative, got {scale}")
    limit = 0x7FFF0000 if max_len is None else min(int(max_len), 0x7FFF0000)
    if q.is_cuda:
        mask = tree_mask if tree_mask is None or tree_mask.stride(-1) == 1 else tree_mask.contiguous()
        with torch.cuda.device(q.device):
            out = nv.decode_calls().kv_attention(_rows(q), k_pages, v_pages, _table(page_table), start, mask, counts, k_scales, v_scales, scale, limit,
                                                 nv.status_ptr(q.device))
        if out is not None:
            return out
    return _attention_plain(q, k_pages, v_pages, page_table, start, tree_mask, counts, k_scales, v_scales, scale, limit)


def tree_mask_of(parents: torch.Tensor) -> torch.Tensor:
    """Which token of a tree is itself or an ancestor of which: bool ``[..., T, T]`` from ``parents [..., T]`` (``parents[i] < i``; the
    root, and a token that starts a tree of its own, has -1)."""
    if parents.is_floating_point():
        raise TypeError("tree_mask_of: parents are integers")
    T = parents.shape[-1]
    i = torch.arange(T, device=parents.device)
    if bool((parents >= i).any()):
        raise ValueError("tree_mask_of: a parent comes before its children")
    seen = (parents[..., None] == i) | torch.eye(T, dtype=torch.bool, device=parents.device)
    for _ in range(max(T - 1, 1).bit_length()):      # ancestors of ancestors, twice as far each time
        seen = torch.matmul(seen.float(), seen.float()) > 0
    return seen


class PagedKVCache:
    """Pages of one or more layers, the sequences that own them, and the calls on them.

    ``dtype`` is ``torch.bfloat16``, ``torch.int8`` or ``torch.float8_e4m3fn``. Heads of 64 or 128 columns, and queries in bf16, take the
    kernels; other heads and types run in PyTorch, which gathers a context in fp32 and waits for the device, so that such steps cannot be
    captured. Every layer has its own pages; the table and the lengths are common. A step is: :meth:`reserve` room for the new tokens of the batch, for each layer :meth:`write` their keys and values and
    :meth:`attend`, then :meth:`advance` the lengths by what is kept (after a verification fewer than were written: the rest is
    written over). Table and lengths are device tensors that are written in place, so a step with ``advance(tensor, most)`` can be captured
    into a graph and replayed while what has been reserved lasts; after one, :meth:`reserve`, :meth:`read` and :meth:`truncate` ask the device for the
    lengths. Places of the batch that have no sequence have no pages: what a batched
    step writes for them is left out, and what it reads is zeros.
    """

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, batch: int, max_len: int, dtype: torch.dtype = torch.bfloat16,
                 page: int = 64, num_pages: int | None = None, device="cuda"):
        if page <= 0 or page % 16:
            raise ValueError("PagedKVCache: pages hold a multiple of 16 tokens")
        if dtype not in _CODES and not (dtype.is_floating_point and dtype.itemsize > 1):
            raise TypeError(f"PagedKVCache: bfloat16, int8 or float8_e4m3fn, got {dtype}")
        self.page, self.batch, self.dtype = page, batch, dtype
        per = -(-max_len // page)
        self.max_len = max_len
        num_pages = batch * per if num_pages is None else num_pages
        shape = (num_pages, num_heads, page, head_dim)
        mk = lambda: torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) if dtype in _CODES else torch.zeros(shape, dtype=dtype, device=device)   # noqa: E731
        self.layers = [(mk(), mk()) for _ in range(num_layers)]
        sc = lambda: torch.zeros(shape[:3], device=device) if dtype in _CODES else None   # noqa: E731
        self.scales = [(sc(), sc()) for _ in range(num_layers)]
        self.page_table = torch.full((batch, per), -1, dtype=torch.int32, device=device)   # -1: no page
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.host_lengths = [0] * batch           # upper bounds: what advance() has been told on the host
        self._replayed = False                    # an advance() has been captured: only the device knows how often it has run
        self._owned: list[list[int]] = [[] for _ in range(batch)]
        self._free = list(range(num_pages - 1, -1, -1))

    def _per_place(self, tokens) -> list[int]:
        tokens = [tokens] * self.batch if isinstance(tokens, int) else [int(t) for t in tokens]
        if len(tokens) != self.batch:
            raise ValueError(f"PagedKVCache: tokens {tokens} for {self.batch} sequences")
        return tokens

    def _capturing(self) -> bool:
        return self.lengths.is_cuda and torch.cuda.is_current_stream_capturing()

    def _bounds(self, exact: bool = False) -> list[int]:
        """``host_lengths``, brought up to date from the device where asked to, and where replays may have changed them."""
        if (exact or self._replayed) and not self._capturing():
            self.host_lengths = self.lengths.tolist()
        return self.host_lengths

    def _ghosts(self, tokens=None) -> bool:
        """Whether a place has a length on the host without pages of its own: a batched step has counted it (then the device has 0), or its table
        names others' pages. ``tokens``: only places that are to get some."""
        return any(n and not own and (tokens is None or tokens[b]) for b, (n, own) in enumerate(zip(self.host_lengths, self._owned)))

    def reserve(self, tokens) -> None:
        """Room for ``tokens`` (an int, or one per sequence) more tokens of every sequence. Raises where the pool or ``max_len`` has none."""
        tokens = self._per_place(tokens)
        for exact in (self._ghosts(tokens), True):   # upper bounds first: what does not fit them is asked of the device
            # places without pages that get no tokens need none
            ends = [n + t if t or own else 0 for n, t, own in zip(self._bounds(exact), tokens, self._owned)]
            need = [max(0, -(-end // self.page) - len(own)) for end, own in zip(ends, self._owned)]
            longest = max(ends, default=0)
            if longest <= self.max_len and sum(need) <= len(self._free):
                break
        if longest > self.max_len:
            raise ValueError(f"PagedKVCache: {longest} tokens in a sequence, room for {self.max_len}")
        if sum(need) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(need)} pages wanted, {len(self._free)} free")
        for b, n in enumerate(need):
            if n:
                new = [self._free.pop() for _ in range(n)]
                at = len(self._owned[b])
                self._owned[b] += new
                self.page_table[b, at:at + n] = torch.tensor(new, dtype=torch.int32, device=self.page_table.device)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None) -> None:
        """:func:`kv_cache_write` behind each sequence's length."""
        (kp, vp), (ks, vs) = self.layers[layer], self.scales[layer]
        kv_cache_write(k, v, kp, vp, self.page_table, self.lengths, counts, ks, vs)

    def attend(self, layer: int, q: torch.Tensor, tree_mask: torch.Tensor | None = None, counts: torch.Tensor | None = None,
               scale: float | None = None) -> torch.Tensor:
        """:func:`kv_cache_attention` of tokens that :meth:`write` has just written."""
        (kp, vp), (ks, vs) = self.layers[layer], self.scales[layer]
        return kv_cache_attention(q, kp, vp, self.page_table, self.lengths, tree_mask, counts, ks, vs, scale)

    def read(self, layer: int, dtype: torch.dtype = torch.bfloat16):
        """All keys and values of a layer, ``[B, longest, H, D]``."""
        (kp, vp), (ks, vs) = self.layers[layer], self.scales[layer]
        return kv_cache_read(kp, vp, self.page_table, self.lengths, max(self._bounds(self._ghosts()), default=0), None, ks, vs, dtype)

    def keep(self, path: torch.Tensor, accepted: torch.Tensor) -> None:
        """Moves the accepted nodes of a tree (:func:`~torsh_b200.ops.speculative.verify_draft`) to the front of the tokens just written,
        in every layer: node ``path[b, i]`` to place ``i``, for ``i <= accepted[b]``. A chain is in place already."""
        B, T = path.shape
        if B * T == 0 or self.layers[0][0].numel() == 0:
            return
        i = torch.arange(T, device=path.device)
        base = self.lengths.long()[:, None]
        src, srow, ok = _slots(self.page_table, self.layers[0][0].shape[0], self.page, base + path.clamp(min=0))
        dst, drow, there = _slots(self.page_table, self.layers[0][0].shape[0], self.page, base + i)
        ok = ok & there & (i <= accepted[:, None]) & (path >= 0)
        # no sizes that depend on the data: places that stay as they are copy themselves, and those without a page repeat one that has one
        src, srow = torch.where(ok, src, dst), torch.where(ok, srow, drow)
        some = there.flatten().int().argmax()[None]
        src, srow, dst, drow = (torch.where(there, x, x.flatten().gather(0, some)) for x in (src, srow, dst, drow))
        for pages, scales in zip(self.layers, self.scales):
            for x in (*map(_bits, pages), *scales):
                if x is not None:
                    x[dst, :, drow] = x[src, :, srow]

    def advance(self, tokens, most: int | None = None) -> None:
        """The last ``tokens`` that were written belong to their sequences now: an int, one per sequence, or a device vector of at most ``most``.
        Places without a sequence stay empty, whatever they are given."""
        taken = (self.page_table >= 0).any(1)
        if isinstance(tokens, torch.Tensor):
            self.lengths += torch.where(taken, tokens.to(torch.int32), 0)
            if most is None:
                self.host_lengths = self.lengths.tolist()
            else:
                self.host_lengths = [n + most for n in self.host_lengths]
            self._replayed = self._replayed or self._capturing()
            return
        tokens = self._per_place(tokens)
        self.lengths += torch.where(taken, torch.tensor(tokens, dtype=torch.int32, device=self.lengths.device), 0)
        self.host_lengths = [n + t for n, t in zip(self.host_lengths, tokens)]

    def truncate(self, lengths) -> None:
        """Shortens the sequences to ``lengths`` (one per sequence; shorter ones stay as they are): what lies behind is written over. Their pages
        stay theirs."""
        lengths = [int(n) for n in lengths]
        have = self._bounds(self._ghosts())
        if len(lengths) != self.batch or any(not 0 <= n <= was for n, was in zip(lengths, have)):
            raise ValueError(f"PagedKVCache: lengths {lengths} of sequences that have {have}")
        # the host may know upper bounds only: nothing gets longer
        self.lengths.copy_(torch.minimum(self.lengths, torch.tensor(lengths, dtype=torch.int32, device=self.lengths.device)))
        self.host_lengths = lengths

    def release(self, b: int) -> None:
        """Gives sequence ``b``'s pages back; its place takes a new sequence from position 0."""
        self._free += reversed(self._owned[b])
        self._owned[b] = []
        self.page_table[b] = -1
        self.lengths[b] = 0
        self.host_lengths[b] = 0
