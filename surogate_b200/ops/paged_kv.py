"""Paged key/value cache of the answering path and the attention that reads it.

A layer's cache is one tensor of pages, ``[pages, 2, kv heads, page size, head size]`` (index 1: keys, values); a row (sequence) owns a list of
pages, its line of ``page_table``, and its token at position ``t`` lies in page ``page_table[row, t // page_size]`` at place ``t % page_size``.
An 8-bit cache (``float8_e4m3fn``) has one fp32 scale for each token, head and key / value: ``scales [pages, 2, kv heads, page size]``.

* ``kv_append(kv, k, v, page_table, start, count, scales)`` writes the keys and values of new tokens.
* ``kv_copy_pages(kv, src, dst, scales)`` copies pages through all layers (forked and moved sequences).
* ``paged_attention(q, kv, page_table, lengths, ...)`` attends from one new token of each row over its pages.
* ``PagedKVCache`` keeps the pages of all layers and who owns them: ``append``, ``fork``, ``free``, ``compact``.

On a GPU they run the kernels of ``csrc/paged_kv_kernels.cu`` and ``csrc/paged_attention.cu`` on the current stream, without a host
synchronisation; elsewhere the PyTorch forms below, which are also the oracle of the kernel tests.  (Attention on a GPU reads bf16, fp16 and
e4m3 caches with heads of 64, 128 or 256; caches of fp32 and of other head sizes can be written and copied there, and read by the caller.)
A page number, position or length outside the cache found by a kernel leaves that token out and is reported by ``check_device_errors``.
"""
from __future__ import annotations

import math
from typing import Dict, List, Optional, Sequence, Tuple

import torch

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -100
ATTENTION_DIMS = (64, 128, 256)


# ---------------------------------------------------------------------------------------------- PyTorch forms
def quantize_e4m3(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 values, fp32 scale) of ``x [..., head size]``: scale = largest magnitude / 448 (1 for zeros), values = x / scale."""
    xf = x.float()
    amax = xf.abs().nan_to_num(nan=0.0, posinf=math.inf).amax(-1)
    # divided by a tensor: by a number, CUDA's element-wise division multiplies by the reciprocal, which is another fp32 value
    scale = torch.where(amax > 0, (amax / torch.full_like(amax, E4M3_MAX)).clamp_min(MIN_SCALE), torch.ones_like(amax))
    return (xf / scale.unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def kv_append_reference(kv, k, v, page_table, start, count=None, scales=None) -> None:
    B, T = k.shape[:2]
    P, pages = kv.shape[3], kv.shape[0]
    for b in range(B):
        for t in range(T if count is None else min(T, int(count[b]))):
            pos = int(start[b]) + t
            if pos < 0 or pos // P >= page_table.shape[1] or not 0 <= int(page_table[b, pos // P]) < pages:
                raise RuntimeError(f"kv_append: position {pos} of row {b} lies outside the cache")
            page, place = int(page_table[b, pos // P]), pos % P
            for i, x in enumerate((k, v)):
                if scales is None:
                    kv[page, i, :, place] = x[b, t].to(kv.dtype)
                else:
                    kv[page, i, :, place], scales[page, i, :, place] = quantize_e4m3(x[b, t])


def kv_copy_pages_reference(kv, src, dst, scales=None) -> None:
    s, d, n = src.tolist(), dst.tolist(), kv.shape[1]
    _check_pairs(s, d, n)
    for part in (kv.view(torch.uint8) if kv.dtype == torch.float8_e4m3fn else kv, scales):   # (8-bit floats cannot be indexed everywhere)
        if part is not None:
            part[:, d] = part[:, s]


def paged_attention_reference(q, kv, page_table, lengths, softmax_scale=None, window: int = 0, softcap: float = 0.0, sinks=None, scales=None):
    """(output, log-sum-exp), computed in fp64 for fp64 inputs and in fp32 for all others."""
    B, Hq, D = q.shape
    _, _, Hkv, P, _ = kv.shape
    ft = torch.float64 if q.dtype == torch.float64 else torch.float32
    out, lse = torch.zeros(B, Hq, D, dtype=ft, device=q.device), torch.full((B, Hq), -math.inf, dtype=ft, device=q.device)
    for b in range(B):
        n = int(lengths[b])
        a = max(0, n - window) if window else 0
        if n > page_table.shape[1] * P or n < 0:
            raise RuntimeError(f"paged_attention: length {n} of row {b} lies outside its pages")
        if n == a:
            continue
        pages = page_table[b, a // P:(n + P - 1) // P].long()
        if bool(((pages < 0) | (pages >= kv.shape[0])).any()):
            raise RuntimeError(f"paged_attention: row {b} has a page outside the cache")
        x = kv[pages].to(ft)                                            # [pages, 2, Hkv, P, D]
        if scales is not None:
            x = x * scales[pages].to(ft).unsqueeze(-1)
        x = x.permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, D)[:, :, a - a // P * P:][:, :, :n - a]
        s = q[b].to(ft).reshape(Hkv, Hq // Hkv, D) @ x[0].transpose(-1, -2) * (D ** -0.5 if softmax_scale is None else softmax_scale)
        if softcap:
            s = torch.tanh(s / softcap) * softcap
        s = s.reshape(Hq, -1)
        lse[b] = torch.logsumexp(s, -1)
        total = lse[b] if sinks is None else torch.logaddexp(lse[b], sinks.to(ft))
        p = torch.exp(s - total.unsqueeze(-1))
        out[b] = (p.reshape(Hkv, Hq // Hkv, -1) @ x[1]).reshape(Hq, D)
    return out.to(q.dtype), lse.to(torch.float64 if ft == torch.float64 else torch.float32)


# ---------------------------------------------------------------------------------------------- entry points
_ext = None


def _kernels():
    """The extension module; kept here because looking it up costs as much as a small launch."""
    global _ext
    if _ext is None:
        from . import ext

        _ext = ext()
    return _ext


def kv_append(kv: torch.Tensor, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor, count: Optional[torch.Tensor] = None,
              scales: Optional[torch.Tensor] = None) -> None:
    """Write the keys and values of new tokens into one layer's pages, in place.

    ``k``, ``v`` ``[rows, T, kv heads, head size]`` (any strides: slices of packed projections are read where they lie) of the cache's type, or
    bf16 / fp16 / fp32 with an e4m3 cache, which then also gets ``scales``; row ``b``'s token ``t`` goes to position ``start[b] + t`` for
    ``t < count[b]`` (all ``T`` without ``count``).  ``page_table`` int32 ``[rows, pages of a row]``, ``start`` and ``count`` int32 ``[rows]``.
    Two tokens of one call must not have the same place."""
    if kv.is_cuda:
        return _kernels().kv_append(kv, k, v, page_table, start, count, scales)
    if kv.dim() != 5 or kv.shape[1] != 2 or k.dim() != 4 or k.shape != v.shape or k.shape[2:] != (kv.shape[2], kv.shape[4]):
        raise RuntimeError("kv_append: kv must be [pages, 2, kv heads, page size, head size], k and v [rows, tokens, kv heads, head size]")
    if (scales is not None) != (kv.dtype == torch.float8_e4m3fn):
        raise RuntimeError("kv_append: scales go with a float8_e4m3fn cache, and only with one")
    if scales is None and k.dtype != kv.dtype:
        raise RuntimeError("kv_append: k and v must have the cache's type")
    kv_append_reference(kv, k, v, page_table, start, count, scales)


def _check_pairs(src: Sequence[int], dst: Sequence[int], pages: int) -> None:
    if len(src) != len(dst):
        raise RuntimeError("kv_copy_pages: as many targets as sources are needed")
    if any(not 0 <= x < pages for x in list(src) + list(dst)):
        raise RuntimeError(f"kv_copy_pages: a page number outside the cache's {pages} pages")
    moved = [(a, b) for a, b in zip(src, dst) if a != b]
    if len(set(dst)) != len(dst) or {a for a, _ in zip(src, dst)} & {b for _, b in moved}:
        raise RuntimeError("kv_copy_pages: a page is copied onto one that another pair of the same call reads or writes")


def kv_copy_pages(kv: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, scales: Optional[torch.Tensor] = None) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every layer of ``kv [layers, pages, 2, kv heads, page size, head size]``, in place, and of
    ``scales [layers, pages, 2, kv heads, page size]`` with them.  ``src``, ``dst`` int32 on the cache's device.  The pairs have no order: no
    page may be a target twice, or a target and another pair's source (a page copied onto itself is no target for the others); pairs that break
    this are left out and reported."""
    if kv.is_cuda:
        return _kernels().kv_copy_pages(kv, src, dst, scales)
    if kv.dim() != 6 or kv.shape[2] != 2:
        raise RuntimeError("kv_copy_pages: kv must be [layers, pages, 2, kv heads, page size, head size]")
    if kv.dtype == torch.float8_e4m3fn and scales is None:
        raise RuntimeError("kv_copy_pages: the scales of a float8_e4m3fn cache are copied with its pages")
    if scales is not None and (scales.shape != kv.shape[:5] or scales.dtype != torch.float32):
        raise RuntimeError("kv_copy_pages: scales must be fp32 [layers, pages, 2, kv heads, page size]")
    kv_copy_pages_reference(kv, src, dst, scales)


def paged_attention(q: torch.Tensor, kv: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *, softmax_scale: Optional[float] = None, window: int = 0,
                    softcap: float = 0.0, sinks: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of one token of each row over the first ``lengths[row]`` tokens of its pages (its own, the last, among them).

    ``q [rows, query heads, head size]`` (64, 128 or 256 on a GPU; query head ``h`` reads key head ``h // (query heads / kv heads)``), of the
    cache's type, or bf16 / fp16 with an e4m3 cache.  ``window`` > 0: only the last ``window`` tokens; ``softcap`` > 0: scores become
    ``softcap * tanh(score / softcap)`` (2^-64 to 2^64); ``sinks`` fp32 ``[query heads]``: logits that take part in the softmax's sum without a value;
    ``softmax_scale`` defaults to ``head size ** -0.5``.  Returns ``[rows, query heads, head size]`` of q's type, with ``return_lse`` also the
    fp32 log-sum-exp of the scores ``[rows, query heads]`` (without the sinks).  A row of length 0 gives zeros and -inf; NaN and infinities in places
    that count make outputs NaN as the formula does, those in other places are not seen.  Scales of an e4m3 cache are positive."""
    if kv.is_cuda:
        out, lse = _kernels().paged_attention(q, kv, page_table, lengths, softmax_scale, window, softcap, sinks, scales, return_lse)
    else:
        if kv.dim() != 5 or kv.shape[1] != 2 or q.dim() != 3 or q.shape[2] != kv.shape[4] or q.shape[1] % kv.shape[2] or window < 0 or softcap < 0:
            raise RuntimeError("paged_attention: kv must be [pages, 2, kv heads, page size, head size], q [rows, query heads, head size]; window and softcap not negative")
        if not (softcap == 0 or 2.0 ** -64 <= softcap <= 2.0 ** 64) or (softmax_scale is not None and not abs(softmax_scale) < 2.0 ** 128):
            raise RuntimeError("paged_attention: softcap must be 0 or within 2^-64 and 2^64, the scale finite in fp32")
        if (scales is not None) != (kv.dtype == torch.float8_e4m3fn):
            raise RuntimeError("paged_attention: scales go with a float8_e4m3fn cache, and only with one")
        out, lse = paged_attention_reference(q, kv, page_table, lengths, softmax_scale, int(window), float(softcap), sinks, scales)
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------------------------- the cache of a model
class PagedKVCache:
    """The pages of all layers, and which sequence owns which.

    Sequences are numbers below ``max_seqs``.  Pages are counted by owner: ``fork`` lets completions of one prompt share its full pages and
    copies only the last, partly filled one.  The books are kept on the host; ``table`` makes the device copy that the kernels read."""

    def __init__(self, n_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, max_seqs: int, dtype: torch.dtype = torch.bfloat16, device=None):
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"the page size must be a multiple of 16, not {page_size}")
        if min(n_layers, num_pages, num_kv_heads, head_dim, max_seqs) <= 0:
            raise ValueError("a cache needs at least one layer, page, head, element and sequence")
        self.page_size, self.num_pages, self.max_seqs = page_size, num_pages, max_seqs
        self.kv = torch.zeros(n_layers, num_pages, 2, num_kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.scales = torch.ones(n_layers, num_pages, 2, num_kv_heads, page_size, device=device) if dtype == torch.float8_e4m3fn else None
        self.device = self.kv.device
        self._free: List[int] = list(range(num_pages - 1, -1, -1))          # pages are handed out from the end: lowest numbers first
        self._owners = [0] * num_pages
        self._pages: Dict[int, List[int]] = {}
        self._length: Dict[int, int] = {}

    # ------------------------------------------------------------------ books
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def sequences(self) -> List[int]:
        return sorted(self._pages)

    def length(self, seq: int) -> int:
        return self._length[seq]

    def pages(self, seq: int) -> List[int]:
        return list(self._pages[seq])

    def _take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise RuntimeError(f"the cache is full: {n} pages needed, {len(self._free)} free")
        got = [self._free.pop() for _ in range(n)]
        for p in got:
            self._owners[p] = 1
        return got

    def _drop(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._owners[p] -= 1
            if self._owners[p] == 0:
                self._free.append(p)
        self._free.sort(reverse=True)

    def _new(self, seq: int) -> None:
        if not 0 <= seq < self.max_seqs:
            raise ValueError(f"sequence {seq} is outside the cache's {self.max_seqs}")
        if seq in self._pages:
            raise ValueError(f"sequence {seq} is in use")

    def reserve(self, counts: Dict[int, int]) -> None:
        """Make room for ``counts[seq]`` more tokens of each sequence (unknown ones start empty), and count them as written: every layer then appends
        them.  A shared last page that new tokens would go to is copied first.  Nothing changes if the cache has not enough free pages."""
        P = self.page_size
        need, split = {}, []
        for seq, n in counts.items():
            if n < 0:
                raise ValueError("a sequence cannot grow by a negative number of tokens")
            if seq not in self._pages:
                self._new(seq)
            have = self._length.get(seq, 0)
            need[seq] = (have + n + P - 1) // P - len(self._pages.get(seq, ()))
            if n and have % P and self._owners[self._pages[seq][-1]] > 1:
                split.append(seq)
        # of the owners of one shared page all but the last to go get a copy
        copies, owners = [], {}
        for seq in split:
            page = self._pages[seq][-1]
            owners.setdefault(page, self._owners[page])
            if owners[page] > 1:
                owners[page] -= 1
                copies.append(seq)
        total = sum(max(0, x) for x in need.values()) + len(copies)
        if total > len(self._free):
            raise RuntimeError(f"the cache is full: {total} pages needed, {len(self._free)} free")
        if copies:
            src, dst = [], self._take(len(copies))
            for seq, page in zip(copies, dst):
                old = self._pages[seq][-1]
                src.append(old)
                self._owners[old] -= 1
                self._pages[seq][-1] = page
            self._copy(src, dst)
        for seq, n in counts.items():
            self._pages.setdefault(seq, []).extend(self._take(max(0, need[seq])))
            self._length[seq] = self._length.get(seq, 0) + n

    def fork(self, seq: int, children: Sequence[int]) -> None:
        """Start ``children`` as copies of ``seq``.  Pages are shared; a partly filled last page is copied when an owner next writes to it."""
        if len(set(children)) != len(children):
            raise ValueError("a sequence can be forked into a child once")
        for c in children:
            self._new(c)
        for c in children:
            self._pages[c] = list(self._pages[seq])
            self._length[c] = self._length[seq]
            for p in self._pages[c]:
                self._owners[p] += 1

    def free(self, seq: int) -> None:
        self._drop(self._pages.pop(seq))
        del self._length[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Forget the tokens of ``seq`` from position ``length`` on."""
        if not 0 <= length <= self._length[seq]:
            raise ValueError(f"sequence {seq} has {self._length[seq]} tokens")
        keep = (length + self.page_size - 1) // self.page_size
        self._drop(self._pages[seq][keep:])
        del self._pages[seq][keep:]
        self._length[seq] = length

    def compact(self) -> int:
        """Move the pages in use to the lowest numbers (so that the end of the cache can be given back); returns how many moved."""
        used = [p for p in range(self.num_pages) if self._owners[p]]
        n = len(used)
        holes = [p for p in range(n) if not self._owners[p]]
        movers = [p for p in used if p >= n]
        to = dict(zip(movers, holes))
        if not to:
            return 0
        self._copy(list(to), list(to.values()))
        for pages in self._pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._owners[b], self._owners[a] = self._owners[a], 0
        self._free = list(range(self.num_pages - 1, n - 1, -1))
        return len(to)

    def _copy(self, src: List[int], dst: List[int]) -> None:
        _check_pairs(src, dst, self.num_pages)
        for i in range(0, len(src), 65535):
            both = torch.tensor([src[i:i + 65535], dst[i:i + 65535]], dtype=torch.int32).to(self.device)
            kv_copy_pages(self.kv, both[0], both[1], self.scales)

    # ------------------------------------------------------------------ device side
    def table(self, seqs: Sequence[int], tokens: int = 0) -> torch.Tensor:
        """int32 ``[len(seqs), pages]`` on the device: the pages of each sequence, -1 behind its last.  Wide enough for ``tokens`` tokens a row."""
        width = max([1, (tokens + self.page_size - 1) // self.page_size] + [len(self._pages[s]) for s in seqs])
        return torch.tensor([self._pages[s] + [-1] * (width - len(self._pages[s])) for s in seqs], dtype=torch.int32).to(self.device)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, count: Optional[torch.Tensor] = None) -> None:
        kv_append(self.kv[layer], k, v, table, start, count, None if self.scales is None else self.scales[layer])

    def attend(self, layer: int, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, **kw):
        return paged_attention(q, self.kv[layer], table, lengths, scales=None if self.scales is None else self.scales[layer], **kw)
