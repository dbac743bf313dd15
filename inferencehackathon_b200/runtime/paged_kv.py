"""A paged KV cache for several sequences: pages and tables for the operators of :mod:`..ops.paged`.

The contiguous caches of the decoder hold one sequence; here sequences of any length share one pool of pages, grow page by page, give
pages back, fork (a common prompt prefix is stored once) and drop rejected draft tokens. All bookkeeping is on the host; a step is
``batch = cache.extend({seq: tokens, ...})``, then per layer ``q = cache.append(layer, qkv, batch, cos, sin, ...)`` and
``out = cache.attend(layer, q, batch)``.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Hashable, List, Mapping, Optional, Sequence

import torch

from ..ops import paged


@dataclass
class PagedBatch:
    """Device-side description of one call: the sequences in token order, ``cu_q`` None when each has one token."""
    seqs: List[Hashable]
    block_table: torch.Tensor
    kv_len: torch.Tensor
    cu_q: Optional[torch.Tensor]
    max_q: int
    n_tokens: int


class _Seq:
    def __init__(self):
        self.pages: List[int] = []
        self.len = 0


class PagedKVCache:
    """``kv="bf16"``: bf16 rows; ``kv="fp8"``: e4m3 rows with one power-of-two scale per (layer, page, head)."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, page_size: int = 64, kv: str = "fp8", device="cuda"):
        if page_size not in paged.PAGE_SIZES:
            raise ValueError(f"page size must be one of {paged.PAGE_SIZES}")
        if kv not in ("bf16", "fp8"):
            raise ValueError('kv must be "bf16" or "fp8"')
        if n_layers < 1 or n_pages < 1 or n_kv_heads < 1:
            raise ValueError("layers, pages and KV heads must be positive")
        dtype = torch.bfloat16 if kv == "bf16" else torch.float8_e4m3fn
        self.page_size, self.n_pages, self.device = page_size, n_pages, torch.device(device)
        shape = (n_layers, n_pages, n_kv_heads, page_size, paged.HEAD_DIM)
        self.k = torch.empty(shape, dtype=dtype, device=self.device)      # rows are written before they are read
        self.v = torch.empty(shape, dtype=dtype, device=self.device)
        self.k_scale = self.v_scale = None
        if kv == "fp8":
            self.k_scale = torch.ones(shape[:3], dtype=torch.float32, device=self.device)
            self.v_scale = torch.ones(shape[:3], dtype=torch.float32, device=self.device)
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._refs = [0] * n_pages
        self._seqs: Dict[Hashable, _Seq] = {}

    # ---- bookkeeping -------------------------------------------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: Hashable) -> int:
        return self._seqs[seq].len

    def pages(self, seq: Hashable) -> List[int]:
        return list(self._seqs[seq].pages)

    def add(self, seq: Hashable) -> None:
        if seq in self._seqs:
            raise ValueError(f"sequence {seq!r} exists")
        self._seqs[seq] = _Seq()

    def free(self, seq: Hashable) -> None:
        for p in self._seqs.pop(seq).pages:
            self._release(p)

    def fork(self, seq: Hashable, new: Hashable) -> None:
        """``new`` starts with the rows of ``seq``. Pages are shared; a partly filled one is copied when either side writes to it."""
        src = self._seqs[seq]
        self.add(new)
        dst = self._seqs[new]
        dst.pages, dst.len = list(src.pages), src.len
        for p in dst.pages:
            self._refs[p] += 1

    def truncate(self, seq: Hashable, length: int) -> None:
        """Drops rows from ``length`` on (rejected draft tokens). The scale of the page that stays partly filled is kept: it holds for
        fewer rows as well."""
        s = self._seqs[seq]
        if not 0 <= length <= s.len:
            raise ValueError(f"sequence {seq!r} has {s.len} rows, cannot keep {length}")
        keep = -(-length // self.page_size)
        for p in s.pages[keep:]:
            self._release(p)
        del s.pages[keep:]
        s.len = length

    def _release(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def _take(self) -> int:
        page = self._free.pop()
        self._refs[page] = 1
        return page

    def _needs(self, s: _Seq, n: int) -> int:
        """Pages that ``n`` more tokens take, a copy of a shared last page included."""
        copy = n > 0 and s.len % self.page_size != 0 and self._refs[s.pages[-1]] > 1
        return -(-(s.len + n) // self.page_size) - len(s.pages) + copy

    # ---- one call ----------------------------------------------------------------------------------------------------------
    def extend(self, new: Mapping[Hashable, int]) -> PagedBatch:
        """Room for ``new[seq]`` more tokens of each sequence (in this order), and the batch that describes the call. Raises before
        anything changes when the pool does not hold them."""
        if not new:
            raise ValueError("no sequences")
        if any(n < 0 for n in new.values()) or sum(new.values()) < 1:
            raise ValueError("token counts must not be negative, and there must be a token")
        need, shared = 0, {}
        for q, n in new.items():
            need += self._needs(self._seqs[q], n)
            s = self._seqs[q]
            if n > 0 and s.len % self.page_size != 0:
                shared[s.pages[-1]] = shared.get(s.pages[-1], 0) + 1
        # the last of several writers of a shared page keeps it
        need -= sum(1 for p, writers in shared.items() if writers == self._refs[p] > 1)
        if need > len(self._free):
            raise RuntimeError(f"KV cache: {need} pages needed, {len(self._free)} free")
        for q, n in new.items():
            s = self._seqs[q]
            if n > 0 and s.len % self.page_size != 0 and self._refs[s.pages[-1]] > 1:
                old, page = s.pages[-1], self._take()
                for t in (self.k, self.v, self.k_scale, self.v_scale):
                    if t is not None:
                        t[:, page] = t[:, old]
                self._release(old)
                s.pages[-1] = page
            while len(s.pages) * self.page_size < s.len + n:
                s.pages.append(self._take())
            s.len += n
        return self._batch(list(new), list(new.values()))

    def _batch(self, seqs: Sequence[Hashable], counts: Sequence[int]) -> PagedBatch:
        width = max(1, max(len(self._seqs[q].pages) for q in seqs))
        table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        for b, q in enumerate(seqs):
            p = self._seqs[q].pages
            if p:
                table[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        lens = torch.tensor([self._seqs[q].len for q in seqs], dtype=torch.int32)
        cu = None
        if any(n != 1 for n in counts):
            cu = torch.zeros(len(seqs) + 1, dtype=torch.int32)
            cu[1:] = torch.tensor(counts, dtype=torch.int32).cumsum(0)
            cu = cu.to(self.device)
        return PagedBatch(list(seqs), table.to(self.device), lens.to(self.device), cu, max(counts), sum(counts))

    def _scales(self, layer: int):
        return (None, None) if self.k_scale is None else (self.k_scale[layer], self.v_scale[layer])

    def append(self, layer: int, qkv: torch.Tensor, batch: PagedBatch, cos_t: torch.Tensor, sin_t: torch.Tensor, *, nq: int,
               q_gamma: Optional[torch.Tensor] = None, k_gamma: Optional[torch.Tensor] = None, eps: float = 1e-6,
               positions: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """K / V rows of the batch's tokens into layer ``layer``; returns the rotated queries (see :func:`..ops.paged.paged_append`)."""
        ks, vs = self._scales(layer)
        return paged.paged_append(qkv, nq, self.k.shape[2], self.k[layer], self.v[layer], batch.block_table, batch.kv_len, cos_t, sin_t,
                                  cu_q=batch.cu_q, positions=positions, q_gamma=q_gamma, k_gamma=k_gamma, eps=eps, k_scale=ks, v_scale=vs,
                                  q_out=q_out, err=self.err)

    def attend(self, layer: int, q: torch.Tensor, batch: PagedBatch, *, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the batch's tokens over layer ``layer`` (see :func:`..ops.paged.paged_attention`)."""
        ks, vs = self._scales(layer)
        return paged.paged_attention(q, self.k[layer], self.v[layer], batch.block_table, batch.kv_len, cu_q=batch.cu_q, max_q=batch.max_q,
                                     mask=mask, k_scale=ks, v_scale=vs, scale=scale, out=out, lse=lse, err=self.err)

    def check_error(self) -> None:
        """Synchronises; raises when a kernel met a page id, a length or a position that does not fit."""
        code = int(self.err.item())
        if code:
            from ..ops.lib import ERR_NAMES
            self.err.zero_()
            raise RuntimeError(f"paged KV cache: device error {code} ({ERR_NAMES.get(code, '?')})")
