"""Paged KV cache: the exact windows of a batch of sequences in pages of one
pool.

The reference keeps one cache per sequence (cache.py:33-57), and
``RFSNBatchedKVCache`` one region of fixed capacity each; here a sequence takes
pages of ``page_size`` tokens from a pool as it grows and returns them when it
ends, so that what is held is what the sequences have, whatever their lengths.

* ``append`` / ``prefill`` write new rows (fp16, or int8 / e4m3 codes with a
  scale per row) and each page's key bounds in one launch;
* ``attention_forward`` attends the newest token of every sequence over all of
  its positions, or over the pages whose bounds promise the largest scores;
* ``prompt_attention`` attends a chunk of one sequence's prompt;
* ``sequence_window`` reads one sequence back.

Rows of K/V heads are as in the other caches: ``num_kv_heads`` heads are stored
and query head ``i`` reads KV head ``i // (Hq // Hkv)``.  Calls belong on one
stream, like those of the other caches.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import kernels as K
from .attention import _blockwise_exact_attention
from .storage import RFSNConfig

PAGE_DTYPES = {"fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class RFSNPagedKVCache:
    """``pages`` pages of ``page_size`` tokens for up to ``batch`` sequences of up to ``max_tokens`` tokens (default:
    the whole pool).  ``page_type``: "fp16", "int8" or "e4m3".  ``bounds``: keep what page selection needs (4 bytes
    per page, KV head and coordinate)."""

    def __init__(self, config: RFSNConfig, batch: int, pages: int, page_size: int = 64, page_type: str = "fp16",
                 max_tokens: Optional[int] = None, bounds: bool = True, device=None):
        if batch <= 0 or pages <= 0:
            raise ValueError("batch and pages must be positive")
        if page_size not in K.PAGE_SIZES:
            raise ValueError(f"page_size must be one of {K.PAGE_SIZES}")
        if page_type not in PAGE_DTYPES:
            raise ValueError(f"page_type must be one of {tuple(PAGE_DTYPES)}")
        if config.head_dim not in (64, 128, 256):
            raise ValueError("paged caches serve head_dim 64, 128 and 256")
        if max_tokens is not None and max_tokens <= 0:
            raise ValueError("max_tokens must be positive")
        self.config = config
        self.batch = batch
        self.H = config.kv_heads
        self.D = config.head_dim
        self.scale = config.head_dim ** -0.5
        self.page_size = page_size
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        width = pages if max_tokens is None else min(pages, -(-max_tokens // page_size))
        self.max_tokens = width * page_size if max_tokens is None else min(max_tokens, width * page_size)
        shape, dtype = (pages, self.H, page_size, self.D), PAGE_DTYPES[page_type]
        new = lambda s, d: torch.zeros(s, dtype=d, device=self.device)
        scales = (None, None) if page_type == "fp16" else (new(shape[:3], torch.float32), new(shape[:3], torch.float32))
        self.pages = K.KVPages(new(shape, dtype), new(shape, dtype), *scales,
                               new((pages, self.H, 2, self.D), torch.float16) if bounds else None)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=self.device)
        self.lens = new((batch,), torch.int32)
        self.num_tokens: List[int] = [0] * batch
        self._held: List[List[int]] = [[] for _ in range(batch)]
        self._free = list(range(pages - 1, -1, -1))
        self._ended = set()  # released, and without tokens since

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _index(self, b: int) -> int:
        if not 0 <= b < self.batch:
            raise ValueError(f"sequence {b} out of range (batch {self.batch})")
        return b

    def _rows(self, x: torch.Tensor, what: str) -> torch.Tensor:
        if x.dim() != 3 or tuple(x.shape[1:]) != (self.H, self.D):
            raise ValueError(f"{what} must be [tokens, {self.H}, {self.D}]")
        return x.to(device=self.device, dtype=torch.float16)

    def _reserve(self, counts: Sequence[int]) -> None:
        """Pages for ``counts`` more tokens, all or none."""
        total = [n + c for n, c in zip(self.num_tokens, counts)]
        if max(total) > self.max_tokens:
            raise ValueError(f"a sequence would pass max_tokens ({self.max_tokens})")
        need = [-(-t // self.page_size) - len(h) for t, h in zip(total, self._held)]
        wanted = sum(n for n in need if n > 0)
        if wanted > len(self._free):
            raise RuntimeError(f"page pool exhausted: {wanted} pages wanted, {len(self._free)} free")
        if not wanted:
            return
        b_at, o_at, page = [], [], []
        for b, n in enumerate(need):
            for _ in range(max(n, 0)):
                b_at.append(b)
                o_at.append(len(self._held[b]))
                page.append(self._free.pop())
                self._held[b].append(page[-1])
        at = torch.tensor([b_at, o_at, page], device=self.device)
        self.table[at[0], at[1]] = at[2].to(torch.int32)

    def append(self, keys: torch.Tensor, values: torch.Tensor, counts: Optional[Sequence[int]] = None) -> None:
        """New rows [N, Hkv, D] of all sequences, ``counts[b]`` of sequence b in
        the order of the batch (default: one each, a decode step).  While a
        released sequence has no successor and others go on, ``counts`` has to be
        given (0 for it): one more token each would start a sequence there."""
        k, v = self._rows(keys, "keys"), self._rows(values, "values")
        each = [1] * self.batch if counts is None else [int(c) for c in counts]
        if len(each) != self.batch or min(each) < 0 or sum(each) != k.shape[0] or v.shape != k.shape:
            raise ValueError(f"{k.shape[0]} key and {v.shape[0]} value rows do not match the counts of "
                             f"{self.batch} sequences")
        if counts is None and self._ended and any(self.num_tokens):
            raise ValueError(f"sequences {sorted(self._ended)} were released: append takes counts until they hold "
                             "tokens again")
        self._reserve(each)
        if counts is None:
            K.paged_append(self.pages, self.table, self.lens, k, v)
            self.lens.add_(1)
        else:
            cu = [0]
            for c in each:
                cu.append(cu[-1] + c)
            on = torch.tensor([cu, each + [0]], dtype=torch.int32).to(self.device)
            K.paged_append(self.pages, self.table, self.lens, k, v, on[0])
            self.lens.add_(on[1, :-1])
        self.num_tokens = [n + c for n, c in zip(self.num_tokens, each)]
        if self._ended:
            self._ended = {b for b in self._ended if not self.num_tokens[b]}

    def prefill(self, b: int, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Rows [T, Hkv, D] behind what sequence b holds (a prompt, or a chunk of one)."""
        self._index(b)
        counts = [0] * self.batch
        counts[b] = int(keys.shape[0])
        self.append(keys, values, counts)

    def release(self, b: int) -> None:
        """Sequence b ends: its pages return to the pool."""
        self._index(b)
        self._free.extend(reversed(self._held[b]))
        self._held[b] = []
        self.num_tokens[b] = 0
        self.table[b].fill_(-1)
        self.lens[b:b + 1].zero_()
        self._ended.add(b)

    def _live_table(self) -> torch.Tensor:
        """The table's columns that some sequence uses."""
        return self.table[:, :max(1, max(len(h) for h in self._held))]

    def attention_forward(self, q: torch.Tensor, sparse_pages: int = 0) -> torch.Tensor:
        """q [B, Hq, D], each sequence's newest token, over the sequence's
        positions -> [B, Hq, D] in q's dtype; an empty sequence gives zeros.
        ``sparse_pages``: over that many of its pages per KV head, the first, the
        newest and those whose bounds promise the largest scores (of keys before
        their rounding to 8 bits)."""
        if q.dim() != 3 or q.shape[0] != self.batch or q.shape[2] != self.D:
            raise ValueError(f"q must be [{self.batch}, heads, {self.D}]")
        qh = q.to(device=self.device, dtype=torch.float16)
        table = self._live_table()
        chosen = None
        if sparse_pages:
            if sparse_pages < 2:
                raise ValueError("sparse_pages must have room for the first and the newest page")
            chosen = K.page_select(qh, self.pages, table, self.lens, sparse_pages)
        held = self.pages.k.shape[0] - len(self._free)
        return K.paged_attention(qh, self.pages, table, self.lens, self.scale, chosen, held).to(q.dtype)

    def prompt_attention(self, b: int, q: torch.Tensor) -> torch.Tensor:
        """q [S, Hq, D], the newest S tokens of sequence b, each over the
        positions up to its own -> [S, Hq, D] in q's dtype.  Rows of 8-bit pages
        are read back as fp16 first at head sizes 64 and 128, while
        ``attention_forward`` takes code * scale as it is."""
        n = self.num_tokens[self._index(b)]
        if q.dim() != 3 or q.shape[2] != self.D or q.shape[0] > n:
            raise ValueError(f"q must be [S, heads, {self.D}] of at most the {n} tokens held")
        if q.shape[0] == 0:
            return torch.zeros_like(q)
        if self.D == 256:  # the blockwise entry serves 64 and 128: each query as a sequence of its own over the same pages
            qh, out = q.to(device=self.device, dtype=torch.float16), []
            ends = torch.arange(n - q.shape[0] + 1, n + 1, dtype=torch.int32, device=self.device)
            for part, lens in zip(qh.split(4096), ends.split(4096)):
                table = self.table[b:b + 1, :len(self._held[b])].expand(part.shape[0], -1)
                out.append(K.paged_attention(part, self.pages, table, lens, self.scale))
            return torch.cat(out).to(q.dtype)
        keys, values = self.sequence_window(b)
        return _blockwise_exact_attention(q.to(self.device), keys, values, self.scale, self.config.block_size_seq,
                                          causal=True, query_positions=torch.arange(n - q.shape[0], n))

    def sequence_window(self, b: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """K and V [T, Hkv, D] fp16 of sequence b."""
        n = self.num_tokens[self._index(b)]
        at = torch.tensor([0, 0, n], dtype=torch.int32).to(self.device)
        return K.paged_read(self.pages, self.table[b:b + 1], at[:1], at[1:], n)

    def memory_usage_bytes(self) -> Dict[str, int]:
        """Bytes of the pool, of the pages in use, and of the table and lengths."""
        size = lambda t: 0 if t is None else t.numel() * t.element_size()
        pool = sum(size(t) for t in self.pages)
        total = self.pages.k.shape[0]
        return {"pool": pool, "in_use": pool // total * (total - len(self._free)),
                "table": size(self.table) + size(self.lens)}
