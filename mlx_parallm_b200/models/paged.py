"""A key-value cache in pages for the Llama-like decoders (DecoderModel.make_paged_cache).

The reference has no such cache: its PagedKVCache (mlx_parallm/models/base.py:93-149) keeps offsets per row on one dense buffer.
Here every layer owns a pool of pages [P, kv heads, page, D], and one book per generation says which pages belong to which row: a
row takes pages as it grows and gives them back, so memory follows what the rows hold and not batch x longest row.  A book may

  - keep only a window of the newest tokens visible, with a few first ones (``window``, ``first``);
  - cut rows that have no room left to the tokens that were attended to most (``keep``, with the ``first`` and the ``recent`` newest ones):
    the layers then add up the attention weight every token receives, and each key head keeps tokens of its own.

Decode steps read the pages (b200p_paged_attn); prompts are attended to through a dense view of their rows (b200p_paged_gather) by the
prompt kernels of dense caches, or token by token once the window hides part of a row.  The device table and counters keep their
addresses, so a captured decode step stays valid while rows grow, shrink and change hands.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from .. import ops
from .base import RowState


OBSERVED_BYTES = 256 << 20        # workspace of a call that adds up the weights of a prompt's last tokens (one token per row at least)


class PagesExhausted(RuntimeError):
    """A step found no room for its tokens in a cache in pages: none of them was appended."""


class PageBook:
    """Which pages belong to which row, for all layers of a generation: the device ``table`` [rows, width] (-1: none), the rows' ``lengths`` (slots in
    use) and ``positions`` (places in the text: larger than the length once tokens were evicted), and the list of free pages."""

    def __init__(self, rows: int, max_tokens: int, device, page: int = 64, pages: Optional[int] = None, window: int = 0, first: int = 0, keep: int = 0,
                 recent: Optional[int] = None, observe: int = 32):
        if page < 16 or page % 16 or page > 4096:
            raise ValueError(f"a page holds a multiple of 16 tokens, 4096 at most: got {page}")
        if rows < 1 or max_tokens < 1:
            raise ValueError("a paged cache has rows, and room for a token in each")
        width = -(-max_tokens // page)
        self.rows, self.page, self.width, self.device = rows, page, width, torch.device(device)
        self.pages = rows * width if pages is None else int(pages)
        if self.pages < 1:
            raise ValueError("a paged cache has at least one page")
        self.window, self.first, self.keep = int(window), int(first), int(keep)
        self.recent = (self.keep - self.first) // 2 if recent is None else int(recent)
        if self.window < 0 or self.first < 0:
            raise ValueError("window and first are counts")
        if self.keep and not (0 <= self.recent and self.first + self.recent <= self.keep < width * page):
            raise ValueError(f"a row of {width * page} tokens cannot be cut to {self.keep}, {self.first} first and {self.recent} recent ones among them")
        self.observe = int(observe)            # a prompt's last tokens, whose weights count when its row is cut
        self.behind = 0                        # tokens of the prompt behind the portion that is being read
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros((rows,), dtype=torch.int32, device=device)
        self.positions = torch.zeros((rows,), dtype=torch.int32, device=device)
        self.row_index = torch.arange(rows, dtype=torch.int32, device=device)      # -1: a row that was given back, whose tokens are idle
        self.live = [True] * rows
        self.free: List[int] = list(range(self.pages - 1, -1, -1))
        self.owned: List[List[int]] = [[] for _ in range(rows)]
        self.evicted = [0] * rows              # how far a row's positions are ahead of its slots
        self.layers: List["PagedLayer"] = []
        self._scratch = {}

    @property
    def max_tokens(self) -> int:
        return self.width * self.page

    def room_for(self, counts: List[int]) -> None:
        """Give every row the pages for ``counts[r]`` tokens (a row that has more keeps them).  All or nothing: PagesExhausted if the pool is short."""
        if max(counts, default=0) > self.max_tokens:
            raise PagesExhausted(f"a row of {max(counts)} tokens does not fit a paged cache of {self.max_tokens} per row")
        need = [max(0, -(-n // self.page) - len(o)) for n, o in zip(counts, self.owned)]
        if sum(need) == 0:
            return
        if sum(need) > len(self.free):
            raise PagesExhausted(f"paged cache exhausted: {sum(need)} pages wanted, {len(self.free)} of {self.pages} free")
        for r, k in enumerate(need):
            if k:
                new = [self.free.pop() for _ in range(k)]
                at = len(self.owned[r])
                self.owned[r] += new
                self.table[r, at:at + k] = torch.tensor(new, dtype=torch.int32).to(self.device)

    def release(self, rows: List[int]) -> None:
        """Rows that are given back are idle until the cache is reset: they take no pages and their counters stay at 0."""
        for r in rows:
            if self.live[r]:
                self.live[r] = False
                self.row_index[r] = -1

    def revive(self) -> None:
        if not all(self.live):
            self.live = [True] * self.rows
            self.row_index.copy_(torch.arange(self.rows, dtype=torch.int32))

    def shrink(self, counts: List[int]) -> None:
        """Take back the pages that rows of ``counts[r]`` tokens do not need."""
        for r, n in enumerate(counts):
            left = -(-n // self.page)
            if left < len(self.owned[r]):
                self.free += reversed(self.owned[r][left:])
                del self.owned[r][left:]
                self.table[r, left:] = -1

    def cut(self, keep: int, first: int, recent: int) -> None:
        """Every row of more than ``keep`` tokens keeps its ``first`` first and ``recent`` newest ones and the most attended ones between (per
        layer and key head); its next tokens go on at their positions in the text."""
        if not self.layers or any(c.mass is None for c in self.layers):
            raise RuntimeError("only a cache that adds up attention weights (keep > 0) can be cut")
        counts = list(self.layers[0]._offsets)
        if max(counts) <= keep:
            return
        for c in self.layers:
            kept = self.scratch("kept", (self.rows, c.n_kv_heads, keep), torch.int32)
            ops.paged_evict(c.kpages, c.vpages, c.mass, self.table, self.lengths, kept, first=first, recent=recent)
        self.lengths.clamp_(max=keep)
        self.evicted = [e + max(0, n - keep) for e, n in zip(self.evicted, counts)]
        counts = [min(n, keep) for n in counts]
        self.shrink(counts)
        for c in self.layers:
            c._offsets = list(counts)
            c.offset = max(counts)

    def scratch(self, name: str, shape, dtype) -> torch.Tensor:
        t = self._scratch.get(name)
        if t is None or t.shape != torch.Size(shape) or t.dtype != dtype:
            t = self._scratch[name] = torch.empty(shape, dtype=dtype, device=self.device)
        return t

    @property
    def weighed(self) -> int:
        """Slots of a row that a token can give a weight to (0: nobody adds them up)."""
        if not self.keep:
            return 0
        return min(self.max_tokens, self.first + self.window + 32) if self.window else self.max_tokens

    def workspace(self, M: int, H: int, G: int, D: int, keys: int) -> torch.Tensor:
        """The workspace of calls of M tokens, which are on one stream (the decode step's stays where a captured step knows it)."""
        need = ops.paged_attn_workspace_bytes(M, H, D, keys, G)
        key = "step" if M == self.rows else "portion"
        t = self._scratch.get(key)
        if t is None or t.numel() < need:
            t = self._scratch[key] = torch.empty((need,), dtype=torch.uint8, device=self.device)
        return t

    def tokens(self, B: int, L: int):
        """(row, slot, position) of the B x L tokens that are about to be appended."""
        if L == 1:
            return self.row_index, self.lengths, self.positions
        M = B * L
        cu = torch.arange(0, M + 1, L, dtype=torch.int32, device=self.device)
        row, slot, pos, off = (torch.empty((M,), dtype=torch.int32, device=self.device) for _ in range(4))
        ops.ragged_plan(cu, self.row_index, self.lengths, row, slot, off, B, M)
        ops.ragged_plan(cu, self.row_index, self.positions, row, pos, off, B, M)
        return row, slot, pos


class PagedLayer(RowState):
    """One layer's entry in the cache list of a paged generation: its pages and, if rows may be cut, the weight their tokens received."""

    def __init__(self, book: PageBook, n_heads: int, n_kv_heads: int, head_dim: int):
        super().__init__(book.rows)
        self.book, self.n_heads, self.n_kv_heads, self.head_dim = book, n_heads, n_kv_heads, head_dim
        self.kpages: Optional[torch.Tensor] = None
        self.vpages: Optional[torch.Tensor] = None
        self.mass: Optional[torch.Tensor] = None
        self.share_lengths(book.lengths)
        book.layers.append(self)

    def buffers(self) -> tuple:
        return (self.kpages, self.vpages, self.mass, self.book.table)

    @property
    def capacity(self) -> int:
        return self.book.max_tokens

    def counters(self) -> tuple:
        return (self.book.lengths, self.book.positions)

    def reset(self, batch_size: Optional[int] = None):
        if batch_size is not None and batch_size != self.batch_size:
            raise ValueError("a paged cache keeps the batch size it was made with")
        self.book.evicted = [0] * self.batch_size
        self.book.behind = 0
        super().reset(None)
        self.book.positions.zero_()
        self.book.shrink([0] * self.batch_size)
        self.book.revive()

    def release_rows_host(self, rows: List[int]):
        if any(not 0 <= r < self.batch_size for r in rows):
            raise ValueError(f"rows of this cache are 0 to {self.batch_size - 1}: got {list(rows)}")
        super().release_rows_host(rows)
        for r in rows:
            self.book.evicted[r] = 0
        self.book.release(rows)
        self.book.shrink(self._offsets)

    def advance_host(self, L: int):
        self._offsets = [o + L if live else 0 for o, live in zip(self._offsets, self.book.live)]
        self.offset = max(self._offsets)

    def _sync_lengths(self):
        super()._sync_lengths()
        self.book.positions.copy_(torch.tensor([n + e for n, e in zip(self._offsets, self.book.evicted)], dtype=torch.int32))

    def ensure_capacity(self, needed: int, dtype, device) -> bool:
        """``needed``: the longest row's tokens after the coming step; the other rows in use grow by as many."""
        moved = False
        if self.kpages is None or self.kpages.dtype != dtype:
            shape = (self.book.pages, self.n_kv_heads, self.book.page, self.head_dim)
            self.kpages = torch.zeros(shape, dtype=dtype, device=device)
            self.vpages = torch.zeros(shape, dtype=dtype, device=device)
            self.mass = torch.zeros(shape[:3], dtype=torch.float32, device=device) if self.book.keep else None
            if self.kpages.is_cuda:                                     # a decode step's workspace: not inside its capture
                self.book.workspace(self.batch_size, self.n_heads, self.n_kv_heads, self.head_dim, self.book.weighed)
            moved = True
        if self is self.book.layers[0]:
            new, room = needed - max(self._offsets), self.book.max_tokens
            if self.book.keep and needed > room:
                left = min(self.book.keep, room - new)
                if left < max(1, self.book.first + self.book.recent):
                    raise PagesExhausted(f"{new} tokens at once do not fit a paged cache of {room} per row beside the {self.book.first} first and "
                                         f"{self.book.recent} recent ones it keeps")
                self.book.cut(left, self.book.first, self.book.recent)
            self.book.room_for([n + new if live else 0 for n, live in zip(self._offsets, self.book.live)])
        return moved

    # -- the layer's part of a step -----------------------------------------------------------------------------------
    def append_and_attend(self, qkv, q, out, tokens, B: int, L: int, heads: int, rates, scale: float, q_norm, k_norm, eps: float, attn_workspace,
                          out_perm: bool):
        """Norms, rotation and append of the step's tokens, then their attention: ``out`` [B L, heads D]."""
        book, G, D = self.book, self.n_kv_heads, self.head_dim
        row, slot, pos = tokens
        ops.paged_append(qkv, q, self.kpages, self.vpages, book.table, row, slot, pos, heads, rates=rates, q_norm_w=q_norm, k_norm_w=k_norm, eps=eps,
                         mass=self.mass)
        observed = min(L, max(0, book.observe - book.behind))
        if L == 1:
            ops.paged_attn(q, self.kpages, self.vpages, book.table, row, slot, out, scale, first=book.first, window=book.window,
                           mass=self.mass if observed or not book.behind else None, workspace=book.workspace(B, heads, G, D, book.weighed),
                           out_perm=out_perm)
            return
        if book.window and max(self._offsets) + L > book.window + book.first:      # (until then the window hides nothing)
            ops.paged_attn(q, self.kpages, self.vpages, book.table, row, slot, out, scale, first=book.first, window=book.window,
                           workspace=book.workspace(B * L, heads, G, D, 0), out_perm=out_perm)
        else:
            cap = -(-(max(self._offsets) + L) // 256) * 256
            dense = book.scratch("dense", (2, B, G, cap, D), self.kpages.dtype)
            ops.paged_gather(self.kpages, self.vpages, book.table, book.row_index, book.lengths, dense[0], dense[1], extra=L)
            ops.attn(q, dense[0], dense[1], book.lengths, out, B, L, heads, G, D, scale, workspace=attn_workspace, out_perm=out_perm)
        if not all(book.live):                                          # (a step's are what they were: finite)
            out.view(B, L, -1)[[not live for live in book.live]] = 0
        if self.mass is not None and observed > 0:                      # what the prompt's last tokens look at
            # as many at once as their scores have room for, every row's in order
            size = lambda n: ops.paged_attn_workspace_bytes(n * B, heads, D, book.weighed, G)
            n = max(1, min(observed, OBSERVED_BYTES // (size(2) - size(1)), 65535 // B))
            for l0 in range(L - observed, L, n):
                part = lambda t: t.view(B, L, -1)[:, l0:l0 + n].reshape(-1, t.numel() // (B * L)).contiguous()
                ql = part(q)
                ops.paged_attn(ql, self.kpages, self.vpages, book.table, part(row).view(-1), part(slot).view(-1), torch.empty_like(ql), scale,
                               first=book.first, window=book.window, mass=self.mass, workspace=book.workspace(ql.shape[0], heads, G, D, book.weighed))
