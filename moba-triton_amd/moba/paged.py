"""Books of a paged cache: which sequence holds which pages.

`PagedCache` gives pages to sequences as they grow, shares them between a
sequence and its forks, and moves them together when sequences have ended; the
work on the pages themselves is `moba.kernels.paged`'s. One decoding step:

    step = cache.grow(ids, [1] * len(ids))
    for i, layer in enumerate(layers):
        q, k, v = layer.project(x)                       # [T, heads, D]
        q = append_tokens(q, k, v, cache.kv.layer(i), *step.args, cos=..., ...)
        o = paged_attention(q, cache.kv.layer(i), step.block_table, step.seq_lens, cfg,
                            cu_seqlens=step.cu_seqlens)
"""

import ctypes
import heapq
from array import array
from dataclasses import dataclass

import torch

from moba.config import MoBAConfig
from moba.kernels.paged import PagedKV, copy_pages


class CacheFull(RuntimeError):
    """The cache has fewer free pages than the call needs; nothing changed."""


@dataclass(frozen=True)
class Step:
    """New tokens of some sequences, as `append_tokens` and `paged_attention`
    take them: int32 tensors on the cache's device."""

    block_table: torch.Tensor
    seq_lens: torch.Tensor
    cu_seqlens: torch.Tensor

    @property
    def args(self) -> tuple:
        return self.block_table, self.seq_lens, self.cu_seqlens


class _Sequence:
    def __init__(self, pages=(), length=0):
        self.pages, self.length = array("i", pages), length


class PagedCache:
    """Pages of every layer, and the sequences on them.

    Args:
        layers, pages: Pages of `cfg.block_size` tokens, in each of `layers`.
        kv_heads, head_dim: Of every layer.
        cfg: Supplies `block_size` and the dtype.
    """

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, cfg: MoBAConfig,
                 device="cuda"):
        self.kv = PagedKV.empty(pages, kv_heads, cfg.block_size, head_dim, cfg.dtype, device,
                                layers=layers)
        self.block_size = cfg.block_size
        self._free = list(range(pages))  # a heap: the lowest page goes first
        self._holders = [0] * pages
        self._sequences: dict[int, _Sequence] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._of(seq).length

    def pages(self, seq: int) -> list[int]:
        """The sequence's pages, in order."""
        return list(self._of(seq).pages)

    def create(self) -> int:
        """A new sequence without tokens."""
        self._sequences[self._next] = _Sequence()
        self._next += 1
        return self._next - 1

    def fork(self, seq: int) -> int:
        """A sequence with the same tokens, on the same pages until either
        grows into a page they share."""
        s = self._of(seq)
        for p in s.pages:
            self._holders[p] += 1
        self._sequences[self._next] = _Sequence(s.pages, s.length)
        self._next += 1
        return self._next - 1

    def free(self, seq: int) -> None:
        """Ends a sequence; pages nobody else holds are free again. Calls in
        flight on the current stream may still read them: a later `grow`'s
        work follows on the same stream."""
        for p in self._of(seq).pages:
            self._drop(p)
        del self._sequences[seq]

    def grow(self, seqs: list[int], new: list[int]) -> Step:
        """Room for `new[i]` more tokens of sequence `seqs[i]`. A partly filled
        last page that others hold too is copied first (one `copy_pages` call
        for all sequences; where that fails, nothing has changed). Does not
        wait for the device.

        Raises:
            CacheFull: With too few free pages; nothing has changed then.
            RuntimeError: While a graph is captured: the books would change
                once, the step's tables with every replay.
            ValueError: If a sequence is named twice or a count is negative.
        """
        self._outside_capture()
        if len(seqs) != len(new) or not seqs:
            raise ValueError(f"{len(seqs)} sequences, {len(new)} counts of new tokens")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        if any(n < 0 for n in new):
            raise ValueError("counts of new tokens must not be negative")
        held = [self._of(s) for s in seqs]
        bs = self.block_size
        # Of a shared page, all holders that write take a copy but the last
        # one to hold it.
        left = {}
        copies = []
        for s, n in zip(held, new):
            if n and s.length % bs:
                last = s.pages[-1]
                left.setdefault(last, self._holders[last])
                if left[last] > 1:
                    left[last] -= 1
                    copies.append(s)
        grown = [-(-(s.length + n) // bs) - len(s.pages) for s, n in zip(held, new)]
        if len(copies) + sum(grown) > len(self._free):
            raise CacheFull(f"{len(copies) + sum(grown)} pages needed, {len(self._free)} free")
        src, dst = [s.pages[-1] for s in copies], [self._take() for _ in copies]
        if src:
            try:
                copy_pages(self.kv, src, dst)
            except Exception:
                for p in dst:
                    self._drop(p)
                raise
        for s, p in zip(copies, dst):
            self._drop(s.pages[-1])
            s.pages[-1] = p
        for s, n, g in zip(held, new, grown):
            s.pages.extend(self._take() for _ in range(g))
            s.length += n
        return self._step(held, new)

    def compact(self) -> int:
        """Moves the pages in use to the front of the cache; returns how many
        moved. Block tables from before are stale. Not in a captured graph."""
        self._outside_capture()
        live = [p for p, n in enumerate(self._holders) if n]
        holes = [p for p in range(len(live)) if not self._holders[p]]
        move = dict(zip((p for p in live if p >= len(live)), holes))
        if not move:
            return 0
        copy_pages(self.kv, list(move), list(move.values()))
        for s in self._sequences.values():
            s.pages = array("i", (move.get(p, p) for p in s.pages))
        for a, b in move.items():
            self._holders[a], self._holders[b] = 0, self._holders[a]
        self._free = list(range(len(live), len(self._holders)))
        return len(move)

    def _outside_capture(self) -> None:
        if self.kv.k.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the books of a cache do not change in a captured graph: grow and "
                               "compact outside of it, and capture the calls on their tables")

    def _of(self, seq: int) -> _Sequence:
        if seq not in self._sequences:
            raise ValueError(f"no sequence {seq}")
        return self._sequences[seq]

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._holders[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._holders[page] -= 1
        if not self._holders[page]:
            heapq.heappush(self._free, page)

    def _step(self, held, new) -> Step:
        width, lens = max(1, max(len(s.pages) for s in held)), len(held)
        rows = lens * width
        tail = array("i", (s.length for s in held))
        tail.append(0)
        for n in new:
            tail.append(tail[-1] + n)
        # One copy to the device for all three, from pinned memory of its own:
        # the host goes on, and the allocator keeps the memory until the copy
        # is done.
        device = self.kv.k.device
        flat = torch.full((rows + 2 * lens + 1,), -1, dtype=torch.int32, pin_memory=device.type == "cuda")
        for at, part in [(i * width, s.pages) for i, s in enumerate(held)] + [(rows, tail)]:
            address, count = part.buffer_info()
            ctypes.memmove(flat.data_ptr() + 4 * at, address, 4 * count)
        flat = flat.to(device, non_blocking=True)
        return Step(flat[:rows].view(lens, width), flat[rows:rows + lens], flat[rows + lens:])
