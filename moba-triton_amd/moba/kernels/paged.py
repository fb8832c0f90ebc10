"""MoBA over a paged cache: new tokens appended, attended over, pages copied.

A page holds one MoBA block of a layer: K and V [pages, H_kv, block_size, D]
(a block of a head is one contiguous run) and the blocks' representatives
[pages, H_kv, D], which the gate reads. A sequence is a row of the block table
(its pages in order) and a length; the new tokens of all sequences are packed
along one token axis. `moba.paged.PagedCache` keeps the books. No counterpart
in the reference, which has no cache.

Values on the device (block table, lengths, cu_seqlens) are checked by the
kernels, which treat what makes no sense as absent (see `append_tokens`).
"""

import ctypes
from dataclasses import dataclass
from operator import index

import torch

from moba import _lib
from moba.config import MoBAConfig
from moba.device import TENSOR_CORE_TILE
from moba.gqa import head_group_size
from moba.kernels.rotary import check_tables, check_weights

HEAD_DIMS = (64, 128, 256)
MAX_BLOCK = 1024
MAX_TAKE = 32  # past blocks per query
MAX_BLOCKS = 1 << 16  # per sequence
_Strides = ctypes.c_int64 * 6


@dataclass(frozen=True)
class PagedKV:
    """A cache's pages, of one layer or (one more leading axis) of several.

    Attributes:
        k, v: [(layers,) pages, H_kv, block_size, D].
        kbar: [(layers,) pages, H_kv, D], valid for full blocks.
    """

    k: torch.Tensor
    v: torch.Tensor
    kbar: torch.Tensor

    def __post_init__(self) -> None:
        k, v, kbar = self.k, self.v, self.kbar
        shape = k.shape
        if len(shape) not in (4, 5) or v.shape != shape:
            raise ValueError(f"pages must be [(layers,) pages, H_kv, block, D], got "
                             f"{tuple(shape)}, {tuple(v.shape)}")
        if kbar.shape != shape[:-2] + shape[-1:]:
            raise ValueError(f"kbar shape {tuple(kbar.shape)} does not match pages "
                             f"{tuple(shape)}")
        if k.dtype is not v.dtype or k.dtype is not kbar.dtype:
            raise ValueError(f"dtype mismatch: {k.dtype}, {v.dtype}, {kbar.dtype}")
        if k.dtype not in _lib.DTYPE_CODE:
            raise ValueError(f"unsupported dtype {k.dtype}")
        if 0 in shape:
            raise ValueError(f"empty cache: {tuple(shape)}")
        if shape[-1] not in HEAD_DIMS:
            raise ValueError(f"paged caches take head_dim {HEAD_DIMS}, got {shape[-1]}")
        if not TENSOR_CORE_TILE <= shape[-2] <= MAX_BLOCK:
            raise ValueError(f"block_size {shape[-2]} must be from {TENSOR_CORE_TILE} to "
                             f"{MAX_BLOCK}")
        for t in (k, v, kbar):
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("pages must be contiguous and 16-byte aligned")

    @classmethod
    def empty(cls, pages: int, h_kv: int, block_size: int, head_dim: int, dtype=torch.bfloat16,
              device="cuda", layers: int | None = None) -> "PagedKV":
        """Uninitialised pages."""
        lead = (pages,) if layers is None else (layers, pages)
        k = torch.empty((*lead, h_kv, block_size, head_dim), dtype=dtype, device=device)
        kbar = torch.empty((*lead, h_kv, head_dim), dtype=dtype, device=device)
        return cls(k, torch.empty_like(k), kbar)

    def layer(self, i: int) -> "PagedKV":
        """One layer's pages (a view)."""
        if self.k.ndim != 5:
            raise ValueError("these pages are one layer's")
        return PagedKV(self.k[i], self.v[i], self.kbar[i])


def _call(q, cache: PagedKV, block_table, seq_lens, cu_seqlens) -> _lib.Paged:
    """The checked call on one layer's pages, without its stage's pointers
    (the device is the caller's to check)."""
    shape, qs = cache.k.shape, q.shape
    if len(shape) != 4:
        raise ValueError("one layer's pages are needed: use PagedKV.layer")
    pages, h_kv, block, d = shape
    if len(qs) != 3 or qs[2] != d:
        raise ValueError(f"queries must be [tokens, H_q, {d}], got {tuple(qs)}")
    if q.dtype is not cache.k.dtype:
        raise ValueError(f"dtype mismatch: {q.dtype}, cache {cache.k.dtype}")
    tokens, h_q, _ = qs
    head_group_size(h_q, h_kv)
    ts, ls = block_table.shape, seq_lens.shape
    if len(ts) != 2 or len(ls) != 1 or 0 in ts or ls[0] != ts[0]:
        raise ValueError(f"block_table must be [sequences, blocks] and seq_lens [sequences], got "
                         f"{tuple(ts)}, {tuple(ls)}")
    seqs, width = ts
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens), ("cu_seqlens", cu_seqlens)):
        if t is not None and (t.dtype is not torch.int32 or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous int32")
    if cu_seqlens is None:
        if tokens % seqs:
            raise ValueError(f"{tokens} tokens do not divide over {seqs} sequences: "
                             "cu_seqlens is needed")
        even, cu = tokens // seqs, None
    elif cu_seqlens.shape != (seqs + 1,):
        raise ValueError(f"cu_seqlens must be [{seqs + 1}], got {tuple(cu_seqlens.shape)}")
    else:
        even, cu = 0, cu_seqlens.data_ptr()
    return _lib.Paged(tokens, seqs, h_q, h_kv, d, block, width, pages, _lib.DTYPE_CODE[q.dtype],
                      even, 0, 0, 0, 0, None, cache.k.data_ptr(), cache.v.data_ptr(),
                      cache.kbar.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), cu)


def _output(out, q):
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype is not q.dtype or out.device != q.device:
        raise ValueError(f"out must be {tuple(q.shape)} {q.dtype} on {q.device}")
    if not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous and 16-byte aligned")
    return out


def append_tokens(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedKV,
                  block_table: torch.Tensor, seq_lens: torch.Tensor,
                  cu_seqlens: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                  sin: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                  k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                  interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """New tokens into the cache: keys normed and rotated (as `norm_rotate`, by
    their positions in their sequences), values as they are, and the
    representatives of blocks that became full, rounded as `pool_blocks` does.

    Args:
        q: [T, H_q, D]; k, v: [T, H_kv, D], any strides.
        cache: One layer's pages.
        block_table: int32 [sequences, blocks], the pages of each sequence. An
            entry outside the cache is no page: tokens there are dropped.
        seq_lens: int32 [sequences], tokens of each sequence with its new ones.
        cu_seqlens: int32 [sequences + 1], where each sequence's new tokens
            begin on the token axis (a sequence may have none); None: the same
            number for each. Tokens behind the last sequence are not read.
            A sequence whose numbers make no sense (outside the token axis,
            falling, more new tokens than `seq_lens`), or that begins before
            an earlier one's end, has no new tokens; the others are served.
        cos, sin, q_weight, k_weight, eps, interleaved: As `norm_rotate`.
        out: Receives the queries; rows of no sequence stay as they are (and
            hold anything without it).

    No gradients (`norm_rotate` has them).

    Returns:
        The normed and rotated queries [T, H_q, D] (`out`).

    A page that is appended to must belong to one sequence only
    (`moba.paged.PagedCache` sees to it).

    Raises:
        ValueError: On mismatched shapes, dtypes, tables or weights.
    """
    if k.ndim != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or \
            k.shape[1] != cache.k.shape[-3] or k.shape[2] != cache.k.shape[-1]:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, v "
                         f"{tuple(v.shape)}, pages {tuple(cache.k.shape)}")
    if q.dtype is not k.dtype or q.dtype is not v.dtype:
        raise ValueError(f"dtype mismatch: {q.dtype}, {k.dtype}, {v.dtype}")
    call = _call(q, cache, block_table, seq_lens, cu_seqlens)
    code = check_weights(q, q_weight, k_weight)
    rotary = check_tables(cos, sin, q.shape[2])
    dev = _lib.require_gpu(q, k, v, cache.k, cache.v, cache.kbar, block_table, seq_lens, cu_seqlens,
                           cos, sin, q_weight, k_weight)
    out = _output(out, q)
    if q.shape[0] == 0:
        return out
    q, k, v = _lib.aligned_rows(q), _lib.aligned_rows(k), _lib.aligned_rows(v)
    length = 0
    if rotary:
        cos, sin = _lib.aligned_contiguous(cos), _lib.aligned_contiguous(sin)
        length = cos.shape[0]
    if q_weight is not None:
        q_weight = q_weight.contiguous()
    if k_weight is not None:
        k_weight = k_weight.contiguous()
    call.q = q.data_ptr()
    strides = _Strides(*_lib.row_strides(q), *_lib.row_strides(k), *_lib.row_strides(v))
    a = _lib.addr
    _lib.call_on(dev, "moba_append_tokens", ctypes.byref(call), k.data_ptr(), v.data_ptr(), strides,
                 out.data_ptr(), a(cos), a(sin), a(q_weight), a(k_weight), rotary, length,
                 bool(interleaved), float(eps), code)
    return out


def _attention_call(q, cache, block_table, seq_lens, cu_seqlens, cfg: MoBAConfig):
    call = _call(q, cache, block_table, seq_lens, cu_seqlens)
    if cfg.block_size != cache.k.shape[2]:
        raise ValueError(f"block_size {cfg.block_size} does not match the pages' "
                         f"{cache.k.shape[2]}")
    if cfg.gate_group > 0:
        raise ValueError("the hierarchical gate (gate_group > 0) takes no paged cache")
    if call.table_width > MAX_BLOCKS:
        raise ValueError(f"block_table has {call.table_width} blocks per sequence, at most {MAX_BLOCKS}")
    call.take = cfg.past_blocks_selected(call.table_width)
    if call.take > MAX_TAKE:
        raise ValueError(f"top_k {cfg.top_k}: at most {MAX_TAKE} past blocks per query")
    # Slots beyond the table's blocks would only hold padding.
    call.slots = max(1, call.take + int(bool(cfg.always_select_current)))
    call.always_current = int(bool(cfg.always_select_current))
    return _lib.require_gpu(q, cache.k, cache.v, cache.kbar, block_table, seq_lens, cu_seqlens), call


def _run(name, dev, call, q, block_idx, out, lse):
    q = _lib.aligned_contiguous(q)
    call.q = q.data_ptr()
    call.block_idx = None if block_idx is None else block_idx.data_ptr()
    call.out = None if out is None else out.data_ptr()
    call.lse = None if lse is None else lse.data_ptr()
    _lib.call("moba_paged_layout", ctypes.byref(call))
    workspace = torch.empty(call.workspace_bytes, device=dev, dtype=torch.uint8)
    call.workspace = workspace.data_ptr()
    _lib.call_on(dev, name, ctypes.byref(call))


def paged_gate_select(q: torch.Tensor, cache: PagedKV, block_table: torch.Tensor,
                      seq_lens: torch.Tensor, cfg: MoBAConfig,
                      cu_seqlens: torch.Tensor | None = None) -> torch.Tensor:
    """Block ids each new token's query heads attend to, by the rules of
    `gate_select`: of each sequence's blocks before the token's own, the best
    by q . kbar, and the own block. Arguments as `paged_attention`.

    Returns:
        int32 [T, H_q, slots], ids within the sequence, ascending, -1 padded
        (all -1 for rows of no sequence); slots is `cfg.slots()`, or fewer
        where the table has fewer blocks.
    """
    dev, call = _attention_call(q, cache, block_table, seq_lens, cu_seqlens, cfg)
    ids = torch.empty((q.shape[0], q.shape[1], call.slots), dtype=torch.int32, device=dev)
    if q.shape[0]:
        _run("moba_paged_gate", dev, call, q, ids, None, None)
    return ids


def paged_attention(q: torch.Tensor, cache: PagedKV, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, cfg: MoBAConfig,
                    cu_seqlens: torch.Tensor | None = None,
                    block_idx: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    return_lse: bool = False):
    """MoBA attention of new tokens over a cache that already holds them
    (`append_tokens`): a chunk of each prompt, or the one token of a decoding
    step. The result is `moba_attention`'s for the same tokens but for
    roundings. A call's sizes decide how its tokens are computed: by float32
    alone, or, in 16-bit chunks, with weights of 16 (bf16) or 22 (float16)
    bits in the product and float32 sums; the same token in a chunk and by
    itself may differ by a step of its type.

    Args:
        q: [T, H_q, D], normed and rotated.
        cache: One layer's pages, block_size `cfg.block_size`.
        block_table, seq_lens, cu_seqlens: As `append_tokens`; pages may be
            shared. Blocks without a page hold no keys and are never selected.
        block_idx: The blocks of `paged_gate_select`, to attend to instead of
            the gate's choice: int32 [T, H_q, slots], no id twice in a row.
        out: Receives the result; rows of no sequence stay as they are (and
            hold anything without it, as their lse does).

    No gradients: the cache's tokens are constants here.

    Returns:
        out [T, H_q, D], plus lse [H_q, T] float32 in log2 units when
        `return_lse` (-inf where a query sees no key; its out is 0).

    Raises:
        ValueError: On mismatched shapes, dtypes or configuration.
    """
    if block_idx is not None and (
            block_idx.ndim != 3 or block_idx.shape[:2] != q.shape[:2] or block_idx.shape[2] == 0 or
            block_idx.dtype != torch.int32):
        raise ValueError(f"block_idx must be int32 [tokens, H_q, slots] for {tuple(q.shape)}, got "
                         f"{block_idx.dtype} {tuple(block_idx.shape)}")
    dev, call = _attention_call(q, cache, block_table, seq_lens, cu_seqlens, cfg)
    out = _output(out, q)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=dev) \
        if return_lse else None
    name = "moba_paged_attention"
    if block_idx is not None:
        _lib.require_gpu(q, block_idx)
        block_idx = block_idx.contiguous()
        call.slots, call.take = block_idx.shape[2], 0
        name = "moba_paged_attend"
    if q.shape[0]:
        _run(name, dev, call, q, block_idx, out, lse)
    return (out, lse) if return_lse else out


def _page_list(pages, name):
    t = pages
    if not isinstance(t, torch.Tensor):
        try:
            t = torch.tensor([index(p) for p in pages], dtype=torch.int32)
        except (TypeError, RuntimeError) as exc:  # no whole numbers, or past 32 bits
            raise ValueError(f"{name} must be a list of pages: {exc}") from None
    if t.ndim != 1 or t.dtype != torch.int32:
        raise ValueError(f"{name} must be a list of pages (int32, one axis)")
    return t.contiguous()


def copy_pages(cache: PagedKV, src, dst) -> None:
    """Pages `src[i]` copied to `dst[i]` in all layers, with their
    representatives: making shared pages a sequence's own, compaction.

    Args:
        cache: Pages of one layer or of all.
        src, dst: Lists, or int32 tensors on the host or the cache's device.
            Destinations distinct, and no page both source and destination;
            one source may have several destinations. Pairs outside the cache
            are skipped where the lists are on the device.

    Raises:
        ValueError: On lists of different lengths and, on the host, on any
            violation of the above or a page outside the cache.
    """
    src, dst = _page_list(src, "src"), _page_list(dst, "dst")
    if src.shape != dst.shape or src.device != dst.device:
        raise ValueError(f"src and dst differ: {tuple(src.shape)} on {src.device}, "
                         f"{tuple(dst.shape)} on {dst.device}")
    host = src.device.type == "cpu"
    pages = cache.k.shape[-4]
    if host:
        s, d = src.tolist(), dst.tolist()
        if any(not 0 <= p < pages for p in s + d):
            raise ValueError(f"pages outside the cache's {pages}")
        if len(set(d)) != len(d):
            raise ValueError("a page is the destination twice")
        if set(s) & set(d):
            raise ValueError("a page is source and destination")
    dev = _lib.require_gpu(cache.k, cache.v, cache.kbar, None if host else src)
    if src.numel() == 0:
        return
    layers = cache.k.shape[0] if cache.k.ndim == 5 else 1
    _, h_kv, block, d = cache.k.shape[-4:]
    _lib.call_on(dev, "moba_copy_pages", *map(_lib.addr, (cache.k, cache.v, cache.kbar, src, dst)),
                 src.numel(), host, layers, pages, h_kv, block, d, _lib.DTYPE_CODE[cache.k.dtype])
