"""Refusals of the paged-cache and rotation calls, and the cache's books, on
the CPU. Every check of values and shapes comes before any GPU work."""

import ctypes
from collections import Counter

import pytest
import torch

from moba import _lib
from moba import paged as P
from moba.config import MoBAConfig
from moba.kernels.paged import (PagedKV, append_tokens, copy_pages, paged_attention,
                                paged_gate_select)
from moba.kernels.rotary import norm_rotate

BF = torch.bfloat16
CFG = MoBAConfig(block_size=16, top_k=3)


def cache(pages=4, h_kv=2, block=16, d=64, dtype=BF, layers=None):
    return PagedKV.empty(pages, h_kv, block, d, dtype, "cpu", layers)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


# -- norm_rotate --------------------------------------------------------------

def qk(h=4, hk=2, d=64, dtype=BF, s=5):
    return torch.zeros(2, s, h, d, dtype=dtype), torch.zeros(2, s, hk, d, dtype=dtype)


TABLE = torch.zeros(8, 32)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(2, 4, 4, 64, dtype=BF)), "shape mismatch"),
    (dict(k=torch.zeros(2, 5, 2, 128, dtype=BF)), "shape mismatch"),
    (dict(k=torch.zeros(2, 5, 2, 64)), "dtype mismatch"),
    (dict(q=torch.zeros(2, 5, 4, 64, dtype=torch.float64),
          k=torch.zeros(2, 5, 2, 64, dtype=torch.float64)), "unsupported dtype"),
    (dict(q=torch.zeros(2, 5, 4, 96, dtype=BF), k=torch.zeros(2, 5, 2, 96, dtype=BF)), "power of two"),
    (dict(q=torch.zeros(2, 5, 4, 32, dtype=BF), k=torch.zeros(2, 5, 2, 32, dtype=BF)), "cache line"),
    (dict(q=torch.zeros(2, 5, 4, 2048, dtype=BF), k=torch.zeros(2, 5, 2, 2048, dtype=BF)), "above 1024"),
    (dict(sin=None), "go together"),
    (dict(sin=torch.zeros(8, 16)), "cos / sin"),
    (dict(cos=torch.zeros(8, 32, dtype=BF), sin=torch.zeros(8, 32, dtype=BF)), "float32"),
    (dict(cos=torch.zeros(8, 12), sin=torch.zeros(8, 12)), "multiple of 16"),
    (dict(cos=torch.zeros(8, 40), sin=torch.zeros(8, 40)), "multiple of 16"),
    (dict(cos=torch.zeros(4, 32), sin=torch.zeros(4, 32)), "cover 4 positions"),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int32)), "positions shape"),
    (dict(positions=torch.zeros(2, 5)), "positions must be"),
    (dict(q_weight=torch.ones(32)), "weight shape"),
    (dict(k_weight=torch.ones(64, dtype=torch.float16)), "weight dtype"),
    (dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=BF)), "dtypes differ"),
])
def test_norm_rotate_refusals(change, match):
    q, k = qk()
    args = dict(q=q, k=k, cos=TABLE, sin=TABLE)
    with pytest.raises(ValueError, match=match):
        norm_rotate(**{**args, **change})


def test_norm_rotate_needs_a_gpu():
    with pytest.raises(RuntimeError, match="GPU tensors"):
        norm_rotate(*qk(), TABLE, TABLE)


# -- pages ----------------------------------------------------------------------

@pytest.mark.parametrize("make,match", [
    (lambda: PagedKV(torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 128), torch.zeros(4, 2, 64)), "pages must be"),
    (lambda: PagedKV(*(torch.zeros(4, 2, 16, 64),) * 2, torch.zeros(4, 64)), "kbar shape"),
    (lambda: PagedKV(*(torch.zeros(4, 2, 16, 64),) * 2, torch.zeros(4, 2, 64, dtype=BF)), "dtype mismatch"),
    (lambda: cache(d=96), "head_dim"),
    (lambda: cache(block=8), "block_size"),
    (lambda: cache(block=1040), "block_size"),
    (lambda: cache(pages=0), "empty cache"),
    (lambda: cache(dtype=torch.float64), "unsupported dtype"),
    (lambda: PagedKV(*(torch.zeros(4, 16, 2, 64).transpose(1, 2),) * 2, torch.zeros(4, 2, 64)), "contiguous"),
    (lambda: cache().layer(0), "one layer"),
])
def test_cache_refusals(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def attention(q=None, kv=None, table=None, lens=None, cfg=CFG, **more):
    q = torch.zeros(3, 4, 64, dtype=BF) if q is None else q
    table = torch.zeros(3, 2, dtype=torch.int32) if table is None else table
    return paged_attention(q, kv or cache(), table, i32(1, 1, 1) if lens is None else lens, cfg, **more)


@pytest.mark.parametrize("change,match", [
    (dict(kv=cache(layers=2)), "PagedKV.layer"),
    (dict(q=torch.zeros(3, 4, 128, dtype=BF)), "queries must be"),
    (dict(q=torch.zeros(3, 256, dtype=BF)), "queries must be"),
    (dict(q=torch.zeros(3, 4, 64)), "dtype mismatch"),
    (dict(q=torch.zeros(3, 3, 64, dtype=BF)), "divisible"),
    (dict(q=torch.zeros(4, 4, 64, dtype=BF)), "do not divide"),
    (dict(lens=i32(1, 1)), "block_table must be"),
    (dict(table=torch.zeros(3, 0, dtype=torch.int32)), "block_table must be"),
    (dict(table=torch.zeros(3, 2, dtype=torch.int64)), "block_table must be contiguous int32"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int32).t()), "block_table must be contiguous int32"),
    (dict(lens=torch.ones(3, dtype=torch.int64)), "seq_lens must be"),
    (dict(cu_seqlens=i32(0, 1, 2)), "cu_seqlens must be"),
    (dict(cfg=MoBAConfig(block_size=32, top_k=3)), "does not match the pages"),
    (dict(cfg=MoBAConfig(block_size=16, top_k=3, gate_group=2, gate_open=1)), "hierarchical"),
    (dict(cfg=MoBAConfig(block_size=16, top_k=40), table=torch.zeros(3, 64, dtype=torch.int32)), "at most 32"),
    (dict(block_idx=torch.zeros(3, 4, dtype=torch.int32)), "block_idx must be"),
])
def test_attention_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        attention(**change)


def test_append_refusals():
    q, k = torch.zeros(3, 4, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), i32(1, 1, 1)
    for bad, match in (((q, k[:2], k[:2]), "shape mismatch"), ((q, k, k[..., :32]), "shape mismatch"),
                       ((q, k, k.float()), "dtype mismatch"), ((q, k[:, :1], k[:, :1]), "shape mismatch")):
        with pytest.raises(ValueError, match=match):
            append_tokens(*bad, cache(), table, lens)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        append_tokens(q, k, k, cache(), table, lens)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        paged_gate_select(q, cache(), table, lens, CFG)


@pytest.mark.parametrize("src,dst,match", [
    ([0], [1, 2], "differ"), ([0, 1], [2, 2], "destination twice"), ([0, 1], [1, 2], "source and destination"),
    ([4], [0], "outside"), ([0], [-1], "outside"),
    (torch.tensor([0]), torch.tensor([1]), "int32"), (i32(0, 1)[None], i32(2, 3)[None], "int32, one axis"),
])
def test_copy_refusals(src, dst, match):
    with pytest.raises(ValueError, match=match):
        copy_pages(cache(), src, dst)


def test_library_refuses_bad_calls_on_the_host():
    lib = _lib.load()

    def rc(text, name="moba_paged_layout", **change):
        call = _lib.Paged(4, 4, 4, 2, 64, 16, 2, 8, 0, 1, 3, 2, 1)
        call.block_table = call.seq_lens = 16  # addresses that are not followed
        for key, value in change.items():
            setattr(call, key, value)
        got = getattr(lib, name)(ctypes.byref(call), *([None] if name != "moba_paged_layout" else []))
        assert got != _lib.MOBA_OK and text in lib.moba_last_error()
        return got

    assert rc(b"non-positive", tokens=0) == _lib.MOBA_ERR_INVALID
    assert rc(b"divisible", h_q=3) == _lib.MOBA_ERR_INVALID
    assert rc(b"head_dim", head_dim=96) == _lib.MOBA_ERR_UNSUPPORTED
    assert rc(b"block_size", block_size=2000) == _lib.MOBA_ERR_UNSUPPORTED
    assert rc(b"2^31", n_pages=1 << 31) == _lib.MOBA_ERR_UNSUPPORTED
    assert rc(b"2^31", table_width=1 << 30) == _lib.MOBA_ERR_UNSUPPORTED
    assert rc(b"dtype", dtype=7) == _lib.MOBA_ERR_UNSUPPORTED
    assert rc(b"same number", even=2) == _lib.MOBA_ERR_INVALID
    assert rc(b"slots", take=3) == _lib.MOBA_ERR_INVALID
    assert rc(b"past blocks", take=33, slots=40) == _lib.MOBA_ERR_UNSUPPORTED
    assert rc(b"65536 blocks", table_width=65537) == _lib.MOBA_ERR_UNSUPPORTED
    assert rc(b"null", block_table=None) == _lib.MOBA_ERR_INVALID
    assert rc(b"null", "moba_paged_attention") == _lib.MOBA_ERR_INVALID
    assert rc(b"unaligned", "moba_paged_gate", q=24, kbar=16, block_idx=16) == _lib.MOBA_ERR_INVALID
    assert rc(b"workspace", "moba_paged_gate", q=16, kbar=16, block_idx=16) == _lib.MOBA_ERR_WORKSPACE
    with pytest.raises(ValueError, match="null"):
        _lib.call("moba_copy_pages", None, None, None, None, None, 1, 1, 1, 4, 2, 16, 64, 0, None)
    with pytest.raises(ValueError, match="multiple of 16"):
        _lib.call("moba_norm_rotate", *[16] * 9, 1, 1, 1, 1, 64, (ctypes.c_int64 * 6)(), 24, 8, 0,
                  1e-6, 0, 2, None)
    with pytest.raises(ValueError, match="16-byte"):
        _lib.call("moba_norm_rotate", *[24] * 4, *[16] * 5, 1, 1, 1, 1, 64, (ctypes.c_int64 * 6)(),
                  32, 8, 0, 1e-6, 0, 2, None)


# -- the books ------------------------------------------------------------------

@pytest.fixture
def books(monkeypatch):
    """A cache on the CPU whose page copies are torch's, one tensor per pair."""
    log = []

    def copy(kv, src, dst):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        log.append((list(src), list(dst)))
        for t in (kv.k, kv.v, kv.kbar):
            t[:, dst] = t[:, src]

    monkeypatch.setattr(P, "copy_pages", copy)
    c = P.PagedCache(2, 12, 2, 64, CFG, device="cpu")
    c.log = log
    for t in (c.kv.k, c.kv.v, c.kv.kbar):
        t.zero_()
    return c


def consistent(c):
    """Holders of every page are those that list it; the others are free."""
    held = Counter(p for s in c._sequences.values() for p in s.pages)
    assert [held.get(p, 0) for p in range(len(c._holders))] == c._holders
    assert sorted(c._free) == [p for p, n in enumerate(c._holders) if not n]
    for s in c._sequences.values():
        assert len(s.pages) == -(-s.length // c.block_size) and len(set(s.pages)) == len(s.pages)


def test_growing_sequences(books):
    a, b = books.create(), books.create()
    step = books.grow([a, b], [17, 0])
    assert step.block_table.tolist() == [[0, 1], [-1, -1]]
    assert step.seq_lens.tolist() == [17, 0] and step.cu_seqlens.tolist() == [0, 17, 17]
    assert all(t.dtype == torch.int32 and t.is_contiguous() for t in step.args)
    step = books.grow([b, a], [16, 15])
    assert step.block_table.tolist() == [[2, -1], [0, 1]] and step.seq_lens.tolist() == [16, 32]
    consistent(books)
    assert books.free_pages == 9 and books.length(a) == 32 and books.pages(a) == [0, 1]


def test_fork_copies_the_shared_part_filled_page_once(books):
    a = books.create()
    books.grow([a], [20])
    books.kv.k[:, 1] = 7
    b, c = books.fork(a), books.fork(a)
    consistent(books)
    step = books.grow([a, b, c], [1, 1, 1])
    # The last of the three that write keeps the page.
    assert books.log == [([1, 1], [2, 3])]
    assert step.block_table.tolist() == [[0, 2], [0, 3], [0, 1]]
    assert bool((books.kv.k[:, [2, 3]] == 7).all())
    consistent(books)
    # A holder that does not write leaves the page shared.
    d = books.fork(c)
    books.grow([c], [1])
    assert books.log[-1] == ([1], [4]) and books.pages(d) == [0, 1]
    consistent(books)
    # A full last page needs no copy.
    books.grow([d], [11])
    e = books.fork(d)
    n = len(books.log)
    books.grow([d, e], [1, 1])
    assert len(books.log) == n and books.pages(d)[:2] == books.pages(e)[:2]
    consistent(books)


def test_a_full_cache_changes_nothing(books):
    a = books.create()
    books.grow([a], [16 * 10 + 1])
    b = books.fork(a)
    before = (books.pages(a), books.pages(b), list(books._holders), sorted(books._free))
    with pytest.raises(P.CacheFull):
        books.grow([a, b], [16, 1])  # a copy and a page: two, with one free
    assert before == (books.pages(a), books.pages(b), list(books._holders), sorted(books._free))
    assert books.length(a) == 161 and not books.log


def test_freeing_and_compaction(books):
    a, b, c = (books.create() for _ in range(3))
    for s, n in ((a, 40), (b, 30), (c, 50)):
        books.grow([s], [n])
    d = books.fork(c)
    for p in range(12):
        books.kv.v[:, p] = p
    books.free(a)
    consistent(books)
    want = [books.kv.v[0, p, 0, 0, 0].item() for p in books.pages(c)]
    assert books.compact() == 3
    consistent(books)
    assert sorted(set(books.pages(b) + books.pages(c))) == list(range(6))
    assert books.pages(d) == books.pages(c)
    assert [books.kv.v[1, p, 0, 0, 0].item() for p in books.pages(c)] == want
    assert books.compact() == 0
    books.free(b)
    books.free(c)
    consistent(books)
    assert books.pages(d) and books.free_pages == 8
    books.free(d)
    assert books.free_pages == 12


def test_refusals_of_the_books(books):
    a = books.create()
    for seqs, new, match in (([a, a], [1, 1], "twice"), ([a], [-1], "negative"), ([a], [1, 1], "counts"),
                             ([], [], "counts"), ([9], [1], "no sequence")):
        with pytest.raises(ValueError, match=match):
            books.grow(seqs, new)
    books.free(a)
    with pytest.raises(ValueError, match="no sequence"):
        books.free(a)
