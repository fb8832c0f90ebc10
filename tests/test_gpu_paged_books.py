"""The books of a paged cache on the GPU: steps that run ahead of the device."""

import pytest
import torch

from moba import paged as P
from moba.config import MoBAConfig

pytestmark = pytest.mark.gpu

CFG = MoBAConfig(block_size=16, top_k=3)


def test_growing_does_not_wait_for_the_device(device):
    """Steps taken while the stream has work for a while, forks that are copied
    among them: the host is through before the work is, and every step has the
    tables of its own time."""
    cache = P.PagedCache(2, 4000, 1, 64, CFG)
    ids = [cache.create() for _ in range(20)]
    cache.grow(ids, [1000 + 7 * i for i in range(20)])
    x = torch.randn(8192, 8192, device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    for _ in range(200):  # about 1 ms each
        x @ x
    done = torch.cuda.Event()
    done.record()
    steps, want = [], []
    for i in range(8):
        if i == 4:
            ids[:3] = [cache.fork(s) for s in ids[:3]]
        steps.append(cache.grow(ids, [i + 1] * 20))
        want.append(([cache.pages(s) for s in ids], [cache.length(s) for s in ids]))
    assert not done.query()
    torch.cuda.synchronize()
    for i, (step, (pages, lengths)) in enumerate(zip(steps, want)):
        width = max(map(len, pages))
        assert step.block_table.tolist() == [p + [-1] * (width - len(p)) for p in pages]
        assert step.seq_lens.tolist() == lengths
        assert step.cu_seqlens.tolist() == [j * (i + 1) for j in range(21)]


def test_books_do_not_change_in_a_captured_graph(device):
    cache = P.PagedCache(1, 10, 1, 64, CFG)
    a, b = cache.create(), cache.create()
    cache.grow([a, b], [20, 20])
    cache.free(a)
    before = cache.pages(b), cache.length(b), cache.free_pages
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x += 1
        for change in (lambda: cache.grow([b], [1]), cache.compact):
            with pytest.raises(RuntimeError, match="captured"):
                change()
    assert before == (cache.pages(b), cache.length(b), cache.free_pages)
