"""What the rotation and paged-cache calls make of their arguments on the host."""

import pytest
import torch

from moba import _lib
from moba import paged as P
from moba.config import MoBAConfig
from moba.kernels.paged import PagedKV, copy_pages

BF = torch.bfloat16


@pytest.mark.parametrize("dtype,piece", [(BF, 8), (torch.float32, 4)])
def test_strides_of_axes_of_size_one(dtype, piece):
    """Rows of a width that is no multiple of 16 bytes: one of them, or one head,
    is read where it lies, at strides that the library takes."""
    wide = torch.arange(3 * 1004 * 2).to(dtype)[:3 * 1006].view(3, 1006)
    for t in (wide[:1, :512].unflatten(1, (4, 128)), wide[0, :512].view(1, 1, 4, 128),
              wide[None, :1, :512].unflatten(2, (4, 128)), torch.zeros(2, 64 * 5, dtype=dtype)[:, None, 64:128]):
        rows = _lib.aligned_rows(t)
        assert rows.data_ptr() == t.data_ptr()
        strides = _lib.row_strides(rows)
        assert len(strides) == t.ndim - 1 and all(s % piece == 0 for s in strides)
        assert torch.equal(torch.as_strided(rows, t.shape, [*strides, 1]), t)
    # Unaligned, or several rows: copied, and read as the copy lies.
    for t in (wide[1:2, 1:513].unflatten(1, (4, 128)), wide[:, :512].unflatten(1, (4, 128)),
              wide[:2, None, 5:69], wide[2:, 3:67].view(1, 1, 1, 64)):
        rows = _lib.aligned_rows(t)
        assert rows.data_ptr() % 16 == 0
        strides = _lib.row_strides(rows)
        assert all(s % piece == 0 for s in strides)
        assert torch.equal(torch.as_strided(rows, t.shape, [*strides, 1], rows.storage_offset()), t)


def test_a_failed_copy_changes_no_books():
    """Page copies need a GPU: `grow` of a forked sequence fails here, and the
    books stay as they were."""
    c = P.PagedCache(2, 12, 2, 64, MoBAConfig(block_size=16, top_k=3), device="cpu")
    a = c.create()
    c.grow([a], [20])
    b = c.fork(a)
    before = (c.pages(a), c.pages(b), c.length(a), c.length(b), list(c._holders), sorted(c._free))
    with pytest.raises(RuntimeError, match="GPU tensors"):
        c.grow([a, b], [1, 40])
    assert before == (c.pages(a), c.pages(b), c.length(a), c.length(b), list(c._holders), sorted(c._free))
    c.free(b)
    assert c.grow([a], [1]).block_table.tolist() == [[0, 1]]


@pytest.mark.parametrize("src,dst", [([0.7], [1]), ([0], [1.9]), ([0], ["1"]), ([0], [None]),
                                     ([2 ** 31], [1]), ([0], [-2 ** 40]), ([[0]], [[1]])])
def test_page_lists_of_no_pages(src, dst):
    with pytest.raises(ValueError, match="must be a list of pages"):
        copy_pages(PagedKV.empty(4, 1, 16, 64, BF, "cpu"), src, dst)
