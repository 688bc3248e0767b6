"""Checks of the paged cache's host side that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from cuda_b200 import _lib, paged


def test_tangents_are_refused():
    x, plain = torch.ones(3), torch.zeros(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        paged.no_grad_needed(plain)
        with pytest.raises(ValueError, match="tangent"):
            paged.no_grad_needed(plain, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            paged.no_grad_needed(dual)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda v: paged.no_grad_needed(v) or v, (x,), (torch.ones(3),))
    paged.no_grad_needed(x)


def test_scratch_of_no_book_is_nothing():
    """A size has no error: 0 for books that every call refuses, a null pointer among them."""
    book = _lib.PageBook(table=16, lengths=16, refs=16, free_pages=16, height=16, slots=4, columns=4, pages=8, page=16)
    scratch = _lib.load().cb_pages_scratch
    assert scratch(ctypes.byref(book), 4) == 4 * (4 + 24) and scratch(None, 1) == 0
    assert scratch(ctypes.byref(book), 5) == 0 and scratch(ctypes.byref(book), -1) == 0
    for name, value in (("pages", 0), ("pages", 2 ** 31), ("slots", 2 ** 30), ("table", None)):
        bad = _lib.PageBook.from_buffer_copy(book)
        setattr(bad, name, value)
        assert scratch(ctypes.byref(bad), 0) == 0


@pytest.mark.parametrize("change", [dict(slots=16, columns=2 ** 27 - 100), dict(pages=2 ** 31 - 1024)])
def test_tables_whose_rounded_entries_pass_32_bits(change):
    book = _lib.PageBook(table=16, lengths=16, refs=16, free_pages=16, height=16, slots=4, columns=4, pages=8, page=16)
    for name, value in change.items():
        setattr(book, name, value)
    assert _lib.load().cb_pages_scratch(ctypes.byref(book), 1) == 0
    book.slots, book.pages = min(book.slots, 8), min(book.pages, 2 ** 30)
    assert _lib.load().cb_pages_scratch(ctypes.byref(book), 1) > 0
