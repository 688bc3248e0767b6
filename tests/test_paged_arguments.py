"""The paged-cache entry points without a GPU: structure layout, refusals of the C
entries (each returns before any CUDA call) and of the Python argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

import test_abi
from cuda_b200 import _lib, paged, speculative


def test_structures_match_the_header(tmp_path, monkeypatch):
    monkeypatch.setattr(test_abi, "STRUCTS", {
        "cb_paged_cache": _lib.PagedCacheArgs, "cb_paged_append_args": _lib.PagedAppendArgs,
        "cb_paged_attention_args": _lib.PagedAttentionArgs, "cb_page_book": _lib.PageBook,
        "cb_page_pools": _lib.PagePools, "cb_verify_args": _lib.VerifyArgs})
    test_abi.test_ctypes_structures_match_the_header(tmp_path)


def cache(**changes):
    c = _lib.PagedCacheArgs(k_pages=16, v_pages=16, k_scale=16, v_scale=16, storage=_lib.I8, kv_heads=2, page=16,
                            head_size=64, pages=8, table=16, lengths=16, slots=2, columns=4)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def append(c, **changes):
    a = _lib.PagedAppendArgs(cache=c, k=16, v=16, dtype=_lib.F32, batch=1, tokens=1)
    for name, value in changes.items():
        setattr(a, name, value)
    return _lib.call("cb_paged_append", ctypes.byref(a), None)


def attend(c, **changes):
    a = _lib.PagedAttentionArgs(cache=c, q=16, out=16, dtype=_lib.F32, batch=1, tokens=1, heads=2, scale=1.0)
    for name, value in changes.items():
        setattr(a, name, value)
    return _lib.call("cb_paged_attention", ctypes.byref(a), 16, 16, None)


@pytest.mark.parametrize("change", [dict(storage=_lib.BF16), dict(head_size=48), dict(page=8), dict(page=24),
                                    dict(page=512), dict(kv_heads=0), dict(pages=0), dict(slots=0), dict(columns=0),
                                    dict(columns=2 ** 31 // 16), dict(k_pages=None), dict(lengths=None),
                                    dict(v_pages=8)])
def test_cache_refusals(change):
    for call in (append, attend):
        with pytest.raises(_lib.KernelError):
            call(cache(**change))


@pytest.mark.parametrize("call, change", [
    (append, dict(dtype=_lib.I32)), (append, dict(k=None)), (append, dict(batch=-1)), (append, dict(batch=65536)),
    (append, dict(tokens=-1)), (append, dict(tokens=2 ** 21)),
    (attend, dict(dtype=_lib.I64)), (attend, dict(heads=3)), (attend, dict(heads=0)), (attend, dict(out=None)),
    (attend, dict(batch=65536)), (attend, dict(tokens=-1))])
def test_call_refusals(call, change):
    with pytest.raises(_lib.KernelError):
        call(cache(), **change)


def test_empty_calls_do_nothing():
    append(cache(), batch=0)
    append(cache(), tokens=0, k=None)
    attend(cache(), batch=0)
    attend(cache(), tokens=0)


def test_page_operation_refusals():
    book = _lib.PageBook(table=16, lengths=16, refs=16, free_pages=16, height=16, slots=4, columns=4, pages=8, page=16)
    pools = _lib.PagePools(k_pages=16, v_pages=16, k_scale=16, v_scale=16, layers=1, pages=8, page_bytes=2048,
                           kv_heads=2)
    ref = ctypes.byref
    bad = [
        ("cb_pages_extend", ref(book), ref(pools), 16, None, 5, 16, None, None),  # more lists than slots
        ("cb_pages_extend", ref(book), ref(pools), None, None, 1, 16, None, None),
        ("cb_pages_extend", ref(book), ref(pools), 16, None, 1, None, None, None),
        ("cb_pages_fork", ref(book), None, 16, 1, None, None),
        ("cb_pages_fork", ref(book), 16, 16, -1, None, None),
        ("cb_pages_truncate", None, None, None, 1, None, None),
        ("cb_pages_compact", ref(book), ref(pools), None, None, None),
        ("cb_pages_copy", ref(pools), None, 16, 1, None, None),
        ("cb_pages_copy", ref(pools), 16, 16, -1, None, None),
    ]
    pools_of_another = _lib.PagePools.from_buffer_copy(pools)
    pools_of_another.pages = 9
    odd = _lib.PagePools.from_buffer_copy(pools)
    odd.page_bytes = 24
    bad += [("cb_pages_compact", ref(book), ref(pools_of_another), 16, None, None),
            ("cb_pages_compact", ref(book), ref(odd), 16, None, None)]
    for name, *args in bad:
        with pytest.raises(_lib.KernelError):
            _lib.call(name, *args)
    _lib.call("cb_pages_extend", ref(book), ref(pools), None, None, 0, None, None, None)
    assert _lib.load().cb_pages_scratch(ref(book), 4) >= 4 * 5 * 4


@pytest.mark.parametrize("change", [dict(dtype=_lib.I32), dict(vocab=0), dict(vocab=2 ** 22 + 1), dict(target=None),
                                    dict(uniforms=None), dict(drafted=None), dict(batch=-1), dict(tokens=-1)])
def test_verify_refusals(change):
    a = _lib.VerifyArgs(target=16, draft=16, dtype=_lib.F32, batch=1, tokens=1, vocab=8, drafted=16, uniforms=16,
                        accepted=16, out=16)
    for name, value in change.items():
        setattr(a, name, value)
    with pytest.raises(_lib.KernelError):
        _lib.call("cb_verify_draft", ctypes.byref(a), None)


def test_python_checks():
    cpu = torch.device("cpu")
    x = torch.zeros(2, 3, 4)
    paged.require(x, "x", cpu, (torch.float32,), (2, None, 4), 1)
    with pytest.raises(TypeError):
        paged.require(x, "x", cpu, (torch.float16,), (2, 3, 4), 1)
    with pytest.raises(ValueError):
        paged.require(x, "x", cpu, (torch.float32,), (2, 4, 4), 1)
    with pytest.raises(ValueError):
        paged.require(x, "x", torch.device("cuda", 0), (torch.float32,), (2, 3, 4), 1)
    with pytest.raises(ValueError):
        paged.require(x.transpose(1, 2), "x", cpu, (torch.float32,), (2, 4, 3), 1)
    with pytest.raises(ValueError):
        paged.no_grad_needed(x, x.clone().requires_grad_())
    with torch.no_grad():
        paged.no_grad_needed(x.clone().requires_grad_())
    with pytest.raises(TypeError):
        paged.tensor_of([1, 2])
    pools = [torch.zeros(1, 2, 1, 16, 32, dtype=torch.int8) for _ in range(2)]
    scales = [torch.zeros(1, 2, 1) for _ in range(2)]
    with pytest.raises(ValueError):
        paged.PagedCache(*pools, *scales, torch.zeros(7, dtype=torch.int32), sequences=1, pages_per_sequence=1)
    with pytest.raises(ValueError):
        speculative.verify(torch.zeros(1, 2, 4), torch.zeros(1, 1, 4), torch.zeros(1, 1, dtype=torch.int64),
                           torch.zeros(1, 2, dtype=torch.float64))


def test_flags_have_errors():
    assert isinstance(_lib.flag_error(_lib.FLAG_PAGES), MemoryError)
    assert isinstance(_lib.flag_error(_lib.FLAG_BOOK), IndexError)
