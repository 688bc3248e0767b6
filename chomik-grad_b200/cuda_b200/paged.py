"""A paged 8-bit KV cache and the operators that serve from it.

The reference keeps one dense float32 cache per program, for one sequence of a
fixed context (chomikgrad/llama.py:436-543).  ``PagedCache`` holds many
sequences of unlike lengths in pages of 16 to 256 tokens, int8 or e4m3 with
one float32 scale for each page and kv head, and pages can be shared:

    cache = PagedCache.allocate(layers=22, pages=4096, kv_heads=4, page_size=64,
                                head_size=64, sequences=32, pages_per_sequence=32)
    cache.extend(counts)                      # room for counts[b] more tokens of slot b
    for layer in range(22):
        cache.append(layer, k, v, counts=counts)        # quantise them into their pages
        out = cache.attend(layer, q, counts=counts)     # attention of the same tokens
    cache.fork([0, 0], [5, 6])                # slots 5 and 6 continue slot 0, sharing its pages
    out = cache.attend_shared(layer, q)       # attend, with the pages that all slots share read once
    cache.truncate(refused)                   # drop the last refused[b] tokens
    cache.release([6])                        # all of slot 6
    cache.compact()                           # move the held pages to the front of the pools

Values are CUDA ``torch.Tensor`` or the device's ``DeviceArray``.  Every call
runs on the current stream and reads lengths and tables on the device.  Counts
and slots are int32 tensors on the device, or lists: a list is copied there
first, which waits for the host's copy.  With tensors no call synchronises with
the host, and a step can be captured in a CUDA graph (lists are refused then).
Arguments that the host can see are checked at the call (``TypeError``,
``ValueError``); what only the device sees (a slot, page, length or count
outside its range, too few free pages) sets the cache's error flag, which
``check_errors`` reads and raises.  There is no backward pass.
"""

from __future__ import annotations

import ctypes
import math
import threading
from typing import Any, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_SIZES = (32, 64, 128)
SHARED_BYTES = 2 ** 27  # of reads that are repeated: a border for ``attend_shared``'s ``least_bytes``
_VALUES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_STORAGE = {torch.int8: _lib.I8, torch.float8_e4m3fn: _lib.E4M3}


def tensor_of(value: Any) -> torch.Tensor:
    """The torch view of a tensor or a ``DeviceArray``."""
    if isinstance(value, torch.Tensor):
        return value
    tensor = getattr(value, "tensor", None)
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"a CUDA tensor or DeviceArray is required, got {type(value).__name__}")
    return tensor[:value.size].view(value.shape)


def require(value: torch.Tensor, name: str, device: torch.device, dtypes, shape: Tuple[Optional[int], ...],
            dense: int) -> None:
    """Checks of one argument: its device, dtype, shape (None: any) and that its last ``dense`` dims are contiguous."""
    if value.device != device:
        raise ValueError(f"{name} is on {value.device}, expected {device}")
    if value.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {value.dtype}, expected one of {', '.join(map(str, dtypes))}")
    if len(value.shape) != len(shape) or any(want is not None and got != want
                                             for got, want in zip(value.shape, shape)):
        raise ValueError(f"{name} has shape {tuple(value.shape)}, expected "
                         f"{tuple('any' if n is None else n for n in shape)}")
    step = 1 if value.numel() else None  # strides of an empty tensor say nothing
    for at in range(len(shape) - 1, len(shape) - 1 - dense, -1):
        if step is None:
            break
        if value.shape[at] != 1 and value.stride(at) != step:
            raise ValueError(f"{name} has to be contiguous in its last {dense} dimension(s)")
        step *= value.shape[at]


def aligned(value: torch.Tensor, name: str) -> None:
    """Check that a tensor begins on 16 bytes, as the kernels' wide accesses need it."""
    if value.data_ptr() % 16:
        raise ValueError(f"{name} has to begin on a multiple of 16 bytes")


def no_grad_needed(*values: torch.Tensor) -> None:
    """Refuse values that a gradient should flow through, backward or as a forward-mode tangent."""
    for value in values:
        if value.requires_grad and torch.is_grad_enabled():
            raise ValueError("an argument requires grad: this operator has no backward pass")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(value).tangent is not None:
            raise ValueError("an argument has a tangent: this operator has no forward-mode derivative")


def current_stream(device: torch.device) -> int:
    """Handle of the current stream of ``device``, which has to be the current device (launches go there).

    (``torch.cuda.current_stream`` makes a stream object first, 3 us of a call that takes 8.)
    """
    if torch.cuda.current_device() != device.index:
        raise ValueError(f"the tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(device.index)


def reach(value: torch.Tensor) -> int:
    """Bytes of memory from a tensor's first element to behind its last."""
    if value.numel() == 0:
        return 0
    return (1 + sum((n - 1) * s for n, s in zip(value.shape, value.stride()))) * value.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the spans of memory that ``a`` and ``b`` reach over meet."""
    return meet(a.data_ptr(), reach(a), b.data_ptr(), reach(b))


def meet(a: int, a_bytes: int, b: int, b_bytes: int) -> bool:
    """Whether two spans of memory, each an address and its bytes, have a byte in common."""
    return a_bytes > 0 and b_bytes > 0 and a < b + b_bytes and b < a + a_bytes


def signature(value: Optional[torch.Tensor]):
    """What the checks of an argument look at: equal signatures pass or fail alike."""
    return None if value is None else (value.shape, value.stride(), value.dtype, value.device)


class Prepared(dict):
    """Checked argument structures by the signatures they were made for, without pointers.

    A call with shapes, strides and types that were seen before skips the
    checks and copies the structure; only the pointers are new.
    """

    LIMIT = 512

    def __setitem__(self, key, value) -> None:
        if len(self) >= self.LIMIT:
            self.clear()
        super().__setitem__(key, value)


class PagedCache:
    """Pools, book and the operators on them (see the module's text).

    ``k_pages`` and ``v_pages`` (layers, pages, kv_heads, page_size, head_size),
    ``k_scale`` and ``v_scale`` (layers, pages, kv_heads) and ``book``, one int32
    tensor of the table (sequences, pages_per_sequence), the lengths
    (sequences), the reference counts (pages), the stack of free pages (pages)
    and its height, are used as they are.  ``allocate`` makes an empty cache.
    """

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 book: torch.Tensor, *, sequences: int, pages_per_sequence: int) -> None:
        if k_pages.device.type != "cuda":
            raise ValueError(f"the cache has to be on a CUDA device, got {k_pages.device}")
        if k_pages.ndim != 5:
            raise ValueError("k_pages has to be (layers, pages, kv_heads, page_size, head_size)")
        self.device = k_pages.device
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_size = map(int, k_pages.shape)
        self.sequences, self.pages_per_sequence = int(sequences), int(pages_per_sequence)
        if self.page_size not in PAGE_SIZES:
            raise ValueError(f"page_size has to be one of {PAGE_SIZES}, got {self.page_size}")
        if self.head_size not in HEAD_SIZES:
            raise ValueError(f"head_size has to be one of {HEAD_SIZES}, got {self.head_size}")
        if min(self.layers, self.pages, self.kv_heads, self.sequences, self.pages_per_sequence) < 1:
            raise ValueError("layers, pages, kv_heads, sequences and pages_per_sequence have to be positive")
        if self.pages_per_sequence * self.page_size >= 2 ** 31:
            raise ValueError("a sequence holds fewer than 2**31 tokens")
        require(k_pages, "k_pages", self.device, tuple(_STORAGE), tuple(k_pages.shape), 5)
        require(v_pages, "v_pages", self.device, (k_pages.dtype,), tuple(k_pages.shape), 5)
        aligned(k_pages, "k_pages")
        aligned(v_pages, "v_pages")
        for name, scale in (("k_scale", k_scale), ("v_scale", v_scale)):
            require(scale, name, self.device, (torch.float32,), tuple(k_pages.shape[:3]), 3)
        rows = self.sequences * self.pages_per_sequence
        require(book, "book", self.device, (torch.int32,), (rows + self.sequences + 2 * self.pages + 1,), 1)
        self.k_pages, self.v_pages, self.k_scale, self.v_scale, self.book = k_pages, v_pages, k_scale, v_scale, book
        self.table, self.lengths, self.refs, self.free, self.height = self.split(book)
        self._flag = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._spans = [(name, t.data_ptr(), t.data_ptr() + t.nbytes) for name, t in (
            ("k_pages", k_pages), ("v_pages", v_pages), ("k_scale", k_scale), ("v_scale", v_scale), ("the book", book),
            ("the error flag", self._flag))]
        self._layer_args = [self._args_of(layer) for layer in range(self.layers)]
        self._book_args, self._pool_args = _lib.PageBook(), _lib.PagePools()
        b, p = self._book_args, self._pool_args
        b.table, b.lengths, b.refs = (t.data_ptr() for t in (self.table, self.lengths, self.refs))
        b.free_pages, b.height = self.free.data_ptr(), self.height.data_ptr()
        b.slots, b.columns, b.pages, b.page = self.sequences, self.pages_per_sequence, self.pages, self.page_size
        p.k_pages, p.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
        p.k_scale, p.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        p.layers, p.pages, p.kv_heads = self.layers, self.pages, self.kv_heads
        p.page_bytes = self.kv_heads * self.page_size * self.head_size
        self._lib = _lib.load()
        self._attend_args, self._append_args, self._lists = Prepared(), Prepared(), Prepared()
        self._scratch_words, self._workspaces, self._calls = Prepared(), Prepared(), threading.Lock()

    @classmethod
    def allocate(cls, *, layers: int, pages: int, kv_heads: int, page_size: int, head_size: int, sequences: int,
                 pages_per_sequence: int, storage: torch.dtype = torch.int8, device: Any = None) -> "PagedCache":
        """An empty cache of ``sequences`` slots on ``device`` (the current CUDA device)."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (layers, pages, kv_heads, page_size, head_size)
        pools = [torch.zeros(shape, dtype=torch.int8, device=device).view(storage) for _ in range(2)]
        scale = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)]
        book = torch.zeros(sequences * pages_per_sequence + sequences + 2 * pages + 1, dtype=torch.int32,
                           device=device)
        cache = cls(*pools, *scale, book, sequences=sequences, pages_per_sequence=pages_per_sequence)
        cache.table.fill_(-1)
        cache.free.copy_(torch.arange(pages - 1, -1, -1, dtype=torch.int32))
        cache.height.fill_(pages)
        return cache

    def split(self, book: torch.Tensor) -> Tuple[torch.Tensor, ...]:
        """Views of a book: table, lengths, reference counts, free pages, height of the free stack."""
        rows = self.sequences * self.pages_per_sequence
        table, lengths, refs, free, height = book.split([rows, self.sequences, self.pages, self.pages, 1])
        return table.view(self.sequences, self.pages_per_sequence), lengths, refs, free, height

    def _args_of(self, layer: int) -> _lib.PagedCacheArgs:
        c = _lib.PagedCacheArgs()
        c.k_pages, c.v_pages = self.k_pages[layer].data_ptr(), self.v_pages[layer].data_ptr()
        c.k_scale, c.v_scale = self.k_scale[layer].data_ptr(), self.v_scale[layer].data_ptr()
        c.storage, c.kv_heads = _STORAGE[self.k_pages.dtype], self.kv_heads
        c.page, c.head_size, c.pages = self.page_size, self.head_size, self.pages
        c.table, c.lengths = self.table.data_ptr(), self.lengths.data_ptr()
        c.slots, c.columns = self.sequences, self.pages_per_sequence
        return c

    def _stream(self) -> int:
        return current_stream(self.device)

    def _ints(self, value: Any) -> Optional[torch.Tensor]:
        """A list of whole numbers as a tensor (host lists are copied to the device)."""
        if value is None or isinstance(value, torch.Tensor):
            return value
        if isinstance(value, (list, tuple)):
            if torch.cuda.is_current_stream_capturing():
                raise ValueError("counts and slots have to be int32 tensors on the device while a graph is captured")
            return torch.tensor(value, dtype=torch.int32, device=self.device)
        return tensor_of(value)

    def _list(self, value: Any, name: str, count: Optional[int]) -> torch.Tensor:
        """An int32 list on the device."""
        value = self._ints(value)
        if value is None:
            raise TypeError(f"{name} are required")
        key = (name, count, signature(value))
        if key not in self._lists:
            require(value, name, self.device, (torch.int32,), (count,), 1)
            self._lists[key] = True
        return value

    def _check_lists(self, counts: Optional[torch.Tensor], sequences: Optional[torch.Tensor], batch: int) -> None:
        if counts is not None:
            self._list(counts, "counts", batch)
        if sequences is not None:
            self._list(sequences, "sequences", batch)
        elif batch > self.sequences:
            raise ValueError(f"{batch} rows, and the cache has {self.sequences} sequences")

    def _layer(self, layer: int) -> _lib.PagedCacheArgs:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        return self._layer_args[layer]

    # -- values ------------------------------------------------------------
    def append(self, layer: int, k: Any, v: Any, *, counts: Any = None, sequences: Any = None) -> None:
        """Quantise new keys and values (batch, tokens, kv_heads, head_size) into ``layer``'s pages.

        Row b's first ``counts[b]`` tokens (all without counts) are the last
        ones of slot ``sequences[b]`` (slot b without), for which ``extend``
        has made room.  float32, bfloat16 or float16, any strides with a
        contiguous head.  See ``cb_paged_append`` for the scales.
        """
        k, v, counts, sequences = tensor_of(k), tensor_of(v), self._ints(counts), self._ints(sequences)
        no_grad_needed(k, v)
        key = (layer, signature(k), signature(v), signature(counts), signature(sequences))
        known = self._append_args.get(key)
        if known is None:
            known = self._append_args[key] = self._prepare_append(layer, k, v, counts, sequences)
        a = _lib.PagedAppendArgs.from_buffer_copy(known)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        if counts is not None:
            a.counts = counts.data_ptr()
        if sequences is not None:
            a.sequences = sequences.data_ptr()
        _lib.check(self._lib.cb_paged_append(ctypes.byref(a), self._stream()), "cb_paged_append")

    def _prepare_append(self, layer: int, k: torch.Tensor, v: torch.Tensor, counts: Optional[torch.Tensor],
                        sequences: Optional[torch.Tensor]) -> _lib.PagedAppendArgs:
        require(k, "k", self.device, tuple(_VALUES), (None, None, self.kv_heads, self.head_size), 1)
        batch, tokens = k.shape[:2]
        require(v, "v", self.device, (k.dtype,), (batch, tokens, self.kv_heads, self.head_size), 1)
        self._check_lists(counts, sequences, batch)
        a = _lib.PagedAppendArgs()
        a.cache = self._layer(layer)
        a.dtype, a.batch, a.tokens = _VALUES[k.dtype], batch, tokens
        a.k_strides[:], a.v_strides[:] = k.stride()[:3], v.stride()[:3]
        a.error_flag = self._flag.data_ptr()
        return a

    def attend(self, layer: int, q: Any, *, counts: Any = None, sequences: Any = None, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q (batch, tokens, heads, head_size), the last tokens of their slots, over ``layer``.

        Each token sees its slot's keys up to its own (``counts`` and
        ``sequences`` as in ``append``; rows past ``counts[b]`` and rows that
        see nothing give zeros).  ``scale`` is 1/sqrt(head_size) without one.
        Returns (batch, tokens, heads, head_size) of q's dtype; ``out`` may be a
        contiguous ``q`` itself and lies over nothing else that the call reads.

        Queries and weights go to the tensor cores as fp16 in two parts (22
        bits) with float32 sums; where more than 8 rows share a kv head,
        bfloat16 outputs take one part (11 bits) of both and float16 outputs one
        of the queries.  A key whose weight is below 2^-30 of another's within
        the same 2048 / head_size keys may be left out.  Every block of rows of a
        slot walks the slot's whole length, also those past ``counts[b]``: one
        long chunk with many single tokens costs less in a call of its own.
        """
        return self._attend(layer, q, counts, sequences, scale, out, None)

    def attend_shared(self, layer: int, q: Any, *, counts: Any = None, sequences: Any = None,
                      scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                      least_bytes: Optional[int] = None) -> torch.Tensor:
        """``attend`` for sequences that begin alike, as ``fork`` leaves them.

        The leading pages that all sequences of the call hold in common (those
        with a count of 0 aside) are found on the device.  Where it pays, they are
        read and multiplied once with the rows of all, each sequence's other keys by
        themselves; elsewhere all is read as by ``attend``, so any sequences may be
        given (looking costs 6 to 8 us where the tables could hold as much).  It pays from 192 MB on that all but three of the sequences would read,
        with kv heads and blocks of rows for a part of the GPU; with ``least_bytes``
        the keys are read once wherever that saves so many bytes of reads.

        Queries and weights of these keys go to the tensor cores as fp16 with float32
        sums: one part (11 bits) of both for bfloat16, two (22 bits) of both for float32 and
        of the weights for float16, whose queries are exact in one. Of 64 keys, one whose
        weight is below 2^-17 (float32: 2^-23) of the largest of them, or 2^-90 of the
        row's, may be left out.
        """
        least = -1 if least_bytes is None else int(least_bytes)  # (below 0: by the library's rule)
        if least_bytes is not None and not 0 <= least < 2 ** 63:
            raise ValueError(f"least_bytes is {least_bytes}, expected 0 or more")
        return self._attend(layer, q, counts, sequences, scale, out, least)

    def _attend(self, layer: int, q: Any, counts: Any, sequences: Any, scale: Optional[float],
                out: Optional[torch.Tensor], least_bytes: Optional[int]) -> torch.Tensor:
        q, counts, sequences = tensor_of(q), self._ints(counts), self._ints(sequences)
        no_grad_needed(q)
        key = (layer, signature(q), signature(counts), signature(sequences), scale, least_bytes)
        known = self._attend_args.get(key)
        if known is None:
            known = self._attend_args[key] = self._prepare_attend(layer, q, counts, sequences, scale, least_bytes)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            require(out, "out", self.device, (q.dtype,), tuple(q.shape), 4)
            aligned(out, "out")
            self._apart(out, q, counts, sequences)
            no_grad_needed(out)
            if not out.is_inference():  # a backward pass that kept what it held notices
                torch.autograd.graph.increment_version(out)
        a = _lib.PagedAttentionArgs.from_buffer_copy(known[0])
        a.q, a.out = q.data_ptr(), out.data_ptr()
        if counts is not None:
            a.counts = counts.data_ptr()
        if sequences is not None:
            a.sequences = sequences.data_ptr()
        stream = self._stream()
        with self._calls:  # (a call's launches share its workspace: none of another thread's come between)
            counters, scratch = self._workspace(stream, known[2], known[1])
            if least_bytes is None:
                _lib.check(self._lib.cb_paged_attention(ctypes.byref(a), scratch, counters, stream),
                           "cb_paged_attention")
            else:
                _lib.check(self._lib.cb_paged_attention_shared(ctypes.byref(a), least_bytes, scratch, counters, stream),
                           "cb_paged_attention_shared")
        return out

    def _apart(self, out: torch.Tensor, q: torch.Tensor, counts: Optional[torch.Tensor],
               sequences: Optional[torch.Tensor]) -> None:
        """Refuse an ``out`` (contiguous) over what other blocks read while it is written; it may be ``q`` itself."""
        at, size = out.data_ptr(), out.nbytes
        for name, start, end in self._spans:
            if start < at + size and at < end and size:
                raise ValueError(f"out shares memory with {name}")
        for name, value in (("q", q), ("counts", counts), ("sequences", sequences)):
            if value is None or (value is q and q.data_ptr() == at and q.is_contiguous()):
                continue
            if meet(at, size, value.data_ptr(), reach(value)):
                raise ValueError(f"out shares memory with {name}")

    def _workspace(self, stream: int, counters: int, words: int) -> Tuple[int, int]:
        """Addresses of zeroed counters, which a call leaves zero, and of scratch for a call on ``stream``.

        Calls of one stream follow one another and share theirs.  A captured
        call may be replayed on any stream, so it has its own, cleared within
        the graph.
        """
        if torch.cuda.is_current_stream_capturing():
            own = self._flag.new_empty(words)  # (the graph's memory pool keeps both)
            return self._flag.new_zeros(counters).data_ptr(), own.data_ptr()
        kept = self._workspaces.get(stream)
        if kept is None or kept[0] < counters or kept[1] < words:
            counts, scratch = self._flag.new_zeros(counters), self._flag.new_empty(words)
            kept = self._workspaces[stream] = (counters, words, counts.data_ptr(), scratch.data_ptr(), counts, scratch)
        return kept[2], kept[3]

    def _prepare_attend(self, layer: int, q: torch.Tensor, counts: Optional[torch.Tensor],
                        sequences: Optional[torch.Tensor], scale: Optional[float],
                        least_bytes: Optional[int]) -> Tuple[_lib.PagedAttentionArgs, int, int]:
        require(q, "q", self.device, tuple(_VALUES), (None, None, None, self.head_size), 1)
        batch, tokens, heads = q.shape[:3]
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads cannot share {self.kv_heads} kv heads")
        self._check_lists(counts, sequences, batch)
        a = _lib.PagedAttentionArgs()
        a.cache = self._layer(layer)
        a.dtype, a.batch, a.tokens, a.heads = _VALUES[q.dtype], batch, tokens, heads
        a.q_strides[:] = q.stride()[:3]
        a.scale = 1.0 / math.sqrt(self.head_size) if scale is None else scale
        a.error_flag = self._flag.data_ptr()
        if least_bytes is None:
            size = self._lib.cb_paged_attention_scratch(ctypes.byref(a))
        else:
            size = self._lib.cb_paged_attention_shared_scratch(ctypes.byref(a), least_bytes)
        return (a, (size + 3) // 4,
                self._lib.cb_paged_attention_counters(ctypes.byref(a)))

    # -- pages -------------------------------------------------------------
    def extend(self, counts: Any, *, sequences: Any = None) -> None:
        """Make room for ``counts[i]`` more tokens of slot ``sequences[i]`` (slot i without).

        Lengths grow, missing pages are taken, and an open last page that
        other slots hold too is copied first.  All or nothing: with too few
        free pages nothing changes and ``check_errors`` raises MemoryError.
        """
        counts, sequences = self._list(counts, "counts", None), self._ints(sequences)
        n = counts.shape[0]
        self._check_lists(None, sequences, n)
        scratch = self._scratch(n)
        _lib.check(self._lib.cb_pages_extend(
            ctypes.byref(self._book_args), ctypes.byref(self._pool_args), counts.data_ptr(),
            None if sequences is None else sequences.data_ptr(), n, scratch.data_ptr(), self._flag.data_ptr(),
            self._stream()), "cb_pages_extend")

    def fork(self, parents: Any, children: Any) -> None:
        """Slot ``children[i]``, which has to be empty, continues slot ``parents[i]`` and shares its pages.

        Each pair by itself: one that is refused changes nothing, the others are done.
        """
        parents = self._list(parents, "parents", None)
        n = parents.shape[0]
        children = self._list(children, "children", n)
        if n > self.sequences:
            raise ValueError(f"{n} forks, and the cache has {self.sequences} sequences")
        _lib.check(self._lib.cb_pages_fork(ctypes.byref(self._book_args), parents.data_ptr(), children.data_ptr(), n,
                                           self._flag.data_ptr(), self._stream()), "cb_pages_fork")

    def truncate(self, counts: Any, *, sequences: Any = None) -> None:
        """Drop the last ``counts[i]`` tokens of slot ``sequences[i]`` and let go of the pages that held only those."""
        counts = self._list(counts, "counts", None)
        self._truncate(counts, sequences, counts.shape[0])

    def release(self, sequences: Any) -> None:
        """Empty the slots ``sequences``."""
        sequences = self._list(sequences, "sequences", None)
        self._truncate(None, sequences, sequences.shape[0])

    def _truncate(self, counts: Optional[torch.Tensor], sequences: Any, n: int) -> None:
        sequences = self._ints(sequences)
        self._check_lists(None, sequences, n)
        if n > self.sequences:
            raise ValueError(f"{n} slots, and the cache has {self.sequences} sequences")
        _lib.check(self._lib.cb_pages_truncate(
            ctypes.byref(self._book_args), None if counts is None else counts.data_ptr(),
            None if sequences is None else sequences.data_ptr(), n, self._flag.data_ptr(), self._stream()),
            "cb_pages_truncate")

    def compact(self) -> None:
        """Move the held pages to the front of the pools (page ids change; the table follows)."""
        scratch = self._scratch(0)
        _lib.check(self._lib.cb_pages_compact(ctypes.byref(self._book_args), ctypes.byref(self._pool_args),
                                              scratch.data_ptr(), self._flag.data_ptr(), self._stream()),
                   "cb_pages_compact")

    def copy_pages(self, source: Any, target: Any) -> None:
        """Copy page ``source[i]`` to page ``target[i]`` in every layer (no page is both)."""
        source = self._list(source, "source", None)
        target = self._list(target, "target", source.shape[0])
        _lib.check(self._lib.cb_pages_copy(ctypes.byref(self._pool_args), source.data_ptr(), target.data_ptr(),
                                           source.shape[0], self._flag.data_ptr(), self._stream()), "cb_pages_copy")

    def _scratch(self, n: int) -> torch.Tensor:
        size = self._scratch_words.get(n)
        if size is None:
            size = self._scratch_words[n] = (self._lib.cb_pages_scratch(ctypes.byref(self._book_args), n) + 3) // 4
        return self._flag.new_empty(size)

    # -- errors ------------------------------------------------------------
    def check_errors(self) -> None:
        """Raise what a call since the last check found on the device (reads one number back)."""
        value = int(self._flag.item())
        if value:
            self._flag.zero_()
            raise _lib.flag_error(value)
