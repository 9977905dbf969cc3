"""Paged KV cache held in 4 bits: the operators an inference engine runs on the
pages that a store keeps.

``KV4Cache`` is a :class:`~cascade_cpp.connector.KVPageConnector` whose pages
hold every layer's keys and values in 4 bits. ``append`` quantises new tokens
into pages, ``attend`` is attention straight over the pages (single tokens, a
few drafted tokens or prompt chunks behind a cached prefix), ``read`` gives
tokens back as 16- or 32-bit values, and ``save`` / ``load`` move pages to and
from the store. Equal tokens give equal page bytes however they were appended,
so full pages of a shared prefix have the same block ID.

``PageTable`` keeps block tables, lengths and the free pages on the GPU:
``plan`` turns the numbers of new tokens of a step into pages, slots and
positions in one launch, without a host round trip.

    table = PageTable(requests=256, columns=512, num_pages=20000)
    cache = KV4Cache(20000, layers=28, kv_heads=4, head_dim=128, store=store)
    plan = table.plan(q_lens, tokens=len(hidden))
    for layer in range(28):
        cache.append(layer, k, v, plan.slots)
        o = cache.attend(layer, q, table.block_table, table.kv_lens, q_start=plan.q_start,
                         max_q=longest)

All calls run on the current stream of the cache's device, allocate only their
outputs (and attend a workspace) from torch's allocator, never wait for the
GPU, and may be captured into a CUDA graph. ``check`` reports what only the GPU
can see: slots, pages or lengths outside the cache, which are skipped.

A value is ``offset + scale * (code - 8)`` with one fp16 pair (scale, offset)
per token, head and ``group`` dimensions: scale = (max - min) / 15 and offset =
min + 8 scale, rounded to fp16 before the codes are taken. Values beyond
+-65000 are stored as +-65000; a NaN makes its group NaN.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Sequence

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

from . import _lib as L
from . import _native_lib
from ._lib import CascadeError
from .connector import KVPageConnector

__all__ = ["KV4Cache", "PageTable", "Plan", "page_bytes"]


def _check(rc: int):
    if rc:
        raise CascadeError(rc, _native_lib().cb_last_error(None).decode(errors="replace"))


def _device(device) -> "torch.device":
    d = torch.device("cuda" if device is None else device)
    if d.type != "cuda":
        raise TypeError("a CUDA device is needed")
    return torch.device("cuda", torch.cuda.current_device()) if d.index is None else d


# torch.cuda.current_stream(device).cuda_stream without the two objects it makes
_raw_stream = getattr(getattr(torch, "_C", None), "_cuda_getCurrentRawStream", None)


def _stream(device):
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _on(t, name: str, device):
    if not isinstance(t, torch.Tensor) or t.get_device() != device.index:  # -1 for the host
        raise TypeError(f"{name} must be a tensor on {device}")


def _vector(t, name: str, dtype, device, n=None):
    """Address of a contiguous 1-D tensor of the device."""
    _on(t, name, device)
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}")
    if t.dim() != 1 or (n is not None and t.numel() != n) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector" + ("" if n is None else f" of {n}"))
    return t.data_ptr()


def _overlap(q, out) -> bool:
    """Whether the dense ``out`` may share memory with ``q [rows, heads, dim]``: it
    does not where it lies before or behind q, or in a gap between two of its rows."""
    rows, heads, dim = q.shape
    if not q.numel():
        return False
    size = q.element_size()
    row, head = q.stride(0), q.stride(1)
    wide = (heads - 1) * head + dim  # elements that a row spans
    at = (out.data_ptr() - q.data_ptr()) // size  # of out, from the first of q
    end = at + -(-out.numel() * out.element_size() // size)
    if end <= 0 or at >= (rows - 1) * row + wide:
        return False
    if rows == 1 or row < wide or at < 0:
        return True
    before = at // row  # the last row that begins at or before out
    return at < before * row + wide or (before + 1 < rows and end > (before + 1) * row)


_forward = getattr(getattr(torch, "autograd", None), "forward_ad", None)


def _plain(t, name: str):
    """Refuses a tensor whose gradient or tangent the call would cut off."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and there is no backward pass: call it under torch.no_grad()")
    if getattr(_forward, "_current_level", 0) >= 0 and _forward.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a tangent, and there is no forward-mode derivative")


def _take_errors(errors) -> int:
    """The error word, which is 0 again afterwards. The calls may be on any stream."""
    torch.cuda.synchronize(errors.device)
    bits = int(errors.item())
    if bits:
        errors.zero_()
        torch.cuda.synchronize(errors.device)  # before a call on another stream sets it
    return bits


def _dtype_code(dtype) -> int:
    if dtype == torch.bfloat16:
        return L.CB_KV4_BF16
    if dtype == torch.float16:
        return L.CB_KV4_F16
    if dtype == torch.float32:
        return L.CB_KV4_F32
    raise TypeError("values must be float16, bfloat16 or float32")


def page_bytes(layers: int, kv_heads: int, head_dim: int, page_size: int = 16, group: int = 64) -> int:
    """Bytes of a page with every layer and head (cb_kv4_page_bytes)."""
    n = int(_native_lib().cb_kv4_page_bytes(int(layers), int(kv_heads), int(head_dim), int(page_size), int(group)))
    if not n:
        raise ValueError("not offered: head_dim is 64, 128 or 256, page_size 16, 32, 64, 128 or 256, "
                         "group 32, 64, 128 or 256 and at most head_dim")
    return n


class KV4Cache(KVPageConnector):
    """Pages ``[num_pages, layers, kv_heads, bytes]`` (``.cache``, uint8) and the
    operators on them. ``store`` is needed for ``save`` and ``load`` only."""

    def __init__(self, num_pages: int, layers: int, kv_heads: int, head_dim: int, page_size: int = 16,
                 group: int = 64, device=None, store=None):
        total = page_bytes(layers, kv_heads, head_dim, page_size, group)
        pages = torch.zeros(int(num_pages), int(layers), int(kv_heads), total // (layers * kv_heads),
                            dtype=torch.uint8, device=_device(device))
        self._bind(store, pages, head_dim, page_size, group)

    @classmethod
    def over(cls, pages, *, head_dim: int, page_size: int = 16, group: int = 64, store=None) -> "KV4Cache":
        """A cache over an existing tensor ``[num_pages, layers, kv_heads, bytes]``
        of uint8, whose pages are contiguous (they may lie apart)."""
        self = cls.__new__(cls)
        self._bind(store, pages, head_dim, page_size, group)
        return self

    def _bind(self, store, pages, head_dim, page_size, group):
        super().__init__(store, pages)
        if pages.dim() != 4 or pages.dtype != torch.uint8:
            raise ValueError("pages must be uint8 [num_pages, layers, kv_heads, bytes]")
        _, layers, heads, n = pages.shape
        if n * layers * heads != page_bytes(layers, heads, head_dim, page_size, group):
            raise ValueError(f"pages have {n} bytes for each layer and head, the form "
                             f"{page_bytes(1, 1, head_dim, page_size, group)}")
        if self.base % 16 or self.stride % 16:
            raise ValueError("pages must start on 16-byte boundaries")
        self.device = pages.device
        self.layers, self.kv_heads, self.head_dim = int(layers), int(heads), int(head_dim)
        self.page_size, self.group = int(page_size), int(group)
        self.errors = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._work: dict = {}
        stride = self.stride if self.num_pages > 1 else max(self.stride, self.page_bytes)
        self._form = L.cb_kv4_cache(self.base, stride, self.errors.data_ptr(), self.num_pages, self.layers,
                                    self.kv_heads, self.head_dim, self.page_size, self.group, self.device.index, 0)

    # ---------------------------------------------------------------- store

    def save(self, pages: Sequence[int], is_prefix: Sequence[bool] | None = None, return_status: bool = False):
        if self.store is None:
            raise ValueError("the cache has no store")
        return super().save(pages, is_prefix, return_status)

    def load(self, ids: Sequence[str], pages: Sequence[int]) -> list[bool]:
        if self.store is None:
            raise ValueError("the cache has no store")
        return super().load(ids, pages)

    # ------------------------------------------------------------ operators

    def _sizes(self, layer: int, sizes: int) -> None:
        """Refuses what the C call's 32 bits would wrap (``sizes``: an or of all)."""
        if not 0 <= layer < self.layers:
            raise CascadeError(L.CB_ERR_ARG, f"layer must be 0 .. {self.layers - 1}")
        if sizes >> 31:
            raise ValueError("sizes must be below 2^31")

    def _values(self, t, name: str):
        _on(t, name, self.device)
        if t.dim() != 3 or t.shape[1] != self.kv_heads or t.shape[2] != self.head_dim or (
                t.stride(2) != 1 and t.numel()):
            raise ValueError(f"{name} must be [tokens, {self.kv_heads}, {self.head_dim}] with contiguous heads")

    def append(self, layer: int, k, v, slots) -> None:
        """Quantises the keys and values ``[n, kv_heads, head_dim]`` (16 or 32
        bits; tokens and heads may be strided, as slices of a fused projection
        are) into ``layer`` of the pages at ``slots`` (int64 ``[n]``, page *
        page_size + offset; negative ones are skipped). A slot may appear once
        in a call. There is no backward pass."""
        self._values(k, "k")
        self._values(v, "v")
        _plain(k, "k")
        _plain(v, "v")
        if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
            raise ValueError("k and v differ in type or length")
        n = k.shape[0]
        self._sizes(layer, n)
        at = _vector(slots, "slots", torch.int64, self.device, n)
        _check(_native_lib().cb_kv4_append(
            self._form, layer, _dtype_code(k.dtype), k.data_ptr(), v.data_ptr(), n, k.stride(0), k.stride(1),
            v.stride(0), v.stride(1), at, _stream(self.device)))

    def read(self, layer: int, slots, dtype=None):
        """Keys and values ``[n, kv_heads, head_dim]`` of the tokens at
        ``slots`` as ``dtype`` (bfloat16 unless given); zeros for a negative
        slot."""
        dtype = torch.bfloat16 if dtype is None else dtype
        code = _dtype_code(dtype)
        at = _vector(slots, "slots", torch.int64, self.device)
        n = slots.shape[0]
        self._sizes(layer, n)
        k = torch.empty((n, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _check(_native_lib().cb_kv4_read(self._form, layer, code, k.data_ptr(), v.data_ptr(), n, at,
                                         _stream(self.device)))
        return k, v

    def attend(self, layer: int, q, block_table, kv_lens, q_start=None, max_q: int | None = None,
               causal: bool = True, scale: float | None = None, out=None, return_lse: bool = False):
        """Attention of the queries ``q [total_q, q_heads, head_dim]`` (fp16 or
        bf16; tokens and heads may be strided) over the cached tokens of
        ``layer``; ``[total_q, q_heads, head_dim]`` of q's type.

        Request i owns the rows ``q_start[i] .. q_start[i+1]`` (int32
        ``[requests + 1]``; without it, one row each) and the first
        ``kv_lens[i]`` tokens of its pages ``block_table[i]``. When ``causal``,
        its last row sees every token and each row before it one fewer; a row
        that sees nothing gets zeros (log-sum-exp -inf). A key that is NaN
        makes the rows that see it NaN, a NaN group of a value its dimensions
        in them. Query heads are in groups of q_heads / kv_heads that share a
        KV head. ``scale`` defaults to 1 / sqrt(head_dim).

        ``max_q`` (rows of a request at most) only helps the choice of kernel:
        the one for more than 64 rows of a KV head rounds keys and values to
        fp16, the one for fewer, which 1 asks for, nothing of the cache. Rows
        of no request (a padded step) are zeros, and left as they were in a
        given ``out``. With ``return_lse`` also the log-sum-exp of each row's
        scores, ``[total_q, q_heads]`` fp32, -inf in rows of no request. There
        is no backward pass."""
        dev, d = self.device, self.head_dim
        _on(q, "q", dev)
        if q.dim() != 3 or q.shape[2] != d or (q.stride(2) != 1 and q.numel()):
            raise ValueError(f"q must be [rows, q_heads, {d}] with contiguous heads")
        _plain(q, "q")
        rows, heads = q.shape[0], q.shape[1]
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"q_heads must be a multiple of {self.kv_heads}")
        code = _dtype_code(q.dtype)
        _on(block_table, "block_table", dev)
        if block_table.dtype is not torch.int32:
            raise TypeError("block_table must be torch.int32")
        if block_table.dim() != 2 or block_table.shape[1] == 0 or (
                block_table.stride(1) != 1 and block_table.shape[1] > 1):
            raise ValueError("block_table must be [requests, columns] with contiguous rows")
        n, columns = block_table.shape
        self._sizes(layer, rows | heads | n | columns)
        lens = _vector(kv_lens, "kv_lens", torch.int32, dev, n)
        start = None if q_start is None else _vector(q_start, "q_start", torch.int32, dev, n + 1)
        if start is None and rows != n:
            raise ValueError("without q_start there is one row for each request")
        fill = L.CB_KV4_FILL_LSE if return_lse else 0
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            fill |= L.CB_KV4_FILL_OUT
        elif (not isinstance(out, torch.Tensor) or out.device != dev or out.dtype != q.dtype
              or out.shape != q.shape or not out.is_contiguous() or out.data_ptr() % 16):
            raise ValueError("out must be contiguous, 16-byte aligned and like q")
        elif out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out may not require a gradient")
        elif _overlap(q, out):
            raise ValueError("out may not overlap q")
        lse = torch.empty((rows, heads), dtype=torch.float32, device=dev) if return_lse else None
        a = L.cb_kv4_attend_args(
            q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), block_table.data_ptr(), lens,
            start, None, 0, block_table.stride(0), q.stride(0), q.stride(1),
            d ** -0.5 if scale is None else scale, layer, code, n, columns, rows, heads,
            (1 if start is None else rows) if max_q is None else min(max_q, rows), causal, fill)
        lib = _native_lib()
        need = self._work.get((heads, a.max_q))  # the sizes that decide it
        if need is None:
            if len(self._work) > 255:
                self._work.clear()
            need = lib.cb_kv4_attend_workspace(self._form, a)
            if need:  # 0: the call below says what is wrong with its arguments
                self._work[heads, a.max_q] = need
        work = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = work.data_ptr(), need
        _check(lib.cb_kv4_attend(self._form, a, _stream(dev)))
        return out if lse is None else (out, lse)

    def check(self) -> None:
        """Waits for the GPU (every stream) and raises if a call since the last
        check was given a slot, page or length outside the cache (those are
        skipped)."""
        bits = _take_errors(self.errors)
        if bits:
            if bits & L.CB_KV4_ERROR_TIMEOUT:
                raise CascadeError(L.CB_ERR_TIMEOUT, "a wait inside a kernel ran out")
            raise CascadeError(L.CB_ERR_DEVICE, "a slot, page or length was outside the cache")


class Plan(NamedTuple):
    """One step of a :class:`PageTable`: where its new tokens go."""

    slots: "torch.Tensor"       # int64 [tokens]: page * page_size + offset, -1 for none
    positions: "torch.Tensor"   # int32 [tokens]: place in the request
    q_start: "torch.Tensor"     # int32 [requests + 1]: first token of each request
    status: "torch.Tensor"      # uint8 [requests]: CB_PUT_STORED, or CB_PUT_FAILED for a refused one
    kv_lens: "torch.Tensor"     # int32 [requests]: lengths with the new tokens
    free_count: "torch.Tensor"  # int32 [1]: free pages left


class PageTable:
    """Block tables ``[requests, columns]``, lengths and free pages on the GPU.

    ``block_table``, ``kv_lens``, ``borrowed`` (leading pages of a row that it
    does not own), ``free`` and ``free_count`` (a stack of page numbers and its
    height) are plain int32 tensors that a program may also write, in place."""

    def __init__(self, requests: int, columns: int, num_pages: int, page_size: int = 16, device=None):
        if requests < 0 or columns <= 0 or num_pages <= 0 or page_size <= 0:
            raise ValueError("requests, columns, num_pages and page_size must be positive")
        if columns * page_size > 1 << 30:
            raise ValueError("a row may not hold more than 2^30 tokens")
        self.device = _device(device)
        self.requests, self.columns, self.num_pages = int(requests), int(columns), int(num_pages)
        self.page_size = int(page_size)
        i32 = {"dtype": torch.int32, "device": self.device}
        self.block_table = torch.zeros(self.requests, self.columns, **i32)
        self.kv_lens = torch.zeros(self.requests, **i32)
        self.borrowed = torch.zeros(self.requests, **i32)
        self.free = torch.arange(self.num_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), self.num_pages, **i32)
        self.errors = torch.zeros(1, **i32)

    def plan(self, q_lens, tokens: int, done=None, commit: bool = True, out: Plan | None = None) -> Plan:
        """Gives row i ``q_lens[i]`` new tokens (int32 ``[requests]``; 0 for a
        row that rests) and says where they go; ``tokens`` is the length of the
        step's token axis, and entries behind the last token get slot -1.

        Rows with ``done`` (bool ``[requests]``) first give back the pages they
        own and start anew at length 0. A row is refused, and keeps its length,
        when its tokens end past ``tokens``, do not fit its columns, or need
        pages that are not there; pages are given in row order, and a refused
        row's count against the rows behind it. ``commit=False`` leaves the
        lengths and the free pages as they were (``done`` cannot be given
        then): the plan says whether the step would fit. ``block_table`` names
        the step's pages behind those that each row holds, where only the
        plan's own ``kv_lens`` reach. ``out`` is an earlier plan of the same
        ``tokens`` whose tensors are written again; the lengths and free count
        of a committed plan are the table's own, which a dry plan does not
        write."""
        n, dev = self.requests, self.device
        i32 = torch.int32
        lens = _vector(q_lens, "q_lens", i32, dev, n)
        if done is not None:
            if not commit:
                raise ValueError("done rows give pages back: commit cannot be False")
            if isinstance(done, torch.Tensor) and done.dtype == torch.bool:
                done = done.view(torch.uint8)
            done = _vector(done, "done", torch.uint8, dev, n)
        tokens = int(tokens)
        if not 0 <= tokens < 1 << 31:
            raise ValueError("tokens must be 0 .. 2^31 - 1")
        kv_lens, count = self.kv_lens, self.free_count
        if out is None:  # the int32 outputs share one allocation
            slots = torch.empty(tokens, dtype=torch.int64, device=dev)
            status = torch.empty(n, dtype=torch.uint8, device=dev)
            if commit:
                positions, q_start = torch.empty(tokens + n + 1, dtype=i32, device=dev).split_with_sizes(
                    (tokens, n + 1))
            else:
                positions, q_start, kv_lens, count = torch.empty(tokens + 2 * n + 2, dtype=i32, device=dev
                                                                 ).split_with_sizes((tokens, n + 1, n, 1))
        else:
            slots, positions, q_start, status = out[:4]
            _vector(slots, "out.slots", torch.int64, dev, tokens)
            _vector(positions, "out.positions", i32, dev, tokens)
            _vector(q_start, "out.q_start", i32, dev, n + 1)
            _vector(status, "out.status", torch.uint8, dev, n)
            if not commit:
                kv_lens, count = out[4:]
                _vector(kv_lens, "out.kv_lens", i32, dev, n)
                _vector(count, "out.free_count", i32, dev, 1)
                if count.data_ptr() == self.free_count.data_ptr() or (
                        n and kv_lens.data_ptr() == self.kv_lens.data_ptr()):
                    kv_lens, count = torch.empty_like(kv_lens), torch.empty_like(count)
        a = L.cb_kv4_plan_args(
            lens, done, self.kv_lens.data_ptr(), kv_lens.data_ptr(), self.borrowed.data_ptr(),
            self.block_table.data_ptr(), self.free.data_ptr(), self.free_count.data_ptr(), count.data_ptr(),
            slots.data_ptr(), positions.data_ptr(), q_start.data_ptr(), status.data_ptr(), self.errors.data_ptr(),
            self.columns, n, self.columns, self.num_pages, self.page_size, tokens, dev.index)
        _check(_native_lib().cb_kv4_plan(a, _stream(dev)))
        return Plan(slots, positions, q_start, status, kv_lens, count)

    def take(self, n: int) -> list[int]:
        """``n`` pages off the free stack, for a program to fill (a prefix loaded
        from the store). Waits for the GPU."""
        have = int(self.free_count.item())
        if n < 0 or n > have:
            raise CascadeError(L.CB_ERR_NOSPACE, f"{n} pages asked for, {have} free")
        pages = self.free[have - n:have].flip(0).tolist()
        self.free_count.sub_(n)
        return pages

    def give(self, pages: Sequence[int]) -> None:
        """Puts pages back on the free stack, each once. Waits for the GPU."""
        have, n = int(self.free_count.item()), len(pages)
        if n and (min(pages) < 0 or max(pages) >= self.num_pages):
            raise IndexError("page index out of range")
        if have + n > self.num_pages:
            raise CascadeError(L.CB_ERR_ARG, "more pages given back than there are")
        back = torch.tensor(list(pages), dtype=torch.int32, device=self.device)
        if len(set(pages)) != n or (n and torch.isin(back, self.free[:have]).any()):
            raise ValueError("a page is given back twice")
        self.free[have:have + n] = back
        self.free_count.add_(n)

    def attach(self, row: int, pages: Sequence[int], tokens: int, borrowed: bool = False) -> None:
        """Starts an empty row with ``tokens`` cached tokens in ``pages``. With
        ``borrowed`` the pages stay someone else's (a prefix that several rows
        share): they do not go to the free stack when the row is done. Further
        tokens go to pages of the row's own, so ``tokens`` must then fill the
        pages. Waits for the GPU."""
        if not 0 <= row < self.requests:
            raise IndexError("row out of range")
        n, tokens = len(pages), int(tokens)
        if n > self.columns or tokens < 0 or n != -(-tokens // self.page_size):
            raise ValueError("tokens do not match the pages, or the pages the columns")
        if borrowed and tokens % self.page_size:
            raise ValueError("a borrowed page must be full")
        if not borrowed and len(set(pages)) != n:
            raise ValueError("a row owns a page once")
        if n and (min(pages) < 0 or max(pages) >= self.num_pages):
            raise IndexError("page index out of range")
        if int(self.kv_lens[row]):
            raise ValueError("the row is not empty")
        if n:
            self.block_table[row, :n] = torch.tensor(list(pages), dtype=torch.int32, device=self.device)
        self.kv_lens[row] = tokens
        self.borrowed[row] = n if borrowed else 0

    def check(self) -> None:
        """Waits for the GPU (every stream) and raises if a plan since the last
        check met a page or length outside the table (a row that was set
        wrongly)."""
        if _take_errors(self.errors):
            raise CascadeError(L.CB_ERR_DEVICE, "a page or length was outside the table")
