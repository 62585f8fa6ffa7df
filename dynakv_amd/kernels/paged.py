"""A paged cache for requests of different lengths, and the attention over it.

The uncompressed baseline keeps one length for all rows of a batch in a buffer allocated for the
longest (``dense_append_``, ``dense_decode_attention``; the reference's baseline,
``scripts/benchmark_throughput.py:17-77``, does the same). Serving has requests that come and go:
each has a length of its own, a prompt goes through in chunks beside other requests' single tokens,
and a request that ends gives its memory back. Here the keys and values are in pages of a pool
(``PagedKVCache``), a step's requests are described by a ``PagedBatch``, and two operators take it:

* ``paged_append`` writes the step's keys and values to their pages and returns its queries, keys and
  queries rotated by their position, with the RMS norm of each head before that for models that have
  one (the reference's second family, ``custom_qwen3.py``);
* ``paged_attention`` lets every new token attend its request's tokens up to itself: prompts, chunks
  and single tokens in one call.

Rows of a step are its requests' new tokens, one request after the other. Rows behind the last
request are neither read nor written (a batch padded for a captured graph); a request may have no
new token. Everything the device buffers of a ``PagedBatch`` hold may change between replays of a
captured call, within the bounds that the ``PagedBatch`` was made with.
"""

from __future__ import annotations

import ctypes
import functools
import math
import operator
from typing import Iterable, Sequence

import torch

from .. import _lib
from .decode import workspace

HEAD_DIM = 128
_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_COUNTERS = 16384  # leading floats of the attention's workspace: its arrival counters
_WORKSPACES: dict = {}  # (device, stream) -> the attention's workspace


class PagedBatch:
    """The requests of one step, on the device. Its buffers' contents may change, the buffers and
    the bounds are fixed.

    ``page_table`` (B, P) int32: the pages of request b in order (entries behind its last page are
    not read; an id outside the pool is a page that is not there: its keys are masked, its tokens
    not stored). ``q_start`` (B + 1,) int32: request b's new tokens are rows ``q_start[b] ..
    q_start[b + 1] - 1``. ``lens`` (B,) int32: its tokens with the new ones. ``rows``: at least
    ``q_start[B]``; ``max_new`` and ``max_len``: at least the largest number of new tokens and the
    largest length; ``min_new``: at most the smallest number of new tokens of a request that has
    any. The host never reads the device buffers, so the bounds are the caller's to keep: new
    tokens past ``max_new`` or keys past ``max_len`` may be left out. They choose the launch: a step
    without single tokens is faster with its own ``min_new`` than with 1, which allows for some (512
    tokens at 8192: 80 us against 128)."""

    __slots__ = ("_page_table", "_q_start", "_lens", "_rows", "_max_new", "_max_len", "_min_new",
                 "_requests", "_args")
    page_table, q_start, lens, rows, max_new, max_len, min_new, requests = (
        property(operator.attrgetter(name)) for name in __slots__[:8])

    def __init__(self, page_table: torch.Tensor, q_start: torch.Tensor, lens: torch.Tensor, *,
                 rows: int, max_new: int, max_len: int, min_new: int = 1):
        self._page_table, self._q_start, self._lens = page_table, q_start, lens
        self._rows, self._max_new, self._max_len, self._min_new = rows, max_new, max_len, min_new
        # what every call passes of the batch (its buffers stay where they are): table pointer, row
        # stride and columns, row starts, lengths, requests, rows, bounds, device
        fast = _lib.tensor_calls()
        self._args = None if fast is None else fast.paged_batch(
            page_table, q_start, lens, rows, max_new, max_len, min_new)
        if self._args is None:
            self._args = self._checked()
        self._requests = self._args[5]

    def _checked(self) -> tuple:
        page_table, q_start, lens = self._page_table, self._q_start, self._lens
        rows, max_new, max_len, min_new = self._rows, self._max_new, self._max_len, self._min_new
        shape, n_start, n_lens = page_table.shape, q_start.shape, lens.shape
        if len(shape) != 2 or len(n_start) != 1 or len(n_lens) != 1:
            raise ValueError("page_table must be (B, P), q_start (B + 1,), lens (B,)")
        B, cols = shape
        if n_lens[0] != B or n_start[0] != B + 1:
            raise ValueError("page_table, q_start and lens disagree on the number of requests")
        if not (page_table.dtype == q_start.dtype == lens.dtype == torch.int32):
            raise ValueError("page_table, q_start and lens must be int32")
        ld, unit = page_table.stride()
        if (not q_start.is_contiguous() or not lens.is_contiguous() or (cols > 1 and unit != 1)
                or (B > 1 and ld < cols)):
            raise ValueError("page_table rows, q_start and lens must be contiguous")
        device = page_table.get_device()
        if not (device == q_start.get_device() == lens.get_device()):
            raise ValueError("page_table, q_start and lens must be on one device")
        if not (0 <= min_new <= max_new <= rows and max_len >= 0):
            raise ValueError("need 0 <= min_new <= max_new <= rows and max_len >= 0")
        return (page_table.data_ptr(), max(ld, cols), cols, q_start.data_ptr(), lens.data_ptr(), B,
                rows, max_new, min_new, max_len, device)


class PagedKVCache:
    """A pool of ``pages`` pages of ``page_size`` tokens for every layer (``k[i]`` and ``v[i]``:
    (pages, kv_heads, page_size, 128)), and the requests that hold them. A page id means the same
    page in every layer, so one ``PagedBatch`` serves a whole step."""

    def __init__(self, layers: int, pages: int, kv_heads: int, *, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two of at least 16")
        if layers < 1 or pages < 1 or kv_heads < 1:
            raise ValueError("layers, pages and kv_heads must be positive")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"unsupported dtype {dtype}")
        self.page_size, self.pages = page_size, pages
        dims = (pages, kv_heads, page_size, HEAD_DIM)
        self.k = [torch.empty(dims, dtype=dtype, device=device)]
        self.device = self.k[0].device  # ("cuda": the device that is current now)
        self.k += [torch.empty(dims, dtype=dtype, device=self.device) for _ in range(layers - 1)]
        self.v = [torch.empty(dims, dtype=dtype, device=self.device) for _ in range(layers)]
        self._free = list(range(pages - 1, -1, -1))
        self._held: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A new request of no tokens; returns its id."""
        r = self._next
        self._next += 1
        self._held[r], self._len[r] = [], 0
        return r

    def length(self, request: int) -> int:
        return self._len[self._known(request)]

    def page_ids(self, request: int) -> list[int]:
        return list(self._held[self._known(request)])

    def truncate(self, request: int, length: int) -> None:
        """Forget a request's tokens from ``length`` on (drafted tokens that were not taken)."""
        self._known(request)
        if not 0 <= length <= self._len[request]:
            raise ValueError(f"request {request} has {self._len[request]} tokens, not {length}")
        keep = -(-length // self.page_size)
        held = self._held[request]
        self._free.extend(reversed(held[keep:]))
        del held[keep:]
        self._len[request] = length

    def free(self, request: int) -> None:
        """End a request: its pages go back to the pool."""
        self.truncate(request, 0)
        del self._held[request], self._len[request]

    def _known(self, request: int) -> int:
        if request not in self._len:
            raise ValueError(f"no request {request}")
        return request

    def batch(self, step: Iterable[tuple[int, int]]) -> PagedBatch:
        """The step that adds ``n`` tokens to each (request, n), in this order: takes the pages they
        need, advances the lengths and returns the batch (one copy to the device). Raises, and
        changes nothing, when the pool has too few pages."""
        step = [(int(r), int(n)) for r, n in step]
        if len({r for r, _ in step}) != len(step):
            raise ValueError("a request can appear once in a step")
        want = []
        for r, n in step:
            self._known(r)
            if n < 0:
                raise ValueError("the number of new tokens cannot be negative")
            want.append(-(-(self._len[r] + n) // self.page_size) - len(self._held[r]))
        if sum(want) > len(self._free):
            raise RuntimeError(f"the step needs {sum(want)} pages, {len(self._free)} are free")
        for (r, n), k in zip(step, want):
            for _ in range(k):
                self._held[r].append(self._free.pop())
            self._len[r] += n
        B = len(step)
        cols = max([len(self._held[r]) for r, _ in step], default=0)
        starts = [0]
        for _, n in step:
            starts.append(starts[-1] + n)
        flat = starts + [self._len[r] for r, _ in step]
        for r, _ in step:
            flat += self._held[r] + [-1] * (cols - len(self._held[r]))
        host = torch.tensor(flat, dtype=torch.int32)
        if self.device.type == "cuda":
            host = host.pin_memory()
        dev = host.to(self.device, non_blocking=True)
        new = [n for _, n in step if n > 0]
        return PagedBatch(dev[2 * B + 1:].view(B, cols), dev[:B + 1], dev[B + 1:2 * B + 1],
                          rows=starts[-1], max_new=max(new, default=0),
                          max_len=max([self._len[r] for r, _ in step], default=0),
                          min_new=min(new, default=0))


@functools.lru_cache(maxsize=64)
def _frequencies(values) -> ctypes.Array:
    """64 host doubles, radians per position of each pair (dims j and j + 64), of a theta or as
    given."""
    if isinstance(values, float):
        if not (values > 0.0 and math.isfinite(values)):
            raise ValueError("theta must be positive and finite")
        values = tuple(values ** (-2.0 * j / HEAD_DIM) for j in range(HEAD_DIM // 2))
    if len(values) != HEAD_DIM // 2 or not all(math.isfinite(f) for f in values):
        raise ValueError(f"inv_freq must hold {HEAD_DIM // 2} finite numbers")
    return (ctypes.c_double * (HEAD_DIM // 2))(*values)


def _frequency_address(theta: float | None, inv_freq: Sequence[float] | None) -> ctypes.Array:
    if (theta is None) == (inv_freq is None):
        raise ValueError("give theta or inv_freq, one of them")
    if theta is not None:
        return _frequencies(float(theta))
    if torch.is_tensor(inv_freq):
        if inv_freq.is_cuda:
            raise ValueError("inv_freq is a host sequence (a device tensor would be read back)")
        inv_freq = inv_freq.tolist()
    return _frequencies(tuple(float(f) for f in inv_freq))


def _pools(k_pages: torch.Tensor, v_pages: torch.Tensor, batch: PagedBatch, dtype: torch.dtype,
           device: int) -> tuple:
    """(KV heads, the pools' arguments of a call), checked against each other and the batch."""
    shape, st = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or shape != v_pages.shape or shape[3] != HEAD_DIM:
        raise ValueError("k_pages / v_pages must be (pages, kv_heads, page_size, 128), alike")
    if st != v_pages.stride() or st[3] != 1 or st[2] != HEAD_DIM:
        raise ValueError("pages must hold a head's tokens back to back, with one layout for K and V")
    if k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise ValueError("page and input dtypes differ")
    if not (k_pages.get_device() == v_pages.get_device() == batch._args[10] == device):
        raise ValueError("inputs, pages and batch must be on one device")
    pages, hkv, ps, _ = shape
    if ps < 16 or ps & (ps - 1):
        raise NotImplementedError("page_size must be a power of two of at least 16")
    if batch._max_len > batch._args[2] * ps:
        raise ValueError(f"max_len {batch._max_len} is past the page table "
                         f"({batch._args[2]} pages of {ps})")
    return hkv, (k_pages.data_ptr(), v_pages.data_ptr(), st[0], st[1], pages, ps)


def _row_strides(t: torch.Tensor) -> tuple[int, int]:
    """The row and head strides of (T, heads, 128); those of a size of one are any number."""
    T, heads, _ = t.shape
    st = t.stride()
    sh = st[1] if heads > 1 else HEAD_DIM
    return (st[0] if T > 1 else sh * heads), sh


def paged_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 batch: PagedBatch, *, heads: int, theta: float | None = None,
                 inv_freq: Sequence[float] | None = None, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Write a step's keys and values to their pages; returns its queries (T, heads, 128).

    ``qkv`` (T, W): rows of the fused projection (``heads`` query heads, then as many key heads as
    the pages have, then the value heads, 128 each). Queries and keys are rotated (rotate-half) at
    their token's position by ``theta`` (frequencies theta^(-2j/128)) or by the 64 host numbers
    ``inv_freq`` (scaled frequencies), the angle formed in 64 bits. With ``q_norm`` / ``k_norm``
    ((128,) of qkv's dtype) each query / key head is first normed, x / sqrt(mean(x^2) + eps) * w.
    Everything in fp32, rounded once where it is stored. ``out``: where the queries go (T, heads,
    128), unit last stride: qkv's own query columns, or memory apart from it. A token whose page is not
    there is not stored."""
    freqs = _frequency_address(theta, inv_freq)
    fast = _lib.tensor_calls()
    if fast is not None and out is None and _lib.is_current(batch._args[10]):
        out = fast.paged_append(_lib.stream_on(batch._args[10]), qkv, k_pages, v_pages, batch._args,
                                heads, ctypes.addressof(freqs), q_norm, k_norm, eps)
        if out is not None:
            return out
    shape, st = qkv.shape, qkv.stride()
    if len(shape) != 2 or st[1] != 1:
        raise ValueError("qkv must be (T, W) with unit last stride")
    T, width = shape
    dt, dev = qkv.dtype, qkv.get_device()
    hkv, pools = _pools(k_pages, v_pages, batch, dt, dev)
    if heads <= 0 or width < (heads + 2 * hkv) * HEAD_DIM:
        raise ValueError(f"qkv must hold {heads} + 2 * {hkv} heads of {HEAD_DIM}")
    if batch._rows > T:
        raise ValueError(f"the batch has {batch._rows} rows, qkv {T}")
    for w in (q_norm, k_norm):
        if w is not None and (w.shape != (HEAD_DIM,) or w.dtype != dt or not w.is_contiguous()
                              or w.get_device() != dev):
            raise ValueError("norm weights must be contiguous (128,) vectors of qkv's dtype")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    stream = _lib.stream_of(qkv)
    if out is None:
        out, o_st = qkv.new_empty(T, heads, HEAD_DIM), (heads * HEAD_DIM, HEAD_DIM)
    elif (out.shape != (T, heads, HEAD_DIM) or out.stride(2) != 1 or out.dtype != dt
          or out.get_device() != dev):
        raise ValueError("out must be (T, heads, 128) of qkv's dtype with unit last stride")
    else:
        o_st = _row_strides(out)
    _lib.check(_lib.call_on(
        dev, _lib.calls().dkv_paged_append, stream, _lib.dtype_code(dt), qkv.data_ptr(),
        st[0] if T > 1 else width, out.data_ptr(), *o_st, *pools, *batch._args[:7], heads, hkv,
        HEAD_DIM, _lib.ptr(q_norm), _lib.ptr(k_norm), float(eps), ctypes.addressof(freqs)),
        "dkv_paged_append")
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    batch: PagedBatch, *, scale: float | None = None,
                    out: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Attention of a step's new tokens over their requests' pages (T, heads, 128).

    ``q`` (T, heads, 128), rotated; query head h reads KV head ``h // (heads / kv_heads)``. The new
    token at position t attends its request's tokens 0 .. t (the pages hold them all: the step's own
    are appended first); one that has none to attend (or scores of -infinity alone) gives 0. ``scale`` defaults to 1 / sqrt(128).
    The output is in q's dtype, or in fp32 before that rounding with ``out_dtype=torch.float32``;
    ``out`` may be q itself, or memory apart from it."""
    fast = _lib.tensor_calls()
    if (fast is not None and out is None and out_dtype is None
            and _lib.is_current(batch._args[10])):
        out = fast.paged_attention(_lib.stream_on(batch._args[10]), q, k_pages, v_pages, batch._args,
                                   _SCALE if scale is None else scale, _attention_workspace)
        if out is not None:
            return out
    shape, st = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM:
        raise ValueError("q must be (T, heads, 128)")
    T, hq, _ = shape
    dt, dev = q.dtype, q.get_device()
    hkv, pools = _pools(k_pages, v_pages, batch, dt, dev)
    if hq % hkv or hq == 0:
        raise ValueError(f"{hq} query heads do not divide among {hkv} KV heads")
    if batch._rows > T:
        raise ValueError(f"the batch has {batch._rows} rows, q {T}")
    if st[2] != 1 or st[0] % 8 or st[1] % 8 or q.data_ptr() % 16:
        q, st = q.clone(memory_format=torch.contiguous_format), (hq * HEAD_DIM, HEAD_DIM)
    odt = out_dtype if out_dtype is not None else (out.dtype if out is not None else dt)
    if odt != dt and odt != torch.float32:
        raise ValueError("out_dtype must be the query dtype or float32")
    stream = _lib.stream_of(q)
    if out is None:
        out = torch.empty_like(q, dtype=odt, memory_format=torch.contiguous_format)
        o_st = hq * HEAD_DIM, HEAD_DIM
    elif (out.shape != shape or out.dtype != odt or out.stride(2) != 1
          or out.get_device() != dev):
        raise ValueError("out must be (T, heads, 128) with unit last stride and the requested dtype")
    else:
        o_st = _row_strides(out)
    lib = _lib.calls()
    bounds = batch._args[7:10]
    need = lib.dkv_paged_workspace_floats(batch._requests, batch._rows, hq, hkv, *bounds)
    ws = _attention_workspace(q, stream, need) if need else None
    _lib.check(_lib.call_on(
        dev, lib.dkv_paged_attention, stream, _lib.dtype_code(dt), q.data_ptr(), st[0], st[1],
        *pools, *batch._args[:7], hq, hkv, HEAD_DIM, *bounds,
        _SCALE if scale is None else float(scale), _lib.ptr(ws), ws.numel() if need else 0,
        out.data_ptr(), _lib.dtype_code(odt), *o_st), "dkv_paged_attention")
    return out


def _attention_workspace(q: torch.Tensor, stream: int, floats: int) -> torch.Tensor:
    """Split records and arrival counters (zero before and after a call). Eager calls of a stream, from
    any threads, share its workspace, in that stream's order: a call of two launches makes them
    together, and no other operator writes there. A call under capture gets one of its own in the
    graph's pool, cleared by the graph itself: two captured graphs may be replayed at once."""
    if _lib.call_on(q.get_device(), torch.cuda.is_current_stream_capturing):
        ws = torch.empty(floats, dtype=torch.float32, device=q.device)
        ws[:_COUNTERS].zero_()
        return ws
    return workspace(q.device, stream, floats, _WORKSPACES)
