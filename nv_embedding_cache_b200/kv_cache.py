"""Paged cache of key and value rows over the C ABI (include/nve_b200_kv.h): the cache a serving model keeps beside
its embedding tables, with the verbs of the embedding cache.

* :meth:`PagedKVCache.append` stores the rows of new tokens, turned by their rotary positions (insert);
* :meth:`PagedKVCache.attend` lets one new token per sequence read all rows of its sequence, weighted by softmax
  (lookup + pool), and adds up the attention every row draws (the counters);
* :meth:`PagedKVCache.evict` keeps the rows that drew the most (replacement);
* :func:`rotary` is the rotation alone, differentiable, for training: positions with one or more axes.

A sequence is a row of ``page_table`` (int32 page ids, entries behind the last row are not read) and a length
(int32).  Pages are the caller's to hand out and to free; sequences may share pages as long as no call writes them
(append, accumulated weights, the new pages of an eviction).  Tensors live on the cache's device; calls run on the
current stream of that device, allocate their outputs and scratch from torch, never synchronise, and can be captured
into CUDA graphs.  Page ids and lengths are checked by the kernels; :meth:`PagedKVCache.check` reports.  The cache is
for serving: its methods have no gradient and refuse tensors that ask for one.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import capi

_E4M3 = torch.float8_e4m3fn
_DTYPES = {torch.float32: capi.DTYPE_FLOAT32, torch.float16: capi.DTYPE_FLOAT16, torch.bfloat16: capi.DTYPE_BFLOAT16,
           _E4M3: capi.DTYPE_E4M3}
_INT32 = torch.int32
_INT32_MAX = 0x7fffffff
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_GROUPS = (None, capi.HeadRows * 1, capi.HeadRows * 2)


def _need(ok: bool, message: str) -> None:
    """For checks outside the calls of a decode step; those spell their messages out only when they fail."""
    if not ok:
        raise ValueError(message)


def _call(fn, device: torch.device, *args) -> None:
    """fn(*args, stream) on `device` and its current stream."""
    index = device.index
    if _current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status != capi.NVE_SUCCESS:
        capi.check(status)


def _int32(t: torch.Tensor, device: torch.device, dims: int, name: str) -> torch.Tensor:
    if t.dtype is not _INT32 or t.device != device or t.dim() != dims:
        raise ValueError(f"{name} must be an int32 tensor with {dims} dimension(s) on {device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"the last dimension of {name} must be dense")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[tokens, heads, width] with dense rows."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _head_rows(t: torch.Tensor, out) -> capi.HeadRows:
    e = t.element_size()
    s = t.stride()
    if out is None:
        return capi.HeadRows(t.data_ptr(), None, s[0] * e, s[1] * e, 0, 0, t.shape[1])
    o = out.stride()
    return capi.HeadRows(t.data_ptr(), out.data_ptr(), s[0] * e, s[1] * e, o[0] * e, o[1] * e, t.shape[1])


class RotaryPlan:
    """Frequencies of a rotation with several axes: pair ``i`` of a head row turns by
    ``positions[pair_axis[i], token] * inv_freq[i]``.

    ``inv_freq``: fp32, one per pair, on the device; ``pair_axis``: int32, the axis each pair follows (None: axis 0);
    pairs are values ``(i, i + pairs)`` of a row, or ``(2 i, 2 i + 1)`` when ``interleaved``.  Values behind the last
    pair are passed through.
    """

    def __init__(self, inv_freq: torch.Tensor, pair_axis: torch.Tensor | None = None, num_axes: int = 1, *,
                 interleaved: bool = False):
        _need(inv_freq.is_cuda and inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous(),
              "inv_freq must be a dense fp32 vector on the GPU")
        _need(num_axes >= 1, "num_axes must be positive")
        if pair_axis is not None:
            _int32(pair_axis, inv_freq.device, 1, "pair_axis")
            _need(pair_axis.numel() == inv_freq.numel(), "pair_axis must have one entry per pair")
        self.inv_freq, self.pair_axis = inv_freq, pair_axis
        self.num_pairs, self.num_axes, self.interleaved = inv_freq.numel(), num_axes, bool(interleaved)
        self.device = inv_freq.device
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._constant = (inv_freq.data_ptr(), None if pair_axis is None else pair_axis.data_ptr(), self.num_pairs,
                          int(self.interleaved), self.status.data_ptr())

    @classmethod
    def sections(cls, pairs_per_axis, *, base: float = 10000.0, restart: bool = False, interleaved: bool = False,
                 device="cuda") -> "RotaryPlan":
        """The axes in turn, ``pairs_per_axis[a]`` pairs each.  One ladder of frequencies
        ``base ** (-i / pairs)`` runs over all of them, or over each axis anew with ``restart``."""
        counts = [int(n) for n in pairs_per_axis]
        _need(bool(counts) and min(counts) >= 0 and sum(counts) > 0, "pairs_per_axis must hold counts")
        axis = [a for a, n in enumerate(counts) for _ in range(n)]
        if restart:
            freq = [base ** (-i / n) for n in counts for i in range(n)]
        else:
            freq = [base ** (-i / len(axis)) for i in range(len(axis))]
        return cls(torch.tensor(freq, dtype=torch.float64).float().to(device),
                   torch.tensor(axis, dtype=torch.int32, device=device), len(counts), interleaved=interleaved)

    def check(self) -> None:
        """Waits for the device and raises RuntimeError if an entry of pair_axis was no axis (its pair did not turn)."""
        if int(self.status.item()):
            self.status.zero_()
            raise RuntimeError("rotary plan: an entry of pair_axis is not in [0, num_axes)")

    def _args(self, positions: torch.Tensor, tokens: int, device: torch.device) -> capi.Rotary:
        if positions.dtype is not _INT32 or positions.device != device or device != self.device:
            raise ValueError(f"positions must be int32 and, like the plan, on {device}")
        if positions.dim() == 1:
            positions = positions[None]
        if tuple(positions.shape) != (self.num_axes, tokens):
            raise ValueError(f"positions must be [{self.num_axes}, {tokens}]")
        s = positions.stride()
        return capi.Rotary(positions.data_ptr(), s[0], s[1], self.num_axes, *self._constant)


def _turn(plan: RotaryPlan, positions: torch.Tensor, tensors, backward: bool):
    """New tensors with the rows of `tensors` ([tokens, heads, width] each) turned."""
    tensors = [_rows(t) for t in tensors]
    outs = [torch.empty_like(t) for t in tensors]
    first = tensors[0]
    shape = first.shape
    groups = _GROUPS[len(outs)](*map(_head_rows, tensors, outs))
    _call(capi.lib.nve_b200_rotary, first.device, plan._args(positions, shape[0], first.device), _DTYPES[first.dtype],
          shape[2], shape[0], groups, len(outs), backward)
    return outs


class _RotaryFunction(torch.autograd.Function):
    """The rotation is linear in its rows and its transpose is the rotation by the negated angles, so the gradient is
    the same function again (and has a gradient in turn)."""

    @staticmethod
    def forward(ctx, plan, positions, backward, *tensors):
        ctx.plan, ctx.turned_back = plan, backward
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        return tuple(_turn(plan, positions, tensors, backward))

    @staticmethod
    def backward(ctx, *grads):
        positions, = ctx.saved_tensors
        out = [None] * len(grads)
        at = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[3 + i]]
        if at:
            taken = [grads[i] for i in at]
            if torch.is_grad_enabled():
                turned = _RotaryFunction.apply(ctx.plan, positions, not ctx.turned_back, *taken)
            else:
                turned = _turn(ctx.plan, positions, taken, not ctx.turned_back)
            for i, g in zip(at, turned):
                out[i] = g
        return (None, None, None, *out)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, plan: RotaryPlan):
    """Queries and keys ([tokens, heads, width], fp32, fp16 or bf16) turned by their positions ([axes, tokens] int32).
    Returns new tensors (q', k'), q' alone when `k` is None.  Differentiable in q and k, any number of times."""
    tensors = (q,) if k is None else (q, k)
    shape, dtype, device = q.shape, q.dtype, q.device
    if not q.is_cuda or len(shape) != 3:
        raise ValueError("q and k must be [tokens, heads, width] on the GPU")
    if dtype not in _DTYPES or dtype is _E4M3:
        raise ValueError("q and k must be fp32, fp16 or bf16")
    if k is not None and (k.dtype is not dtype or k.device != device or k.dim() != 3 or k.shape[0] != shape[0]
                          or k.shape[2] != shape[2]):
        raise ValueError("q and k must agree in type, device, tokens and width")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _RotaryFunction.apply(plan, positions, False, *tensors)
    else:
        out = _turn(plan, positions, tensors, False)
    return out[0] if k is None else tuple(out)


class PagedKVCache:
    """Key and value rows in pages, ``keys`` and ``values`` [num_pages, page_size, heads, width] with any strides
    (a page may hold its rows head by head: a permuted view), fp16, bf16 or E4M3 (``torch.float8_e4m3fn``, stored value =
    value / scale of the head; ``key_scale`` / ``value_scale`` fp32 [heads]).  ``weights`` fp32
    [num_pages, heads, page_size]: the attention every row has drawn since it was stored (None: not kept)."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, weights: torch.Tensor | None = None, *,
                 key_scale: torch.Tensor | None = None, value_scale: torch.Tensor | None = None):
        _need(keys.is_cuda and keys.dim() == 4 and keys.dtype in _DTYPES and keys.dtype != torch.float32,
              "keys must be [num_pages, page_size, heads, width] in fp16, bf16 or E4M3 on the GPU")
        _need(values.shape == keys.shape and values.dtype == keys.dtype and values.device == keys.device,
              "values must match keys")
        _need(keys.numel() > 0 and keys.stride(3) == 1 and values.stride(3) == 1, "rows must be dense and not empty")
        pages, size, heads, width = keys.shape
        self.keys, self.values, self.weights = keys, values, weights
        self.key_scale, self.value_scale = key_scale, value_scale
        self.num_pages, self.page_size, self.num_heads, self.head_width = pages, size, heads, width
        self.dtype, self.device = keys.dtype, keys.device
        if weights is not None:
            _need(weights.dtype == torch.float32 and weights.device == keys.device and weights.is_contiguous()
                  and tuple(weights.shape) == (pages, heads, size),
                  "weights must be dense fp32 [num_pages, heads, page_size]")
        for s in (key_scale, value_scale):
            if s is not None:
                _need(s.dtype == torch.float32 and s.device == keys.device and s.is_contiguous()
                      and tuple(s.shape) == (heads,), "scales must be dense fp32 [heads]")
                _need(keys.dtype == torch.float8_e4m3fn, "scales belong to E4M3 caches")
        self.status = torch.zeros(1, dtype=torch.int32, device=keys.device)
        e = keys.element_size()

        def strides(t):
            return (C.c_int64 * 3)(*[t.stride(i) * e for i in range(3)])

        def address(t):
            return None if t is None else t.data_ptr()

        self._view = capi.KvCache(keys.data_ptr(), values.data_ptr(), strides(keys), strides(values), address(weights),
                                  address(key_scale), address(value_scale), _DTYPES[keys.dtype], pages, size, heads,
                                  width, self.status.data_ptr())
        self._scratch_sizes = {}

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_heads: int, head_width: int, dtype: torch.dtype, *,
                 device="cuda", weights: bool = True, key_scale: torch.Tensor | None = None,
                 value_scale: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache of its own, rows head by head inside a page: one head's part of a page is one piece of memory."""
        shape = (num_pages, num_heads, page_size, head_width)
        k, v = (torch.empty(shape, dtype=dtype, device=device).permute(0, 2, 1, 3) for _ in range(2))
        w = torch.zeros((num_pages, num_heads, page_size), device=device) if weights else None
        return cls(k, v, w, key_scale=key_scale, value_scale=value_scale)

    def check(self) -> None:
        """Waits for the device and raises RuntimeError if a kernel met a bad page id or length since the last call."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = [text for bit, text in ((capi.KV_BAD_PAGE, "a page id outside the pool"),
                                           (capi.KV_BAD_LENGTH, "a length outside the page table or max_length"),
                                           (capi.KV_TIMED_OUT, "a wait that ran into its limit"))
                    if bits & bit]
            raise RuntimeError("paged cache: " + " and ".join(what))

    def _table(self, page_table: torch.Tensor, lengths: torch.Tensor) -> int:
        _int32(page_table, self.device, 2, "page_table")
        _int32(lengths, self.device, 1, "lengths")
        n = page_table.shape[0]
        if lengths.shape[0] != n:
            raise ValueError("page_table and lengths must have one row per sequence")
        return n

    def _most_rows(self, pages: int, max_length: int | None) -> int:
        rows = pages * self.page_size
        if max_length is None:
            max_length = rows
        if not 0 <= max_length <= rows or rows > _INT32_MAX:
            raise ValueError(f"max_length must be in [0, {rows}], the rows of the page table, which must be below 2^31")
        return max_length

    def _row_dtype(self, t: torch.Tensor, name: str) -> int:
        if t.device != self.device or t.dim() != 3 or t.shape[2] != self.head_width:
            raise ValueError(f"{name} must be [.., heads, {self.head_width}] on {self.device}")
        dtype = t.dtype
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient, which the cache does not give: call under torch.no_grad()")
        if dtype is _E4M3 or (dtype is not self.dtype and (self.dtype is not _E4M3 or dtype not in _DTYPES
                                                           or dtype is torch.float32)):
            raise ValueError(f"{name} must have the cache's type, or fp16 or bf16 for an E4M3 cache")
        return _DTYPES[dtype]

    def append(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
               q: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
               positions: torch.Tensor | None = None, rotary: RotaryPlan | None = None):
        """Stores the rows of new tokens behind the ``lengths`` rows their sequences hold.  ``k``, ``v`` (and ``q``):
        [tokens, heads, width], sequence after sequence; ``offsets`` int32 [sequences + 1]: where each begins (None:
        the same number each).  Keys and queries are turned by ``rotary`` at ``positions`` ([axes, tokens]).  Tokens
        outside ``offsets`` are padding: nothing of theirs is stored and their queries are zero.  Returns (turned
        queries or None, new lengths); a sequence that outgrows its page table keeps what fits (:meth:`check`)."""
        n = self._table(page_table, lengths)
        dtype = self._row_dtype(k, "k")
        tokens = k.shape[0]
        self._row_dtype(v, "v")
        if v.dtype is not k.dtype or v.shape != k.shape or k.shape[1] != self.num_heads:
            raise ValueError("k and v must agree and have the cache's heads")
        k, v = _rows(k), _rows(v)
        turned = None
        if q is None:
            q_rows = capi.HeadRows()
        else:
            self._row_dtype(q, "q")
            if q.dtype is not k.dtype or q.shape[0] != tokens:
                raise ValueError("q must have the type and the tokens of k")
            q = _rows(q)
            turned = torch.empty_like(q)
            q_rows = _head_rows(q, turned)
        if offsets is not None:
            _int32(offsets, self.device, 1, "offsets")
            if offsets.shape[0] != n + 1:
                raise ValueError("offsets must have one entry more than there are sequences")
        if (rotary is None) != (positions is None):
            raise ValueError("positions and rotary go together")
        turn = None if rotary is None else C.pointer(rotary._args(positions, tokens, self.device))
        new_lengths = torch.empty_like(lengths, memory_format=torch.contiguous_format)
        args = capi.KvAppend(dtype, tokens, q_rows, _head_rows(k, None), _head_rows(v, None), turn,
                             page_table.data_ptr(), page_table.stride(0), page_table.shape[1], n, lengths.data_ptr(),
                             None if offsets is None else offsets.data_ptr(), new_lengths.data_ptr(), 1)
        _call(capi.lib.nve_b200_kv_append, self.device, self._view, args)
        return turned, new_lengths

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
               max_length: int | None = None, accumulate_weights: bool = False, return_lse: bool = False):
        """Attention of one new token per sequence over its rows; ``q`` [sequences, query heads, width], query head i
        reads key head ``i // (query heads / heads)``.  Returns out (like q), or (out, lse) with lse fp32 [sequences,
        query heads], the natural log of the sum of exponentials: what joins this result with another cache's.  An
        empty sequence gives zeros and -inf.  ``max_length`` (the page table's rows if None) bounds the lengths and
        with it the scratch; ``accumulate_weights`` adds each row's probabilities to ``weights``."""
        n = self._table(page_table, lengths)
        dtype = self._row_dtype(q, "q")
        if q.shape[0] != n:
            raise ValueError("q must have one row per sequence")
        heads, width, device = q.shape[1], self.head_width, self.device
        pages = page_table.shape[1]
        max_length = self._most_rows(pages, max_length)
        q = _rows(q)
        e = q.element_size()
        s = q.stride()
        if q.data_ptr() % 16 or s[0] * e % 16 or s[1] * e % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            s = q.stride()
        out = torch.empty((n, heads, width), dtype=q.dtype, device=device)
        lse = torch.empty((n, heads), dtype=torch.float32, device=device) if return_lse else None
        args = capi.KvAttend(dtype, n, heads, q.data_ptr(), s[0] * e, s[1] * e, out.data_ptr(), heads * width * e,
                             width * e, None if lse is None else lse.data_ptr(), page_table.data_ptr(),
                             page_table.stride(0), pages, lengths.data_ptr(), max_length,
                             1.0 / math.sqrt(width) if scale is None else scale, accumulate_weights)
        key = (n, heads, max_length, accumulate_weights)
        size = self._scratch_sizes.get(key)
        if size is None:
            size = C.c_size_t()
            _call(capi.lib.nve_b200_kv_attend, device, self._view, args, None, size)
            if len(self._scratch_sizes) >= 4096:
                self._scratch_sizes.clear()
            self._scratch_sizes[key] = size
        if n:
            scratch = torch.empty(size.value, dtype=torch.uint8, device=device)
            _call(capi.lib.nve_b200_kv_attend, device, self._view, args, scratch.data_ptr(), size)
        return (out, lse) if return_lse else out

    def evict(self, page_table: torch.Tensor, lengths: torch.Tensor, new_page_table: torch.Tensor, budget: int, *,
              sinks: int = 0, recent: int = 0, max_length: int | None = None):
        """Presses every sequence to at most ``budget`` rows, each head on its own: the first ``sinks`` and the last
        ``recent`` rows stay, and of the others those with the largest weight (equal ones: the earliest).  The rows
        that stay are copied, in order and with their weights, to the pages of ``new_page_table``, which must not be
        pages that are read; the old pages are the caller's to free.  Returns (kept [sequences, heads, budget] int32:
        the old row of each new one, -1 behind the last; new lengths)."""
        n = self._table(page_table, lengths)
        _int32(new_page_table, self.device, 2, "new_page_table")
        if new_page_table.shape[0] != n:
            raise ValueError("new_page_table must have one row per sequence")
        if not 0 < budget <= _INT32_MAX or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError("budget must be positive and hold sinks + recent rows")
        pages = page_table.shape[1]
        max_length = self._most_rows(pages, max_length)
        kept = torch.empty((n, self.num_heads, budget), dtype=_INT32, device=self.device)
        new_lengths = torch.empty_like(lengths, memory_format=torch.contiguous_format)
        args = capi.KvEvict(n, page_table.data_ptr(), page_table.stride(0), pages, lengths.data_ptr(), max_length,
                            new_page_table.data_ptr(), new_page_table.stride(0), new_page_table.shape[1], budget, sinks,
                            recent, kept.data_ptr(), new_lengths.data_ptr())
        _call(capi.lib.nve_b200_kv_evict, self.device, self._view, args)
        return kept, new_lengths
