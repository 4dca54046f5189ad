"""A paged key/value cache, exact attention over it, and eviction.

Keys and values of many sequences live in pages of a fixed number of slots:
``k_pages``, ``v_pages`` ``[num_pages, page_size, h_kv, d]`` (any strides with a
contiguous last dimension; :class:`PagedCache` keeps a head's rows of a page
side by side).  Slot ``j`` of sequence ``s`` is row ``j % page_size`` of page
``page_table[s, j // page_size]``, and ``kv_lens[s]`` slots are filled.

A call takes a ragged batch: ``q_starts [B + 1]`` splits the new rows among the
sequences, and the rows of a sequence are its last cached positions
(``kv_lens`` counts them).  The lengths stay on the device -- no op copies them
back or waits -- so a call can be captured in a CUDA graph and replayed with
other lengths.

The reference keeps no cache.  These ops are exact attention for what runs
next to its sparse attention: dense layers, prompts too short to route, and
caches that must not grow (:func:`paged_evict`).  They serve; they have no
gradient: a backward pass that reaches :func:`paged_attention` raises, and what was
appended is cut off from its history.

Errors in the data (a page number outside the cache, lengths that do not fit)
are found on the device and raised by a later op call or by
:func:`ssa_b200.check_errors`.
"""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib as L
from . import _status as S
from .ops import _dtype_code, _last_contig, _require_cuda

_APPEND, _ATTEND, _EVICT = range(3)


_raw_stream = torch._C._cuda_getCurrentRawStream      # torch.cuda.current_stream(i).cuda_stream, without the object
_i32, _f32 = torch.int32, torch.float32


def _index(t: torch.Tensor, name: str, key: int, rows: int) -> torch.Tensor:
    """An int32 vector of ``rows`` entries (any number: -1) on device ``key``."""
    if t.dtype is _i32 and t.dim() == 1 and t.get_device() == key and (rows < 0 or t.shape[0] == rows):
        return t if t.stride(0) == 1 else t.contiguous()
    return _refuse_index(t, name, key, 1, rows)


def _table(t: torch.Tensor, name: str, key: int, rows: int) -> torch.Tensor:
    """An int32 page table ``[rows, *]`` on device ``key``."""
    if t.dtype is _i32 and t.dim() == 2 and t.get_device() == key and t.shape[0] == rows:
        return t if t.stride(1) == 1 else t.contiguous()
    return _refuse_index(t, name, key, 2, rows)


def _refuse_index(t, name, key, dims, rows):
    if t.get_device() != key:
        raise RuntimeError(f"tensors on different devices: cuda:{key} and {t.device} ({name})")
    if t.dtype is not _i32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    want = ", ".join([str(rows) if rows >= 0 else "*"] + ["*"] * (dims - 1))
    raise ValueError(f"{name} must have shape [{want}], got {list(t.shape)}")


def _check_rows(t, name, key, dtype, shape):
    """``[rows, heads, d]`` of the cache's device and type, last dimension contiguous."""
    if t.get_device() != key:
        _require_cuda(t)
        raise RuntimeError(f"tensors on different devices: cuda:{key} and {t.device} ({name})")
    if t.dtype is not dtype:
        raise TypeError(f"{name} ({t.dtype}) must have the cache's dtype {dtype}")
    return _last_contig(t)


def _cache_args(k_pages, v_pages, page_table, kv_lens, weights, op):
    """The device's number, the filled :class:`SsaPagedCache` (with the op's error
    word), whether to wait for errors, and the index tensors the struct points into."""
    key = k_pages.get_device()
    if not k_pages.is_cuda or v_pages.get_device() != key:
        _require_cuda(k_pages, v_pages)
    shape = k_pages.shape
    if len(shape) != 4 or shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must both be [num_pages, page_size, h_kv, d], got "
                         f"{list(shape)} and {list(v_pages.shape)}")
    if k_pages.dtype is not v_pages.dtype:
        raise TypeError(f"k_pages, v_pages dtypes differ: {k_pages.dtype}, {v_pages.dtype}")
    kp, kn, kh, kd = k_pages.stride()
    vp, vn, vh, vd = v_pages.stride()
    # the pages are written in place, so a copy would be of no use
    if kd != 1 or vd != 1:
        raise ValueError("the last dimension of k_pages and v_pages must be contiguous")
    kv_lens = _index(kv_lens, "kv_lens", key, -1)
    batch = kv_lens.shape[0]
    page_table = _table(page_table, "page_table", key, batch)
    w, wp, wn, wh = None, 0, 0, 0
    if weights is not None:
        if weights.get_device() != key:
            raise RuntimeError(f"tensors on different devices: cuda:{key} and {weights.device} (weights)")
        if weights.dtype is not _f32:
            raise TypeError(f"weights must be float32, got {weights.dtype}")
        if weights.shape != shape[:3]:
            raise ValueError(f"weights must be [num_pages, page_size, h_kv] = {list(shape[:3])}, got "
                             f"{list(weights.shape)}")
        w, (wp, wn, wh) = weights.data_ptr(), weights.stride()
    num_pages, page_size, h_kv, d = shape
    word, sync = S.host_word(key, op)
    c = L.SsaPagedCache(batch, page_table.shape[1], page_size, h_kv, d, _dtype_code(k_pages), num_pages,
                        k_pages.data_ptr(), kp, kn, kh, v_pages.data_ptr(), vp, vn, vh, w, wp, wn, wh,
                        page_table.data_ptr(), page_table.stride(0), kv_lens.data_ptr(), word)
    return key, c, sync, (page_table, kv_lens)


def _finish(key, sync, name, code):
    if code:
        L.check(name, code)
    if sync:
        S.host_word_done(torch.device("cuda", key))


def _launch(key, fn, *args):
    if torch.cuda.current_device() == key:
        return fn(*args, _raw_stream(key))
    with torch.cuda.device(key):
        return fn(*args, _raw_stream(key))


def _call(key, sync, fn, *args):
    _finish(key, sync, fn.__name__, _launch(key, fn, *args))


# One workspace per (device, stream), kept: calls on a stream follow one another,
# also those of several threads, which take turns to launch (S.Workspace).
# A capture takes its own (its graph owns that memory), and so do rare large
# ones.  The head of a workspace is zero before a call and after it.
_KEPT = 96 << 20


def _new_workspace(nbytes: int, like: torch.Tensor) -> S.Workspace:
    ws = like.new_empty((nbytes,), dtype=torch.uint8)
    ws[:L.SSA_PAGED_ZEROED].zero_()
    return S.Workspace(ws)


def _workspace(key: int, nbytes: int, like: torch.Tensor) -> S.Workspace:
    if nbytes > _KEPT or torch.cuda.is_current_stream_capturing():
        return _new_workspace(nbytes, like)
    at = key, _raw_stream(key)
    ws = S.workspaces.get(at)
    if ws is None or ws.buffer.numel() < nbytes:
        with torch.cuda.device(key):
            ws = _new_workspace(nbytes, like)
        S.workspaces[at] = ws            # only now: another thread may take it at once
    return ws


def paged_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, q_starts: torch.Tensor, kv_lens: torch.Tensor,
                 weights: Optional[torch.Tensor] = None) -> None:
    """Writes new keys and values into the cache, in place.

    Args:
        k_new, v_new: ``[T, h_kv, d]``, the rows of all sequences one after another.
        k_pages, v_pages: ``[num_pages, page_size, h_kv, d]``, written.
        page_table: ``[B, max_pages]`` int32.
        q_starts: ``[B + 1]`` int32: rows ``q_starts[s] .. q_starts[s + 1] - 1`` are
            sequence ``s``'s and go to its slots ``kv_lens[s] - n .. kv_lens[s] - 1``.
        kv_lens: ``[B]`` int32, the lengths with the new rows counted.
        weights: optional ``[num_pages, page_size, h_kv]`` float32 slot weights;
            those of the written slots become 0.
    """
    if k_pages.is_cuda:
        # the plain case in one step; whatever it does not take is looked at below
        key = k_pages.get_device()
        word, sync = S.host_word(key, _APPEND)
        code = L.paged_call().append(k_new, v_new, k_pages, v_pages, page_table, q_starts, kv_lens, weights, word)
        if code is not None:
            return _finish(key, sync, "ssa_paged_append", code)
    key, c, sync, keep = _cache_args(k_pages, v_pages, page_table, kv_lens, weights, _APPEND)
    dtype, shape = k_pages.dtype, k_new.shape
    k_new = _check_rows(k_new, "k_new", key, dtype, shape)
    v_new = _check_rows(v_new, "v_new", key, dtype, shape)
    if shape != v_new.shape or len(shape) != 3 or shape[1] != c.h_kv or shape[2] != c.d:
        raise ValueError(f"k_new and v_new must be [rows, {c.h_kv}, {c.d}], got {list(shape)} and {list(v_new.shape)}")
    q_starts = _index(q_starts, "q_starts", key, c.batch + 1)
    kn, kh, _ = k_new.stride()
    vn, vh, _ = v_new.stride()
    a = L.SsaPagedAppendArgs(shape[0], q_starts.data_ptr(), k_new.data_ptr(), kn, kh, v_new.data_ptr(), vn, vh)
    _call(key, sync, L.lib().ssa_paged_append, c, a)


class _NoGradient(torch.autograd.Function):
    """Hands a result on as one of its inputs' that fails where a gradient is asked of it."""

    @staticmethod
    def forward(ctx, result, *inputs):
        ctx.mark_dirty(result)
        return result

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("paged_attention has no gradient (it serves): train with sparse_exact_attention or "
                           "dense_attention, or run it under torch.no_grad()")


def _results(q, k_pages, v_pages, out, lse):
    """What paged_attention returns (``lse`` None: not asked for)."""
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        out = _NoGradient.apply(out, q, k_pages, v_pages)
        lse = None if lse is None else _NoGradient.apply(lse, q, k_pages, v_pages)
    return out if lse is None else (out, lse)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    q_starts: torch.Tensor, kv_lens: torch.Tensor, scale: Optional[float] = None,
                    is_causal: bool = True, weights: Optional[torch.Tensor] = None, return_lse: bool = False
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Softmax attention of a ragged batch of new rows over the paged cache.

    Args:
        q: ``[T, h_q, d]``, the rows of all sequences one after another, split by
            ``q_starts`` as in :func:`paged_append`; query head ``e`` reads KV head
            ``e // (h_q // h_kv)``.
        scale: logits are ``(q . k) / scale``; default ``sqrt(d)`` (a divisor, as in
            :func:`ssa_b200.sparse_exact_attention`).
        is_causal: row ``i`` of a sequence's ``n`` sees the slots
            ``j <= kv_lens[s] - n + i``; otherwise every filled slot.
        weights: optional ``[num_pages, page_size, h_kv]`` float32; every slot's
            weight grows, in place, by the attention it receives in this call,
            summed over the sequence's rows and the heads of its group.  A page
            shared by several sequences of the call collects from all of them
            (in no fixed order of additions).
        return_lse: also return the rows' log-sum-exp of the logits.

    Returns ``[T, h_q, d]`` in ``q``'s dtype (and ``[T, h_q]`` float32).  A row that
    sees no slot gets zeros (and ``-inf``).  Rows outside ``q_starts`` are not
    written.  There is no gradient: a backward pass through the results raises
    ``RuntimeError``.

    Sums and statistics are float32.  A 16-bit call of more than 16 rows (new rows x
    heads of a group) per sequence on average holds the softmax weights in ``q``'s
    dtype for their product with the values, smaller calls in two such terms: so a
    row's last bits can differ with what else is in its batch.  Threads that share a
    stream take turns to launch.
    """
    if k_pages.is_cuda:
        key = k_pages.get_device()
        word, sync = S.host_word(key, _ATTEND)            # before the look-up: it drops workspaces left unfit
        ws = S.workspaces.get((key, _raw_stream(key)))
        if ws is not None and not torch.cuda.is_current_stream_capturing():
            with ws.launching:
                done = L.paged_call().attend(q, k_pages, v_pages, page_table, q_starts, kv_lens, scale, is_causal,
                                             weights, return_lse, word, ws.buffer)
            if done is not None:
                code, out, lse = done
                _finish(key, sync, "ssa_paged_attn", code)
                return _results(q, k_pages, v_pages, out, lse)
    key, c, sync, keep = _cache_args(k_pages, v_pages, page_table, kv_lens, weights, _ATTEND)
    shape = q.shape
    q = _check_rows(q, "q", key, k_pages.dtype, shape)
    if len(shape) != 3 or shape[2] != c.d:
        raise ValueError(f"q must be [rows, h_q, {c.d}], got {list(shape)}")
    rows, h_q, d = shape
    if c.h_kv < 1 or h_q % c.h_kv:
        raise ValueError("num_q_heads must be divisible by num_kv_heads")
    q_starts = _index(q_starts, "q_starts", key, c.batch + 1)
    qn, qh, _ = q.stride()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((rows, h_q), dtype=_f32) if return_lse else None
    a = L.SsaPagedAttnArgs(rows, q_starts.data_ptr(), h_q, 1 if is_causal else 0,
                           math.sqrt(d) if scale is None else float(scale), q.data_ptr(), qn, qh, out.data_ptr(),
                           h_q * d, d, lse.data_ptr() if return_lse else None)
    lib = L.lib()
    nbytes = lib.ssa_paged_attn_workspace_size(c, a)
    ws = _workspace(key, nbytes, q)
    with ws.launching:
        code = _launch(key, lib.ssa_paged_attn, c, a, ws.buffer.data_ptr(), nbytes)
    _finish(key, sync, "ssa_paged_attn", code)
    return _results(q, k_pages, v_pages, out, lse)


def _check_budget(budget: int, recent: int) -> None:
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"budget {budget}, recent {recent}: need budget >= 1 and 0 <= recent <= budget")


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, weights: torch.Tensor, page_table: torch.Tensor,
                kv_lens: torch.Tensor, new_table: torch.Tensor, budget: int, recent: int = 0
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cuts every sequence's cache back to ``budget`` slots per KV head.

    Each (sequence, KV head) keeps ``min(kv_len, budget)`` slots: its last ``recent``
    and the heaviest of the others by ``weights`` (the lower slot first among equal
    weights).  Keys, values and weights of the kept slots are copied, in order, to
    the first slots of the pages ``new_table [B, *]`` names; these must not be pages
    that ``page_table`` uses, which stay as they are (other sequences may share them).

    Returns ``kept [B, h_kv, budget]`` int32, the kept slots in ascending order
    followed by -1, and the new lengths ``[B]`` int32.
    """
    if weights is None:
        raise ValueError("weights is needed: eviction ranks slots by them")
    budget, recent = int(budget), int(recent)
    if k_pages.is_cuda:
        key = k_pages.get_device()
        word, sync = S.host_word(key, _EVICT)
        done = L.paged_call().evict(k_pages, v_pages, weights, page_table, kv_lens, new_table, budget, recent, word)
        if done is not None:
            code, kept, new_lens = done
            _finish(key, sync, "ssa_paged_evict", code)
            return kept, new_lens
    key, c, sync, keep = _cache_args(k_pages, v_pages, page_table, kv_lens, weights, _EVICT)
    _check_budget(budget, recent)
    new_table = _table(new_table, "new_table", key, c.batch)
    kept = kv_lens.new_empty((c.batch, c.h_kv, budget))
    new_lens = kv_lens.new_empty((c.batch,))
    a = L.SsaPagedEvictArgs(budget, recent, new_table.shape[1], new_table.data_ptr(), new_table.stride(0),
                            kept.data_ptr(), new_lens.data_ptr())
    _call(key, sync, L.lib().ssa_paged_evict, c, a)
    return kept, new_lens


class PagedBatch:
    """The sequences of one step: index tensors of the three ops, made once and
    used by every layer."""

    __slots__ = ("ids", "q_lens", "kv_lens_host", "page_table", "q_starts", "kv_lens")

    def __init__(self, ids, q_lens, kv_lens, page_table, q_starts, kv_lens_dev):
        self.ids, self.q_lens, self.kv_lens_host = ids, q_lens, kv_lens
        self.page_table, self.q_starts, self.kv_lens = page_table, q_starts, kv_lens_dev


class PagedCache:
    """Pages, and which of them hold which sequence, for ``num_layers`` layers on one GPU.

    A step: :meth:`extend` makes room for the new rows of some sequences and
    returns their :class:`PagedBatch`; then each layer calls :meth:`append` and
    :meth:`attend` with it.  :meth:`evict` cuts sequences back to a budget (with
    ``track_weights=True``, where :meth:`attend` counts the attention every slot
    receives).  Page numbers are handed out on the host; pages given back are
    reused at once, which is safe for work on one stream."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, num_layers: int = 1,
                 dtype=torch.bfloat16, device="cuda", track_weights: bool = False):
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.num_pages, self.num_layers = page_size, num_pages, num_layers
        # zeros, not garbage: slots past a length are loaded (and masked) with their tile
        shape = (num_layers, num_pages, num_kv_heads, page_size)
        self.k_pages = torch.zeros(shape + (head_dim,), dtype=dtype, device=self.device).transpose(2, 3)
        self.v_pages = torch.zeros(shape + (head_dim,), dtype=dtype, device=self.device).transpose(2, 3)
        self.weights = (torch.zeros(shape, dtype=torch.float32, device=self.device).transpose(2, 3)
                        if track_weights else None)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages = {}
        self._len = {}
        self._next = 0

    # -- sequences ---------------------------------------------------------
    def add(self) -> int:
        """A new, empty sequence's id."""
        sid, self._next = self._next, self._next + 1
        self._pages[sid], self._len[sid] = [], 0
        return sid

    def remove(self, sid: int) -> None:
        """Gives the sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(sid)))
        del self._len[sid]

    def length(self, sid: int) -> int:
        return self._len[sid]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _pages_for(self, n: int) -> int:
        return -(-n // self.page_size)

    def _upload(self, pages: Sequence[List[int]], *vectors: Sequence[int]):
        """Page lists as a padded table, and integer vectors, in one copy."""
        width = max([len(p) for p in pages] + [1])
        flat = [x for p in pages for x in p + [0] * (width - len(p))]
        for v in vectors:
            flat.extend(v)
        dev = torch.tensor(flat, dtype=torch.int32).pin_memory().to(self.device, non_blocking=True)
        at = len(pages) * width
        parts = [dev[:at].view(len(pages), width)]
        for v in vectors:
            parts.append(dev[at:at + len(v)])
            at += len(v)
        return parts

    def extend(self, ids: Sequence[int], new_rows: Sequence[int]) -> PagedBatch:
        """Room for ``new_rows[i]`` more rows of sequence ``ids[i]``; nothing changes
        when the free pages do not suffice (``RuntimeError``)."""
        ids, q_lens = list(ids), [int(n) for n in new_rows]
        if len(ids) != len(q_lens) or len(set(ids)) != len(ids):
            raise ValueError("ids must be distinct and match new_rows")
        if any(n < 0 for n in q_lens):
            raise ValueError("new_rows must not be negative")
        kv = [self._len[s] + n for s, n in zip(ids, q_lens)]
        need = [self._pages_for(n) - len(self._pages[s]) for s, n in zip(ids, kv)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"paged cache full: {sum(need)} pages needed, {len(self._free)} free")
        for s, n, more in zip(ids, kv, need):
            self._pages[s].extend(self._free.pop() for _ in range(more))
            self._len[s] = n
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        table, q_starts, kv_dev = self._upload([self._pages[s] for s in ids], starts, kv)
        return PagedBatch(ids, q_lens, kv, table, q_starts, kv_dev)

    # -- one layer of a step -------------------------------------------------
    def append(self, batch: PagedBatch, k_new: torch.Tensor, v_new: torch.Tensor, layer: int = 0) -> None:
        """:func:`paged_append` of the batch's rows to one layer."""
        paged_append(k_new, v_new, self.k_pages[layer], self.v_pages[layer], batch.page_table, batch.q_starts,
                     batch.kv_lens, None if self.weights is None else self.weights[layer])

    def attend(self, batch: PagedBatch, q: torch.Tensor, layer: int = 0, scale: Optional[float] = None,
               is_causal: bool = True) -> torch.Tensor:
        """:func:`paged_attention` of the batch's rows over one layer (weights
        counted where the cache tracks them)."""
        return paged_attention(q, self.k_pages[layer], self.v_pages[layer], batch.page_table, batch.q_starts,
                               batch.kv_lens, scale, is_causal, None if self.weights is None else self.weights[layer])

    # -- between steps ---------------------------------------------------------
    def evict(self, ids: Sequence[int], budget: int, recent: int = 0) -> List[int]:
        """Cuts the sequences longer than ``budget`` back to it in every layer
        (:func:`paged_evict`); returns their ids.  The copies go to free pages,
        so at least one sequence's budget of them must be free; as many
        sequences as fit are cut at a time.  Where a call fails, the sequences
        not yet cut in every layer keep their pages and lengths."""
        if self.weights is None:
            raise ValueError("the cache keeps no weights: make it with track_weights=True")
        ids, budget, recent = list(ids), int(budget), int(recent)
        if len(set(ids)) != len(ids):
            raise ValueError("ids must be distinct")
        _check_budget(budget, recent)
        todo = [s for s in ids if self._len[s] > budget]
        done, need = list(todo), self._pages_for(budget)
        if todo and len(self._free) < need:
            raise RuntimeError(f"paged cache full: eviction copies to {need} free pages, {len(self._free)} are")
        while todo:
            now = todo[:len(self._free) // need]
            todo = todo[len(now):]
            old = [self._pages[s] for s in now]
            new = [[self._free.pop() for _ in range(need)] for _ in now]
            try:
                table, lens = self._upload(old, [self._len[s] for s in now])
                new_table, = self._upload(new)
                for layer in range(self.num_layers):
                    paged_evict(self.k_pages[layer], self.v_pages[layer], self.weights[layer], table, lens, new_table,
                                budget, recent)
            except BaseException:
                # the old pages are as they were
                self._free.extend(p for pages in reversed(new) for p in reversed(pages))
                raise
            for s, o, p in zip(now, old, new):
                self._free.extend(reversed(o))
                self._pages[s], self._len[s] = p, budget
        return done
