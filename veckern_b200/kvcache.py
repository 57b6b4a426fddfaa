"""Paged key/value cache over the C ABI (vk_kv_*, include/vk_abi.h): what a retrieval user's model does after the search.
The keys and values of retrieved passages and of the model's own tokens live in fixed-size pages; a page table per
sequence, made e.g. from a search's ids, says which pages it reads.

    cache = PagedCache(k_pages, v_pages)                          # [pages, page_size, kv_heads, head_dim], f16 or bf16
    cache.append(k, v, offsets, table, lens)                      # new tokens behind their sequences
    out, lse = cache.attend(q, offsets, table, lens, scores=s)    # their attention over all slots
    kept, lens, s = cache.evict(table, lens, new_table, keep, recent, s)

Slot s of a sequence is entry s % page_size of its page s // page_size: every page but the last is full. Passages that pages
are shared by therefore have to fill whole pages; slots that a passage leaves over in the middle of a sequence would be
attended to as well.

All tensors are torch tensors on the cache's device. Sequence b of a call has the new tokens offsets[b]:offsets[b + 1]
(int32, [batch + 1]), lens[b] slots with the new tokens included (int32, [batch]) and the pages table[b] (int32,
[batch, width]; entries past its last slot are not read). Calls are asynchronous on `stream` (a torch.cuda.Stream or raw
handle; default: the current stream), which the results they make belong to as well: another stream waits before it reads
them. sync() waits and raises what the kernels found wrong. The calls of one stream share their working memory, those captured
into CUDA graphs on it too: such graphs are replayed in any order, one after the other, and not while eager calls of that
stream run. No derivatives: a cache is for inference.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading

from . import _native as N
from ._native import VkError, check, lib

# The argument structs (N.KvBatch, N.KvAttend, N.KvEvict), packed in one step: a call's fields set one by one take longer
# than its launch. Every call packs its own: the C entries run without the interpreter's lock, beside other threads' calls.
_BATCH, _ATTEND, _EVICT = struct.Struct("@iiqqPPP"), struct.Struct("@PqqPqqPPqqqiiifPN"), struct.Struct("@PqiiiPqqqPPP")
_STRIDES = struct.Struct("@qq")  # of append's keys or values
assert [x.size for x in (_BATCH, _ATTEND, _EVICT)] == [C.sizeof(x) for x in (N.KvBatch, N.KvAttend, N.KvEvict)]

# Attention's working memory by (device, stream): the calls of a stream share it, one at a time; it grows, and its start is
# zero between calls. What was outgrown is kept: a captured graph may hold its address.
_WORK: dict = {}
_OUTGROWN: list = []  # (device, working memory)
_GROWING = threading.Lock()
_ZEROED = 8192  # VK_KV_WORKSPACE_ZEROED


class _Work:
    """Working memory of a stream. `lock` is held while a call is issued: a call may be two launches, and another thread's
    call on the stream must not come between them."""

    def __init__(self, torch, device, stream: int, size: int):
        self.size, self.lock = size, threading.Lock()
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
            if torch.cuda.is_current_stream_capturing():
                # The graph's own pool will not do: what a graph records there (clearing it, or another node's use of the
                # same memory) happens when that graph is replayed, while other graphs and eager calls of the stream use
                # the memory too. It is made outside the capture, cleared, and kept for good.
                at = C.c_void_p()
                check(lib().vk_kv_workspace_create(device.index, size, C.byref(at)), "attend (working memory, while capturing)")
                self.at = at.value
            else:
                self._memory = torch.empty((size,), dtype=torch.uint8, device=device)
                self._memory[:_ZEROED].zero_()
                self.at = self._memory.data_ptr()


def _workspace(torch, device, stream: int, need: int) -> _Work:
    """Larger working memory for a stream."""
    key = (device.index, stream)
    with _GROWING:
        work = _WORK.get(key)
        if work is not None:
            if work.size >= need:  # another thread was here first
                return work
            _OUTGROWN.append((device.index, work))
            need = max(need, work.size * 3 // 2)
        work = _WORK[key] = _Work(torch, device, stream, need)
    return work


def _clear_all(torch, device) -> None:
    """Clears the device's working memory after a wait ran out: the call may have been on any stream, and captured graphs
    hold what was outgrown."""
    with _GROWING:
        works = [(key[0], work) for key, work in _WORK.items()] + _OUTGROWN
        for index, work in works:
            if index == device.index:
                with work.lock:
                    torch.cuda.synchronize(device)
                    check(lib().vk_kv_workspace_clear(index, work.at), "sync (clearing working memory)")


_DTYPES = {"torch.float16": N.VK_KV_F16, "torch.bfloat16": N.VK_KV_BF16}


def _want(t, name: str, dtype, ndim: int, device) -> None:
    if t.dtype != dtype or t.dim() != ndim or t.device != device:
        raise ValueError(f"{name} must be a {ndim}-dimensional {dtype} tensor on {device}, got {t.dim()}-dimensional "
                         f"{t.dtype} on {t.device}")


class PagedCache:
    """k_pages and v_pages: [pages, page_size, kv_heads, head_dim], any strides that are multiples of 8 elements with
    the last dimension contiguous (a [pages, kv_heads, page_size, head_dim] tensor is passed transposed). The cache
    refers to the tensors, it does not copy them. page_size: a power of two in [8, 1024]; head_dim: a multiple of 8 up to
    128. Threads may call a cache at the same time, on one stream or on several."""

    def __init__(self, k_pages, v_pages):
        import torch

        self._torch, self._i32, self._f32, self._lib = torch, torch.int32, torch.float32, lib()
        self._h = C.c_void_p()
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            if t.dim() != 4 or t.shape != k_pages.shape or t.dtype != k_pages.dtype or t.device != k_pages.device:
                raise ValueError(f"{name} must be [pages, page_size, kv_heads, head_dim], k_pages and v_pages alike")
            if not t.is_cuda:
                raise ValueError(f"{name} must be on a GPU")
            if t.stride(3) != 1:
                raise ValueError(f"{name}: the last dimension must be contiguous")
        if str(k_pages.dtype) not in _DTYPES:
            raise ValueError("pages must be float16 or bfloat16")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.pages, self.page_size, self.kv_heads, self.head_dim = k_pages.shape
        self.dtype, self.device = k_pages.dtype, k_pages.device
        self._scale = self.head_dim ** -0.5
        d = N.KvDesc(device=self.device.index, dtype=_DTYPES[str(self.dtype)], page_size=self.page_size,
                     kv_heads=self.kv_heads, head_dim=self.head_dim, pages=self.pages, k=k_pages.data_ptr(),
                     k_stride=(C.c_int64 * 3)(*k_pages.stride()[:3]), v=v_pages.data_ptr(),
                     v_stride=(C.c_int64 * 3)(*v_pages.stride()[:3]))
        check(lib().vk_kv_create(C.byref(d), C.byref(self._h)), "vk_kv_create")
        self._sizes = {}  # bytes of attention's working memory by what they depend on

    def _sequences(self, table, lens, offsets=None, tokens: int = 0):
        """Checks a call's sequences; (N.KvBatch packed, sequences, table width)."""
        i32, dev = self._i32, self.device
        if table.dtype != i32 or table.dim() != 2 or table.device != dev:
            _want(table, "table", i32, 2, dev)
        if lens.dtype != i32 or lens.dim() != 1 or lens.device != dev:
            _want(lens, "lens", i32, 1, dev)
        n, width = table.shape
        stride, step = table.stride()
        if lens.shape[0] != n or not lens.is_contiguous() or (step != 1 and width > 1):
            raise ValueError("lens must be contiguous, one per row of table, and table's rows contiguous")
        at = 0
        if offsets is not None:
            if offsets.dtype != i32 or offsets.dim() != 1 or offsets.device != dev:
                _want(offsets, "offsets", i32, 1, dev)
            if offsets.shape[0] != n + 1 or not offsets.is_contiguous():
                raise ValueError("offsets must be contiguous [batch + 1]")
            at = offsets.data_ptr()
        return _BATCH.pack(n, width, stride, tokens, at, table.data_ptr(), lens.data_ptr()), n, width

    def _rows(self, t, name: str, heads: int):
        """Checks rows of tokens; their strides."""
        if t.dtype != self.dtype or t.dim() != 3 or t.device != self.device:
            _want(t, name, self.dtype, 3, self.device)
        strides = t.stride()
        if t.shape[1] != heads or t.shape[2] != self.head_dim or strides[2] != 1:
            raise ValueError(f"{name} must be [tokens, {heads}, {self.head_dim}] with the last dimension contiguous")
        return strides

    def _stream(self, stream):
        if stream is None:
            return self._torch._C._cuda_getCurrentRawStream(self.device.index)
        return getattr(stream, "cuda_stream", stream)

    def _empty(self, shape, strides, dtype, stream):
        """A tensor for results whose memory is that of the call's stream (as the caller gave it): memory of the current
        one may have kernels of that stream still to write it."""
        torch = self._torch
        if stream is not None:
            raw = getattr(stream, "cuda_stream", stream)
            if raw != torch._C._cuda_getCurrentRawStream(self.device.index):
                with torch.cuda.stream(torch.cuda.ExternalStream(raw, device=self.device)):
                    return torch.empty_strided(shape, strides, dtype=dtype, device=self.device)
        return torch.empty_strided(shape, strides, dtype=dtype, device=self.device)

    def append(self, k, v, offsets, table, lens, *, stream=None) -> None:
        """New token t of sequence b (of T) is written to slot lens[b] - T + t. k, v: [tokens, kv_heads, head_dim],
        strides multiples of 8 elements (slices of one projection's output are fine)."""
        k_token, k_head, _ = self._rows(k, "k", self.kv_heads)
        v_token, v_head, _ = self._rows(v, "v", self.kv_heads)
        tokens = k.shape[0]
        if v.shape[0] != tokens:
            raise ValueError("k and v must have the same number of tokens")
        batch, _, _ = self._sequences(table, lens, offsets, tokens)
        code = self._lib.vk_kv_append(self._h, batch, k.data_ptr(), _STRIDES.pack(k_token, k_head), v.data_ptr(),
                                      _STRIDES.pack(v_token, v_head), self._stream(stream))
        if code:
            check(code, "append")

    def attend(self, q, offsets, table, lens, *, causal: bool = True, scale: float | None = None, scores=None,
               max_q: int = 0, out=None, lse=None, stream=None):
        """Attention of new tokens q [tokens, heads, head_dim] over their sequences' slots: (out like q, lse [tokens,
        heads] float32). Token t of T sees slots up to lens[b] - T + t when causal, all lens[b] otherwise; a row that
        sees none gets zeros and -inf. out, if given, is not q itself. scale defaults to head_dim ** -0.5. scores,
        [batch, kv_heads, width] float32 with the last dimension contiguous: the attention weights of a sequence's
        tokens and of a kv head's query heads are added to its slots. max_q: an upper bound of a sequence's new tokens,
        where the caller knows it (a decoding step: 1). Where it says that no sequence has more than 16 rows (new
        tokens x query heads of a kv head) the kernel for few rows takes the call; without it (0) any sequence may have
        all of the tokens, and the kernel for chunks takes it (a decoding batch of 32 over up to 8,192 slots: 132 us
        where it takes 120, with weights 291 where it takes 141)."""
        torch = self._torch
        if q.dim() != 3:
            raise ValueError("q must be [tokens, heads, head_dim]")
        tokens, heads, dim = q.shape
        q_token, q_head, _ = self._rows(q, "q", heads)
        batch, n, width = self._sequences(table, lens, offsets, tokens)
        if out is None:
            o_token, o_head = heads * dim, dim
            out = self._empty((tokens, heads, dim), (o_token, o_head, 1), self.dtype, stream)
        else:
            o_token, o_head, _ = self._rows(out, "out", heads)
            if out.shape[0] != tokens:
                raise ValueError("out must have q's shape")
        if lse is None:
            lse = self._empty((tokens, heads), (heads, 1), self._f32, stream)
        else:
            _want(lse, "lse", self._f32, 2, self.device)
            if lse.shape != (tokens, heads) or not lse.is_contiguous():
                raise ValueError("lse must be contiguous [tokens, heads]")
        s_at = s_seq = s_head = s_width = 0
        if scores is not None:
            s_seq, s_head = self._check_scores(scores, n)
            s_at, s_width = scores.data_ptr(), scores.shape[2]
        if scale is None:
            scale = self._scale
        stream = self._stream(stream)

        def pack(work: int, size: int) -> bytes:
            return _ATTEND.pack(q.data_ptr(), q_token, q_head, out.data_ptr(), o_token, o_head, lse.data_ptr(), s_at, s_seq,
                                s_head, s_width, heads, max_q, bool(causal), scale, work, size)

        sizes = (n, width, tokens, heads, max_q, s_width)
        need = self._sizes.get(sizes)
        if need is None:
            size = C.c_size_t()
            check(lib().vk_kv_attend_workspace(self._h, batch, pack(0, 0), C.byref(size)), "attend")
            if len(self._sizes) >= 4096:
                self._sizes.clear()
            need = self._sizes[sizes] = size.value
        work = _WORK.get((self.device.index, stream))
        if work is None or work.size < need:
            work = _workspace(torch, self.device, stream, need)
        args = pack(work.at, work.size)
        with work.lock:
            code = self._lib.vk_kv_attend(self._h, batch, args, stream)
        if code:
            check(code, "attend")
        return out, lse

    def evict(self, table, lens, new_table, keep: int, recent: int, scores, *, stream=None):
        """Cuts every sequence back to at most `keep` slots for each kv head: its last `recent` ones and, of the others,
        those with the largest scores (ties to the lower slot), in slot order, copied to the pages of new_table (which
        no sequence of the call reads). Returns (kept [batch, kv_heads, keep] int32: the old slots, -1 behind the last;
        new lens [batch] int32; new scores like scores, contiguous, 0 behind the last)."""
        batch, n, _ = self._sequences(table, lens)
        s_seq, s_head = self._check_scores(scores, n)
        if new_table.dtype != self._i32 or new_table.dim() != 2 or new_table.device != self.device:
            _want(new_table, "new_table", self._i32, 2, self.device)
        new_stride, new_step = new_table.stride()
        if new_table.shape[0] != n or (new_step != 1 and new_table.shape[1] > 1):
            raise ValueError("new_table must have one row per sequence, rows contiguous")
        if not 0 <= recent <= keep:
            raise ValueError("keep and recent must satisfy 0 <= recent <= keep")
        heads, width = self.kv_heads, scores.shape[2]
        kept = self._empty((n, heads, keep), (heads * keep, keep, 1), self._i32, stream)
        new_lens = self._empty((n,), (1,), self._i32, stream)
        new_scores = self._empty((n, heads, width), (heads * width, width, 1), self._f32, stream)
        args = _EVICT.pack(new_table.data_ptr(), new_stride, new_table.shape[1], keep, recent, scores.data_ptr(), s_seq,
                           s_head, width, new_scores.data_ptr(), kept.data_ptr(), new_lens.data_ptr())
        code = self._lib.vk_kv_evict(self._h, batch, args, self._stream(stream))
        if code:
            check(code, "evict")
        return kept, new_lens, new_scores

    def _check_scores(self, scores, n: int):
        """Checks scores; their first two strides."""
        if scores.dtype != self._f32 or scores.dim() != 3 or scores.device != self.device:
            _want(scores, "scores", self._f32, 3, self.device)
        seq, head, step = scores.stride()
        if scores.shape[0] != n or scores.shape[1] != self.kv_heads or (step != 1 and scores.shape[2] > 1):
            raise ValueError(f"scores must be [batch, {self.kv_heads}, width] with the last dimension contiguous")
        return seq, head

    def sync(self, stream=None) -> None:
        """Waits for the cache's work on the stream and raises VkError for anything its kernels found wrong, on other streams
        too. With the code VK_ERR_DEVICE a bounded wait ran out: what attend gave since the last sync is void, and so is
        what other caches' calls on the stream gave (their sync says so). The device's working memory is then cleared; no
        graph with a captured attend may be running."""
        try:
            check(lib().vk_kv_sync(self._h, self._stream(stream)), "sync")
        except VkError as e:
            if e.code == N.VK_ERR_DEVICE:
                _clear_all(self._torch, self.device)
            raise

    def close(self) -> None:
        if self._h:
            lib().vk_kv_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
