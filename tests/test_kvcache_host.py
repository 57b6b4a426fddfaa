"""CPU: what PagedCache does on the host around the C entries (streams, working memory, threads), with torch and the native
library replaced by stand-ins that write down what they are asked for."""
import ctypes as C
import sys
import threading
import types

import pytest
import torch

from veckern_b200 import _native as N
from veckern_b200 import kvcache


class Device:
    index = 0


class Tensor:
    """Sizes, strides and an address; `made_on` is the stream that was current when it was made."""

    def __init__(self, fake, shape, strides=None, dtype=torch.float32):
        self.shape, self.dtype, self.device, self.is_cuda = tuple(shape), dtype, fake.device, True
        if strides is None:
            strides, step = [], 1
            for n in reversed(self.shape):
                strides.insert(0, step)
                step *= n
        self.strides, self.made_on, self.at = tuple(strides), fake.current, fake.address()
        fake.made.append(self)

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.at


class Fake(types.ModuleType):
    """The torch functions that PagedCache calls, and the C entries; streams are numbers."""

    def __init__(self):
        super().__init__("torch")
        self.device, self.current, self.made, self.calls, self.next = Device(), 3, [], [], 1 << 20
        self.inside = None  # called by an entry before it reads its arguments: the interpreter's lock is free then
        self.capturing, self.cleared, self.need, self.sync_code = set(), [], 1000, N.VK_OK
        self.int32, self.float32, self.uint8 = torch.int32, torch.float32, torch.uint8
        self.float16, self.bfloat16 = torch.float16, torch.bfloat16
        outer = self

        class Cuda:
            @staticmethod
            def ExternalStream(raw, device=None):
                return types.SimpleNamespace(cuda_stream=raw)

            class stream:
                def __init__(self, s):
                    self.raw = s.cuda_stream

                def __enter__(self):
                    self.before, outer.current = outer.current, self.raw

                def __exit__(self, *exc):
                    outer.current = self.before

            @staticmethod
            def is_current_stream_capturing():
                return outer.current in outer.capturing

            @staticmethod
            def synchronize(device=None):
                outer.calls.append(("synchronize",))

        self.cuda = Cuda
        self._C = types.SimpleNamespace(_cuda_getCurrentRawStream=lambda index: outer.current)

    def address(self):
        self.next += 1 << 16
        return self.next

    def empty_strided(self, shape, strides, dtype, device):
        return Tensor(self, shape, strides, dtype)

    def empty_like(self, x):
        return Tensor(self, x.shape, x.strides, x.dtype)

    def empty(self, shape, dtype, device):
        t = Tensor(self, shape, None, dtype)
        t.zeroed_on = []

        class Start:
            def zero_(_):
                t.zeroed_on.append("graph" if self.current in self.capturing else self.current)

        t.__class__ = type("Work", (Tensor,), {"__getitem__": lambda _, i: Start()})
        return t

    # ---- the C entries
    def vk_kv_create(self, desc, out):
        return N.VK_OK

    def vk_kv_destroy(self, h):
        return N.VK_OK

    def vk_kv_workspace_create(self, device, size, out):
        out = C.cast(out, C.POINTER(C.c_void_p))
        out[0] = self.address()
        self.cleared.append(out[0])
        return N.VK_OK

    def vk_kv_workspace_clear(self, device, at):
        self.calls.append(("clear", at))
        return N.VK_OK

    def vk_kv_attend_workspace(self, h, batch, args, size):
        C.cast(size, C.POINTER(C.c_size_t))[0] = self.need
        return N.VK_OK

    def vk_kv_append(self, h, batch, k, k_stride, v, v_stride, stream):
        self.enter()
        pair = C.c_int64 * 2
        self.calls.append(("append", read(N.KvBatch, batch), (k, *read(pair, k_stride), v, *read(pair, v_stride)), stream))
        return N.VK_OK

    def enter(self):
        if self.inside:
            then, self.inside = self.inside, None
            then()

    def vk_kv_attend(self, h, batch, args, stream):
        self.enter()
        self.calls.append(("attend", read(N.KvBatch, batch), read(N.KvAttend, args), stream))
        return N.VK_OK

    def vk_kv_evict(self, h, batch, args, stream):
        self.enter()
        self.calls.append(("evict", read(N.KvBatch, batch), read(N.KvEvict, args), stream))
        return N.VK_OK

    def vk_kv_sync(self, h, stream):
        return self.sync_code


def read(kind, x):
    """A C struct behind what a call passes: an address or packed bytes."""
    return kind.from_buffer_copy(x if isinstance(x, bytes) else C.string_at(x, C.sizeof(kind)))


@pytest.fixture
def fake(monkeypatch):
    f = Fake()
    monkeypatch.setitem(sys.modules, "torch", f)
    monkeypatch.setattr(kvcache, "lib", lambda: f)
    monkeypatch.setattr(kvcache, "_WORK", {})
    monkeypatch.setattr(kvcache, "_OUTGROWN", [])
    return f


def make(fake, batch=2, heads=4):
    """A cache, and a call's tensors: (cache, q, offsets, table, lens, scores)."""
    pages = Tensor(fake, (8, 16, 2, 64), dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32)
    return (kvcache.PagedCache(pages, pages), Tensor(fake, (batch, heads, 64), dtype=torch.bfloat16),
            Tensor(fake, (batch + 1,), **i32), Tensor(fake, (batch, 4), **i32), Tensor(fake, (batch,), **i32),
            Tensor(fake, (batch, 2, 64)))


@pytest.mark.parametrize("stream", [None, 3, 7])
def test_results_are_made_on_the_stream_that_writes_them(fake, stream):
    """Memory that another stream still uses, or will use as soon as a result is dropped, must not become a result."""
    cache, q, offsets, table, lens, scores = make(fake)
    want = 3 if stream is None else stream
    out, lse = cache.attend(q, offsets, table, lens, stream=stream)
    kept, new_lens, new_scores = cache.evict(table, lens, table, 8, 2, scores, stream=stream)
    assert [x.made_on for x in (out, lse, kept, new_lens, new_scores)] == [want] * 5
    assert [c[3] for c in fake.calls] == [want] * 2 and fake.current == 3
    assert kept.shape == (2, 2, 8) and new_lens.shape == (2,) and new_scores.shape == (2, 2, 64)


def test_working_memory_made_under_capture_is_clear_at_once(fake):
    """A graph that was never replayed has cleared nothing: neither a second graph nor an eager call may depend on it."""
    cache, q, offsets, table, lens, _ = make(fake)
    fake.capturing.add(9)
    cache.attend(q, offsets, table, lens, stream=9)
    fake.need = 5000  # grows within the capture
    cache.attend(Tensor(fake, (3, 4, 64), dtype=torch.bfloat16), offsets, table, lens, stream=9)
    fake.capturing.clear()
    cache.attend(q, offsets, table, lens, stream=9)
    used = [c[2].workspace for c in fake.calls]
    assert used[0] != used[1] == used[2]
    assert set(used) <= set(fake.cleared), "cleared by a node of the graph alone"
    assert not any("graph" in x.zeroed_on for x in fake.made if hasattr(x, "zeroed_on"))


def test_working_memory_of_a_stream(fake):
    """Outside a capture it is torch's, cleared in the stream's order, and shared by the stream's calls while it suffices."""
    cache, q, offsets, table, lens, _ = make(fake)
    for stream in (None, 3, 8, 8):
        cache.attend(q, offsets, table, lens, stream=stream)
    used = [c[2].workspace for c in fake.calls]
    assert used[0] == used[1] != used[2] == used[3] and not fake.cleared
    work = {x.at: x for x in fake.made if hasattr(x, "zeroed_on")}
    assert work[used[0]].zeroed_on == [3] and work[used[0]].made_on == 3 and work[used[2]].zeroed_on == [8]


@pytest.mark.parametrize("op", ["append", "attend", "evict"])
def test_threads_do_not_share_arguments(fake, op):
    """A C entry reads its arguments without the interpreter's lock: another thread may call the same cache meanwhile."""
    cache, q, offsets, table, lens, scores = make(fake)
    more = make(fake, batch=5)[1:]

    def run(q, offsets, table, lens, scores, stream):
        if op == "append":
            cache.append(Tensor(fake, (q.shape[0], 2, 64), dtype=torch.bfloat16),
                         Tensor(fake, (q.shape[0], 2, 64), (256, 64, 1), torch.bfloat16), offsets, table, lens, stream=stream)
        elif op == "attend":
            cache.attend(q, offsets, table, lens, stream=stream)
        else:
            cache.evict(table, lens, table, q.shape[0], 1, scores, stream=stream)

    def beside():
        t = threading.Thread(target=run, args=(*more, 9))
        t.start()
        t.join()

    fake.inside = beside
    run(q, offsets, table, lens, scores, 3)
    (_, batch9, args9, s9), (_, batch3, args3, s3) = fake.calls
    assert (s9, s3) == (9, 3)
    for (x, tensors, n), args in (((batch3, (table, lens), 2), args3), ((batch9, (more[2], more[3]), 5), args9)):
        assert (x.batch, x.table, x.lens) == (n, tensors[0].at, tensors[1].at)
        if op == "append":
            assert args[1:3] == (128, 64) and args[4:] == (256, 64) and x.tokens == n
        elif op == "attend":
            assert args.q == (q if n == 2 else more[0]).at
        else:
            assert args.keep == n and args.scores == (scores if n == 2 else more[4]).at


def test_calls_that_share_working_memory_are_issued_one_at_a_time(fake):
    """A call may be two launches: no other call of the stream comes between them."""
    cache, q, offsets, table, lens, _ = make(fake)
    other = make(fake)[0]
    threads, order = [], []

    def start(c, name, stream):
        def run():
            c.attend(q, offsets, table, lens, stream=stream)
            order.append(name)

        threads.append(threading.Thread(target=run))
        threads[-1].start()

    def beside():
        start(other, "same stream", 3)
        start(cache, "another stream", 9)
        threads[1].join()
        threads[0].join(0.2)
        order.append("first")

    cache.attend(q, offsets, table, lens)
    fake.inside = beside
    cache.attend(q, offsets, table, lens)
    threads[0].join()
    assert order == ["another stream", "first", "same stream"]


@pytest.mark.parametrize("code", [N.VK_OK, N.VK_ERR_INVALID, N.VK_ERR_DEVICE])
def test_sync_clears_all_working_memory_after_a_wait_ran_out(fake, code):
    """The status word is the cache's, working memory the stream's: the call that gave up may have been any of the cache's
    streams', and a graph may hold what was outgrown."""
    cache, q, offsets, table, lens, _ = make(fake)
    cache.attend(q, offsets, table, lens)
    cache.attend(q, offsets, table, lens, stream=9)
    fake.need = 5000
    cache.attend(Tensor(fake, (3, 4, 64), dtype=torch.bfloat16), offsets, table, lens, stream=9)
    used = {c[2].workspace for c in fake.calls}
    assert len(used) == 3
    fake.calls.clear()
    fake.sync_code = code
    if code == N.VK_OK:
        cache.sync()
    else:
        with pytest.raises(N.VkError) as e:
            cache.sync()
        assert e.value.code == code
    if code != N.VK_ERR_DEVICE:
        assert not fake.calls
        return
    assert {c[1] for c in fake.calls if c[0] == "clear"} == used, "memory whose flags may be anything stays in use"
    for i, c in enumerate(fake.calls):  # no call that is under way may still use it
        assert c[0] != "clear" or fake.calls[i - 1][0] == "synchronize"
    fake.calls.clear()
    cache.attend(q, offsets, table, lens, stream=9)
    assert fake.calls[0][2].workspace in used


def test_workspace_entries_refuse_null():
    assert N.lib().vk_kv_workspace_clear(0, None) == N.VK_ERR_INVALID and "workspace" in N.last_error()
    assert N.lib().vk_kv_workspace_create(0, 1 << 20, None) == N.VK_ERR_INVALID and "out" in N.last_error()
    assert N.lib().vk_kv_workspace_destroy(0, None) == N.VK_OK
    assert N.lib().vk_kv_wait_limit(None, 5) == N.VK_ERR_INVALID and "cache" in N.last_error()


def test_kernels_do_not_read_through_the_read_only_path():
    """They start while the kernel before them runs; that path, and hoisting its loads over the wait, is for memory that
    nobody writes while a kernel lives."""
    from pathlib import Path

    found = {}
    for f in (Path(kvcache.__file__).parent / "csrc").glob("kv_*.cu*"):
        lines = [x.split("//")[0] for x in f.read_text().splitlines()]
        found[f.name] = [x for x in lines if "__ldg" in x or "ld.global.nc" in x or "__restrict__" in x]
    assert found and not any(found.values()), found
