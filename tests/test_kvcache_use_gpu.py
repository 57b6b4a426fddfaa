"""GPU: the paged key/value cache as a serving program uses it: several streams, graphs, threads and caches at once."""
import pytest

from test_kvcache_gpu import Cache, check_attend

pytestmark = pytest.mark.gpu

STEP, CHUNK = [1, 1, 1], [70, 33, 128]  # new tokens: the step kernel and the chunk kernel


def wait_on_current(ms=20):
    """Keeps the current stream busy."""
    import torch

    torch.cuda._sleep(int(ms * 1.5e6))


def call(c, counts, heads=8, seed=1):
    """(q, offsets, zero scores) of a call."""
    torch = c.t
    return c.random(sum(counts), heads, c.dim, scale=2.0), c.offsets(counts), \
        torch.zeros((len(counts), c.kv_heads, max(c.lens_list)), device="cuda")


@pytest.mark.parametrize("counts", [STEP, CHUNK])
def test_results_on_another_stream(counts):
    """A block that the current stream has still to write when it is given back must not become a result of a call on
    another stream, nor a dropped result of that call become a tensor of the current one."""
    import torch

    c = Cache([900, 700, 300], 32, 2, 128, seed=3, extra=3)
    q, off, s0 = call(c, counts)
    want, want_lse = c.cache.attend(q, off, c.table, c.lens)
    c.cache.sync()
    check_attend(c, q, counts, want, want_lse, True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    c.cache.attend(q, off, c.table, c.lens, stream=st)  # the stream's working memory
    torch.cuda.synchronize()
    junk = [torch.empty_like(want) for _ in range(4)] + [torch.empty_like(want_lse) for _ in range(4)]
    wait_on_current()
    for x in junk:
        x.fill_(7.0)  # after the wait
    del junk, x
    out, lse = c.cache.attend(q, off, c.table, c.lens, stream=st)
    st.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    # the other way round: the call waits, its results are dropped, the current stream makes tensors of their sizes
    with torch.cuda.stream(st):
        wait_on_current()
    c.cache.attend(q, off, c.table, c.lens, stream=st)
    mine = [torch.full_like(want, 5.0) for _ in range(4)] + [torch.full_like(want_lse, 5.0) for _ in range(4)]
    torch.cuda.synchronize()
    assert all((x == 5).all() for x in mine)
    # eviction's results
    new = c.spare[:3, None].contiguous()
    scores = torch.rand((3, 2, 900), generator=c.g, device="cuda")
    kept0, lens0, scores0 = c.cache.evict(c.table, c.lens, new, 32, 4, scores)
    torch.cuda.synchronize()
    junk = [torch.empty_like(x) for x in (scores0, lens0, kept0) for _ in range(4)]
    wait_on_current()
    for x in junk:
        x.fill_(7)
    del junk, x
    kept, new_lens, new_scores = c.cache.evict(c.table, c.lens, new, 32, 4, scores, stream=st)
    st.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(kept, kept0) and torch.equal(new_lens, lens0) and torch.equal(new_scores, scores0)
    c.cache.sync(st)


@pytest.mark.parametrize("counts", [STEP, CHUNK])
@pytest.mark.parametrize("first", [0, 1, None])
def test_graphs_in_any_order(monkeypatch, counts, first):
    """Two graphs captured on one stream that never ran a call before: either may be replayed first, or neither before an
    eager call on that stream."""
    import torch

    from veckern_b200 import kvcache

    c = Cache([4000, 2500, 700], 64, 2, 128, seed=2)
    q, off, s0 = call(c, counts)
    want, want_lse = c.cache.attend(q, off, c.table, c.lens, scores=s0)
    c.cache.sync()
    dirt = torch.full((64 << 20,), 0x01010101, dtype=torch.int32, device="cuda")  # what is allocated next is not zero
    del dirt
    torch.cuda.empty_cache()
    monkeypatch.setattr(kvcache, "_WORK", {})
    st = torch.cuda.Stream()
    graphs, got = [], []
    for _ in range(2):
        s = torch.zeros_like(s0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out, lse = c.cache.attend(q, off, c.table, c.lens, scores=s)
        graphs.append(g)
        got.append((out, lse, s))
    order = [] if first is None else [first, 1 - first]
    if first is None:
        s = torch.zeros_like(s0)
        torch.cuda.synchronize()
        out, lse = c.cache.attend(q, off, c.table, c.lens, scores=s, stream=st)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(s, s0)
    for i in order + order:
        got[i][2].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(got[i][0], want) and torch.equal(got[i][1], want_lse) and torch.equal(got[i][2], s0)
    c.cache.sync(st)


@pytest.mark.parametrize("kinds", [(STEP, STEP), (CHUNK, CHUNK), (STEP, CHUNK)])
def test_calls_on_two_streams_at_once(kinds):
    """Calls whose segments are cut between many CTAs, on two streams beside kernels that keep the SMs busy: whoever waits
    for a part waits for a CTA that has started, so that neither call can keep the other from ending."""
    import torch

    caches = [Cache([9000, 5000, 700], 32, 2, 128, seed=11 + i) for i in range(2)]
    sides = []
    for c, counts in zip(caches, kinds):
        q, off, s0 = call(c, counts)
        out, lse = c.cache.attend(q, off, c.table, c.lens, scores=s0, max_q=max(counts))
        c.cache.sync()
        sides.append((c, q, off, s0, out, lse, max(counts)))
    streams = [torch.cuda.Stream() for _ in range(3)]
    x = torch.randn((4096, 4096), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    got = []
    for _ in range(40):
        with torch.cuda.stream(streams[2]):
            x @ x
        for (c, q, off, s0, _, _, most), st in zip(sides, streams):
            with torch.cuda.stream(st):
                s = torch.zeros_like(s0)
                got.append((*c.cache.attend(q, off, c.table, c.lens, scores=s, max_q=most), s))
    torch.cuda.synchronize()
    for st, (c, *_) in zip(streams, sides):
        c.cache.sync(st)
    for i, (out, lse, s) in enumerate(got):
        _, _, _, s0, want, want_lse, _ = sides[i % 2]
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(s, s0)


def test_threads_with_a_stream_each():
    """Two threads call one cache with other sizes, other tensors and streams of their own."""
    import threading

    import torch

    c = Cache([2000, 1500, 700], 32, 2, 128, seed=7)
    work = []
    for counts in (STEP, CHUNK):
        q, off, s = call(c, counts)
        out, lse = c.cache.attend(q, off, c.table, c.lens, scores=s, max_q=max(counts))
        work.append((counts, q, off, s, out, lse))
    torch.cuda.synchronize()
    wrong = []

    def run(counts, q, off, s0, want, want_lse):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(150):
                s = torch.zeros_like(s0)
                out, lse = c.cache.attend(q, off, c.table, c.lens, scores=s, max_q=max(counts))
                kept, _, _ = c.cache.evict(c.table, c.lens, c.table[:, :0], 0, 0, s0)
                if not (torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(s, s0) and kept.numel() == 0):
                    wrong.append(counts)
        st.synchronize()

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    c.cache.sync()
    assert not wrong


def test_working_memory_that_a_wait_has_left_unfinished():
    """A call whose wait ran out leaves its mark and any flags in the stream's working memory (both are set here by hand).
    Later calls with it report that they are void, of another cache too; sync clears it, and nothing sticks."""
    import torch

    from veckern_b200 import _native as N
    from veckern_b200 import kvcache

    a, b = (Cache([9000, 5000, 700], 32, 2, 128, seed=21 + i) for i in range(2))
    st = torch.cuda.Stream()
    for c in (a, b):
        c.made = call(c, CHUNK)
        c.want = c.cache.attend(*c.made[:2], c.table, c.lens)
        c.cache.sync()
    st.wait_stream(torch.cuda.current_stream())
    a.cache.attend(*a.made[:2], a.table, a.lens, stream=st)
    a.cache.sync(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        captured = a.cache.attend(*a.made[:2], a.table, a.lens)
    flags = kvcache._WORK[(0, st.cuda_stream)]._memory[:kvcache._ZEROED].view(torch.int32)
    assert not flags.any()
    flags[:16] = 1
    flags[-2] = 1
    torch.cuda.synchronize()
    a.cache.sync(st)  # of cache a nothing is void yet
    b.cache.attend(*b.made[:2], b.table, b.lens, stream=st)
    with pytest.raises(N.VkError, match="workspace") as e:
        b.cache.sync(st)
    assert e.value.code == N.VK_ERR_DEVICE and not flags.any()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(captured, a.want))
    for c in (a, b):
        got = c.cache.attend(*c.made[:2], c.table, c.lens, stream=st)
        c.cache.sync(st)
        assert all(torch.equal(x, y) for x, y in zip(got, c.want))


@pytest.mark.parametrize("counts", [STEP, CHUNK])
@pytest.mark.parametrize("dim", [64, 128])
def test_waits_that_run_out(counts, dim):
    """With a limit of one cycle the first wait for a copy runs out: the call ends at once, what it had in flight has landed
    when it does, sync says so, and the next call with the usual limit is right."""
    import torch

    from veckern_b200 import _native as N

    c = Cache([9000, 5000, 700], 32, 2, dim, seed=31)
    q, off, s0 = call(c, counts)
    want, want_lse = c.cache.attend(q, off, c.table, c.lens, scores=s0, max_q=max(counts))
    c.cache.sync()
    for _ in range(3):
        assert N.lib().vk_kv_wait_limit(c.cache._h, 1) == N.VK_OK
        c.cache.attend(q, off, c.table, c.lens, scores=torch.zeros_like(s0), max_q=max(counts))
        with pytest.raises(N.VkError, match=r"wait ran out.*status (1|9)\)") as e:
            c.cache.sync()
        assert e.value.code == N.VK_ERR_DEVICE
        assert N.lib().vk_kv_wait_limit(c.cache._h, 0) == N.VK_OK
        s = torch.zeros_like(s0)
        out, lse = c.cache.attend(q, off, c.table, c.lens, scores=s, max_q=max(counts))
        c.cache.sync()
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(s, s0)
    assert N.lib().vk_kv_wait_limit(c.cache._h, -1) == N.VK_ERR_INVALID


def test_offsets_that_count_the_tokens_again_and_again():
    """Offsets that do not ascend give many sequences the same tokens: 2,200 x 131,072 x 8 units, more than 32 bits count.
    The call is reported and does nothing."""
    import torch

    from veckern_b200 import PagedCache
    from veckern_b200 import _native as N

    tokens, batch = 2048, 4400
    pages = torch.zeros((2, 1024, 8, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((1, 128), dtype=torch.int32, device="cuda").expand(batch, -1)
    lens = torch.full((batch,), 128 * 1024, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, tokens], dtype=torch.int32, device="cuda").repeat(batch // 2 + 1)[:batch + 1].contiguous()
    out = torch.full((tokens, 128, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    with PagedCache(pages, pages) as cache:
        cache.attend(torch.zeros_like(out), offsets, table, lens, causal=False, out=out)
        with pytest.raises(N.VkError, match="out of range"):
            cache.sync()
        assert (out == 7).all()
        ascending = torch.full((batch + 1,), 5, dtype=torch.int32, device="cuda")
        ascending[0] = 0
        cache.attend(torch.zeros_like(out), ascending, table, lens // 1024, causal=False, out=out)
        cache.sync()
        assert (out[:5] == 0).all() and (out[5:] == 7).all()


@pytest.mark.parametrize("counts", [[1, 1], [40, 33]])
def test_results_whose_rows_overlap_are_refused(counts):
    """Scores that sequences or heads share would be added to by several threads without an order; the same of out."""
    import torch

    from veckern_b200 import _native as N

    c = Cache([300, 200], 16, 2, 64, seed=5)
    q, off, _ = call(c, counts, heads=4)
    room = torch.zeros((2, 2, 400), device="cuda")
    for s in (room[:1].expand(2, -1, -1), room[:, :1].expand(-1, 2, -1), room.as_strided((2, 2, 300), (600, 299, 1)),
              room.as_strided((2, 2, 300), (300, 300, 1))):
        with pytest.raises(N.VkError, match="scores: rows overlap"):
            c.cache.attend(q, off, c.table, c.lens, scores=s)
    n = sum(counts)
    for out in (torch.zeros((1, 4, 64), dtype=c.dtype, device="cuda").expand(n, -1, -1),
                torch.zeros((n, 1, 64), dtype=c.dtype, device="cuda").expand(-1, 4, -1)):
        with pytest.raises(N.VkError, match="out: rows overlap"):
            c.cache.attend(q, off, c.table, c.lens, out=out)
    want, want_lse = c.cache.attend(q, off, c.table, c.lens)
    for s in (room[:, :, :300], room[:, :, 50:350].transpose(0, 1), torch.zeros((2, 9, 300), device="cuda")[:, ::5]):
        before = s.clone()
        head_major = torch.empty((4, n, 64), dtype=c.dtype, device="cuda").transpose(0, 1)
        out, lse = c.cache.attend(q, off, c.table, c.lens, scores=s, out=head_major)
        c.cache.sync()
        check_attend(c, q, counts, out, lse, True, None, s, before)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    one = Cache([300], 16, 1, 64, seed=6)  # one row: its strides say nothing
    q, off, _ = call(one, [5])
    s = torch.zeros((1, 1, 300), device="cuda").as_strided((1, 1, 300), (0, 0, 1))
    one.cache.attend(q, off, one.table, one.lens, scores=s)
    one.cache.sync()


def test_a_new_cache_reports_what_its_first_call_finds():
    """The status word is clear when the cache is made, not when the default stream comes to it: work that is pending there
    must not clear what a call on another stream has found meanwhile."""
    import torch

    from veckern_b200 import PagedCache
    from veckern_b200 import _native as N

    c = Cache([300, 200], 16, 2, 64, seed=5)
    q, off, _ = call(c, [1, 1])
    st = torch.cuda.Stream()
    bad = c.table.clone()
    bad[0, 1] = -1
    c.cache.attend(q, off, c.table, c.lens, stream=st)
    torch.cuda.synchronize()
    wait_on_current(100)
    with PagedCache(c.k, c.v) as cache:
        cache.attend(q, off, bad, c.lens, stream=st)
        torch.cuda.synchronize()
        with pytest.raises(N.VkError, match="out of range"):
            cache.sync(st)
        cache.sync(st)


def same(x, y):
    """Bit for bit (NaN included)."""
    import torch

    return torch.equal(x.contiguous().view(torch.int16), y.contiguous().view(torch.int16))


def refused(c, what="attention read .* as zeros"):
    from veckern_b200 import _native as N

    with pytest.raises(N.VkError, match=f"out of range: {what}"):
        c.cache.sync()


@pytest.mark.parametrize("counts", [[1, 1, 1], [20, 1, 30]])
def test_what_is_refused_changes_nothing_else(counts):
    """Page numbers, lengths and offsets out of range: an attention gives the other sequences what it gave before, and reads a
    page that is not there as zeros; an append writes the slots that it can and no others."""
    import torch

    c = Cache([100, 60, 90], 16, 2, 64, seed=6, extra=3)
    q, off, _ = call(c, counts, heads=4)
    good, good_lse = c.cache.attend(q, off, c.table, c.lens, causal=False)
    c.cache.sync()
    check_attend(c, q, counts, good, good_lse, False)
    k0, v0 = c.k.clone(), c.v.clone()
    at = [0, counts[0], sum(counts[:2]), sum(counts)]
    others = [i for i in range(at[3]) if not at[1] <= i < at[2]]
    for wrong in (-5, -1, c.k.shape[0], 2 ** 31 - 1):
        t = c.table.clone()
        t[1, 2] = wrong
        out, lse = c.cache.attend(q, off, t, c.lens, causal=False)
        refused(c)
        assert torch.equal(out[others], good[others]) and torch.equal(lse[others], good_lse[others])
        zeros = Cache.__new__(Cache)
        zeros.__dict__.update(c.__dict__)
        zeros.k, zeros.v = torch.cat([c.k, torch.zeros_like(c.k[:1])]), torch.cat([c.v, torch.zeros_like(c.v[:1])])
        zeros.table = torch.where(t == wrong, c.k.shape[0], t).to(torch.int32)
        zeros.table[c.table == 2 ** 31 - 1] = 2 ** 31 - 1
        check_attend(zeros, q, counts, out, lse, False)
        # the last of sequence 1's slots 60 - count .. 59 lie in the page that is not there (slots 32 .. 47) or behind it
        t = c.table.clone()
        t[1, 3] = wrong
        ones = torch.ones((at[3], 2, 64), dtype=c.dtype, device="cuda")
        c.cache.append(ones, ones, off, t, c.lens)
        refused(c, ".* nothing was written")
        own = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
        for b, (n, cnt) in enumerate(zip(c.lens_list, counts)):
            j = torch.arange(n - cnt, n, device="cuda")
            if b == 1:
                j = j[j < 48]
            own[c.table[b].long()[j // 16], j % 16] = True
        for x, x0 in ((c.k, k0), (c.v, v0)):
            assert (x[own] == 1).all() and same(x[~own], x0[~own])
            x.copy_(x0)
    # lengths: below zero none, past the table all of its slots (their page numbers lie past the sequence's)
    for length in (-1, 10 ** 9):
        lens = c.lens.clone()
        lens[1] = length
        out, lse = c.cache.attend(q, off, c.table, lens, causal=False)
        refused(c)
        assert torch.equal(out[others], good[others]) and torch.equal(lse[others], good_lse[others])
        if length < 0:
            assert (out[at[1]:at[2]] == 0).all() and (lse[at[1]:at[2]] == -torch.inf).all()
    # offsets: sequences whose own pair is in range and ascends keep their results
    for bad, kept in (([0, at[1], at[2], 10 ** 6], [0, 1]), ([-3, at[1], at[2], at[3]], [1, 2]), ([0, at[2], at[1], at[1]], [])):
        o = torch.tensor(bad, dtype=torch.int32, device="cuda")
        out, lse = c.cache.attend(q, o, c.table, c.lens, causal=False)
        refused(c)
        for b in kept:
            assert torch.equal(out[at[b]:at[b + 1]], good[at[b]:at[b + 1]])
    # more new tokens than slots: the last ones are written
    new = torch.arange(9, device="cuda", dtype=c.dtype)[:, None, None].expand(-1, 2, 64).contiguous()
    c.cache.append(new, new, c.offsets([9]), c.table[:1], torch.tensor([5], dtype=torch.int32, device="cuda"))
    refused(c, ".* nothing was written")
    first = int(c.table[0, 0])
    assert torch.equal(c.k[first, :5], new[4:]) and torch.equal(c.v[first, :5], new[4:])
    c.k[first, :5], c.v[first, :5] = k0[first, :5], v0[first, :5]
    assert same(c.k, k0) and same(c.v, v0)
    again, again_lse = c.cache.attend(q, off, c.table, c.lens, causal=False)
    c.cache.sync()
    assert torch.equal(again, good) and torch.equal(again_lse, good_lse)


def test_working_memory_goes_by_the_scores():
    """Tables are often as wide as the longest sequence that may ever come: kept scores take memory for the slots that have a
    score, not for all of the table's."""
    import torch

    from veckern_b200 import kvcache

    c = Cache([300, 200], 16, 2, 64, seed=5)
    q, off, s = call(c, [1, 1])
    wide = torch.full((2, 1 << 16), 2 ** 31 - 1, dtype=torch.int32, device="cuda")  # a million slots
    wide[:, :c.table.shape[1]] = c.table
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    out, lse = c.cache.attend(q, off, wide, c.lens, scores=s, max_q=1, stream=st)
    c.cache.sync(st)
    check_attend(c, q, [1, 1], out, lse, True, None, s, torch.zeros_like(s))
    small = kvcache._WORK[(0, st.cuda_stream)].size
    c.cache.attend(q, off, c.table, c.lens, scores=s, max_q=1, stream=st)
    c.cache.sync(st)
    assert kvcache._WORK[(0, st.cuda_stream)].size == small < 16 << 20


def test_more_tokens_than_32_bits_count_are_refused():
    """A sequence's tokens are rounded up to pairs of row tiles (up to 256 tokens) in 32 bits."""
    import ctypes as C

    from veckern_b200 import _native as N

    c = Cache([30], 8, 1, 64)
    at = c.table.data_ptr()
    strides = (C.c_int64 * 2)(0, 0)
    for tokens, code in ((2 ** 31 - 1, N.VK_ERR_INVALID), (2 ** 31 - 1023, N.VK_ERR_INVALID), (-1, N.VK_ERR_INVALID),
                         (0, N.VK_OK)):
        b = N.KvBatch(batch=1, table_width=4, table_stride=4, tokens=tokens, offsets=at, table=at, lens=at)
        assert N.lib().vk_kv_append(c.cache._h, C.byref(b), at, strides, at, strides, None) == code
        if code:
            assert "tokens" in N.last_error()
