"""GPU: the paged key/value cache (PagedCache over vk_kv_*, include/vk_abi.h) against its definition in 64 bits.

Every slot that no sequence owns holds NaN, and table entries past a sequence's last page hold numbers of no page, so a
kernel that lets either through shows it. Tolerances follow from the arithmetic the header promises, with u the unit
roundoff of the 16-bit type (2^-11 for float16, 2^-8 for bfloat16) and e = 2^-24 that of the 32-bit sums:
  s_j    products of 16-bit values are exact in 32 bits; a sum of D terms in any order errs by at most
         D e sum_d |q_d k_d| scale, to which the scaling and the exponential's argument (|s_j| (1 + log2(e)) e) add:
         ds = 2 (D + 8) e scale max_j sum_d |q_d k_d|
  lse    ds, plus the exponentials' and the n-term sum's relative error; a running sum over tiles of 128 slots, joined
         over parts, errs by less than (n / 32 + 64) e; plus the rounding of lse itself
  out    each weight is off by (2 ds + that) relative, and by u from its own rounding (float16 weights below 2^-14 of
         the row's maximum: by 2^-25 of it, absolute); the value sum's 32-bit error is covered by (n / 32 + 64) e of
         sum_j p_j |v_j|; the result is rounded once more: u |out|
  scores each weight as above without the rounding to 16 bits; the sum over rows errs by (rows / 8 + 64) e of it
"""
import numpy as np
import pytest

from veckern_b200 import _native as N

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
NO_PAGE = 2 ** 31 - 1


class Cache:
    """Random pages with NaN in every slot that no sequence owns, and its sequences' tables in shuffled order."""

    def __init__(self, lens, page, kv_heads, dim, dtype="bfloat16", layout="slot", seed=0, extra=2, shared=0, scale=1.0):
        import torch

        from veckern_b200 import PagedCache

        self.t = torch
        self.dtype = getattr(torch, dtype)
        self.u = 2.0 ** -11 if dtype == "float16" else 2.0 ** -8
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-n // page) for n in lens]
        shared = min([shared] + [n // page for n in lens])
        pages = sum(need) - shared * (len(need) - 1) + extra if need else extra
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), max(need + [0]) + 1), NO_PAGE, dtype=torch.int32, device="cuda")
        own = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
        at = shared
        for b, (n, w) in enumerate(zip(lens, need)):
            self.table[b, :shared] = order[:shared]
            self.table[b, shared:w] = order[at:at + w - shared]
            at += w - shared
            j = torch.arange(n, device="cuda")
            own[self.table[b].long()[j // page], j % page] = True
        self.spare = order[at:]

        def fill():
            x = torch.randn((pages, page, kv_heads, dim), generator=g, device="cuda") * scale
            x[~own] = float("nan")
            x = x.to(self.dtype)
            return x if layout == "slot" else x.transpose(1, 2).contiguous().transpose(1, 2)

        self.k, self.v = fill(), fill()
        self.page, self.kv_heads, self.dim, self.lens_list = page, kv_heads, dim, list(lens)
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.cache = PagedCache(self.k, self.v)

    def offsets(self, counts):
        return self.t.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), device="cuda")

    def random(self, *shape, scale=1.0):
        return (self.t.randn(shape, generator=self.g, device="cuda") * scale).to(self.dtype)

    def rows(self, x, b, n, head):
        j = self.t.arange(n, device="cuda")
        return x[self.table[b].long()[j // self.page], j % self.page, head].double()


def check_attend(c, q, counts, out, lse, causal, scale=None, scores=None, before=None):
    """Compares with the 64-bit definition under the tolerances above."""
    torch = c.t
    heads = q.shape[1]
    group = heads // c.kv_heads
    scale = c.dim ** -0.5 if scale is None else scale
    at = 0
    for b, (n, cnt) in enumerate(zip(c.lens_list, counts)):
        gathered = None if scores is None else torch.zeros((c.kv_heads, n), dtype=torch.float64, device="cuda")
        tol_g = None if scores is None else torch.zeros_like(gathered)
        for h in range(heads):
            kk, vv = c.rows(c.k, b, n, h // group), c.rows(c.v, b, n, h // group)
            x = q[at:at + cnt, h].double()
            s = x @ kk.T * scale
            seen = torch.ones((cnt, n), dtype=torch.bool, device="cuda")
            if causal:
                seen = torch.arange(n, device="cuda")[None] <= (torch.arange(cnt, device="cuda") + n - cnt)[:, None]
            mag = torch.where(seen, x.abs() @ kk.abs().T * abs(scale), 0.0)
            s = torch.where(seen, s, -torch.inf)
            want_lse = torch.logsumexp(s, 1) if n else torch.full((cnt,), -torch.inf, dtype=torch.float64, device="cuda")
            empty = want_lse == -torch.inf
            p = torch.where(empty[:, None], 0.0, torch.exp(s - want_lse[:, None]))
            want = p @ vv
            ds = 2 * (c.dim + 8) * E * (mag.amax(1) if n else mag.sum(1))
            sums = (n / 32 + 64) * E
            err = (lse[at:at + cnt, h].double() - want_lse).abs()
            assert torch.equal(lse[at:at + cnt, h] == -torch.inf, empty), f"empty rows, sequence {b} head {h}"
            bad = (err > ds + sums + 2 * E * want_lse.abs())[~empty]
            assert not bad.any(), f"lse: sequence {b} head {h}: {err[~empty].max().item():.3g}"
            got = out[at:at + cnt, h].double()
            tiny = 2.0 ** -25 * p.amax(1, keepdim=True) * vv.abs().sum(0) if n and c.dtype == torch.float16 else 0.0
            tol = c.u * want.abs() + (c.u + 4 * ds[:, None] + 2 * sums) * (p @ vv.abs()) + tiny + 2.0 ** -24
            assert torch.isfinite(got).all(), f"out: sequence {b} head {h} is not finite"
            over = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
            assert over <= 0, f"out: sequence {b} head {h}: over the tolerance by {over:.3g}"
            if scores is not None:
                gathered[h // group] += p.sum(0)
                tol_g[h // group] += ((4 * ds[:, None] + 2 * sums + (cnt * group / 8 + 64) * E) * p).sum(0)
        if scores is not None:
            w = scores.shape[2]
            want_s = before[b].double()
            want_s[:, :min(n, w)] += gathered[:, :w]
            tol = 2 * E * want_s.abs()
            tol[:, :min(n, w)] += tol_g[:, :w]
            over = ((scores[b].double() - want_s).abs() - tol).max().item()
            assert over <= 0, f"scores of sequence {b}: over the tolerance by {over:.3g}"
        at += cnt


def attend_and_check(c, counts, heads, causal, with_scores=False, max_q=0, width=None, qscale=2.0, scale=None):
    torch = c.t
    q = c.random(sum(counts), heads, c.dim, scale=qscale)
    scores = before = None
    if with_scores:
        width = max(c.lens_list + [1]) if width is None else width
        scores = torch.rand((len(counts), c.kv_heads, width), generator=c.g, device="cuda")
        before = scores.clone()
    out, lse = c.cache.attend(q, c.offsets(counts), c.table, c.lens, causal=causal, scores=scores, max_q=max_q, scale=scale)
    c.cache.sync()
    check_attend(c, q, counts, out, lse, causal, scale, scores, before)
    return q, out, lse


# (lens, new tokens, heads, kv heads, dim, page): steps, drafts and chunks; lengths 0 and 1, around tile and page ends
SHAPES = [
    ([1], [1], 1, 1, 8, 8),
    ([0, 1, 2, 7, 8, 9], [1, 1, 1, 1, 1, 1], 4, 4, 64, 8),
    ([15, 16, 17, 31, 33, 63, 64, 65], [1] * 8, 8, 1, 128, 16),
    ([127, 128, 129, 255, 257, 1023], [1] * 6, 32, 8, 128, 32),
    ([3001, 17, 0, 900], [1, 1, 1, 1], 12, 4, 96, 64),
    ([5000], [1], 64, 4, 128, 1024),
    ([777, 300, 40], [1, 1, 1], 24, 1, 80, 16),      # 24 query heads to one kv head
    ([500, 129], [1, 1], 128, 1, 64, 128),
    ([700, 64, 5], [2, 5, 3], 6, 2, 72, 16),
    ([1000, 1000], [4, 16], 8, 2, 128, 128),
    ([9, 40, 130], [9, 40, 130], 4, 2, 64, 8),        # prompts with nothing before them
    ([5, 0, 20], [9, 4, 33], 4, 2, 128, 16),          # more new tokens than slots: rows that see nothing
    ([600, 513, 1], [100, 257, 1], 10, 2, 112, 64),   # 5 heads to a group: tiles of 125 rows
    ([1500], [700], 3, 3, 128, 256),
    ([400, 333], [130, 200], 16, 1, 40, 32),
    ([2100, 3, 650, 0, 90], [1, 3, 300, 0, 64], 16, 4, 128, 64),  # steps, chunks and nothing in one call
]


@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,layout", [("bfloat16", "slot"), ("float16", "head")])
def test_attend_matches_definition(shape, causal, dtype, layout):
    lens, counts, heads, kv_heads, dim, page = shape
    c = Cache(lens, page, kv_heads, dim, dtype, layout, seed=len(lens) * 100 + dim)
    attend_and_check(c, counts, heads, causal, with_scores=True)
    attend_and_check(c, counts, heads, causal, max_q=max(counts))


@pytest.mark.parametrize("counts", [[1, 1, 1], [90, 64, 7]])
def test_attend_peaked_and_uniform_weights(counts):
    """Scales that make one weight of nearly one (maxima that keep growing along the slots) and all weights equal."""
    c = Cache([1111, 640, 300], 32, 2, 128, "float16", seed=5)
    c.k *= c.t.linspace(0.1, 3.0, c.k.shape[0], device="cuda")[:, None, None, None].to(c.dtype)
    attend_and_check(c, counts, 8, True, with_scores=True, qscale=12.0)
    attend_and_check(c, counts, 8, True, with_scores=True, qscale=0.0)
    attend_and_check(c, counts, 8, False, with_scores=True, scale=-0.25)


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [33, 70, 20, 128]])
def test_attend_shared_pages_and_narrow_scores(counts):
    """Sequences that begin with the same pages; fewer scores than slots."""
    c = Cache([640, 700, 513, 900], 64, 2, 64, seed=9, shared=6)
    attend_and_check(c, counts, 8, False, with_scores=True, width=200)


@pytest.mark.parametrize("counts", [[1, 1], [40, 81]])
def test_attend_strided_rows(counts):
    """q as a slice of one projection's output, out inside a larger tensor, a table that is part of a wider one."""
    torch = __import__("torch")
    c = Cache([300, 517], 16, 2, 64, seed=3)
    fused = c.random(sum(counts), 6 + 4, 64, scale=2.0)
    q = fused[:, 2:8]
    room = torch.full((sum(counts), 9, 64), 7.0, dtype=c.dtype, device="cuda")
    wide = torch.full((2, c.table.shape[1] + 5), NO_PAGE, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table
    out, lse = c.cache.attend(q, c.offsets(counts), wide[:, :c.table.shape[1]], c.lens, out=room[:, 1:7])
    c.cache.sync()
    check_attend(c, q, counts, out, lse, True)
    assert (room[:, 0] == 7).all() and (room[:, 7:] == 7).all(), "rows beside out were written"


def test_attend_ignores_other_rows_nan():
    """NaN in one sequence's rows stays there: the others' results and weights do not change by a bit."""
    torch = __import__("torch")
    counts = [70, 1, 50]
    c = Cache([300, 200, 260], 32, 2, 128, seed=8)
    q = c.random(sum(counts), 8, 128)
    s1, s2 = (torch.zeros((3, 2, 300), device="cuda") for _ in range(2))
    o1, l1 = c.cache.attend(q, c.offsets(counts), c.table, c.lens, scores=s1)
    bad = q.clone()
    bad[70] = float("nan")
    o2, l2 = c.cache.attend(bad, c.offsets(counts), c.table, c.lens, scores=s2)
    c.cache.sync()
    keep = torch.arange(121, device="cuda") != 70
    assert torch.equal(o1[keep], o2[keep]) and torch.equal(l1[keep], l2[keep])
    assert torch.equal(s1[0], s2[0]) and torch.equal(s1[2], s2[2])


@pytest.mark.parametrize("counts,heads", [([1, 1, 1], 16), ([128, 300, 9], 8)])
def test_attend_repeats_bit_for_bit(counts, heads):
    """Equal calls give equal bits, on another stream and from a captured graph too."""
    torch = __import__("torch")
    c = Cache([4000, 2500, 700], 64, 2, 128, seed=2)
    q = c.random(sum(counts), heads, 128)
    off = c.offsets(counts)
    s0 = torch.zeros((3, 2, 4000), device="cuda")
    o0, l0 = c.cache.attend(q, off, c.table, c.lens, scores=s0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        s1 = torch.zeros_like(s0)
        torch.cuda.synchronize()
        o1, l1 = c.cache.attend(q, off, c.table, c.lens, scores=s1, stream=st)
        st.synchronize()
        assert torch.equal(o0, o1) and torch.equal(l0, l1) and torch.equal(s0, s1)
    s2 = torch.zeros_like(s0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, l2 = c.cache.attend(q, off, c.table, c.lens, scores=s2)
    for _ in range(2):
        s2.zero_()
        o2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o0, o2) and torch.equal(l0, l2) and torch.equal(s0, s2)
    c.cache.sync()


@pytest.mark.parametrize("counts", [[1, 1], [40, 33]])
def test_offsets_beyond_32_bits(counts):
    """Pages whose elements lie past 2^31 (keys and values in one tensor to save memory)."""
    torch = __import__("torch")

    from veckern_b200 import PagedCache

    c = Cache([150, 90], 64, 64, 128, seed=4)
    pages = 2 ** 31 // (64 * 64 * 128) + 8
    big = torch.zeros((pages, 64, 64, 128), dtype=c.dtype, device="cuda")
    last = torch.arange(pages - c.k.shape[0], pages, device="cuda")
    big[last] = c.k
    big[last[0] - 1] = float("nan")
    table = torch.where(c.table == NO_PAGE, NO_PAGE, c.table + int(last[0])).to(torch.int32)
    assert int(last[-1]) * 64 * 64 * 128 > 2 ** 31
    with PagedCache(big, big) as cache:
        q = c.random(sum(counts), 64, 128)
        s = torch.zeros((2, 64, 150), device="cuda")
        before = s.clone()
        out, lse = cache.attend(q, c.offsets(counts), table, c.lens, scores=s)
        cache.sync()
        c.v = c.k
        check_attend(c, q, counts, out, lse, True, None, s, before)
        k = c.random(sum(counts), 64, 128)
        cache.append(k, k, c.offsets(counts), table, c.lens)
        cache.sync()
        for b, cnt in enumerate(counts):
            n = c.lens_list[b]
            j = torch.arange(n - cnt, n, device="cuda")
            at = sum(counts[:b])
            assert torch.equal(big[table[b].long()[j // 64], j % 64], k[at:at + cnt])
        new = torch.tensor([[int(last[0]) - 1], [int(last[0]) - 2]], dtype=torch.int32, device="cuda")
        kept, _, _ = cache.evict(table, c.lens, new, 50, 10, torch.rand((2, 64, 150), device="cuda"))
        cache.sync()
        for b in range(2):
            for h in (0, 63):
                j = kept[b, h].long()
                assert torch.equal(big[new[b, 0].long(), :50, h], big[table[b].long()[j // 64], j % 64, h])


@pytest.mark.parametrize("most", [1, 40])
def test_attend_many_short_sequences(most):
    """More sequences than a block has threads, of all small lengths, some without new tokens."""
    rng = np.random.default_rng(most)
    lens = [int(x) for x in rng.integers(0, 70, 1500)]
    counts = [int(x) for x in rng.integers(0, most + 1, 1500)]
    c = Cache(lens, 8, 1, 32, "float16", seed=most)
    heads = 2
    q = c.random(sum(counts), heads, 32, scale=2.0)
    s = c.t.zeros((1500, 1, 70), device="cuda")
    before = s.clone()
    out, lse = c.cache.attend(q, c.offsets(counts), c.table, c.lens, scores=s, max_q=most)
    c.cache.sync()
    check_attend(c, q, counts, out, lse, True, None, s, before)


def test_attend_reports_a_bound_that_does_not_hold():
    """A sequence with more new tokens than max_q says is left out, and reported."""
    torch = __import__("torch")
    c = Cache([100, 60], 16, 1, 64, seed=6)
    counts = [1, 5]
    q = c.random(6, 4, 64)
    for s in (None, torch.zeros((2, 1, 100), device="cuda")):
        c.cache.attend(q, c.offsets(counts), c.table, c.lens, max_q=1, scores=s)
        with pytest.raises(N.VkError, match="out of range"):
            c.cache.sync()


def test_attend_no_tokens_and_no_sequences():
    torch = __import__("torch")
    c = Cache([30], 8, 1, 64)
    out, lse = c.cache.attend(c.random(0, 2, 64), c.offsets([0]), c.table, c.lens)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    none = torch.zeros((0,), dtype=torch.int32, device="cuda")
    c.cache.attend(c.random(0, 2, 64), c.offsets([]), c.table[:0], none)
    c.cache.append(c.random(0, 1, 64), c.random(0, 1, 64), c.offsets([]), c.table[:0], none)
    c.cache.sync()
    # sequences without slots, through a table without columns
    empty = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    s = torch.ones((2, 1, 4), device="cuda")
    out, lse = c.cache.attend(c.random(41, 2, 64), c.offsets([1, 40]), empty, torch.zeros(2, dtype=torch.int32, device="cuda"),
                              scores=s)
    c.cache.sync()
    assert (out == 0).all() and (lse == -torch.inf).all() and (s == 1).all()


@pytest.mark.parametrize("dtype,layout", [("bfloat16", "slot"), ("float16", "head")])
@pytest.mark.parametrize("lens,counts,dim,page", [([1, 9, 40], [1, 1, 1], 64, 8), ([300, 17, 64, 5], [120, 17, 0, 2], 128, 16),
                                                  ([2000], [1999], 72, 1024)])
def test_append_writes_its_slots_only(lens, counts, dim, page, dtype, layout):
    torch = __import__("torch")
    c = Cache(lens, page, 3, dim, dtype, layout, seed=dim)
    fused = c.random(sum(counts), 2, 3, dim)
    k, v = fused[:, 0], fused[:, 1]
    want_k, want_v = c.k.clone(), c.v.clone()
    at = 0
    for b, (n, cnt) in enumerate(zip(lens, counts)):
        j = torch.arange(n - cnt, n, device="cuda")
        pages = c.table[b].long()[j // page]
        want_k[pages, j % page], want_v[pages, j % page] = k[at:at + cnt], v[at:at + cnt]
        at += cnt
    c.cache.append(k, v, c.offsets(counts), c.table, c.lens)
    c.cache.sync()
    for got, want in ((c.k, want_k), (c.v, want_v)):
        assert torch.equal(got.contiguous().view(torch.int16), want.contiguous().view(torch.int16))


def evict_plain(scores, n, keep, recent):
    """Old slots kept for one (sequence, head), by numpy's stable sort."""
    k = min(n, keep)
    r = min(recent, k)
    s = np.zeros(n, np.float32)
    w = min(n, scores.shape[0])
    s[:w] = scores[:w]
    s = np.where(np.isnan(s), -np.inf, s)[:n - r]
    lowest = np.isnan(scores[:n - r][:w]) if w else np.zeros(0, bool)
    key = np.zeros(n - r, [("s", "f4"), ("nan", "?")])
    key["s"] = s
    key["nan"][:lowest.shape[0]] = lowest
    order = np.lexsort((np.arange(n - r), key["nan"], -key["s"]))  # larger score first, NaN last, then the lower slot
    return np.concatenate([np.sort(order[:k - r]), np.arange(n - r, n)]).astype(np.int32)


EVICTS = [
    # lens, kv heads, dim, page, keep, recent, kind of scores
    ([10], 1, 8, 8, 4, 2, "random"),
    ([0, 1, 5, 33, 100], 2, 64, 8, 16, 4, "random"),
    ([1087], 8, 128, 16, 1024, 64, "random"),
    ([3000, 2999, 64, 1500], 3, 96, 64, 1000, 0, "ties"),
    ([2500, 700], 2, 128, 32, 600, 600, "random"),       # the latest alone
    ([2500, 700], 2, 72, 32, 699, 1, "same"),            # all equal: the first ones
    ([9000], 2, 64, 128, 4000, 100, "special"),          # NaN, infinities, signed zeros, negatives
    ([40000, 100], 1, 64, 64, 20001, 33, "random"),
    ([400, 300], 2, 64, 16, 0, 0, "random"),
    ([5000], 1, 64, 64, 1200, 10, "narrow"),             # fewer scores than slots
    ([150000], 1, 8, 1024, 70000, 1024, "ties"),
]


@pytest.mark.parametrize("case", EVICTS, ids=[f"{c[6]}{i}" for i, c in enumerate(EVICTS)])
@pytest.mark.parametrize("dtype,layout", [("bfloat16", "slot"), ("float16", "head")])
def test_evict_keeps_the_right_slots(case, dtype, layout):
    torch = __import__("torch")
    lens, kv_heads, dim, page, keep, recent, kind = case
    fresh = [-(-min(n, keep) // page) for n in lens]
    c = Cache(lens, page, kv_heads, dim, dtype, layout, seed=keep, extra=sum(fresh) + 1)
    width = max(lens) if kind != "narrow" else max(lens) // 2
    rng = np.random.default_rng(len(lens) + keep)
    s = rng.exponential(size=(len(lens), kv_heads, width)).astype(np.float32)
    if kind == "ties":
        s = np.floor(s * 4)
    elif kind == "same":
        s[:] = 0.5
    elif kind == "special":
        s[..., ::3] *= -1
        s[..., 1::50] = np.nan
        s[..., 2::60] = np.inf
        s[..., 3::70] = -np.inf
        s[..., 4::9], s[..., 5::9] = 0.0, -0.0
    new_table = torch.full((len(lens), max(fresh) + 1), NO_PAGE, dtype=torch.int32, device="cuda")
    at = 0
    for b, w in enumerate(fresh):
        new_table[b, :w] = c.spare[at:at + w]
        at += w
    k0, v0 = c.k.clone(), c.v.clone()
    kept, new_lens, new_scores = c.cache.evict(c.table, c.lens, new_table, keep, recent, torch.from_numpy(s).cuda())
    c.cache.sync()
    kept_h, new_h = kept.cpu().numpy(), new_scores.cpu().numpy()
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    for b, n in enumerate(lens):
        for h in range(kv_heads):
            want = evict_plain(s[b, h], n, keep, recent)
            k = want.shape[0]
            assert np.array_equal(kept_h[b, h, :k], want) and (kept_h[b, h, k:] == -1).all(), f"sequence {b} head {h}"
            full = np.zeros(max(n, width), np.float32)
            full[:width] = s[b, h]
            want_s = np.zeros(width, np.float32)
            want_s[:min(k, width)] = full[want][:width]
            assert np.array_equal(new_h[b, h], want_s, equal_nan=True)
            if k:
                old = torch.from_numpy(want).cuda().long()
                to = torch.arange(k, device="cuda")
                p0, p1 = c.table[b].long()[old // page], new_table[b].long()[to // page]
                for x, x0 in ((c.k, k0), (c.v, v0)):
                    assert torch.equal(x[p1, to % page, h], x0[p0, old % page, h])
    # nothing else was written
    for x, x0 in ((c.k, k0), (c.v, v0)):
        same = x.contiguous().view(torch.int16) == x0.contiguous().view(torch.int16)
        own = torch.zeros(x.shape[:2], dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            to = torch.arange(min(n, keep), device="cuda")
            own[new_table[b].long()[to // page], to % page] = True
        assert same.all(-1).all(-1)[~own].all()


def test_what_the_kernels_refuse():
    """Page numbers, lengths and offsets out of range are reported by sync, name no memory, and do not stick."""
    torch = __import__("torch")
    c = Cache([100, 60], 16, 2, 64, seed=6)
    q = c.random(2, 4, 64)
    off = c.offsets([1, 1])
    good, _ = c.cache.attend(q, off, c.table, c.lens, causal=False)
    c.cache.sync()
    for counts in ([1, 1], [20, 1]):
        many = c.random(sum(counts), 4, 64)
        for wrong in (-5, c.k.shape[0], NO_PAGE):
            t = c.table.clone()
            t[0, 2] = wrong
            s = torch.zeros((2, 2, 100), device="cuda")
            out, lse = c.cache.attend(many, c.offsets(counts), t, c.lens, causal=False, scores=s)
            with pytest.raises(N.VkError, match="out of range"):
                c.cache.sync()
            assert torch.isfinite(out).all()
            c.cache.append(c.random(sum(counts), 2, 64), c.random(sum(counts), 2, 64), c.offsets(counts), t - 1000000, c.lens)
            with pytest.raises(N.VkError, match="out of range"):
                c.cache.sync()
        for lens in ([-1, 60], [100, 10 ** 9]):
            bad = torch.tensor(lens, dtype=torch.int32, device="cuda")
            t = torch.zeros_like(c.table)
            c.cache.attend(many, c.offsets(counts), t, bad, causal=False)
            with pytest.raises(N.VkError, match="out of range"):
                c.cache.sync()
        for o in ([0, 5, 2], [-3, 1, 2], [0, 1, 10 ** 6]):
            bad = torch.tensor(o, dtype=torch.int32, device="cuda")
            c.cache.attend(many, bad, c.table, c.lens, causal=False)
            with pytest.raises(N.VkError, match="out of range"):
                c.cache.sync()
    c.cache.append(c.random(9, 2, 64), c.random(9, 2, 64), c.offsets([9]), c.table[:1], c.t.tensor([5], dtype=torch.int32, device="cuda"))
    with pytest.raises(N.VkError, match="out of range"):
        c.cache.sync()
    again, _ = c.cache.attend(q, off, c.table, c.lens, causal=False)
    c.cache.sync()


def test_what_python_refuses():
    torch = __import__("torch")
    from veckern_b200 import PagedCache

    c = Cache([100, 60], 16, 2, 64, seed=6)
    q, off = c.random(2, 4, 64), c.offsets([1, 1])
    ok = dict(causal=True)
    for args in ((q.float(), off, c.table, c.lens), (q[0], off, c.table, c.lens), (q[:, :, :32], off, c.table, c.lens),
                 (q, off.long(), c.table, c.lens), (q, off[:2], c.table, c.lens), (q, off, c.table.long(), c.lens),
                 (q, off, c.table, c.lens[:1]), (q, off, c.table.T, c.lens), (q.cpu(), off, c.table, c.lens)):
        with pytest.raises(ValueError):
            c.cache.attend(*args, **ok)
    with pytest.raises(N.VkError, match="multiple of kv_heads"):
        c.cache.attend(c.random(2, 3, 64), off, c.table, c.lens)
    with pytest.raises(N.VkError, match="scale"):
        c.cache.attend(q, off, c.table, c.lens, scale=float("nan"))
    with pytest.raises(N.VkError, match="max_q"):
        c.cache.attend(q, off, c.table, c.lens, max_q=-1)
    with pytest.raises(N.VkError, match="aligned|strides"):
        c.cache.attend(torch.zeros((2, 4, 65), dtype=c.dtype, device="cuda")[:, :, 1:], off, c.table, c.lens)
    for s in (torch.zeros((2, 3, 100), device="cuda"), torch.zeros((2, 2, 100), device="cuda").half(),
              torch.zeros((2, 2, 100, 2), device="cuda")[..., 0]):
        with pytest.raises(ValueError):
            c.cache.attend(q, off, c.table, c.lens, scores=s)
    s = torch.zeros((2, 2, 100), device="cuda")
    with pytest.raises(ValueError):
        c.cache.evict(c.table, c.lens, c.table, 4, 5, s)
    with pytest.raises(ValueError):
        c.cache.append(c.random(2, 3, 64), c.random(2, 2, 64), off, c.table, c.lens)
    with pytest.raises(ValueError):
        c.cache.append(c.random(2, 2, 64), c.random(1, 2, 64), off, c.table, c.lens)
    x = torch.zeros((4, 16, 2, 64), dtype=torch.float16, device="cuda")
    for k, v in ((x.float(), x.float()), (x, x[:2]), (x, x.bfloat16()), (x.cpu(), x.cpu()), (x[..., ::2], x[..., ::2])):
        with pytest.raises(ValueError):
            PagedCache(k, v)
    for k in (x[:, :12], x[..., :4], x[:, :4], torch.zeros((4, 16, 2, 136), dtype=torch.float16, device="cuda"),
              torch.zeros((4, 16, 2, 65), dtype=torch.float16, device="cuda")[..., :64]):
        with pytest.raises(N.VkError):
            PagedCache(k, k)


def test_example_reads_what_it_found():
    """The example's path: search, read, forget, go on. The passage that a question is made of is found, gathers the
    largest weight, and its slots are what is kept of the passages; the last step agrees with the definition."""
    torch = __import__("torch")
    from veckern_b200.examples import retrieval_memory as ex

    r = ex.run(passages=1500, questions=9, steps=3, seed=3)
    hit = r["ids"] == r["about"][:, None]
    assert hit.any(1).all(), "the index missed a question's passage"
    assert torch.equal(r["read"].argmax(1), hit.int().argmax(1))
    assert r["lens"].tolist() == [r["keep"] + 3] * 9
    kept = r["kept"]
    assert (kept[:, :, -r["asked"]:] == torch.arange(8 * 64, 8 * 64 + r["asked"], device="cuda")).all()
    c = Cache.__new__(Cache)
    c.t, c.dtype, c.u = torch, r["k"].dtype, 2.0 ** -8
    c.k, c.v, c.table, c.page, c.kv_heads, c.dim = r["k"], r["v"], r["table"], ex.PAGE, ex.KV_HEADS, ex.DIM
    c.lens_list = r["lens"].tolist()
    check_attend(c, r["q"], [1] * 9, r["out"], r["lse"], True)
    r["cache"].close()
