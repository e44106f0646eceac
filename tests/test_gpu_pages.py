"""llmk_pages_update, llmk_pages_compact and llmk_pages_copy on the GPU against
the rows taken one after another in plain Python (pages_util.py): tables,
lengths, counts, free pages, what each row was granted, and every page's
contents, all equal."""
import numpy as np
import pytest
import torch

import llmk
from llmk import _lib
from pages_util import Plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampler():
    s = llmk.HipSampler(max_batch=1, max_vocab=1024)
    yield s
    s.close()


def dev(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32).to("cuda:0")


def host(t):
    return t.cpu().numpy().astype(np.int64)


def used_pages(cache):
    words = cache.used.cpu().numpy().view(np.uint32)
    return np.unpackbits(words.view(np.uint8), bitorder="little")[:cache.num_pages].astype(bool)


class Pair:
    """A cache on the GPU beside its plain form; page p of every pool is filled
    with words made from one number."""

    def __init__(self, sampler, rows, max_pages, page_tokens, num_pages, page_words=(4,), offset=0):
        self.plain = Plain(rows, max_pages, page_tokens, num_pages)
        self.sampler, self.pools = sampler, []
        for w in page_words:
            base = torch.zeros(num_pages * w + 8, dtype=torch.uint8, device="cuda:0")
            self.pools.append(base[offset:offset + num_pages * w].view(num_pages, w))
        for i, p in enumerate(self.pools):
            p.copy_(self.bytes_of(np.arange(num_pages), i, p.shape[1]))
        self.cache = llmk.PageCache(sampler, rows, max_pages, page_tokens, num_pages, self.pools)

    @staticmethod
    def bytes_of(numbers, pool, width):
        n = torch.as_tensor(numbers)[:, None] * 7919 + torch.arange(width)[None, :] * 31 + pool * 101
        return ((n ^ (n >> 7)) & 255).to(torch.uint8).to("cuda:0")

    def same(self):
        c, p = self.cache, self.plain
        assert np.array_equal(host(c.lengths), p.lengths)
        assert np.array_equal(host(c.refs), p.refs)
        assert np.array_equal(host(c.table), p.table)
        assert np.array_equal(used_pages(c), p.refs > 0)
        held = np.nonzero(p.refs > 0)[0]
        for i, t in enumerate(self.pools):
            assert torch.equal(t[torch.as_tensor(held).to("cuda:0")],
                               self.bytes_of(p.contents[held], i, t.shape[1]))
        # nothing is left over from one call to the next
        N, work = c.num_pages, c._work
        moves = 4 + 2 * max(c.rows, N // 2 + 1)
        assert not work[2:4].any()
        assert not work[moves:moves + 2 * N].any()

    def update(self, new=None, parents=None):
        g, invalid, full = self.plain.update(new, parents)
        got = self.cache.update(None if new is None else dev(new), None if parents is None else dev(parents))
        assert np.array_equal(host(got), g)
        want = (_lib.LLMK_STATUS_INVALID_PARAMS if invalid else 0) | (_lib.LLMK_STATUS_PAGES_FULL if full else 0)
        assert self.sampler.status() == want
        self.same()
        return g

    def compact(self):
        to = self.plain.compact()
        assert np.array_equal(host(self.cache.compact()), to)
        assert self.sampler.status() == 0
        self.same()


@pytest.mark.parametrize("rows,max_pages,page_tokens,num_pages,seed", [
    (1, 1, 1, 1, 0), (3, 4, 4, 7, 1), (16, 20, 16, 200, 2), (16, 20, 16, 64, 3), (70, 9, 1, 333, 4),
    (1500, 3, 5, 2100, 5), (1100, 4, 3, 900, 6)])
def test_random_steps(sampler, rows, max_pages, page_tokens, num_pages, seed):
    """Steps of any mix of forks, ends, cuts and growth, with enough pages and
    with too few, invalid requests among them; more rows than a workgroup has
    threads; rows that share a page on both sides of that."""
    rng = np.random.default_rng(seed)
    c = Pair(sampler, rows, max_pages, page_tokens, num_pages, page_words=(16, 5))
    most = max_pages * page_tokens
    for step in range(14):
        new = rng.integers(-1, most + 1, rows)
        kind = rng.random(rows)
        grow = np.minimum(c.plain.lengths + rng.integers(0, 3, rows), most)
        new = np.where(kind < 0.5, grow, np.where(kind < 0.65, 0, np.where(kind < 0.9, -1, new)))
        # children of few parents, so that many share a last page
        few = rng.integers(0, rows, 3)
        par = np.where((c.plain.lengths == 0) & (rng.random(rows) < 0.7), rng.choice(few, rows), -1)
        par[few] = -1
        child = par >= 0
        new = np.where(child & (rng.random(rows) < 0.7), np.minimum(c.plain.lengths[np.maximum(par, 0)] + 1, most), new)
        if step % 4 == 3:  # invalid requests
            at = rng.integers(0, rows, 3)
            par[at] = [rows, rng.integers(0, rows), at[2]]
            new[rng.integers(0, rows)] = most + 1
        c.update(new if step % 5 != 4 else None, par if step % 3 != 2 or step % 5 == 4 else None)
        if step % 6 == 5:
            c.compact()


def test_all_rows_that_share_a_page_grow(sampler):
    """Each takes a copy but the last; with one more holder that waits, every
    one does; with too few pages, the first ones do."""
    for wait in (False, True):
        for pages in (40, 12):
            c = Pair(sampler, 20, 4, 8, pages, page_words=(8,))
            c.update([13] + [-1] * 19)
            c.update(None, [-1] + [0] * 19)
            new = [14] * 20
            if wait:
                new[7] = -1
            g = c.update(new)
            assert g.sum() == (20 if pages == 40 else 10 + (1 if wait else 0))


def test_rows_that_pass_a_thousand_share_one_page(sampler):
    c = Pair(sampler, 2500, 2, 4, 2600, page_words=(12,))
    c.update([3] + [-1] * 2499)
    c.update(None, [-1] + [0] * 2499)
    c.update(np.where(np.arange(2500) % 3 == 0, 4, -1))
    c.update(np.full(2500, 5))


def test_long_rows(sampler):
    """A prompt of thousands of pages begins, is forked, and ends."""
    c = Pair(sampler, 4, 5000, 2, 12000, page_words=(8,))
    c.update([9999, 700, -1, -1])
    c.update([-1, -1, 8001, -1], [-1, -1, 0, -1])
    c.update([10000, 0, 9001, 5000])
    c.update([1, -1, 0, -1])
    c.compact()


@pytest.mark.parametrize("num_pages", [1, 31, 32, 33, 1024, 1025, 40000])
def test_number_of_pages(sampler, num_pages):
    """All pages taken, all given back, every second one kept, moved down."""
    rows = 8
    per = -(-num_pages // rows)
    c = Pair(sampler, rows, num_pages, 1, num_pages, page_words=(4,))
    c.update([min(per, max(0, num_pages - per * r)) for r in range(rows)])
    assert (c.plain.refs == 1).all()
    c.compact()
    c.update([0 if r % 2 == 0 else -1 for r in range(rows)])
    c.compact()
    c.update([0] * rows)
    c.compact()


@pytest.mark.parametrize("words", [(1,), (3,), (4, 7), (16,), (17,), (4096,), (16384, 100), (65552, 20000)])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_copies_of_any_size_and_alignment(sampler, words, offset):
    rng = np.random.default_rng(sum(words))
    n = 12 if words[0] > 10000 else 300
    pools = []
    for w in words:
        base = torch.randint(0, 256, (n * w + 40,), dtype=torch.uint8, device="cuda:0")
        pools.append((base, base[offset + 16:offset + 16 + n * w].view(n, w)))
    at = rng.permutation(n)
    k = n // 3
    src, dst = at[:k].copy(), at[k:2 * k]
    src[1] = src[0]  # one source for two copies
    want = []
    for base, p in pools:
        b = base.clone()
        b[offset + 16:offset + 16 + n * p.shape[1]].view(n, -1)[torch.as_tensor(dst).cuda()] = \
            p[torch.as_tensor(src).cuda()]
        want.append(b)
    sampler.copy_pages(llmk.PagePools([p for _, p in pools]), dev(src), dev(dst))
    torch.cuda.synchronize()
    for (base, _), b in zip(pools, want):
        assert torch.equal(base, b)
    assert sampler.status() == 0


def test_copies_of_pages_that_are_none(sampler):
    p = torch.arange(40, dtype=torch.int32, device="cuda:0").view(10, 4)
    want = p.clone()
    want[3] = want[2]
    sampler.copy_pages(llmk.PagePools([p]), dev([10, 2, 1, -1]), dev([0, 3, 2**31 - 1, 4]))
    assert torch.equal(p, want)
    assert sampler.status() == _lib.LLMK_STATUS_INVALID_PARAMS
    sampler.copy_pages(llmk.PagePools([p]), dev([]), dev([]))


def test_pages_past_32_bit_offsets(sampler):
    """Pools of more than 4 GiB: the last page copied, grown into and moved."""
    n, words = 1200, 1 << 20  # 4 MiB a page
    pool = torch.zeros(n, words, dtype=torch.int32, device="cuda:0")
    c = llmk.PageCache(sampler, 3, n, 1, n, [pool])
    assert host(c.update(dev([n - 1, 1, -1]))).all()
    pool[n - 1] = 5
    c.update(dev([0, -1, -1]))
    to = host(c.compact())
    assert to[n - 1] == 0 and c.table[1, 0].item() == 0 and bool((pool[0] == 5).all())
    pool[7] = 9
    c.copy(dev([7]), dev([n - 1]))
    assert bool((pool[n - 1] == 9).all()) and not bool(pool[n - 2].any())
    del pool, c
    torch.cuda.empty_cache()


def test_a_cache_that_was_not_kept(sampler):
    """Entries that are no pages, pages nobody holds, lengths past the table:
    bounded, and reported."""
    c = llmk.PageCache(sampler, 6, 4, 4, 10, [torch.zeros(10, 16, dtype=torch.uint8, device="cuda:0")])
    c.update(dev([16, 16, -1, -1, -1, -1]))
    c.table[0, 1], c.table[1, 3] = 77, -1
    c.lengths[5] = 1000
    g = host(c.update(dev([0, -1, 10, 10, -1, 3]), dev([-1, -1, 1, 5, -1, -1])))
    assert g[3] == 0  # no such prefix to fork
    assert sampler.status() & _lib.LLMK_STATUS_INVALID_PARAMS
    c.compact()
    torch.cuda.synchronize()
    sampler.status()


def test_load_and_snapshots(sampler):
    a = Pair(sampler, 12, 6, 4, 90, page_words=(8,))
    rng = np.random.default_rng(3)
    a.update(rng.integers(0, 25, 12))
    a.update([0] * 6 + [-1] * 6)
    a.update([-1] * 12, [6, 7, 8] + [-1] * 9)
    b = llmk.PageCache(sampler, 12, 6, 4, 90)
    b.load(a.cache.table, a.cache.lengths)
    assert torch.equal(a.cache.state, b.state)
    saved = b.state.clone()
    b.update(dev([24] * 12))
    b.state.copy_(saved)
    assert np.array_equal(host(b.update(dev([5] * 12))), a.update([5] * 12))
    assert torch.equal(a.cache.state, b.state)
    with pytest.raises(llmk.SamplerError, match="out of range"):
        b.load(torch.full((12, 6), 90), torch.full((12,), 3))
    with pytest.raises(llmk.SamplerError, match="table must be"):
        b.load(torch.zeros(12, 5), torch.zeros(12))


def test_refusals(sampler):
    pool = torch.zeros(8, 4, device="cuda:0")
    c = llmk.PageCache(sampler, 2, 4, 4, 8, [pool])
    for call, word in ((lambda: c.update(), "nothing"),
                       (lambda: c.update(dev([1])), "entry per row"),
                       (lambda: c.update(torch.zeros(2, device="cuda:0")), "contiguous"),
                       (lambda: c.update(torch.zeros(2, dtype=torch.int32)), "is on cpu"),
                       (lambda: c.copy(dev([1]), dev([1, 2])), "differ"),
                       (lambda: llmk.PageCache(sampler, 2, 4, 4, 9, [pool]), "num_pages 9"),
                       (lambda: llmk.PageCache(sampler, 0, 4, 4, 9), "rows"),
                       (lambda: llmk.PageCache(sampler, 2, 2**20, 2**12, 9).update(dev([1, 1])), "2.31"),
                       (lambda: llmk.PagePools([pool, torch.zeros(9, 4, device="cuda:0")]), "pools must"),
                       (lambda: llmk.PagePools([pool.t()]), "pools must"),
                       (lambda: llmk.PageCache(sampler, 2, 4, 4, 9).copy(dev([1]), dev([2])), "no pools")):
        with pytest.raises(llmk.SamplerError, match=word):
            call()


def test_graph_replays(sampler):
    """A step captured once, replayed as the rows' requests change on the device,
    with eager calls on another cache between the replays; every replay against
    the plain form."""
    c = Pair(sampler, 10, 8, 4, 60, page_words=(32,))
    other = Pair(sampler, 5, 4, 4, 30, page_words=(8,))
    new, par = dev([-1] * 10), dev([-1] * 10)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c.cache.update(new, par)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        granted = c.cache.update(new, par)
        moved = c.cache.compact()
    rng = np.random.default_rng(1)
    for i in range(8):
        n = np.minimum(c.plain.lengths + rng.integers(-1, 5, 10), 32)
        p = np.where(c.plain.lengths == 0, (np.arange(10) + 1) % 10, -1) if i % 2 else np.full(10, -1)
        new.copy_(dev(n))
        par.copy_(dev(p))
        g.replay()
        want, invalid, full = c.plain.update(n, p)
        to = c.plain.compact()
        assert np.array_equal(host(granted), want) and np.array_equal(host(moved), to)
        c.same()
        assert sampler.status() == (_lib.LLMK_STATUS_INVALID_PARAMS if invalid else 0) | \
            (_lib.LLMK_STATUS_PAGES_FULL if full else 0)
        other.update(rng.integers(0, 17, 5))


def test_another_stream(sampler):
    c = Pair(sampler, 10, 8, 4, 60, page_words=(32,))
    st = torch.cuda.Stream()
    new, par = dev([9] + [-1] * 9), dev([-1] + [0] * 9)
    torch.cuda.synchronize()
    g0 = c.cache.update(new, stream=st)
    g1 = c.cache.update(parents=par, stream=st)
    g2 = c.cache.update(dev([10] * 10), stream=st)
    m = c.cache.compact(stream=st)
    st.synchronize()
    c.plain.update([9] + [-1] * 9)
    c.plain.update(None, [-1] + [0] * 9)
    c.plain.update([10] * 10)
    assert np.array_equal(host(m), c.plain.compact())
    assert host(g0).all() and host(g1).all() and host(g2).all()
    c.same()


def test_a_serving_step(sampler):
    """What a step does on the device around the sampling call: a prompt's row
    is forked into three samples with its history, each samples its own token
    from processed logits, appends it, and its pages grow; one sample ends."""
    s = llmk.HipSampler(max_batch=4, max_vocab=500)
    V, cap, B = 500, 64, 4
    rng = np.random.default_rng(0)
    prompt = rng.integers(0, V, 21)
    c = Pair(s, B, 8, 8, 24, page_words=(64,))
    hist = torch.zeros(B, cap, dtype=torch.int32, device="cuda:0")
    hist[0, :21] = dev(prompt)
    lens = dev([21, 0, 0, 0])
    off = dev(np.arange(B) * cap)
    c.update([21, -1, -1, -1])
    # the fork: pages by reference, history rows and lengths by copy
    c.update(None, [-1, 0, 0, 0])
    s.copy_pages(llmk.PagePools([hist]), dev([0, 0, 0]), dev([1, 2, 3]))
    s.copy_pages(llmk.PagePools([lens]), dev([0, 0, 0]), dev([1, 2, 3]))
    seen = [list(prompt) for _ in range(B)]
    alive = np.ones(B, bool)
    for step in range(12):
        lg = torch.as_tensor(rng.normal(0, 3, (B, V)).astype(np.float32)).cuda()
        lb = llmk.LogitsBatch(logits=lg, hist_offsets=off, hist_tokens=hist.view(-1), hist_lengths=lens,
                              repetition_penalty=torch.full((B,), 1.3, device="cuda:0"),
                              frequency_penalty=torch.full((B,), 0.2, device="cuda:0"))
        x = s.process_logits(lb)
        u = torch.as_tensor(rng.random(B).astype(np.float32)).cuda()
        d = s.sample_batch(llmk.DeviceBatch(logits=x, uniforms=u,
                                            top_k=torch.full((B,), 5, dtype=torch.int32, device="cuda:0")))
        r = s.logprobs(x, d.tokens, top_n=5)
        assert (r.ranks < 5).all()
        s.history_append(off, lens, hist.view(-1), cap, d.tokens)
        if step == 6:
            alive[2] = False
        c.update(np.where(alive, c.plain.lengths + 1, 0))
        # the plain form of the penalties on each row's own tokens
        for b in range(B):
            n = np.bincount(seen[b], minlength=V)
            v = lg[b].double().cpu().numpy()
            y = np.where(n > 0, np.where(v > 0, v / np.float32(1.3), v * np.float32(1.3)) - n * np.float32(0.2), v)
            assert np.abs(y - x[b].double().cpu().numpy()).max() < 30 * 8 * 2.0 ** -24 * 1.3
            seen[b].append(int(d.tokens[b]))
        assert np.array_equal(host(hist)[1, :host(lens)[1]], seen[1])
    s.close()


def test_more_pages_than_the_words_kept_in_shared_memory(sampler):
    """200000 pages (past 131072 their words stay in memory), rows of tens of
    thousands of them (more than the list of free pages kept there), given up,
    grown, moved."""
    c = Pair(sampler, 6, 60000, 4, 200000, page_words=(8,))
    c.update([4 * 40000, 4 * 30000 + 1, 17, 4 * 20000, -1, -1])
    c.update([0, -1, 4 * 5000, -1, -1, -1])
    c.update([-1, 4 * 30000 + 2, -1, 4 * 100, 4 * 30000 + 3, 4 * 50000], [-1, -1, -1, -1, 1, -1])
    c.update([4 * 60000] * 6)
    c.compact()
    c.update([1, 2, 3, 4, 5, 6])
    c.compact()


@pytest.mark.parametrize("rows", [511, 512, 513])
def test_rows_about_the_threads_of_a_workgroup(sampler, rows):
    c = Pair(sampler, rows, 3, 4, 2 * rows, page_words=(8,))
    c.update([(r * 7) % 13 for r in range(rows)])
    new = c.plain.lengths + 1
    new[::5] = 0
    c.update(new)
    par = np.where(c.plain.lengths == 0, 1, -1)
    c.update(np.where(par >= 0, c.plain.lengths[1] + 1, -1), par)
    c.compact()
