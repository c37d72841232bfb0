"""KVPages without a GPU: against lists of tokens, with a cache of plain numbers in the place of
the device's."""
import ctypes

import numpy as np
import pytest
import torch

import jhq_gpu_amd as jg


class Batch:
    def __init__(self, pages, kv_len, cu_q, n_tokens, max_q, max_kv):
        # as they are when a kernel that is enqueued now runs
        self.pages, self.kv_len, self.cu_q = (x.numpy().copy() for x in (pages, kv_len, cu_q))
        self.n_tokens, self.max_q, self.max_kv = n_tokens, max_q, max_kv
        assert max_kv <= self.pages.shape[1] * Cache.page_size
        assert self.cu_q[-1] == n_tokens and (np.diff(self.cu_q) >= 0).all()
        assert np.diff(self.cu_q).max(initial=0) <= max_q and self.kv_len.max(initial=0) <= max_kv


class Cache:
    """A token is a number in a slot."""
    page_size = 4
    device = torch.device("cpu")

    def __init__(self, num_pages):
        self.num_pages = num_pages
        self.slots = np.full((num_pages, self.page_size), -1, np.int64)
        self.copied = 0

    def batch(self, *a):
        return Batch(*a)

    def new_slots(self, b):
        out = []
        for s in range(len(b.kv_len)):
            q, n = b.cu_q[s + 1] - b.cu_q[s], b.kv_len[s]
            for j in range(n - q, n):
                out.append((b.pages[s, j // self.page_size], j % self.page_size))
        return out

    def write(self, tokens, b):
        at = self.new_slots(b)
        assert len(at) == len(tokens) and len(set(at)) == len(at), "a slot is written twice"
        for (p, i), t in zip(at, tokens):
            self.slots[p, i] = t

    def copy_pages(self, src, dst):
        src, dst = src.numpy(), dst.numpy()
        assert len(set(dst.tolist())) == len(dst) and not set(src.tolist()) & set(dst.tolist())
        self.slots[dst] = self.slots[src]
        self.copied += len(dst)

    def copy(self, slots, b):
        at = self.new_slots(b)
        src = slots.numpy()
        assert src.dtype == np.int64 and len(at) == len(src)
        flat = {int(p) * self.page_size + int(i) for p, i in at}
        assert len(flat) == len(at) and not flat & set(src.tolist())
        got = self.slots.reshape(-1)[src].copy()
        for (p, i), t in zip(at, got):
            self.slots[p, i] = t

    def read(self, b):
        return [int(self.slots[p, i]) for p, i in self.new_slots(b)]


def _check(pages, cache, model):
    assert [pages.length(s) for s in range(len(model))] == [len(m) for m in model]
    assert cache.read(pages.everything()) == sum(model, [])
    held = [p for s in range(len(model)) for p in pages.pages_of(s)]
    assert pages.free_pages == cache.num_pages - len(set(held))
    assert pages.free_pages == len(set(pages._free)) and not set(pages._free) & set(held)
    assert (pages._refs == np.bincount(np.array(held, np.int64), minlength=cache.num_pages)).all()


@pytest.mark.parametrize("seed", range(30))
def test_against_lists(seed):
    rng = np.random.default_rng(seed)
    n_seq, most = int(rng.integers(1, 7)), 40
    cache = Cache(int(rng.integers(5, 60)))
    pages = jg.KVPages(cache, n_seq, most)
    model = [[] for _ in range(n_seq)]
    token, full = 0, 0
    for _ in range(150):
        what = rng.choice(["extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        s = int(rng.integers(0, n_seq))
        if what == "extend":
            new = rng.integers(0, int(rng.choice([2, 2, 9])), n_seq)
            new = np.minimum(new, most - np.array([len(m) for m in model]))
            before = (pages._table.copy(), pages._refs.copy(), pages._len.copy(), list(pages._free))
            try:
                b = pages.extend(new)
            except RuntimeError as e:
                assert "full" in str(e)
                full += 1
                assert all(np.array_equal(x, y) for x, y in
                           zip(before, (pages._table, pages._refs, pages._len, pages._free)))
                continue
            tokens = list(range(token, token + int(new.sum())))
            token += len(tokens)
            cache.write(tokens, b)
            for m, a in zip(model, new):
                m += tokens[:a]
                tokens = tokens[a:]
        elif what == "fork":
            d = int(rng.integers(0, n_seq))
            if d == s or model[d]:
                with pytest.raises(ValueError):
                    pages.fork(s, d)
            else:
                pages.fork(s, d)
                model[d] = list(model[s])
        elif what == "truncate":
            n = int(rng.integers(0, len(model[s]) + 1))
            pages.truncate(s, n)
            model[s] = model[s][:n]
        elif what == "free":
            if rng.random() < 0.3:
                pages.free(s)
                model[s] = []
        else:
            keep = {}
            for d in range(n_seq):
                if rng.random() < 0.5:
                    keep[d] = np.nonzero(rng.random(len(model[d])) < rng.choice([0.2, 0.8, 1.0]))[0]
            try:
                pages.compact(keep)
            except RuntimeError:
                continue
            for d, at in keep.items():
                model[d] = [model[d][i] for i in at]
        _check(pages, cache, model)
    assert token > 20


def _grown(lens, num_pages=60, forks=()):
    cache = Cache(num_pages)
    pages = jg.KVPages(cache, len(lens), 100)
    b = pages.extend(lens)
    cache.write(list(range(sum(lens))), b)
    for a, d in forks:
        pages.fork(a, d)
    return cache, pages


def test_pages_are_shared_until_they_are_written():
    cache, pages = _grown([10, 0, 0, 0], forks=[(0, 1), (0, 2)])
    assert pages.free_pages == 57 and pages.pages_of(0) == pages.pages_of(2) == [0, 1, 2]
    pages.extend([1, 1, 1, 0])
    # the last one to write keeps the page
    assert cache.copied == 2 and pages.pages_of(2) == [0, 1, 2]
    assert pages.pages_of(0)[:2] == [0, 1] and pages.free_pages == 55
    pages.extend([1, 0, 0, 0])  # its own by now (and full with it)
    assert cache.copied == 2
    pages.extend([1, 0, 0, 0])  # a page of its own from the start
    assert cache.copied == 2 and pages.free_pages == 54


def test_a_full_page_is_not_copied():
    cache, pages = _grown([8, 0], forks=[(0, 1)])
    pages.extend([1, 5])
    assert cache.copied == 0 and pages.pages_of(0)[:2] == pages.pages_of(1)[:2]


def test_truncation_into_a_shared_page():
    cache, pages = _grown([8, 0], forks=[(0, 1)])
    pages.truncate(1, 5)
    b = pages.extend([0, 2])
    cache.write([100, 101], b)
    assert cache.copied == 1
    assert cache.read(pages.everything()) == list(range(8)) + [0, 1, 2, 3, 4, 100, 101]


def test_compaction_keeps_whole_pages_in_front():
    cache, pages = _grown([30, 3], forks=[])
    before = pages.pages_of(0)
    keep = list(range(9)) + [11, 20, 29]
    pages.compact({0: keep, 1: [0, 1]})
    assert pages.pages_of(0)[:2] == before[:2] and pages.pages_of(0)[2] not in before
    assert cache.read(pages.everything()) == keep + [30, 31]
    pages.compact({0: [], 1: np.array([1])})
    assert pages.length(0) == 0 and cache.read(pages.everything()) == [31]


def test_compaction_of_a_shared_sequence():
    cache, pages = _grown([12, 0], forks=[(0, 1)])
    pages.compact({1: [1, 2, 11]})
    assert cache.read(pages.everything()) == list(range(12)) + [1, 2, 11]


def test_prefix_groups():
    cache, pages = _grown([10, 0, 0, 9, 0, 0], forks=[(0, 1), (0, 2), (3, 4)])
    with pytest.raises(RuntimeError, match="changed"):
        pages.prefix()
    pages.extend([1, 2, 0, 1, 3, 5])
    p = pages.prefix()
    # 0 and 1, 3 and 4, and 5 alone with nothing
    assert p.kv_len.tolist() == [8, 8, 0] and p.cu_q.tolist() == [0, 3, 7, 12]
    assert p.pages[0].tolist() == pages.pages_of(0)[:2] and p.pages[1].tolist() == pages.pages_of(3)[:2]
    assert p.n_tokens == 12 and p.max_q == 5 and p.max_kv == 8
    assert pages.prefix(least=3) is None
    pages.truncate(0, 1)
    with pytest.raises(RuntimeError, match="changed"):
        pages.prefix()
    # new tokens that begin inside the common pages end the prefix before them
    cache, pages = _grown([12, 0], forks=[(0, 1)])
    pages.truncate(1, 7)
    pages.extend([1, 1])
    assert pages.prefix().kv_len.tolist() == [4]


def test_bounds():
    _, pages = _grown([10, 3])
    b = pages.extend([1, 2])
    assert (b.max_q, b.max_kv) == (2, 11)
    b = pages.extend([1, 0], max_q=1, max_kv=100)
    assert (b.max_q, b.max_kv) == (1, 100)
    for kw in (dict(max_q=0), dict(max_kv=11), dict(max_kv=101), dict(max_q=(1 << 30) + 1)):
        with pytest.raises(ValueError, match="max_"):
            pages.extend([1, 0], **kw)
    assert pages.length(0) == 12


def test_nothing_shared():
    _, pages = _grown([10, 10])
    assert pages.prefix() is None
    pages.extend([0, 0])
    assert pages.prefix() is None


@pytest.mark.parametrize("call", [
    lambda p: p.extend([1]), lambda p: p.extend([1, -1, 0]), lambda p: p.extend([0.5, 1, 0]),
    lambda p: p.extend([101, 0, 0]), lambda p: p.extend([95, 0, 0]), lambda p: p.extend([1 << 40, 0, 0]),
    lambda p: p.fork(0, 0), lambda p: p.fork(0, 1), lambda p: p.fork(0, 3), lambda p: p.fork(-1, 2),
    lambda p: p.truncate(0, 11), lambda p: p.truncate(0, -1), lambda p: p.free(7),
    lambda p: p.compact({0: [1, 1]}), lambda p: p.compact({0: [2, 1]}), lambda p: p.compact({0: [10]}),
    lambda p: p.compact({0: [-1]}), lambda p: p.compact({0: [[1]]}), lambda p: p.compact({0: [0.5]}),
    lambda p: p.compact({5: []}),
])
def test_refusals(call):
    cache, pages = _grown([10, 3, 0])
    before = cache.read(pages.everything())
    with pytest.raises(ValueError):
        call(pages)
    assert cache.read(pages.everything()) == before and pages.free_pages == 60 - 4


@pytest.mark.parametrize("n_seq,most", [(0, 5), (1, 0), (1, (1 << 30) + 1)])
def test_sizes_are_refused(n_seq, most):
    with pytest.raises(ValueError):
        jg.KVPages(Cache(4), n_seq, most)


def test_a_full_cache_changes_nothing():
    cache, pages = _grown([10, 0], num_pages=4, forks=[(0, 1)])
    with pytest.raises(RuntimeError, match="full: 2 pages"):
        pages.extend([3, 1])
    with pytest.raises(RuntimeError, match="full"):
        pages.compact({0: [0, 2, 3, 4, 5, 6]})
    assert cache.read(pages.everything()) == list(range(10)) * 2
    pages.free(1)
    pages.extend([3, 0])
    assert pages.free_pages == 0


def test_the_copies_refuse():
    """What the host can see, before anything is launched (addresses that are never used)."""
    L, F = jg.lib(), 1 << 20
    p, o = (ctypes.byref(jg._KvParams(8, 2, d, 64, 10)) for d in (128, 64))
    b = ctypes.byref(jg._KvBatch(1, 4, F, F, F, 9, 4, 200))

    def err(rc, msg):
        assert rc == jg.JHQ_EINVAL and msg in L.jhq_last_error().decode()
    err(L.jhq_k_kv_copy_pages(p, None, F, F, 1, None), "null cache")
    err(L.jhq_k_kv_copy_pages(p, F + 8, F, F, 1, None), "aligned")
    err(L.jhq_k_kv_copy_pages(p, F, F, F, -1, None), "negative")
    err(L.jhq_k_kv_copy_pages(p, F, None, F, 1, None), "null pages")
    err(L.jhq_k_kv_copy_pages(p, F, F, F, 1 << 40, None), "more work")
    err(L.jhq_k_kv_copy(p, F, F, p, None, b, None), "null cache")
    err(L.jhq_k_kv_copy(p, None, F, p, F, b, None), "null source")
    err(L.jhq_k_kv_copy(p, F + 4, F, p, F, b, None), "aligned")
    err(L.jhq_k_kv_copy(o, F, F, p, F, b, None), "other bits")
    err(L.jhq_k_kv_copy(p, F, None, p, F, b, None), "null slots")
    err(L.jhq_k_kv_copy(None, F, F, p, F, b, None), "null parameters")


class Failing(Cache):
    """A cache whose calls named in `fail` raise, as they do where there is no memory."""
    fail = ()

    def batch(self, *a):
        if "batch" in self.fail:
            raise MemoryError("batch")
        return super().batch(*a)

    def copy_pages(self, src, dst):
        if "copy_pages" in self.fail:
            raise MemoryError("copy_pages")
        super().copy_pages(src, dst)

    def copy(self, slots, b):
        if "copy" in self.fail:
            raise MemoryError("copy")
        super().copy(slots, b)


def _failing(lens, num_pages=60, forks=()):
    cache = Failing(num_pages)
    pages = jg.KVPages(cache, len(lens), 100)
    b = pages.extend(lens)
    cache.write(list(range(sum(lens))), b)
    for a, d in forks:
        pages.fork(a, d)
    return cache, pages


def _model(lens, forks=()):
    at = np.concatenate([[0], np.cumsum(lens)])
    model = [list(range(a, b)) for a, b in zip(at[:-1], at[1:])]
    for a, d in forks:
        model[d] = list(model[a])
    return model


@pytest.mark.parametrize("fail", ["copy_pages", "batch", "upload"])
def test_an_extend_that_fails_changes_nothing(fail, monkeypatch):
    lens, forks = [10, 0, 0, 7], [(0, 1), (0, 2)]
    cache, pages = _failing(lens, forks=forks)
    model = _model(lens, forks)
    before = (pages._table.copy(), pages._refs.copy(), pages._len.copy(), sorted(pages._free))
    with monkeypatch.context() as m:
        if fail == "upload":
            m.setattr(pages, "_upload", lambda *a: (_ for _ in ()).throw(MemoryError("upload")))
        cache.fail = (fail,)
        with pytest.raises(MemoryError):
            pages.extend([1, 9, 1, 30])
    cache.fail = ()
    held = [pages.pages_of(s) for s in range(4)]
    assert held == [before[0][s, :-(-len(m) // 4)].tolist() for s, m in enumerate(model)]
    for x, y in zip(before[1:], (pages._refs, pages._len, sorted(pages._free))):
        assert np.array_equal(x, y)
    _check(pages, cache, model)
    b = pages.extend([1, 9, 1, 30])
    cache.write(list(range(100, 141)), b)
    for m, x in zip(model, np.split(np.arange(100, 141), [1, 10, 11])):
        m += x.tolist()
    _check(pages, cache, model)


@pytest.mark.parametrize("fail", ["copy", "batch", "upload"])
def test_a_compaction_that_fails_changes_nothing(fail, monkeypatch):
    lens, forks = [30, 0, 9, 6], [(0, 1)]
    cache, pages = _failing(lens, forks=forks)
    model = _model(lens, forks)
    keep = {0: list(range(1, 30, 2)), 2: [0, 1, 5, 8], 3: [0, 1]}
    before = (pages._table.copy(), pages._refs.copy(), pages._len.copy(), list(pages._free))
    with monkeypatch.context() as m:
        if fail == "upload":
            m.setattr(pages, "_to_device", lambda *a: (_ for _ in ()).throw(MemoryError("upload")))
        cache.fail = (fail,)
        with pytest.raises(MemoryError):
            pages.compact(keep)
    cache.fail = ()
    for x, y in zip(before, (pages._table, pages._refs, pages._len, pages._free)):
        assert np.array_equal(x, y)
    _check(pages, cache, model)
    pages.compact(keep)
    for s, at in keep.items():
        model[s] = [model[s][i] for i in at]
    _check(pages, cache, model)


def _compacted(lens, keep, num_pages, forks=()):
    cache, pages = _grown(lens, num_pages, forks)
    model = _model(lens, forks)
    pages.compact(keep)
    for s, at in keep.items():
        model[s] = [model[s][i] for i in at]
    _check(pages, cache, model)
    return pages


def test_compaction_in_a_full_cache():
    """Pages that keep nothing take what follows; without one, one free page is enough, over and over."""
    whole = list(range(32, 64))
    assert _compacted([64], {0: whole}, 16).free_pages == 8
    assert _compacted([40, 40], {0: range(20, 40), 1: range(1, 40)}, 20).free_pages == 5
    # every page keeps something, one page is free
    assert _compacted([60], {0: np.arange(1, 60)}, 16).free_pages == 1
    assert _compacted([60], {0: np.arange(0, 60, 2)}, 16).free_pages == 8
    assert _compacted([28, 28], {0: np.arange(1, 28, 3), 1: np.arange(28)[np.arange(28) % 4 > 0]}, 15).free_pages == 6
    # what one sequence gives back serves the next, and what is only cut off serves both
    assert _compacted([30, 30, 0], {0: np.arange(20, 30), 1: np.arange(4, 30, 2)}, 17, forks=[(0, 2)]).free_pages == 2
    assert _compacted([30, 30], {0: np.arange(1, 30), 1: np.arange(3)}, 16).free_pages == 7


def test_a_compaction_that_finds_no_page_changes_nothing():
    for num_pages, lens, keep, forks in ((15, [60], {0: np.arange(1, 60)}, []),
                                         (8, [30, 0], {0: np.arange(1, 30)}, [(0, 1)]),
                                         (12, [30, 0], {0: np.arange(1, 30)}, [(0, 1)]),
                                         # 8 for what another holds too, 1 + 4 are to be had
                                         (17, [30, 30, 0], {0: np.arange(1, 30), 1: np.arange(4, 30, 2)}, [(0, 2)])):
        cache, pages = _grown(lens, num_pages, forks)
        before = (pages._table.copy(), pages._refs.copy(), pages._len.copy(), list(pages._free))
        with pytest.raises(RuntimeError, match="full"):
            pages.compact(keep)
        for x, y in zip(before, (pages._table, pages._refs, pages._len, pages._free)):
            assert np.array_equal(x, y)
        _check(pages, cache, _model(lens, forks))


@pytest.mark.parametrize("seed", range(40))
def test_compaction_with_few_free_pages(seed):
    """Against lists: whatever is shared, with as many pages as are held and a few more."""
    rng = np.random.default_rng(seed)
    lens = [int(x) for x in rng.integers(0, 60, 5)]
    lens[4] = 0
    forks = [(int(rng.integers(0, 4)), 4)] if rng.random() < 0.6 else []
    held = sum(-(-n // 4) for n in lens)
    cache, pages = _grown(lens, max(1, held) + int(rng.integers(0, 3)), forks)
    model = _model(lens, forks)
    for _ in range(3):
        keep = {s: np.nonzero(rng.random(len(m)) < rng.choice([0.1, 0.5, 0.9, 1.0]))[0]
                for s, m in enumerate(model) if rng.random() < 0.7}
        try:
            pages.compact(keep)
        except RuntimeError:
            # only pages that others hold, or no free one at all, stand in the way
            assert forks or pages.free_pages == 0
        else:
            for s, at in keep.items():
                model[s] = [model[s][i] for i in at]
        _check(pages, cache, model)


def test_batches_say_where_places_are_not_positions():
    cache, pages = _grown([20, 10, 6, 0])
    assert not pages.extend([1, 1, 1, 0]).moved and not pages.everything().moved
    pages.compact({0: np.arange(15), 2: np.arange(7)})  # beginnings: nothing moves
    assert not pages.extend([1, 1, 1, 0]).moved
    pages.compact({0: np.r_[0:9, 11:16]})  # token 11 becomes 9
    assert pages.everything().moved
    assert not pages.extend([0, 1, 1, 0]).moved  # of sequences without new tokens nothing is turned
    assert pages.extend([1, 0, 0, 0]).moved
    pages.fork(0, 3)
    assert pages.extend([0, 0, 0, 1]).moved
    pages.truncate(0, 10)
    assert pages.extend([1, 0, 0, 0]).moved
    pages.truncate(0, 9)  # the last token that was moved goes
    assert not pages.extend([1, 0, 0, 0]).moved
    pages.compact({3: np.arange(5, 16)})
    pages.compact({3: np.arange(0)})
    assert not pages.extend([1, 1, 1, 1]).moved
    # moved once, and compacted again: in front of it, behind it, cut off before it
    for keep, moved in ((np.r_[0:20, 22:26], True), (np.r_[0:2, 3:26], True), (np.arange(26), True),
                        (np.arange(11), True), (np.arange(10), False)):
        cache, pages = _grown([30])
        pages.compact({0: np.r_[0:10, 14:30]})
        pages.compact({0: keep})
        assert pages.extend([1]).moved == moved
    pages.free(0)
    assert not pages.extend([3]).moved
