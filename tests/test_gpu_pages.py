"""Pages and tokens copied on the device: byte for byte what the cache held, and nothing else; KVPages
with the cache, its copies and attention."""
import numpy as np
import pytest

import kv_ref as ref

import jhq_gpu_amd as jg

pytestmark = pytest.mark.gpu

SHAPES = [(8, 128, 2, 64), (8, 64, 3, 16), (8, 256, 1, 32), (4, 128, 2, 16), (4, 64, 5, 128),
          (4, 256, 2, 1024)]


def _i32(gpu, a):
    import torch
    return torch.tensor(np.asarray(a, np.int32), device=gpu)


def _filled(gpu, bits, D, H, page, num_pages, seed=0):
    """A cache whose every slot holds a row of its own, some of them NaN and some zero."""
    import torch
    c = jg.KVCache(num_pages, page, H, D, bits=bits, device=gpu)
    n = num_pages * page
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(2, n, H, D, generator=g).bfloat16().unbind(0)
    k[3], v[5, :, 7], v[6], k[7, 0, 0] = 0, float("inf"), 0, float("nan")
    table = torch.arange(num_pages, dtype=torch.int32, device=gpu)[None]
    c.write(k.to(gpu), v.to(gpu), c.batch(table, _i32(gpu, [n]), _i32(gpu, [0, n]), n, n, n))
    return c


def _all(c):
    """Every slot's rows."""
    import torch
    n = c.num_pages * c.page_size
    table = torch.arange(c.num_pages, dtype=torch.int32, device=c.device)[None]
    return c.read(c.batch(table, _i32(c.device, [n]), _i32(c.device, [0, n]), n, n, n))


def _same(a, b):
    import torch
    return torch.equal(torch.nan_to_num(a, nan=1e30), torch.nan_to_num(b, nan=1e30))


@pytest.mark.parametrize("bits,D,H,page", SHAPES)
@pytest.mark.parametrize("n", [1, 2, 7])
def test_whole_pages(gpu, bits, D, H, page, n):
    import torch
    c = _filled(gpu, bits, D, H, page, 3 * n + 4)
    pb = c.data.numel() // c.num_pages
    order = np.random.default_rng(n).permutation(c.num_pages)
    src, dst = order[:n], order[n:2 * n]
    src[-1] = src[0]  # one page may be copied to several
    want = c.data.clone().view(-1, pb)
    want[torch.from_numpy(dst).to(gpu)] = want[torch.from_numpy(src).to(gpu)]
    c.copy_pages(_i32(gpu, src), _i32(gpu, dst))
    assert torch.equal(c.data.view(-1, pb), want)
    # pairs that name no page, or one page twice
    c.copy_pages(_i32(gpu, [-1, 0, c.num_pages, 0, 2 ** 31 - 1, 1]),
                 _i32(gpu, [0, -1, 0, c.num_pages, 1, 1]))
    c.copy_pages(_i32(gpu, []), _i32(gpu, []))
    assert torch.equal(c.data.view(-1, pb), want)


@pytest.mark.parametrize("how", ["random", "runs", "reverse", "one", "ascending"])
@pytest.mark.parametrize("bits,D,H,page", SHAPES)
def test_tokens(gpu, bits, D, H, page, how):
    """Sequences of every kind of end inside a group and a page, in two steps that split
    groups: rows equal the source's, slots of nobody keep every byte."""
    import torch
    lens = [1, 16, 0, 17, 33, 5, 64, 131, 2]
    per = [-(-n // page) for n in lens]
    src = _filled(gpu, bits, D, H, page, -(-400 // page), seed=1)
    n_src = src.num_pages * page
    dst = _filled(gpu, bits, D, H, page, sum(per) + 2, seed=2)
    rng = np.random.default_rng(D + page)
    order = rng.permutation(dst.num_pages)
    table, at = np.full((len(lens), max(per)), -1, np.int32), 0
    for b, p in enumerate(per):
        table[b, :p] = order[at:at + p]
        at += p
    T = sum(lens)
    slots = {"random": rng.integers(0, n_src, T), "runs": (np.arange(T) * 7 // 20 * 20 + np.arange(T)) % n_src,
             "reverse": n_src - 1 - np.arange(T), "one": np.full(T, 5),
             "ascending": np.sort(rng.choice(n_src, T, replace=False))}[how].astype(np.int64)
    before = dst.data.clone()
    old_k, old_v = _all(dst)
    first = [n * 2 // 3 for n in lens]
    cu = np.concatenate([[0], np.cumsum(lens)])
    for new, upto in ((first, first), ([n - f for n, f in zip(lens, first)], lens)):
        rows = np.concatenate([np.arange(a + n - q, a + n) for a, n, q in zip(cu, upto, new)])
        b = dst.batch(_i32(gpu, table), _i32(gpu, upto), _i32(gpu, np.concatenate([[0], np.cumsum(new)])),
                      sum(new), max(new), max(upto))
        dst.copy(torch.from_numpy(slots[rows]).to(gpu), b, source=src)
    sk, sv = _all(src)
    dk, dv = _all(dst)
    place = np.concatenate([table[b, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
                            for b, n in enumerate(lens)])
    pick, put = torch.from_numpy(slots).to(gpu), torch.from_numpy(place).to(gpu)
    assert _same(dk[put], sk[pick]) and _same(dv[put], sv[pick])
    rest = torch.ones(dk.shape[0], dtype=torch.bool, device=gpu)
    rest[put] = False
    assert _same(dk[rest], old_k[rest]) and _same(dv[rest], old_v[rest])
    pb = dst.data.numel() // dst.num_pages
    for p in order[at:]:
        assert torch.equal(dst.data.view(-1, pb)[p], before.view(-1, pb)[p])


@pytest.mark.parametrize("bits,D", [(8, 128), (4, 64)])
def test_slots_that_are_none(gpu, bits, D):
    """A slot outside the source becomes NaN; pages that the destination does not have, and
    sequences past their bounds, are not written."""
    import torch
    c = _filled(gpu, bits, D, 2, 16, 8, seed=3)
    k0, v0 = _all(c)
    slots = torch.tensor([0, -1, 8 * 16, 1, 2 ** 40, -2 ** 40, 2, 9], device=gpu)
    table = _i32(gpu, [[5, 99], [6, 0], [7, 0]])
    b = c.batch(table, _i32(gpu, [20, 2, 40]), _i32(gpu, [0, 6, 8, 8]), 8, 6, 20)
    c.copy(slots, b)  # tokens 14 .. 19 of the first: 14, 15 in page 5, the others in no page
    k, v = _all(c)
    want_k, want_v = k0.clone(), v0.clone()
    want_k[5 * 16 + 14], want_v[5 * 16 + 14] = k0[0], v0[0]
    want_k[5 * 16 + 15], want_v[5 * 16 + 15] = float("nan"), float("nan")
    want_k[96:98], want_v[96:98] = k0[[2, 9]], v0[[2, 9]]
    assert _same(k, want_k) and _same(v, want_v)
    data = c.data.clone()
    c.copy(slots, c.batch(table, _i32(gpu, [20, 2, 40]), _i32(gpu, [0, 6, 8, 8]), 8, 1, 1))
    assert torch.equal(c.data, data)


def test_between_caches_of_other_pages(gpu):
    import torch
    a = _filled(gpu, 8, 64, 2, 128, 2, seed=4)
    b = _filled(gpu, 8, 64, 2, 16, 9, seed=5)
    slots = torch.arange(100, 230, device=gpu)
    table = _i32(gpu, [[3, 1, 4, 0, 5, 8, 2, 6, 7]])
    to = b.batch(table, _i32(gpu, [130]), _i32(gpu, [0, 130]), 130, 130, 130)
    b.copy(slots, to, source=a)
    k, v = b.read(to)
    ak, av = _all(a)
    assert _same(k, ak[100:230]) and _same(v, av[100:230])
    for other in (jg.KVCache(2, 16, 2, 64, bits=4, device=gpu), jg.KVCache(2, 16, 1, 64, device=gpu),
                  jg.KVCache(2, 16, 2, 128, device=gpu)):
        with pytest.raises(ValueError, match="source"):
            b.copy(slots, to, source=other)


def test_ragged_copies(gpu):
    """The launch that numbers runs of sequences of very different lengths."""
    import torch
    src = _filled(gpu, 8, 128, 1, 16, 40, seed=6)
    new = [1] * 40 + [500]
    per = [1] * 40 + [32]
    table = np.zeros((41, 32), np.int32)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = np.arange(at, at + p)
        at += p
    dst = jg.KVCache(at, 16, 1, 128, device=gpu)
    to = dst.batch(_i32(gpu, table), _i32(gpu, new), _i32(gpu, np.concatenate([[0], np.cumsum(new)])), 540,
                   500, 500)
    slots = torch.randint(0, 640, (540,), device=gpu)
    dst.copy(slots, to, source=src)
    k, v = dst.read(to)
    sk, sv = _all(src)
    assert _same(k, sk[slots]) and _same(v, sv[slots])


def test_far_pages(gpu):
    """Offsets past 32 bits: 9 GB of pages."""
    import torch
    c = jg.KVCache(130000, 16, 16, 256, bits=8, device=gpu)
    assert c.data.numel() > 1 << 33
    pb = c.data.numel() // c.num_pages
    view = c.data.view(-1, pb)
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(2, 16, 16, 256, generator=g).bfloat16().to(gpu).unbind(0)

    def one(page):
        return c.batch(_i32(gpu, [[page]]), _i32(gpu, [16]), _i32(gpu, [0, 16]), 16, 16, 16)
    c.write(k, v, one(129998))
    c.copy_pages(_i32(gpu, [129998]), _i32(gpu, [129999]))
    assert torch.equal(view[129998], view[129999])
    slots = 129999 * 16 + torch.arange(15, -1, -1, device=gpu)
    c.copy(slots, one(129997))
    a, b = c.read(one(129999)), c.read(one(129997))
    assert torch.equal(a[0], b[0].flip(0)) and torch.equal(a[1], b[1].flip(0))
    assert torch.isfinite(a[0]).all() and a[0].abs().max() > 0


def test_streams_and_graphs(gpu):
    import torch
    c = _filled(gpu, 8, 64, 2, 16, 12, seed=7)
    src, dst = _i32(gpu, [0, 1]), _i32(gpu, [8, 9])
    slots = torch.arange(16, 36, device=gpu)
    b = c.batch(_i32(gpu, [[10, 11]]), _i32(gpu, [20]), _i32(gpu, [0, 20]), 20, 20, 20)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c.copy_pages(src, dst, stream=s)
    c.copy(slots, b, stream=s)
    torch.cuda.synchronize()
    k0, v0 = _all(c)
    assert _same(k0[128:160], k0[:32]) and _same(v0[160:180], v0[16:36])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.copy_pages(src, dst)
        c.copy(slots, b)
    for i in range(3):
        src.add_(1)
        slots.add_(8)
        graph.replay()
        k, v = _all(c)
        assert _same(k[128:144], k[16 * (1 + i):16 * (2 + i)])
        assert _same(v[160:180], v[24 + 8 * i:44 + 8 * i])


def test_refusals(gpu):
    import torch
    c = _filled(gpu, 8, 64, 2, 16, 4)
    b = c.batch(_i32(gpu, [[3]]), _i32(gpu, [4]), _i32(gpu, [0, 4]), 4, 4, 4)
    good = torch.zeros(4, dtype=torch.int64, device=gpu)
    p = _i32(gpu, [0, 1])
    for bad in (lambda: c.copy(good.int(), b), lambda: c.copy(good[:3], b), lambda: c.copy(good.cpu(), b),
                lambda: c.copy(good[None], b),
                lambda: c.copy(torch.zeros(8, dtype=torch.int64, device=gpu)[::2], b),
                lambda: c.copy_pages(p, p[:1]), lambda: c.copy_pages(p.long(), p),
                lambda: c.copy_pages(p.cpu(), p), lambda: c.copy_pages(p[None], p[None]),
                lambda: c.copy_pages(_i32(gpu, [0, 1, 2, 3])[::2], p)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("bits", [8, 4])
def test_sequences_that_fork_grow_and_shrink(gpu, bits):
    """A serving program's life against lists of rows: what each sequence reads back, and attention
    over it."""
    import torch
    H, D, page, n_seq = 2, 64, 16, 5
    rng = np.random.default_rng(bits)
    cache = jg.KVCache(90, page, H, D, bits=bits, device=gpu)
    cache.data.fill_(0xff)
    pages = jg.KVPages(cache, n_seq, 300)
    held = [(np.zeros((0, H, D)), np.zeros((0, H, D))) for _ in range(n_seq)]

    def grow(new):
        b = pages.extend(new)
        k, v = (torch.randn(sum(new), H, D, generator=torch.Generator().manual_seed(int(rng.integers(1 << 30))))
                .bfloat16() for _ in range(2))
        cache.write(k.to(gpu), v.to(gpu), b)
        at = 0
        for s, a in enumerate(new):
            held[s] = tuple(np.concatenate([h, ref.value32(x[at:at + a].float().numpy(), bits)])
                            for h, x in zip(held[s], (k, v)))
            at += a
        return b

    def check(b=None, new=None):
        k, v = cache.read(pages.everything())
        assert np.array_equal(k.cpu().numpy(), np.concatenate([h[0] for h in held]))
        assert np.array_equal(v.cpu().numpy(), np.concatenate([h[1] for h in held]))
        if b is None:
            return
        q = torch.randn(sum(new), 4, D, generator=torch.Generator().manual_seed(1)).half()
        out = cache.attend(q.to(gpu), b).float().cpu().numpy()
        at = 0
        for s, a in enumerate(new):
            o, _, tol, _ = ref.attend(q[at:at + a].double().numpy(), held[s][0].astype(np.float64),
                                      held[s][1].astype(np.float64), D ** -0.5, unit=ref.UNIT["f16"])
            assert (np.abs(out[at:at + a] - o) <= tol).all()
            at += a

    new = [100, 0, 37, 0, 1]
    check(grow(new), new)
    pages.fork(0, 1)
    pages.fork(2, 3)
    held[1], held[3] = held[0], held[2]
    for _ in range(3):
        new = [1, 1, 1, 1, 0]
        check(grow(new), new)
    keep = np.nonzero(rng.random(103) < 0.6)[0]
    pages.compact({1: keep, 0: np.arange(50), 3: np.r_[0:20, 30:40]})
    held[1] = tuple(h[keep] for h in held[1])
    held[0] = tuple(h[:50] for h in held[0])
    held[3] = tuple(h[np.r_[0:20, 30:40]] for h in held[3])
    check()
    pages.free(2)
    held[2] = tuple(h[:0] for h in held[2])
    new = [3, 20, 5, 1, 40]
    check(grow(new), new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pages.compact({4: np.arange(1, 41)}, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    held[4] = tuple(h[1:41] for h in held[4])
    check()
    for s in range(n_seq):
        pages.free(s)
    assert pages.free_pages == 90


def test_a_captured_step_is_replayed_as_sequences_grow(gpu):
    """Positions, write and attention in one graph: extend moves what it reads."""
    import torch
    H, D, G, n_seq = 2, 64, 2, 3
    cache = jg.KVCache(40, 16, H, D, device=gpu)
    pages = jg.KVPages(cache, n_seq, 200)
    rope = jg.Rotary(D, device=gpu)
    g = torch.Generator().manual_seed(5)

    def rows(n, h):
        return torch.randn(n, h, D, generator=g).bfloat16().to(gpu)
    prompt = pages.extend([30, 0, 9])
    cache.write(rows(39, H), rows(39, H), prompt, rotary=rope)
    pages.fork(0, 1)
    b = pages.extend([1, 1, 1], max_kv=200)
    q, k, v = rows(3, H * G), rows(3, H), rows(3, H)
    turned, out = torch.zeros_like(q), torch.zeros_like(q)
    work = torch.zeros(cache.work_bytes(b, H * G), dtype=torch.uint8, device=gpu)

    def step():
        rope.apply(q, b, out=turned)
        cache.write(k, v, b, rotary=rope)
        cache.attend(turned, b, out=out, work=work)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):  # over the end of a page, and of the page that two hold
        now = pages.extend([1, 1, 1], max_kv=200)
        for x, h in ((q, H * G), (k, H), (v, H)):
            x.copy_(rows(3, h))
        graph.replay()
        got, seen = out.clone(), turned.clone()
        assert torch.equal(rope.apply(q, now), seen)
        assert torch.equal(cache.attend(seen, now), got)
    assert pages.length(1) == 51 and torch.isfinite(out).all()


def test_a_captured_step_writes_where_extend_says(gpu):
    """A captured step's replays against lists of rows: every token of every sequence as it reads back, keys
    at the positions that they had when their replay ran, and attention over them.  Slots that nothing was
    written into read as NaN."""
    import torch
    H, D, G, n_seq = 2, 64, 2, 3
    cache = jg.KVCache(40, 16, H, D, device=gpu)
    cache.data.fill_(0xff)
    pages = jg.KVPages(cache, n_seq, 200)
    rope = jg.Rotary(D, device=gpu)
    gen = torch.Generator().manual_seed(6)
    held = [[np.zeros((0, H, D))] * 2 for _ in range(n_seq)]

    def rows(n, h):
        return torch.randn(n, h, D, generator=gen).bfloat16().to(gpu)

    plain = jg.KVCache(3, 16, H, D, device=gpu)

    def hold(new, k, v):
        """The rows as a cache holds them that they enter as one sequence, keys turned before, to positions
        that are counted here."""
        T = sum(new)
        pos = np.concatenate([len(h[0]) + np.arange(a) for h, a in zip(held, new)])
        b = plain.batch(_i32(gpu, [[2, 0, 1]]), _i32(gpu, [T]), _i32(gpu, [0, T]), T, T, T)
        plain.write(rope.apply(k.float(), torch.from_numpy(pos).to(gpu)), v.float(), b)
        at, kv = 0, [x.cpu().numpy() for x in plain.read(b)]
        for h, a in zip(held, new):
            h[:] = [np.concatenate([x, y[at:at + a]]) for x, y in zip(h, kv)]
            at += a
    k, v = rows(39, H), rows(39, H)
    cache.write(k, v, pages.extend([30, 0, 9]), rotary=rope)
    hold([30, 0, 9], k, v)
    pages.fork(0, 1)
    held[1] = list(held[0])
    b = pages.extend([1, 1, 1], max_kv=200)
    q, k, v = rows(3, H * G), rows(3, H), rows(3, H)
    turned, out = torch.zeros_like(q), torch.zeros_like(q)
    work = torch.zeros(cache.work_bytes(b, H * G), dtype=torch.uint8, device=gpu)

    def step():
        rope.apply(q, b, out=turned)
        cache.write(k, v, b, rotary=rope)
        cache.attend(turned, b, out=out, work=work)
    step()
    hold([1] * n_seq, k, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):  # over the end of a page, and of the page that two hold
        pages.extend([1, 1, 1], max_kv=200)
        for x, h in ((q, H * G), (k, H), (v, H)):
            x.copy_(rows(3, h))
        graph.replay()
        hold([1] * n_seq, k, v)
        got = out.clone()
        at = torch.tensor([len(h[0]) - 1 for h in held], device=gpu)
        assert torch.equal(rope.apply(q, at), turned)
        for x, y in zip(cache.read(pages.everything()), zip(*held)):
            assert np.array_equal(x.cpu().numpy(), np.concatenate(y))
        for s in range(n_seq):
            o, _, tol, _ = ref.attend(turned[s:s + 1].double().cpu().numpy(), *held[s], D ** -0.5,
                                      unit=ref.UNIT["bf16"])
            assert (np.abs(got[s:s + 1].double().cpu().numpy() - o) <= tol).all()


@pytest.mark.parametrize("bits,D,H", [(8, 128, 2), (4, 64, 3)])
def test_compaction_in_a_full_cache(gpu, bits, D, H):
    """In as many copies as the pages that become empty ask for: rows read back as they were."""
    import torch
    lens = [600, 333, 50]
    rng = np.random.default_rng(D)
    for keep, spare in (([np.arange(300, 600), np.arange(0, 333, 2), np.arange(50)], 0),
                        ([np.arange(1, 600), np.sort(rng.choice(333, 300, replace=False)), np.arange(20)], 1),
                        ([np.sort(rng.choice(600, 200, replace=False)), np.arange(3, 333), np.arange(1, 50)], 3)):
        cache = jg.KVCache(sum(-(-n // 16) for n in lens) + spare, 16, H, D, bits=bits, device=gpu)
        cache.data.fill_(0xff)
        pages = jg.KVPages(cache, 3, 700)
        k, v = torch.randn(2, sum(lens), H, D, generator=torch.Generator().manual_seed(D)).bfloat16().unbind(0)
        cache.write(k.to(gpu), v.to(gpu), pages.extend(lens))
        before = cache.read(pages.everything())
        pages.compact(dict(enumerate(keep)))
        rows = torch.from_numpy(np.concatenate([a + n for a, n in zip(keep, (0, 600, 933))])).to(gpu)
        for x, y in zip(before, cache.read(pages.everything())):
            assert torch.equal(x[rows], y)


def test_moved_tokens_are_not_turned_to_their_places(gpu):
    """What a compacted sequence holds stands elsewhere than at its positions: write(rotary=) and apply refuse
    its batches, and nothing is written."""
    import torch
    cache = jg.KVCache(9, 16, 1, 64, device=gpu)
    pages, rope = jg.KVPages(cache, 2, 60), jg.Rotary(64, device=gpu)
    x = torch.randn(50, 1, 64, generator=torch.Generator().manual_seed(7)).bfloat16().to(gpu)
    cache.write(x, x, pages.extend([30, 20]), rotary=rope)
    pages.compact({0: np.arange(4, 30)})
    b = pages.extend([1, 1])
    before = cache.data.clone()
    with pytest.raises(ValueError, match="moved"):
        cache.write(x[:2], x[:2], b, rotary=rope)
    with pytest.raises(ValueError, match="moved"):
        rope.apply(x[:2], b)
    assert torch.equal(cache.data, before)
    turned = rope.apply(x[:2], torch.tensor([30, 20], device=gpu))
    cache.write(turned, x[:2], b)
    b = pages.extend([0, 1])  # the other sequence's places are its positions
    cache.write(x[:1], x[:1], b, rotary=rope)
    assert torch.equal(rope.apply(x[:1], b), rope.apply(x[:1], torch.tensor([21], device=gpu)))
