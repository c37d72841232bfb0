"""Attention of sequences that share a prefix, against attention over all of their tokens in
float64 (kv_ref): every kernel that sizes choose for the prefix and for what stands behind it."""
import numpy as np
import pytest

import kv_ref as ref

import jhq_gpu_amd as jg

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def _np(t):
    return t.float().cpu().numpy()


class Shared:
    """groups: [(prefix tokens, [(new, own tokens with the new ones), ..]), ..], in a cache whose pages are
    in random order; whole pages of a prefix are held once."""

    def __init__(self, gpu, groups, H, D, bits=8, page=16, dtype="bf16", seed=0):
        import torch
        self.gpu, self.groups, self.H, self.D, self.bits, self.page, self.dtype = (
            gpu, groups, H, D, bits, page, dtype)
        rng = np.random.default_rng(seed)
        whole = [p // page for p, _ in groups]
        need = sum(-(-p // page) + sum(-(-(p + n) // page) - w for _, n in s)
                   for (p, s), w in zip(groups, whole))
        order = list(rng.permutation(need + 2))
        self.cache = jg.KVCache(need + 2, page, H, D, bits=bits, device=gpu)
        self.cache.data.fill_(0xff)
        g = torch.Generator().manual_seed(seed)

        def rows(n):
            size = torch.exp(torch.randn(n, 1, 1, generator=g))
            return [(torch.randn(n, H, D, generator=g) * x).to(_dt(dtype)) for x in (size, size.flip(0))]

        def put(table, lo, kv):
            n = lo + len(kv[0])
            if n == lo:
                return
            b = self.cache.batch(self.i32([table]), self.i32([n]), self.i32([0, n - lo]), n - lo, n - lo, n)
            self.cache.write(kv[0].to(gpu), kv[1].to(gpu), b)
        self.tables, self.leads, self.new, self.lens, self.kv = [], [], [], [], []
        for (p, seqs), w in zip(groups, whole):
            lead = [order.pop() for _ in range(-(-p // page))]
            pk, pv = rows(p)
            put(lead, 0, (pk, pv))
            self.leads.append(lead)
            for a, n in seqs:
                table = lead[:w] + [order.pop() for _ in range(-(-(p + n) // page) - w)]
                ok, ov = rows(n)
                k, v = torch.cat([pk, ok]), torch.cat([pv, ov])
                put(table, w * page, (k[w * page:], v[w * page:]))
                self.tables.append(table)
                self.new.append(a)
                self.lens.append(p + n)
                self.kv.append([ref.value32(_np(x), bits).astype(np.float64) for x in (k, v)])

    def i32(self, a):
        import torch
        return torch.tensor(np.asarray(a, np.int32), device=self.gpu)

    def batch(self, n_tokens=None, first=0, max_q=None, max_kv=None):
        width = max(1, max(len(t) for t in self.tables))
        table = np.full((len(self.tables), width), -1, np.int32)
        for b, t in enumerate(self.tables):
            table[b, :len(t)] = t
        cu = np.concatenate([[0], np.cumsum(self.new)]) + first
        return self.cache.batch(self.i32(table), self.i32(self.lens), self.i32(cu),
                                int(cu[-1]) if n_tokens is None else n_tokens,
                                max(self.new) if max_q is None else max_q,
                                max(self.lens) if max_kv is None else max_kv)

    def prefix(self, n_tokens=None, first=0, max_q=None, max_kv=None, lens=None):
        width = max(1, max(len(t) for t in self.leads), -(-(max_kv or 0) // self.page))
        table = np.full((len(self.leads), width), -1, np.int32)
        for b, t in enumerate(self.leads):
            table[b, :len(t)] = t
        rows = [sum(a for a, _ in s) for _, s in self.groups]
        lens = [p for p, _ in self.groups] if lens is None else lens
        cu = np.concatenate([[0], np.cumsum(rows)]) + first
        return self.cache.batch(self.i32(table), self.i32(lens), self.i32(cu),
                                int(cu[-1]) if n_tokens is None else n_tokens,
                                max(rows) if max_q is None else max_q, max(lens) if max_kv is None else max_kv)

    def queries(self, Hq, seed=1, T=None):
        import torch
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(sum(self.new) if T is None else T, Hq, self.D, generator=g) * 1.5).to(_dt(self.dtype))

    def check(self, q, out, lse=None, causal=True, scale=None, skip=()):
        got = _np(out)
        at = 0
        for s, (a, n) in enumerate(zip(self.new, self.lens)):
            if s not in skip:
                o, l, tol, ltol = ref.attend(_np(q[at:at + a]).astype(np.float64), *self.kv[s],
                                             self.D ** -0.5 if scale is None else scale, causal, 0,
                                             ref.UNIT[self.dtype])
                err = np.abs(got[at:at + a] - o)
                assert (err <= tol).all(), (s, a, n, (err / np.maximum(tol, 1e-300)).max())
                if lse is not None:
                    x = lse[at:at + a].cpu().numpy()
                    e = np.isinf(l)
                    assert np.array_equal(x[e], l[e])
                    assert (np.abs(x[~e] - l[~e]) <= ltol[~e]).all(), (s, a, n)
            at += a

    def attend(self, Hq, causal=True, scale=None, **kw):
        import torch
        q = self.queries(Hq)
        b, p = self.batch(**kw), self.prefix()
        lse = torch.full(q.shape[:2], 7.0, device=self.gpu)
        out = self.cache.attend(q.to(self.gpu), b, causal=causal, scale=scale, lse=lse, prefix=p, once=True)
        assert out.dtype == q.dtype and out.shape == q.shape
        assert torch.equal(out, self.cache.attend(q.to(self.gpu), b, causal=causal, scale=scale, prefix=p,
                                                  once=True))
        self.check(q, out, lse, causal, scale)
        # as the bounds choose
        self.check(q, self.cache.attend(q.to(self.gpu), b, causal=causal, scale=scale, prefix=p), None, causal,
                   scale)
        return q, out


SHAPES = [(8, 128, 2, 64), (8, 64, 3, 16), (8, 256, 1, 32), (4, 128, 2, 16), (4, 64, 2, 128), (4, 256, 2, 16)]
# prefixes and sequences: few rows and many, short and long before and behind
GROUPS = {
    "few_short": [(77, [(1, 1), (1, 20), (1, 64)]), (64, [(1, 5), (1, 70)])],
    "few_long_before": [(1500, [(1, 3), (1, 130)])],
    "few_long_behind": [(100, [(1, 1500), (1, 20)])],
    "many_short": [(130, [(1, 1 + 3 * i) for i in range(40)])],
    "many_long": [(1900, [(1, 1 + 7 * i) for i in range(30)]), (333, [(1, 9)] * 12)],
    "chunks": [(200, [(5, 9), (8, 8), (1, 40)]), (31, [(7, 100), (3, 3)])],
    "wide_chunks": [(600, [(20, 25), (17, 200), (30, 30)]), (100, [(25, 26)])],
}


@pytest.mark.parametrize("G", [1, 4, 7])
@pytest.mark.parametrize("groups", GROUPS)
@pytest.mark.parametrize("bits,D,H,page", SHAPES)
def test_groups(gpu, bits, D, H, page, groups, G):
    w = Shared(gpu, GROUPS[groups], H, D, bits, page, "f16" if G == 4 else "bf16", seed=D + bits)
    w.attend(H * G)


@pytest.mark.parametrize("bound", [300, 5000])
@pytest.mark.parametrize("groups", ["few_short", "many_short", "chunks"])
def test_bounds_choose_the_kernels(gpu, groups, bound):
    """The same batch under wide bounds, which choose the kernels for long contexts."""
    w = Shared(gpu, GROUPS[groups], 2, 64, 8, 16, "bf16", seed=3)
    q = w.queries(8)
    b = w.batch()
    width = -(-bound // 16)
    import torch
    table = torch.full((len(w.tables), width), -1, dtype=torch.int32, device=gpu)
    table[:, :b.pages.shape[1]] = b.pages
    wide = w.cache.batch(table, b.kv_len, b.cu_q, b.n_tokens, b.max_q, bound)
    p = w.prefix()
    ptable = torch.full((len(w.leads), width), -1, dtype=torch.int32, device=gpu)
    ptable[:, :p.pages.shape[1]] = p.pages
    wp = w.cache.batch(ptable, p.kv_len, p.cu_q, p.n_tokens, p.max_q, bound)
    for x, y in ((wide, p), (b, wp), (wide, wp)):
        w.check(q, w.cache.attend(q.to(gpu), x, prefix=y, once=True))


@pytest.mark.parametrize("groups", ["few_short", "many_long", "chunks", "wide_chunks"])
@pytest.mark.parametrize("bits", [8, 4])
def test_everything_visible(gpu, groups, bits):
    w = Shared(gpu, GROUPS[groups], 2, 64, bits, 16, "f16", seed=5)
    w.attend(8, causal=False, scale=0.2)


@pytest.mark.parametrize("new", [8, 33, 70, 200])
@pytest.mark.parametrize("G", [1, 4])
def test_long_chunks(gpu, new, G):
    """From where a sequence's rows fill tiles of their own on, with other kernels."""
    w = Shared(gpu, [(700, [(new, new), (max(1, new // 3), new), (new, new + 100)])], 2, 128, 8, 64, "f16",
               seed=new)
    w.attend(2 * G)


@pytest.mark.parametrize("bits,D,G", [(8, 128, 4), (4, 64, 8), (8, 256, 2)])
def test_long_prefix(gpu, bits, D, G):
    """Cut into many parts, and a short one beside it."""
    w = Shared(gpu, [(20011, [(1, 40), (1, 300), (2, 3)]), (50, [(1, 2)])], 1, D, bits, 64, "f16", seed=bits)
    w.attend(G)


def test_many_groups(gpu):
    """More groups and sequences than a wave has lanes, groups without a prefix, of one sequence,
    sequences without new tokens and without tokens."""
    rng = np.random.default_rng(4)
    groups = []
    for i in range(90):
        p = int(rng.choice([0, 0, 5, 16, 64, 100]))
        groups.append((p, [(a, a + int(b) if a or b else 0) for a, b in
                           zip(rng.choice([0, 1, 1, 2], rng.integers(1, 4)), rng.choice([0, 1, 30], 3))]))
    groups[0] = (0, [(0, 0)])
    groups[3] = (40, [(0, 0), (0, 0)])
    groups[-1] = (33, [(1, 1), (0, 5)])
    w = Shared(gpu, groups, 2, 64, 8, 16, "f16", seed=6)
    w.attend(4)


def test_no_prefix_at_all(gpu):
    import torch
    w = Shared(gpu, [(0, [(1, 50), (1, 700)]), (0, [(3, 9)])], 2, 128, 8, 16, "bf16", seed=7)
    q, out = w.attend(8)
    b = w.batch()
    assert torch.equal(out, w.cache.attend(q.to(gpu), b))  # nothing is shared: the same kernels
    # no tokens in any: the prefixes' kernel has nothing to do
    wide = w.prefix(max_kv=16)
    w.check(q, w.cache.attend(q.to(gpu), b, prefix=wide, once=True))
    empty = w.cache.batch(w.i32(np.zeros((0, 1))), w.i32([]), w.i32([0]), b.n_tokens, 0, 0)
    assert torch.equal(out, w.cache.attend(q.to(gpu), b, prefix=empty, once=True))


def test_rows_of_no_group(gpu):
    """Sequences in front of and behind the groups, and rows of no sequence, which stay."""
    import torch
    w = Shared(gpu, [(0, [(1, 30), (2, 9)]), (90, [(1, 5), (1, 8)]), (0, [(1, 200)])], 2, 64, 8, 16, "f16", seed=8)
    T = sum(w.new)
    q = w.queries(4, T=T + 9)
    b = w.batch(n_tokens=T + 9, first=4)
    p = w.cache.batch(w.i32([w.leads[1]]), w.i32([90]), w.i32([4 + 3, 4 + 5]), T + 9, 2, 90)
    out = torch.full_like(q, 7.0).to(gpu)
    lse = torch.full((T + 9, 4), 7.0, device=gpu)
    assert w.cache.attend(q.to(gpu), b, prefix=p, out=out, lse=lse, once=True) is out
    assert (out[:4] == 7).all() and (out[T + 4:] == 7).all() and (lse[:4] == 7).all() and (lse[T + 4:] == 7).all()
    w.check(q[4:T + 4], out[4:T + 4], lse[4:T + 4])
    fresh = w.cache.attend(q.to(gpu), b, prefix=p, once=True)
    assert (fresh[:4] == 0).all() and torch.equal(fresh[4:T + 4], out[4:T + 4])


def test_rows_that_see_nothing(gpu):
    """More new tokens than tokens, in a sequence without a prefix: 0 and -inf."""
    import torch
    w = Shared(gpu, [(0, [(6, 2)]), (40, [(1, 3), (1, 1)])], 2, 64, 8, 16, "f16", seed=9)
    q = w.queries(4)
    lse = torch.zeros(8, 4, device=gpu)
    out = w.cache.attend(q.to(gpu), w.batch(), prefix=w.prefix(), lse=lse, once=True)
    assert (out[:4] == 0).all() and torch.isneginf(lse[:4]).all()
    assert torch.isfinite(lse[4:]).all() and (out[4:] != 0).any()
    w.check(q, out, lse)


def test_not_finite(gpu):
    """A NaN in the prefix reaches every row of its group and no other; one in a sequence its rows;
    rows whose every score is -inf come out as NaN."""
    import torch
    groups = [(50, [(1, 9), (1, 9)]), (70, [(1, 30), (2, 4)])]
    w = Shared(gpu, groups, 2, 64, 8, 16, "f16", seed=10)
    bad = torch.full((1, 2, 64), float("nan"), dtype=torch.float16, device=gpu)
    ok = torch.ones_like(bad)
    # token 20 of the first group's prefix, token 71 of the last sequence
    for table, n, kv in ((w.leads[0], 21, (ok, bad)), (w.tables[3], 72, (bad, ok))):
        w.cache.write(*kv, w.cache.batch(w.i32([table]), w.i32([n]), w.i32([0, 1]), 1, 1, n))
    q = w.queries(4)
    out = w.cache.attend(q.to(gpu), w.batch(), prefix=w.prefix(), once=True)
    assert torch.isnan(out[:2]).all() and torch.isnan(out[3:]).all()
    assert torch.isfinite(out[2]).all()
    w.check(q, out, skip=(0, 1, 3))
    q2 = q.clone()
    q2[2, 1, 3] = float("inf")
    out2 = w.cache.attend(q2.to(gpu), w.batch(), prefix=w.prefix(), once=True)
    assert torch.isnan(out2[2, 1]).all() and torch.equal(out2[2, [0, 2, 3]], out[2, [0, 2, 3]])


def test_contradictions(gpu):
    """A prefix that reaches into new tokens, groups that cut a sequence, bounds below what the arrays say:
    NaN in the rows concerned, the others as ever."""
    import torch
    groups = [(64, [(1, 9), (2, 9)]), (70, [(1, 30), (1, 4)])]
    w = Shared(gpu, groups, 2, 64, 8, 16, "f16", seed=11)
    q = w.queries(4)
    b = w.batch()

    def call(p, b=b):
        return w.cache.attend(q.to(gpu), b, prefix=p, once=True)
    good = call(w.prefix())
    w.check(q, good)
    far = w.prefix(lens=[73, 70], max_kv=80)  # the first sequences' new tokens begin at 72 and 71
    out = call(far)
    assert torch.isnan(out[:3]).all() and torch.equal(out[3:], good[3:])
    p = w.prefix()
    cut = w.cache.batch(p.pages, p.kv_len, w.i32([0, 2, 5]), 5, 3, 70)
    out = call(cut)
    assert torch.isnan(out[1:3]).all() and torch.isfinite(out[0]).all()
    w.check(q, out, skip=(1, 2, 3))
    out = call(w.prefix(max_kv=66))
    assert torch.isnan(out[3:]).all()
    w.check(q, out, skip=(2, 3))
    out = call(w.prefix(max_q=2))
    assert torch.isnan(out[:3]).all()
    w.check(q, out, skip=(0, 1))
    out = call(w.prefix(), w.batch(max_kv=80))
    assert torch.isnan(out[3]).all()
    w.check(q, out, skip=(2,))
    bad = p.pages.clone()
    bad[1, 2] = 1 << 20
    out = call(w.cache.batch(bad, p.kv_len, p.cu_q, 5, 3, 70))
    assert torch.isnan(out[3:]).all() and torch.equal(out[:3], good[:3])


@pytest.mark.parametrize("new", [1, 30])
def test_rows_out_of_order(gpu, new):
    """cu_q that does not ascend, in the batch and in the prefix: any sequence may be left out, and
    nothing else is written."""
    import torch
    w = Shared(gpu, [(100, [(new, new + 3)] * 6)], 2, 64, 8, 16, "f16", seed=14)
    T = 6 * new
    q = w.queries(4)
    b, p = w.batch(), w.prefix()
    buf = torch.full((T + 2, 4, 64), 7.0, dtype=q.dtype, device=gpu)
    data = w.cache.data.clone()
    for cu in ([0, T, 0, T, 0, T, T], [T, new, 0, 2 * new, T, 0, T], [0, -5, new, 1 << 30, 0, T, 2 * new]):
        for pcu in ([0, T], [T, 0], [-3, T], [0, 1 << 30]):
            x = w.cache.batch(b.pages, b.kv_len, w.i32(cu), T, T, b.max_kv)
            y = w.cache.batch(p.pages, p.kv_len, w.i32(pcu), T, T, p.max_kv)
            w.cache.attend(q.to(gpu), x, prefix=y, out=buf[1:-1], once=True)
            assert (buf[0] == 7).all() and (buf[-1] == 7).all()
    assert torch.equal(w.cache.data, data)
    w.check(q, w.cache.attend(q.to(gpu), b, prefix=p, once=True))


def test_strides_streams_and_graphs(gpu):
    """Queries inside a projection and on no boundary; another stream; a captured call replayed while
    lengths, rows and tables change."""
    import torch
    groups = [(150, [(1, 9), (1, 40), (1, 3)]), (33, [(1, 30), (1, 4)])]
    w = Shared(gpu, groups, 2, 128, 8, 16, "bf16", seed=12)
    q = w.queries(8).to(gpu)
    b, p = w.batch(), w.prefix()
    want = w.cache.attend(q, b, prefix=p, once=True)
    fused = torch.zeros(5, 12, 128, dtype=q.dtype, device=gpu)
    fused[:, 2:10] = q
    odd = torch.zeros(5 * (8 * 128 + 3) + 1, dtype=q.dtype, device=gpu)[1:].view(5, -1)[:, :1024].unflatten(1, (8, 128))
    odd.copy_(q)
    for x in (fused[:, 2:10], odd, q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(w.cache.attend(x, b, prefix=p, once=True), want)
    buf = torch.zeros(q.numel() + 1, dtype=q.dtype, device=gpu)[1:].view_as(q)
    assert torch.equal(w.cache.attend(q, b, prefix=p, once=True, out=buf), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = w.cache.attend(q, b, prefix=p, once=True, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(q)
    work = torch.full((w.cache.work_bytes(b, 8, prefix=p, once=True),), 0xff, dtype=torch.uint8, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.cache.attend(q, b, prefix=p, once=True, out=out, work=work)
    full = (b.kv_len.clone(), p.kv_len.clone())
    for i in range(4):
        b.kv_len.copy_(full[0] - torch.tensor([i, 2 * i, 0, i, 0], dtype=torch.int32, device=gpu))
        p.kv_len.copy_(full[1] - 7 * i)  # less of it shared: the same attention
        graph.replay()
        work.fill_(0xff)
        assert torch.equal(out, w.cache.attend(q, b, prefix=p, once=True, work=work))
        keep = w.kv, w.lens
        w.lens = b.kv_len.tolist()
        w.kv = [[x[:n] for x in kv] for kv, n in zip(w.kv, w.lens)]
        w.check(q.cpu(), out)
        w.kv, w.lens = keep


def test_refusals(gpu):
    import torch
    w = Shared(gpu, [(40, [(1, 3), (1, 1)])], 2, 64, 8, 16, "f16", seed=13)
    q = w.queries(4).to(gpu)
    b, p = w.batch(), w.prefix()
    for bad in (lambda: w.cache.attend(q, b, prefix=p, window=5), lambda: w.cache.work_bytes(b, 4, 5, prefix=p),
                lambda: w.cache.attend(q, b, prefix=w.prefix(n_tokens=3)),
                lambda: w.cache.work_bytes(b, 4, prefix=w.prefix(n_tokens=3)),
                lambda: w.cache.attend(q, b, prefix=p, once=True, work=torch.empty(16, dtype=torch.uint8, device=gpu)),
                lambda: w.cache.attend(q[:, :3], b, prefix=p)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("new,P,seqs,G,pays", [(1, 16000, 24, 4, True), (1, 60000, 4, 8, True),
                                               (9, 24000, 12, 4, True), (40, 9000, 12, 2, False)])
def test_where_it_pays(gpu, new, P, seqs, G, pays):
    """The bounds choose to read the prefix once, or by every sequence: the results of one way or the
    other, and both within rounding of the same values."""
    import torch
    w = Shared(gpu, [(P, [(new, new + 11 * i) for i in range(seqs)])], 4, 128, 8, 64, "bf16", seed=seqs)
    q = w.queries(4 * G).to(gpu)
    b, p = w.batch(), w.prefix()
    out = w.cache.attend(q, b, prefix=p)
    once, alone = w.cache.attend(q, b, prefix=p, once=True), w.cache.attend(q, b)
    assert torch.equal(out, once if pays else alone)
    assert w.cache.work_bytes(b, 4 * G, prefix=p) == w.cache.work_bytes(
        b, 4 * G, **(dict(prefix=p, once=True) if pays else {}))
    rows = slice(sum(w.new[:-1]), None)  # the last sequence against float64
    w.new, w.lens, w.kv = w.new[-1:], w.lens[-1:], w.kv[-1:]
    w.check(q[rows].cpu(), once[rows])
    w.check(q[rows].cpu(), alone[rows])


def test_two_calls_at_once(gpu):
    """On two streams, with a workspace each: each its own results, every time."""
    import torch
    w = Shared(gpu, [(900, [(1, 40 + i) for i in range(20)]), (300, [(2, 9)] * 3)], 2, 128, 8, 16, "bf16", seed=15)
    b, p = w.batch(), w.prefix()
    qs = [w.queries(8, seed=s).to(gpu) for s in (1, 2)]
    want = [w.cache.attend(q, b, prefix=p, once=True) for q in qs]
    n = w.cache.work_bytes(b, 8, prefix=p, once=True)
    streams = [torch.cuda.Stream() for _ in qs]
    works = [torch.empty(n, dtype=torch.uint8, device=gpu) for _ in qs]
    outs = [[torch.zeros_like(q) for _ in range(10)] for q in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i in range(10):
        for q, s, x, o in zip(qs, streams, works, outs):
            w.cache.attend(q, b, prefix=p, once=True, work=x, out=o[i], stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for os, y in zip(outs, want) for o in os)


def test_a_workspace_inside_others(gpu):
    """No byte outside the workspace is written, and every byte of it may be anything before."""
    import torch
    for groups, G in ((GROUPS["many_long"], 4), (GROUPS["few_short"], 1), (GROUPS["wide_chunks"], 4)):
        w = Shared(gpu, groups, 2, 64, 8, 16, "f16", seed=16)
        q = w.queries(2 * G).to(gpu)
        b, p = w.batch(), w.prefix()
        n = w.cache.work_bytes(b, 2 * G, prefix=p, once=True)
        buf = torch.full((n + 512,), 0xff, dtype=torch.uint8, device=gpu)
        out = w.cache.attend(q, b, prefix=p, once=True, work=buf[256:256 + n])
        assert (buf[:256] == 0xff).all() and (buf[256 + n:] == 0xff).all()
        w.check(q.cpu(), out)


@pytest.mark.parametrize("new,G", [(3, 4), (40, 4)])
def test_sequences_that_reach_into_a_group(gpu, new, G):
    """A sequence that begins outside of a group with a prefix and has rows in it: these are NaN, whatever
    stands in front of the group (a group without a prefix, or none); all other rows are as ever."""
    import torch
    w = Shared(gpu, [(0, [(new, 90)]), (64, [(1, 9), (2, 9)])], 2, 64, 8, 16, "f16", seed=17)
    T = new + 3
    q = w.queries(2 * G)
    b, p = w.batch(), w.prefix()
    first = ref.attend(_np(q[:new]).astype(np.float64), *w.kv[0], 64 ** -0.5, True, 0, ref.UNIT["f16"])
    table = {0: [-1] * p.pages.shape[1], 64: p.pages[1].tolist()}
    for cu, lens in (([0, new - 1, T], [0, 64]), ([1, T], [64]), ([0, 1, 2, T], [0, 64, 0])):
        y = w.cache.batch(w.i32([table[n] for n in lens]), w.i32(lens), w.i32(cu), T, T, 64)
        lse = torch.zeros(T, 2 * G, device=gpu)
        out = w.cache.attend(q.to(gpu), b, prefix=y, lse=lse, once=True)
        g = lens.index(64)
        cut = np.array([cu[g] <= t < cu[g + 1] for t in range(new)])
        assert torch.isnan(out[:new][cut]).all() and torch.isnan(lse[:new][cut]).all(), cu
        o, l, tol, ltol = (x[~cut] for x in first)
        assert (np.abs(_np(out[:new])[~cut] - o) <= tol).all(), cu
        assert (np.abs(lse[:new].cpu().numpy()[~cut] - l) <= ltol).all(), cu
        w.check(q, out, lse, skip=(0,))
