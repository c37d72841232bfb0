"""The quantised key/value cache on the device against its definition in float64
(kv_ref): what is written reads back exactly, and attention stays within the
bounds of its own roundings."""
import numpy as np
import pytest

import kv_ref as ref

import jhq_gpu_amd as jg

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _np(t):
    return t.float().cpu().numpy()


class World:
    """A cache, its page table in random order and the sequences' tokens."""

    def __init__(self, gpu, lens, H, D, bits=8, page=16, dtype="bf16", seed=0, spare=2, junk=0xff):
        import torch
        self.gpu, self.H, self.D, self.bits, self.page, self.dtype = gpu, H, D, bits, page, dtype
        self.lens = list(lens)
        rng = np.random.default_rng(seed)
        per = [-(-n // page) for n in lens]
        P = sum(per) + spare
        order = rng.permutation(P)
        self.table = np.full((len(lens), max(max(per), 1)), -1, np.int32)
        at = 0
        for b, p in enumerate(per):
            self.table[b, :p] = order[at:at + p]
            at += p
        self.cache = jg.KVCache(P, page, H, D, bits=bits, device=gpu)
        self.cache.data.fill_(junk)  # what lies there before must not matter
        N = sum(lens)
        g = torch.Generator().manual_seed(seed)
        size = torch.exp(torch.randn(N, 1, 1, generator=g))
        self.k = (torch.randn(N, H, D, generator=g) * size).to(_dt(dtype))
        self.v = (torch.randn(N, H, D, generator=g) * size.flip(0)).to(_dt(dtype))
        self.at = np.concatenate([[0], np.cumsum(lens)])

    def i32(self, a):
        import torch
        return torch.tensor(np.asarray(a, np.int32), device=self.gpu)

    def batch(self, new, lens=None, table=None, max_q=None, max_kv=None):
        lens = self.lens if lens is None else lens
        return self.cache.batch(self.i32(self.table if table is None else table), self.i32(lens),
                                self.i32(np.concatenate([[0], np.cumsum(new)])), int(sum(new)),
                                max(new) if max_q is None else max_q,
                                max(lens) if max_kv is None else max_kv)

    def rows(self, new, lens=None):
        """Rows of the last new[b] tokens of each sequence's first lens[b]."""
        lens = self.lens if lens is None else lens
        return np.concatenate([np.arange(a + n - q, a + n)
                               for a, n, q in zip(self.at, lens, new)]).astype(np.int64)

    def fill(self):
        self.cache.write(self.k.to(self.gpu), self.v.to(self.gpu), self.batch(self.lens))

    def held(self):
        """float64 values of all tokens."""
        return [ref.value32(_np(x), self.bits).astype(np.float64) for x in (self.k, self.v)]


SHAPES = [(8, 128, 2, 64), (8, 64, 3, 16), (8, 256, 1, 32), (4, 128, 2, 16), (4, 64, 5, 128),
          (4, 256, 2, 16)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,D,H,page", SHAPES)
def test_written_rows_read_back(gpu, bits, D, H, page, dtype):
    """Sequences of every kind of end inside a group and a page, written in two
    steps that split groups; rows equal the definition's bit for bit."""
    import torch
    lens = [1, 16, 0, 17, 33, 5, 64, 131, 2]
    w = World(gpu, lens, H, D, bits, page, dtype, seed=bits + D)
    first = [n * 2 // 3 for n in lens]
    r = w.rows(first, first)
    w.cache.write(w.k[r].to(gpu), w.v[r].to(gpu), w.batch(first, first))
    before = w.cache.data.clone()
    rest = [n - f for n, f in zip(lens, first)]
    r = w.rows(rest)
    w.cache.write(w.k[r].to(gpu), w.v[r].to(gpu), w.batch(rest))
    k, v = w.cache.read(w.batch(lens), dtype=torch.float32)
    assert np.array_equal(_np(k), ref.value32(_np(w.k), bits))
    assert np.array_equal(_np(v), ref.value32(_np(w.v), bits))
    k16, v16 = w.cache.read(w.batch(lens), dtype=_dt(dtype))
    assert torch.equal(k16, k.to(_dt(dtype))) and torch.equal(v16, v.to(_dt(dtype)))
    # pages of no sequence keep every byte
    pb = w.cache.data.numel() // w.cache.num_pages
    used = set(w.table[w.table >= 0].tolist())
    for p in range(w.cache.num_pages):
        if p not in used:
            assert torch.equal(w.cache.data[p * pb:(p + 1) * pb], before[p * pb:(p + 1) * pb])
    # a single token back
    one = [min(n, 1) for n in lens]
    k1, _ = w.cache.read(w.batch(one))
    assert np.array_equal(_np(k1), ref.value32(_np(w.k), bits)[w.rows(one)])


@pytest.mark.parametrize("bits", [8, 4])
def test_strides_and_alignment(gpu, bits):
    """Rows inside a fused projection, heads outermost, and rows that start on no
    16-byte boundary; read into unaligned rows too."""
    import torch
    H, D = 2, 128
    lens = [37, 20]
    w = World(gpu, lens, H, D, bits, 16, "bf16", seed=3)
    T = sum(lens)
    want = [ref.value32(_np(x), bits) for x in (w.k, w.v)]
    fused = torch.zeros(T, 3 * H, D, dtype=torch.bfloat16, device=gpu)
    fused[:, H:2 * H], fused[:, 2 * H:] = w.k.to(gpu), w.v.to(gpu)
    odd = torch.zeros(2, T * (H * D + 3) + 1, dtype=torch.bfloat16, device=gpu)
    ko, vo = (o[1:].view(T, H * D + 3)[:, :H * D].unflatten(1, (H, D)) for o in odd)
    ko.copy_(w.k), vo.copy_(w.v)
    kt, vt = (x.to(gpu).transpose(0, 1).contiguous().transpose(0, 1) for x in (w.k, w.v))
    for k, v in ((fused[:, H:2 * H], fused[:, 2 * H:]), (ko, vo), (kt, vt)):
        w.cache.data.fill_(0xff)
        w.cache.write(k, v, w.batch(lens))
        got = w.cache.read(w.batch(lens))
        assert all(np.array_equal(_np(a), b) for a, b in zip(got, want))
        buf = torch.zeros(2, T * H * D + 1, dtype=torch.float16, device=gpu)
        a, b = (x[1:].view(T, H, D) for x in buf)
        w.cache.read(w.batch(lens), k_out=a, v_out=b)
        assert torch.equal(a, got[0].half()) and torch.equal(b, got[1].half())


@pytest.mark.parametrize("bits", [8, 4])
def test_float32_rows(gpu, bits):
    """float32 rows: the scale exactly, each element within half a step (and the
    quotient's float32 error)."""
    import torch
    H, D, lens = 2, 128, [50]
    w = World(gpu, lens, H, D, bits, 16, "f32", seed=5)
    w.fill()
    k, v = w.cache.read(w.batch(lens))
    top = 127 if bits == 8 else 7
    for got, x in ((k, w.k), (v, w.v)):
        x = _np(x).astype(np.float64)
        step = np.abs(x).max(-1, keepdims=True) / top
        assert (np.abs(_np(got) - x) <= step * (0.5 + 2.0 ** -15)).all()
        assert np.allclose(np.abs(_np(got)).max(-1, keepdims=True), step * top, rtol=2.0 ** -22)


@pytest.mark.parametrize("bits", [8, 4])
def test_ties_zeros_and_extremes(gpu, bits):
    """Halves between codes go to the even one; rows of zeros, below the floor,
    at the type's ends, and rows with an infinity or a NaN."""
    import torch
    D, top = 64, 127 if bits == 8 else 7
    x = torch.zeros(12, 1, D)
    x[0, 0, :top + 1] = torch.arange(top + 1)[:D] if top + 1 <= D else torch.arange(D)
    x[1, 0] = torch.linspace(-1, 1, D)
    x[1, 0, 0], x[1, 0, 1] = -1.0, 0.5       # amax / 2 is a tie (63.5, 3.5)
    x[2, 0, :3] = torch.tensor([2.0 ** -61, -2.0 ** -62, 0])   # below the floor: zeros
    x[3, 0, :3] = torch.tensor([2.0 ** -60, 2.0 ** -61, 0])    # at the floor: held
    x[4, 0, :3] = torch.tensor([3.0e38, -1.5e38, 1.0e38])
    x[5, 0, 7] = float("inf")
    x[6, 0, 9] = float("nan")
    x[7, 0, 3], x[7, 0, 4] = float("-inf"), float("nan")
    x[8, 0] = torch.where(torch.arange(D) % 2 == 0, 254.0, 1.0)   # (2i + 1) / 254 halves
    x[8, 0, 1::2] = torch.arange(D // 2).float() * 2 + 1
    x[9, 0] = -x[8, 0]
    x[10, 0, 0], x[10, 0, 1:8] = 14.0, torch.arange(7).float() * 2 + 1
    x = x.bfloat16()
    n = x.shape[0]
    w = World(gpu, [n], 1, D, bits, 16, "bf16")
    w.k, w.v = x, x.flip(0)
    w.fill()
    k, v = w.cache.read(w.batch([n]))
    for got, src in ((k, w.k), (v, w.v)):
        want = ref.value32(_np(src), bits)
        assert np.array_equal(_np(got), want, equal_nan=True)
        assert np.isnan(want).all(-1).sum() == 3 and np.isnan(want).any(-1).sum() == 3


def test_contradictions_touch_nothing_else(gpu):
    """Pages outside the buffer, sequences past max_kv or max_q and rows outside
    n_tokens: NaN where they are read, nothing written, neighbours intact."""
    import torch
    H, D, lens = 2, 64, [40, 40, 40, 20]
    w = World(gpu, lens, H, D, 8, 16, "bf16", seed=9)
    w.fill()
    want = ref.value32(_np(w.k), 8)
    table = w.table.copy()
    table[1, 1], table[2, 0] = 1 << 20, -5
    k, v = (_np(t) for t in w.cache.read(w.batch(lens, table=table)))
    bad = np.zeros(sum(lens), bool)
    bad[40 + 16:40 + 32] = bad[80:96] = True
    assert np.isnan(k[bad]).all() and np.isnan(v[bad]).all()
    assert np.array_equal(k[~bad], want[~bad])
    before = w.cache.data.clone()
    other = w.batch(lens, table=np.where(table == table[1, 1], 1 << 20, -1), max_kv=40)
    w.cache.write(torch.ones_like(w.k).to(gpu), torch.ones_like(w.k).to(gpu), other)
    assert torch.equal(before, w.cache.data)
    # max_kv and max_q below what the arrays say
    for b in (w.batch(lens, max_kv=30), w.batch(lens, max_q=30, max_kv=40)):
        w.cache.write(torch.ones_like(w.k).to(gpu), torch.ones_like(w.k).to(gpu), b)
        w.cache.write(w.k[120:].to(gpu), w.v[120:].to(gpu),
                      w.batch([0, 0, 0, 20]))  # the one that was within the bounds
        assert torch.equal(before, w.cache.data)
        k, _ = w.cache.read(b)
        k = _np(k)
        assert np.isnan(k[:30]).all() and np.array_equal(k[120:], want[120:])
        q = torch.randn(140, 4, D, device=gpu, dtype=torch.bfloat16)
        o = _np(w.cache.attend(q, b))
        assert np.isnan(o[:30]).all() and np.isfinite(o[120:]).all()
    # cu_q past n_tokens: that sequence has no rows here
    b = w.cache.batch(w.i32(w.table), w.i32(lens), w.i32([0, 40, 80, 120, 150]), 140, 40, 40)
    k, _ = w.cache.read(b)
    assert np.array_equal(_np(k)[:120], want[:120]) and not _np(k)[120:].any()


def _check(w, new, Hq, causal=True, window=0, scale=None, lens=None, q=None, seed=1, **kw):
    import torch
    lens = w.lens if lens is None else lens
    T = sum(new)
    if q is None:
        g = torch.Generator().manual_seed(seed)
        q = (torch.randn(T, Hq, w.D, generator=g) * 1.5).to(_dt(w.dtype))
    lse = torch.full((T, Hq), 7.0, device=w.gpu)
    b = w.batch(new, lens)
    out = w.cache.attend(q.to(w.gpu), b, causal=causal, window=window, scale=scale, lse=lse, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape
    again = w.cache.attend(q.to(w.gpu), b, causal=causal, window=window, scale=scale)
    assert torch.equal(out, again), "not the same twice"
    k, v = w.held()
    got, gl = _np(out), lse.cpu().numpy()
    at = 0
    for s, (a, n) in enumerate(zip(new, lens)):
        sl = slice(w.at[s], w.at[s] + n)
        qq = _np(q[at:at + a]).astype(np.float64)
        o, l, tol, ltol = ref.attend(qq, k[sl], v[sl], w.D ** -0.5 if scale is None else scale,
                                     causal, window, ref.UNIT[w.dtype])
        err = np.abs(got[at:at + a] - o)
        assert (err <= tol).all(), (s, a, n, (err / np.maximum(tol, 1e-300)).max())
        e = np.isinf(l)
        assert np.array_equal(gl[at:at + a][e], l[e])
        assert (got[at:at + a][e] == 0).all()
        assert (np.abs(gl[at:at + a][~e] - l[~e]) <= ltol[~e]).all(), (s, a, n)
        at += a
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,D,H,page", SHAPES)
@pytest.mark.parametrize("G", [1, 4, 7])
def test_single_tokens(gpu, bits, D, H, page, dtype, G):
    lens = [1, 2, 15, 16, 0, 17, 63, 64, 65, 130, 700]
    w = World(gpu, lens, H, D, bits, page, dtype, seed=D + bits)
    w.fill()
    _check(w, [min(n, 1) for n in lens], H * G)


@pytest.mark.parametrize("bits,D,H,page", SHAPES)
@pytest.mark.parametrize("G", [1, 3, 8])
def test_chunks(gpu, bits, D, H, page, G):
    """Chunks of a few tokens and of many, over nothing, a little and much."""
    lens = [1, 70, 33, 0, 200, 16, 519]
    new = [1, 70, 5, 0, 129, 2, 300]
    w = World(gpu, lens, H, D, bits, page, "f16" if G == 3 else "bf16", seed=D + G)
    w.fill()
    _check(w, new, H * G)


@pytest.mark.parametrize("n_seq", [3, 64, 65, 150])
def test_chunks_of_many_ragged_sequences(gpu, n_seq):
    """Sequences with no tile beside ones with several, fewer and more of them than a
    wave has lanes."""
    rng = np.random.default_rng(n_seq)
    new = [int(x) for x in rng.choice([0, 0, 1, 31, 33, 63, 64, 65, 129, 200], n_seq)]
    new[0], new[-1] = 0, 130
    lens = [q + int(x) for q, x in zip(new, rng.choice([0, 1, 50, 130], n_seq))]
    w = World(gpu, lens, 2, 64, 8, 16, "f16", seed=n_seq)
    w.fill()
    _check(w, new, 4)
    _check(w, new, 4, window=40)


@pytest.mark.parametrize("window", [1, 15, 64, 100, 5000])
@pytest.mark.parametrize("new", [[1, 1, 1], [200, 40, 3], [20, 20, 2]])
def test_windows(gpu, window, new):
    lens = [400, 40, 777]
    w = World(gpu, lens, 2, 128, 8, 32, "bf16", seed=window)
    w.fill()
    _check(w, new, 8, window=window)


@pytest.mark.parametrize("new", [6, 40, 200])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1])
def test_windows_longer_than_any_sequence(gpu, window, new):
    """Such a window hides nothing, also where new tokens stand far before position 0
    (more of them than tokens)."""
    import torch
    w = World(gpu, [3], 2, 64, 8, 16, "bf16", seed=6)
    w.fill()
    q = torch.randn(new, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(gpu)
    b = w.cache.batch(w.i32(w.table), w.i32([3]), w.i32([0, new]), new, new, 3)
    lse = [torch.zeros(new, 4, device=gpu) for _ in range(2)]
    out = w.cache.attend(q, b, window=window, lse=lse[0])
    assert torch.equal(out, w.cache.attend(q, b, lse=lse[1])) and torch.equal(*lse)
    assert torch.isfinite(lse[0][-3:]).all() and torch.isneginf(lse[0][:-3]).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [120, 40, 9], [400, 40, 70]])
def test_everything_visible(gpu, new):
    lens = [400, 40, 131]
    w = World(gpu, lens, 3, 64, 4, 16, "f16", seed=2)
    w.fill()
    _check(w, new, 6, causal=False)


@pytest.mark.parametrize("bits,G", [(8, 4), (4, 8), (8, 1)])
def test_long_contexts(gpu, bits, G):
    """Long enough that the tokens are split over workgroups and joined."""
    lens = [20011, 300, 0, 9000]
    w = World(gpu, lens, 1, 128, bits, 64, "f16", seed=bits)
    w.fill()
    _check(w, [1, 1, 0, 1], G)
    _check(w, [3, 40, 0, 2], G)
    _check(w, [1, 1, 0, 1], G, window=7000)


def test_rows_that_see_nothing(gpu):
    """More new tokens than tokens: the rows before position 0 see nothing (they
    come first), beside ordinary rows of the same sequence."""
    import torch
    w = World(gpu, [40, 30], 2, 64, 8, 16, "bf16", seed=4)
    w.fill()
    T, Hq = 100, 4
    q = torch.randn(T, Hq, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    b = w.cache.batch(w.i32(w.table), w.i32([40, 30]), w.i32([0, 60, 100]), T, 60, 40)
    lse = torch.zeros(T, Hq, device=gpu)
    out = _np(w.cache.attend(q.to(gpu), b, lse=lse))
    k, v = w.held()
    for (r0, r1), (t0, t1) in (((0, 60), (0, 40)), ((60, 100), (40, 70))):
        n, a = t1 - t0, r1 - r0
        o, l, tol, _ = ref.attend(_np(q[r1 - n:r1]).astype(np.float64), k[t0:t1], v[t0:t1], 0.125,
                                  unit=ref.UNIT["bf16"])
        assert (out[r0:r1 - n] == 0).all() and np.isneginf(lse[r0:r1 - n].cpu().numpy()).all()
        assert (np.abs(out[r1 - n:r1] - o) <= tol).all()
    # read and write leave such rows alone
    w.cache.write(w.k.new_ones(T, 2, 64).to(gpu) * float("nan"),
                  w.k.new_ones(T, 2, 64).to(gpu), w.cache.batch(
                      w.i32(w.table), w.i32([0, 0]), w.i32([0, 60, 100]), T, 60, 40))
    kk, _ = w.cache.read(w.batch([40, 30]))
    assert np.array_equal(_np(kk), ref.value32(_np(w.k), 8))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("new", [[20, 1], [150, 64]])
def test_nan_rows_reach_only_what_sees_them(gpu, bits, new):
    """A token whose key or value is not finite: the rows that see it are NaN, all
    others as if it were not there; the same for a query that is not finite."""
    import torch
    lens = [170, 64]
    w = World(gpu, lens, 1, 128, bits, 16, "bf16", seed=6)
    hot = 165
    w.v[hot, 0, 5] = float("inf")
    w.k[hot + 3, 0, 1] = float("nan")
    w.fill()
    clean_k, clean_v = w.k.clone(), w.v.clone()
    g = torch.Generator().manual_seed(1)
    q = torch.randn(sum(new), 4, 128, generator=g).bfloat16()
    q[2, 1, 0] = float("inf")
    out = _np(w.cache.attend(q.to(gpu), w.batch(new)))
    k, v = w.held()
    pos = np.concatenate([np.arange(n - a, n) for n, a in zip(lens, new)])
    seq = np.repeat([0, 1], new)
    nan = np.zeros(out.shape[:2], bool)
    nan[(seq == 0) & (pos >= hot)] = True
    nan[2, 1] = True
    assert np.isnan(out[nan]).all()
    assert np.isfinite(out[~nan]).all()
    for s, (a, n) in enumerate(zip(new, lens)):
        sl, at = slice(w.at[s], w.at[s] + n), sum(new[:s])
        kk, vv = np.nan_to_num(k[sl], nan=0.0), np.nan_to_num(v[sl], nan=0.0)
        qq = _np(q[at:at + a]).astype(np.float64)
        o, _, tol, _ = ref.attend(np.where(np.isfinite(qq), qq, 0), kk, vv, 128 ** -0.5,
                                  unit=ref.UNIT["bf16"])
        ok = ~nan[at:at + a]
        assert (np.abs(out[at:at + a] - o)[ok] <= tol[ok]).all()
    del clean_k, clean_v


@pytest.mark.parametrize("new", [[1], [130]])
def test_values_of_very_different_sizes(gpu, new):
    """Rows of zero values that draw most of the weight, values many orders of
    magnitude apart, and sharp and flat softmax rows."""
    import torch
    n = 150
    w = World(gpu, [n], 2, 64, 8, 16, "bf16", seed=8)
    w.v[::3] = 0
    w.v[1::3] = (w.v[1::3].float() * 1e-12).bfloat16()
    w.v[2::7] = (w.v[2::7].float() * 1e6).bfloat16()
    w.k[:2] = (w.k[:2].float() * 30).bfloat16()
    w.fill()
    for s in (0.125, 2.0, 0.0, -0.3):
        _check(w, new, 4, scale=s)
    # all values tiny: the output is not lost
    w.v = (w.v.float().clamp(-1, 1) * 1e-9).bfloat16()
    w.fill()
    got = _check(w, new, 4)
    assert np.abs(got).max() > 0
    q = (torch.randn(sum(new), 4, 64, generator=torch.Generator().manual_seed(2)) * 1e30).bfloat16()
    out = w.cache.attend(q.to(gpu), w.batch(new), scale=1e-30)
    small = w.cache.attend((q.float() * 2.0 ** -100).bfloat16().to(gpu), w.batch(new),
                           scale=1e-30 * 2.0 ** 100)
    assert torch.equal(out, small)  # powers of two in q and scale cancel


@pytest.mark.parametrize("new,D,bits", [([2], 128, 8), ([9], 64, 4), ([100], 128, 8), ([70], 256, 4)])
def test_queries_of_very_different_sizes(gpu, new, D, bits):
    """Rows 2^-50 to 2^90 apart in one tile: none costs another its precision."""
    import torch
    w = World(gpu, [300], 1, D, bits, 16, "bf16", seed=11)
    w.fill()
    T, Hq = new[0], 4
    q = torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(6)) * 1.5
    size = torch.tensor([1.0, 2.0 ** 90, 2.0 ** -50, 2.0 ** -14]).repeat(T)[torch.randperm(4 * T)]
    size = size.view(T, Hq, 1)
    _check(w, new, Hq, q=(q * size).bfloat16())  # bounds are each row's own


@pytest.mark.parametrize("new", [1, 5, 80])
def test_very_negative_scores(gpu, new):
    """Scores of -1e36 are scores: a row whose tokens are all alike gets their value."""
    import torch
    D, n = 64, 90
    w = World(gpu, [n], 1, D, 8, 16, "bf16")
    w.k = torch.full((n, 1, D), -1e18).bfloat16()
    w.v = torch.linspace(-1, 1, D).expand(n, 1, D).bfloat16()
    w.fill()
    out = w.cache.attend(torch.full((new, 2, D), 1e18, device=gpu).bfloat16(), w.batch([new]))
    want = torch.tensor(w.held()[1][0, 0]).bfloat16()
    assert torch.equal(out.cpu(), want.expand(new, 2, D))


def test_strided_queries_outputs_and_streams(gpu):
    """Queries inside a fused projection and on no 16-byte boundary, own output,
    workspace and stream."""
    import torch
    lens, new, Hq, D = [300, 5000], [70, 3], 4, 128
    w = World(gpu, lens, 2, D, 8, 64, "bf16", seed=10)
    w.fill()
    T = sum(new)
    q = torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(3)).bfloat16().to(gpu)
    want = w.cache.attend(q, w.batch(new))
    fused = torch.zeros(T, Hq + 4, D, dtype=torch.bfloat16, device=gpu)
    fused[:, 2:2 + Hq] = q
    odd = torch.zeros(T * (Hq * D + 5) + 1, dtype=torch.bfloat16, device=gpu)
    qo = odd[1:].view(T, Hq * D + 5)[:, :Hq * D].unflatten(1, (Hq, D))
    qo.copy_(q)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (fused[:, 2:2 + Hq], qo, qt):
        assert torch.equal(w.cache.attend(x, w.batch(new)), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = w.batch(new)
    s.wait_stream(torch.cuda.current_stream())
    outs = [w.cache.attend(q, b, stream=s) for _ in range(4)]
    odd_out = torch.zeros(T * Hq * D + 1, dtype=torch.bfloat16, device=gpu)
    with torch.cuda.stream(s):
        work = torch.empty(w.cache.work_bytes(b, Hq), dtype=torch.uint8, device=gpu)
        odd_out.zero_()
        got = w.cache.attend(q, b, out=odd_out[1:].view(T, Hq, D), work=work)
    s.synchronize()
    assert all(torch.equal(o, want) for o in outs) and torch.equal(got, want)


def test_graph_replays(gpu):
    """A captured step (write, attend) replayed with lengths and tokens changed in
    place equals the eager step."""
    import torch
    H, Hq, D, n0 = 2, 8, 128, [4000, 60]
    w = World(gpu, [5000, 200], H, D, 8, 64, "bf16", seed=12)
    w.cache.write(w.k.to(gpu), w.v.to(gpu), w.batch([5000, 200]))
    kv = w.i32(n0)
    b = w.cache.batch(w.i32(w.table), kv, w.i32([0, 1, 2]), 2, 1, 5000)
    k, v = (torch.zeros(2, H, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    q = torch.zeros(2, Hq, D, dtype=torch.bfloat16, device=gpu)
    out = torch.zeros_like(q)
    work = torch.empty(w.cache.work_bytes(b, Hq), dtype=torch.uint8, device=gpu)

    def step():
        w.cache.write(k, v, b)
        w.cache.attend(q, b, out=out, work=work)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    gen = torch.Generator().manual_seed(5)
    for i in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen))
        kv.add_(7 * i + 1)
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.isfinite(got).all() and torch.equal(got, out), i


def test_offsets_past_32_bits(gpu):
    """Pages that lie more than 2^32 bytes into the buffer."""
    import torch
    H, D, page = 8, 128, 1024
    P = (9 << 29) // (H * page * (2 * D + 8)) + 2  # 4.5 GiB
    c = jg.KVCache(P, page, H, D, device=gpu)
    assert c.data.numel() > 1 << 32
    n = 1500
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(n, H, D, generator=g).bfloat16() for _ in range(2))
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    b = c.batch(i32([[P - 1, P - 2]]), i32([n]), i32([0, n]), n, n, n)
    c.write(k.to(gpu), v.to(gpu), b)
    gk, gv = c.read(b)
    assert np.array_equal(_np(gk), ref.value32(_np(k), 8))
    assert np.array_equal(_np(gv), ref.value32(_np(v), 8))
    q = torch.randn(1, H, D, generator=g).bfloat16()
    out = _np(c.attend(q.to(gpu), c.batch(i32([[P - 1, P - 2]]), i32([n]), i32([0, 1]), 1, 1, n)))
    o, _, tol, _ = ref.attend(_np(q).astype(np.float64), ref.value32(_np(k), 8).astype(np.float64),
                              ref.value32(_np(v), 8).astype(np.float64), D ** -0.5,
                              unit=ref.UNIT["bf16"])
    assert (np.abs(out - o) <= tol).all()


def test_python_refusals(gpu):
    import torch
    w = World(gpu, [20], 2, 64, 8, 16, "bf16")
    b = w.batch([20])
    k, v, q = w.k.to(gpu), w.v.to(gpu), torch.zeros(20, 4, 64, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError):
        jg.KVCache(4, 16, 2, 80, device=gpu)
    with pytest.raises(ValueError):
        jg.KVCache(4, 24, 2, 64, device=gpu)
    for bad in (k[:10], k[:, :1], k.double(), k.cpu(), k.float(), k[:, :, :32]):
        with pytest.raises(ValueError):
            w.cache.write(bad, v, b)
    with pytest.raises(ValueError):
        w.cache.write(k.transpose(1, 2).contiguous().transpose(1, 2), v, b)
    for bad in (q.float(), q[:, :3], q[:5], q[:, :, :32]):
        with pytest.raises(ValueError):
            w.cache.attend(bad, b)
    with pytest.raises(ValueError):
        w.cache.attend(q, b, causal=False, window=3)
    with pytest.raises(ValueError):
        w.cache.attend(q, b, out=torch.zeros(20, 4, 64, device=gpu))
    with pytest.raises(ValueError):
        w.cache.attend(q, b, lse=torch.zeros(20, 2, device=gpu))
    with pytest.raises(ValueError):
        w.cache.read(b, k_out=torch.zeros(20, 2, 64, device=gpu))
    with pytest.raises(ValueError):
        w.cache.batch(w.i32(w.table).long(), w.i32([20]), w.i32([0, 20]), 20, 20, 20)
    with pytest.raises(ValueError):
        w.cache.batch(w.i32(w.table), w.i32([20]), w.i32([0, 20]), 20, 20, 1000)
