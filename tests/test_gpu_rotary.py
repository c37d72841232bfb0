"""Rotary positions on the device against the formula in float64 (rotary_ref), and the
cache's write with them."""
import numpy as np
import pytest

import rotary_ref as ref

import jhq_gpu_amd as jg

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _np(t):
    return t.double().cpu().numpy()


def _rows(T, h, D, dtype, seed=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, h, D, generator=g) * torch.exp(torch.randn(T, 1, D, generator=g))).to(_dt(dtype))


def _check(rope, got, x, pos, dtype, inverse=False):
    y, tol = ref.turn(_np(x), pos, rope.frequencies, rope.rot_dim, rope.interleaved, rope.amplitude,
                      inverse, ref.UNIT[dtype])
    err = np.abs(_np(got) - y)
    assert (err <= tol).all(), (err - tol).max()


SHAPES = [  # head_dim, rot_dim, heads, tokens
    (64, 64, 1, 1), (64, 64, 3, 37), (64, 32, 5, 9), (128, 128, 40, 3), (128, 128, 18, 1), (128, 64, 2, 70),
    (256, 256, 7, 5), (256, 64, 12, 11), (80, 80, 6, 10), (80, 20, 3, 33), (96, 48, 9, 4), (192, 192, 2, 3),
    (1024, 1024, 2, 3), (1024, 2, 1, 4), (2, 2, 1, 130), (6, 4, 70, 3), (66, 34, 2, 5), (520, 520, 3, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,h,T", SHAPES)
def test_turns(gpu, D, rot, h, T, interleaved, dtype):
    import torch
    rope = jg.Rotary(D, rot_dim=rot, interleaved=interleaved, device=gpu)
    x = _rows(T, h, D, dtype, seed=D + rot)
    rng = np.random.default_rng(T)
    pos = rng.integers(0, 9000, T)
    p = torch.from_numpy(pos).to(gpu)
    for inverse in (False, True):
        got = rope.apply(x.to(gpu), p, inverse=inverse)
        _check(rope, got, x, pos, dtype, inverse)
        assert torch.equal(got, rope.apply(x.to(gpu), p.int(), inverse=inverse))
        same = x.to(gpu)
        assert rope.apply(same, p, inverse=inverse, out=same) is same
        assert torch.equal(same, got)


@pytest.mark.parametrize("pos", [[0, 1, 2 ** 20, 2 ** 30 + 3, 2 ** 31 - 1], [-1, -70000, 2 ** 40 + 1, 5]])
@pytest.mark.parametrize("scaling", [None, dict(kind="linear", factor=8), dict(kind="ntk", factor=4),
                                     dict(kind="yarn", factor=16, length=4096),
                                     dict(kind="bands", factor=8, length=8192)])
def test_far_positions_and_scalings(gpu, pos, scaling):
    """float32 rows: an angle's error is the frequency's rounding alone, |p| 2^-65 turns, which the
    bound covers up to 2^40 (2^-25 turns, 2^-22.3 radians)."""
    import torch
    rope = jg.Rotary(128, rot_dim=128, base=500000.0, scaling=scaling, device=gpu)
    x = _rows(len(pos), 2, 128, "f32", seed=7)
    got = rope.apply(x.to(gpu), torch.tensor(pos, device=gpu))
    y, tol = ref.turn(_np(x), pos, rope.frequencies, 128, False, rope.amplitude, False, ref.UNIT["f32"])
    pair = np.abs(_np(x)[..., :64]) + np.abs(_np(x)[..., 64:])
    far = np.abs(np.array(pos, np.float64))[:, None, None] * 2.0 ** -65 * 2 * np.pi
    tol += np.concatenate([pair, pair], -1) * far * 2 * rope.amplitude
    assert (np.abs(_np(got) - y) <= tol).all()


def test_own_frequencies_and_amplitude(gpu):
    import torch
    freq = [0.0, 1.0, -2.5, 1e-9, 3.0e5, 0.1, 0.2, 0.3]
    rope = jg.Rotary(32, rot_dim=16, frequencies=freq, amplitude=-1.75, device=gpu)
    x = _rows(5, 3, 32, "f32")
    pos = [0, 1, 17, 4000, 10 ** 6]
    _check(rope, rope.apply(x.to(gpu), torch.tensor(pos, device=gpu)), x, pos, "f32")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_and_alignment(gpu, dtype):
    """Rows inside a projection, heads outermost, rows on no boundary, rows that share memory,
    into strided outputs."""
    import torch
    T, h, D = 19, 5, 128
    rope = jg.Rotary(D, device=gpu)
    x = _rows(T, h, D, dtype).to(gpu)
    pos = torch.arange(T, device=gpu) * 37
    want = rope.apply(x, pos)
    fused = torch.zeros(T, 3 * h, D, dtype=x.dtype, device=gpu)
    fused[:, h:2 * h] = x
    odd = torch.zeros(T * (h * D + 3) + 1, dtype=x.dtype, device=gpu)[1:].view(T, -1)[:, :h * D] \
        .unflatten(1, (h, D))
    odd.copy_(x)
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    for y in (fused[:, h:2 * h], odd, turned):
        assert torch.equal(rope.apply(y, pos), want)
        out = torch.zeros(h, T, D, dtype=x.dtype, device=gpu).transpose(0, 1)
        assert rope.apply(y, pos, out=out) is out and torch.equal(out, want)
        rope.apply(y, pos, out=y)
        assert torch.equal(y, want)
    assert (fused[:, :h] == 0).all() and (fused[:, 2 * h:] == 0).all()
    # queries and keys of one projection in one call, in place
    fused[:, :h] = x
    fused[:, h:2 * h] = x
    rope.apply(fused[:, :2 * h], pos, out=fused[:, :2 * h])
    assert torch.equal(fused[:, :h], want) and torch.equal(fused[:, h:2 * h], want)
    one = x[:, :1].expand(T, h, D)
    assert torch.equal(rope.apply(one, pos), rope.apply(one.contiguous(), pos))
    row = x[:1].expand(T, h, D)
    assert torch.equal(rope.apply(row, pos), rope.apply(row.contiguous(), pos))


def _batch(gpu, lens, new, n_tokens=None, first=0):
    import torch
    cache = jg.KVCache(4, 1024, 1, 64, device=gpu)

    def i32(a):
        return torch.tensor(np.asarray(a, np.int32), device=gpu)
    cu = np.concatenate([[0], np.cumsum(new)]) + first
    return cache.batch(torch.zeros(len(lens), 32, dtype=torch.int32, device=gpu), i32(lens), i32(cu),
                       int(cu[-1]) if n_tokens is None else n_tokens, max(new), max(lens))


@pytest.mark.parametrize("heads,D", [(1, 64), (3, 128), (40, 128), (2, 80)])
def test_positions_of_a_batch(gpu, heads, D):
    """Idle sequences, single tokens and chunks, more new tokens than tokens (positions below 0);
    rows before the first and behind the last sequence stay as they were."""
    import torch
    lens = [700, 0, 5, 9, 0, 20000, 3, 131]
    new = [1, 0, 5, 2, 0, 77, 6, 1]
    T = sum(new)
    rope = jg.Rotary(D, device=gpu)
    x = _rows(T + 9, heads, D, "bf16").to(gpu)
    pos = np.concatenate([np.arange(n - q, n) for n, q in zip(lens, new)])
    b = _batch(gpu, lens, new, n_tokens=T + 9, first=4)
    out = torch.full_like(x, 7.0)
    rope.apply(x, b, out=out)
    assert (out[:4] == 7).all() and (out[T + 4:] == 7).all()
    assert torch.equal(out[4:T + 4], rope.apply(x[4:T + 4], torch.from_numpy(pos).to(gpu)))
    fresh = rope.apply(x, b)
    assert (fresh[:4] == 0).all() and torch.equal(fresh[4:T + 4], out[4:T + 4])


def test_many_sequences(gpu):
    import torch
    rng = np.random.default_rng(3)
    new = [int(a) for a in rng.integers(0, 4, 300)]
    lens = [a + int(b) for a, b in zip(new, rng.integers(0, 5000, 300))]
    rope = jg.Rotary(64, device=gpu)
    x = _rows(sum(new), 1, 64, "f32").to(gpu)
    pos = np.concatenate([np.arange(n - q, n) for n, q in zip(lens, new)])
    assert torch.equal(rope.apply(x, _batch(gpu, lens, new)), rope.apply(x, torch.from_numpy(pos).to(gpu)))


def test_gradient(gpu):
    """The inverse is the transposed map: against the formula's gradient and against differences of
    sum(g * apply(x)), which is linear in x (so a step of 1 has no error but float32's)."""
    import torch
    rope = jg.Rotary(64, rot_dim=32, scaling=dict(kind="yarn", factor=4, length=128), device=gpu)
    x, g = _rows(6, 2, 64, "f32", 1).to(gpu), _rows(6, 2, 64, "f32", 2).to(gpu)
    pos = [3, 0, 100, 5000, 77, 12]
    p = torch.tensor(pos, device=gpu)
    dx = rope.apply(g, p, inverse=True)
    _check(rope, dx, g.cpu(), pos, "f32", inverse=True)
    rng = np.random.default_rng(0)
    base = _np(rope.apply(x, p))
    for _ in range(20):
        i = tuple(int(rng.integers(0, n)) for n in x.shape)
        y = x.clone()
        y[i] += 1.0
        diff = ((_np(rope.apply(y, p)) - base) * _np(g)).sum()
        row = np.abs(_np(g)[i[0], i[1]])
        # two outputs of the pair, each within a few roundings of float32 of its terms
        big = (np.abs(_np(x)[i[0], i[1]]).max() + 1) * rope.amplitude * 16 * 2.0 ** -24
        assert abs(diff - float(dx[i])) <= big * 2 * row.max() + abs(float(dx[i])) * 2.0 ** -22


def test_not_finite(gpu):
    """Infinities and NaN stay in their pair."""
    import torch
    rope = jg.Rotary(64, device=gpu)
    x = _rows(3, 2, 64, "bf16")
    x[0, 0, 3], x[1, 1, 40], x[2, 0, 0] = float("nan"), float("inf"), float("-inf")
    got = rope.apply(x.to(gpu), torch.tensor([5, 6, 7], device=gpu)).cpu()
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    for t, h, e in ((0, 0, 3), (1, 1, 40), (2, 0, 0)):
        want[t, h, e % 32] = want[t, h, e % 32 + 32] = True
    assert torch.equal(bad, want)


def test_streams_and_graphs(gpu):
    import torch
    rope = jg.Rotary(128, device=gpu)
    x = _rows(20, 4, 128, "bf16").to(gpu)
    pos = torch.arange(20, device=gpu)
    want = rope.apply(x, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = rope.apply(x, pos, stream=s)
    with torch.cuda.stream(s):
        more = rope.apply(x, pos)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(more, want)
    out = torch.zeros_like(x)
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope.apply(x, pos, out=out)
    for i in range(3):
        pos.add_(11)  # read when the graph runs
        graph.replay()
        assert torch.equal(out, rope.apply(x, pos))


def test_refusals(gpu):
    import torch
    rope = jg.Rotary(64, device=gpu)
    x, pos = torch.zeros(4, 2, 64, device=gpu), torch.arange(4, device=gpu)
    for bad in (lambda: rope.apply(x[0], pos), lambda: rope.apply(x[..., :32], pos),
                lambda: rope.apply(x.double(), pos), lambda: rope.apply(x.cpu(), pos),
                lambda: rope.apply(x, pos[:3]), lambda: rope.apply(x, pos.float()),
                lambda: rope.apply(x, pos.cpu()), lambda: rope.apply(x, torch.arange(8, device=gpu)[::2]),
                lambda: rope.apply(x, pos, out=x.half()), lambda: rope.apply(x, pos, out=x[:3]),
                lambda: rope.apply(x.transpose(1, 2), pos),
                lambda: rope.apply(x, pos, out=x[:, :1].expand(4, 2, 64)),
                lambda: rope.apply(x, _batch(gpu, [9], [3]))):
        with pytest.raises(ValueError):
            bad()
    assert rope.apply(x[:0], pos[:0]).shape == (0, 2, 64)
    assert rope.apply(x[:, :0], pos).shape == (4, 0, 64)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bits,D,rot", [(8, 128, 128), (8, 64, 32), (8, 256, 64), (4, 128, 64), (4, 64, 64),
                                        (4, 256, 256), (8, 128, 20), (4, 64, 6), (8, 256, 250)])
def test_write(gpu, bits, D, rot, interleaved, dtype):
    """Keys that write turns are held byte for byte as keys turned in float32 before, values as
    ever; what reads back is within half a step of the formula."""
    import torch
    H, page, lens, new = 3, 16, [40, 1, 0, 33, 70], [40, 1, 0, 5, 20]
    T = sum(new)
    rope = jg.Rotary(D, rot_dim=rot, interleaved=interleaved, amplitude=1.25, device=gpu)
    k, v = (_rows(T, H, D, dtype, s).to(gpu) for s in (1, 2))
    per = [-(-n // page) for n in lens]
    table = np.zeros((len(lens), max(per)), np.int32)
    table[:] = np.arange(table.size).reshape(table.shape)

    def i32(a):
        return torch.tensor(np.asarray(a, np.int32), device=gpu)
    caches = []
    for _ in range(3):
        c = jg.KVCache(table.size, page, H, D, bits=bits, device=gpu)
        c.data.fill_(0x5a)
        b = c.batch(i32(table), i32(lens), i32(np.concatenate([[0], np.cumsum(new)])), T, max(new), max(lens))
        caches.append((c, b))
    caches[0][0].write(k, v, caches[0][1], rotary=rope)
    k32 = rope.apply(k.float(), caches[1][1])
    caches[1][0].write(k32, v.float(), caches[1][1])
    assert torch.equal(caches[0][0].data, caches[1][0].data)
    # rows that start on no boundary
    odd = torch.zeros(2, T * (H * D + 3) + 1, dtype=k.dtype, device=gpu)
    ko, vo = (o[1:].view(T, H * D + 3)[:, :H * D].unflatten(1, (H, D)) for o in odd)
    ko.copy_(k), vo.copy_(v)
    caches[2][0].write(ko, vo, caches[2][1], rotary=rope)
    assert torch.equal(caches[0][0].data, caches[2][0].data)
    back, _ = caches[0][0].read(caches[0][1])
    pos = np.concatenate([np.arange(n - q, n) for n, q in zip(lens, new)])
    y, tol = ref.turn(_np(k), pos, rope.frequencies, rot, interleaved, rope.amplitude)
    top = 127 if bits == 8 else 7
    step = np.abs(y).max(-1, keepdims=True) / top
    far = tol.max(-1, keepdims=True)
    assert (np.abs(_np(back) - y) <= step * (0.5 + 2.0 ** -15) + 2 * far).all()


def test_write_of_ragged_batches(gpu):
    """The launch that numbers runs of sequences of very different lengths."""
    import torch
    new = [1] * 30 + [300]
    lens = [a + 3 * i for i, a in enumerate(new)]
    rope = jg.Rotary(64, device=gpu)
    c = [jg.KVCache(40 * 8, 64, 2, 64, device=gpu) for _ in range(2)]
    table = torch.arange(31 * 8, device=gpu, dtype=torch.int32).view(31, 8)

    def i32(a):
        return torch.tensor(np.asarray(a, np.int32), device=gpu)
    k, v = (_rows(sum(new), 2, 64, "bf16", s).to(gpu) for s in (3, 4))
    b = [x.batch(table, i32(lens), i32(np.concatenate([[0], np.cumsum(new)])), sum(new), 300, max(lens))
         for x in c]
    c[0].data.zero_(), c[1].data.zero_()
    c[0].write(k, v, b[0], rotary=rope)
    c[1].write(rope.apply(k.float(), b[1]), v.float(), b[1])
    assert torch.equal(c[0].data, c[1].data)
    with pytest.raises(ValueError):
        c[0].write(k, v, b[0], rotary=jg.Rotary(128, device=gpu))


def test_not_finite_keys(gpu):
    """A key that turns to an infinity is held as NaN, alone."""
    import torch
    rope = jg.Rotary(64, device=gpu)
    c = jg.KVCache(2, 16, 1, 64, device=gpu)
    k = _rows(3, 1, 64, "bf16").to(gpu)
    k[1, 0, 5] = float("inf")
    i = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([[0]], [3], [0, 3])]
    b = c.batch(*i, 3, 3, 3)
    c.write(k, k, b, rotary=rope)
    back, _ = c.read(b)
    assert torch.isnan(back[1]).all() and torch.isfinite(back[[0, 2]]).all()
