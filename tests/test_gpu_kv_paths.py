"""Every attention kernel that the sizes of a call can choose, on the device: rows of a key head and
contexts on both sides of each rule, many sequences, tiles in parts, within the bounds of
kv_tight."""
import numpy as np
import pytest

import kv_ref as ref
import kv_tight

import jhq_gpu_amd as jg
from test_gpu_kv import SHAPES, World, _dt, _np

pytestmark = pytest.mark.gpu


def _check(w, new, Hq, causal=True, window=0, seed=1):
    """At the usual scale, where few tokens have most of the weight, and at a twentieth, where all
    count."""
    import torch
    T = sum(new)
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(T, Hq, w.D, generator=g) * 1.5).to(_dt(w.dtype))
    k, v = w.held()
    codes = ref.held(_np(w.v), w.bits)[0]
    for scale in (w.D ** -0.5, 0.05 * w.D ** -0.5):
        lse = torch.full((T, Hq), 7.0, device=w.gpu)
        out = _np(w.cache.attend(q.to(w.gpu), w.batch(new), scale=scale, causal=causal,
                                 window=window, lse=lse))
        lse = lse.cpu().numpy()
        at = 0
        for s, (a, n) in enumerate(zip(new, w.lens)):
            sl, rows = slice(w.at[s], w.at[s] + n), slice(at, at + a)
            o, l, tol, ltol = kv_tight.attend(_np(q[rows]).astype(np.float64), k[sl], v[sl],
                                              codes[sl], scale, causal, window, ref.UNIT[w.dtype])
            err = np.abs(out[rows] - o)
            assert (err <= tol).all(), (s, a, n, (err / np.maximum(tol, 1e-300)).max())
            e = np.isinf(l)
            assert np.array_equal(lse[rows][e], l[e]) and (out[rows][e] == 0).all()
            assert (np.abs(lse[rows][~e] - l[~e]) <= ltol[~e]).all(), (s, a, n)
            at += a


@pytest.mark.parametrize("bits,D,H,page", SHAPES)
@pytest.mark.parametrize("new,G", [(1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (2, 16), (5, 3), (11, 3)])
@pytest.mark.parametrize("n", [900, 3000])
def test_rows_on_both_sides_of_the_rules(gpu, bits, D, H, page, new, G, n):
    """15 to 33 rows of a key head, short and longer contexts, idle and short sequences
    between."""
    H = min(H, 2)
    w = World(gpu, [n, 70, 0, n // 2 + 1], H, D, bits, page, "f16" if G % 2 else "bf16", seed=n + G)
    w.fill()
    _check(w, [new, 1, 0, min(new, 2)], H * G)


@pytest.mark.parametrize("bits,D", [(8, 64), (4, 64), (8, 128), (4, 128), (8, 256), (4, 256)])
@pytest.mark.parametrize("n_seq", [65, 150])
def test_more_sequences_than_lanes(gpu, bits, D, n_seq):
    """Single tokens of more sequences than a wave has lanes, some idle, over contexts that waves
    share."""
    rng = np.random.default_rng(n_seq + D)
    lens = [int(x) for x in rng.choice([0, 0, 1, 64, 200, 700, 1500], n_seq)]
    lens[-1], lens[63], lens[64] = 1300, 0, 1025
    w = World(gpu, lens, 2, D, bits, 16, "bf16", seed=n_seq)
    w.fill()
    new = [min(n, 1) for n in lens]
    _check(w, new, 8)
    _check(w, new, 8, window=333)


@pytest.mark.parametrize("bits,D,H,page", SHAPES)
@pytest.mark.parametrize("window,causal", [(700, True), (1700, True), (0, True), (0, False)])
def test_tiles_in_parts(gpu, bits, D, H, page, window, causal):
    """Chunks of many rows cut into parts, with windows that cut their tokens and without a causal
    mask."""
    w = World(gpu, [3000, 0, 1100], 1, D, bits, page, "bf16", seed=D + bits)
    w.fill()
    _check(w, [90, 0, 130], 2, causal=causal, window=window)


@pytest.mark.parametrize("D,bits,H,G,new,n,window,causal", [
    # few rows in one workgroup, up to its last step and one token past it
    (64, 8, 2, 4, 1, 900, 0, True), (128, 4, 1, 32, 1, 1024, 0, True), (256, 8, 2, 8, 2, 1000, 77, True),
    (64, 4, 1, 17, 1, 63, 0, True), (128, 8, 1, 5, 5, 129, 0, False),
    # few rows cut among the chip's waves
    (64, 8, 2, 4, 1, 1025, 0, True), (128, 8, 1, 32, 1, 5000, 0, True), (256, 4, 2, 16, 1, 70001, 0, True),
    (64, 4, 3, 11, 2, 70001, 0, True), (128, 4, 2, 4, 8, 30000, 9001, True), (64, 8, 1, 7, 3, 4000, 0, False),
    # many rows, in one part and in several
    (128, 8, 1, 1, 40, 500, 0, True), (256, 4, 2, 2, 150, 3000, 1700, True), (64, 8, 1, 4, 130, 9000, 0, False),
    # parts of 4096 tokens, where the last round of workgroups would be part empty
    (128, 8, 4, 16, 600, 20000, 0, True),
    (128, 8, 4, 16, 600, 20000, 0, False),
    (128, 4, 4, 16, 600, 20000, 9000, True),
    (256, 8, 2, 8, 700, 21000, 0, True),
    (64, 4, 4, 16, 900, 13000, 0, True),
])
def test_every_step_counts_once(gpu, D, bits, H, G, new, n, window, causal):
    """With scale 0 all weights are alike: each step of 64 tokens has a value of its own, so that
    a step or a part that is left out or counted twice shows in its element.

    Bound: weights 1 are exact, their sums of at most 2^20 too; one division and the rounding of the
    result, and half a unit of the log-sum-exp's float32."""
    import torch
    c = jg.KVCache(-(-n // 64), 64, H, D, bits=bits, device=gpu)
    step = np.arange(n) // 64 % D
    v = np.zeros((n, D), np.float32)
    v[np.arange(n), step] = 1
    vt = torch.from_numpy(v).half().to(gpu)[:, None].expand(n, H, D)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    pages = torch.randperm(c.num_pages, generator=torch.Generator().manual_seed(1)).int()[None]
    pages = pages.to(gpu)
    c.write(torch.ones_like(vt), vt, c.batch(pages, i32([n]), i32([0, n]), n, n, n))
    q = torch.randn(new, H * G, D, generator=torch.Generator().manual_seed(2)).half().to(gpu)
    lse = torch.zeros(new, H * G, device=gpu)
    out = _np(c.attend(q, c.batch(pages, i32([n]), i32([0, new]), new, new, n), scale=0.0,
                       causal=causal, window=window, lse=lse))
    hi = np.arange(n - new, n) + 1 if causal else np.full(new, n)
    lo = np.maximum(0, hi - window) if window else np.zeros_like(hi)
    upto = np.concatenate([np.zeros((1, D)), np.cumsum(v, 0, dtype=np.float64)])
    want = ((upto[hi] - upto[lo]) / (hi - lo)[:, None])[:, None]
    assert (np.abs(out - want) <= want * (2.0 ** -11 + 2.0 ** -20) + 2.0 ** -25).all()
    assert (np.abs(lse.cpu().numpy() - np.log(hi - lo)[:, None]) <= 1e-5).all()
