"""The quantised key/value cache on the device with batches whose sequences differ much:
bounds far above most lengths, a long chunk beside single tokens, many idle slots."""
import numpy as np
import pytest

import kv_ref as ref

import jhq_gpu_amd as jg
from test_gpu_kv import World, _check, _np

pytestmark = pytest.mark.gpu


def test_attend_within_wide_bounds(gpu):
    """128 sequences with 512 new tokens in all, whose bounds allow 8192 each over 16384 (as a
    captured call's do): the call is sized by its rows, and its results are those of tight
    bounds within both runs' roundings."""
    import torch
    rng = np.random.default_rng(4)
    new = [int(x) for x in rng.integers(0, 8, 128)]
    new[5], new[77] = 0, 40
    while sum(new) > 512:
        new[int(rng.integers(128))] = 0
    lens = [q + int(x) for q, x in zip(new, rng.integers(0, 60, 128))]
    w = World(gpu, lens, 8, 128, 8, 64, "bf16", seed=4)
    w.fill()
    table = np.full((128, 16384 // 64), -1, np.int32)
    table[:, :w.table.shape[1]] = w.table
    b = w.cache.batch(w.i32(table), w.i32(lens), w.i32(np.concatenate([[0], np.cumsum(new)])), 512,
                      8192, 16384)
    q = torch.randn(512, 64, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    lse = torch.full((512, 64), 7.0, device=gpu)
    out = _np(w.cache.attend(q.to(gpu), b, lse=lse))
    lse = lse.cpu().numpy()
    k, v = w.held()
    at = 0
    for s, (a, n) in enumerate(zip(new, lens)):
        sl = slice(w.at[s], w.at[s] + n)
        o, l, tol, ltol = ref.attend(_np(q[at:at + a]).astype(np.float64), k[sl], v[sl], 128 ** -0.5,
                                     unit=ref.UNIT["bf16"])
        assert (np.abs(out[at:at + a] - o) <= tol).all(), s
        assert (np.abs(lse[at:at + a] - l) <= ltol).all(), s
        at += a
    assert not out[at:].any() and (lse[at:] == 7.0).all()  # rows of no sequence


@pytest.mark.parametrize("n_seq", [3, 71, 4200])
@pytest.mark.parametrize("D,bits,G", [(64, 8, 3), (128, 4, 4), (256, 8, 2)])
@pytest.mark.parametrize("chunk", [1, 9, 150])
def test_one_chunk_beside_single_tokens(gpu, n_seq, D, bits, G, chunk):
    """A chunk over a longer context beside single tokens and idle slots, more of them than
    the waves of a search look at in one round, in two and in three; at the lowest count the
    chunk's tokens are split into parts."""
    rng = np.random.default_rng(n_seq + chunk)
    new = [int(x) for x in rng.random(n_seq) < 60 / n_seq]
    lens = [q and int(x) for q, x in zip(new, rng.integers(1, 40, n_seq))]
    for at, n in ((n_seq // 2, 2300), (n_seq - 1, 1100)):
        new[at], lens[at] = chunk, n
    new[0] = lens[0] = 0
    w = World(gpu, lens, 1, D, bits, 16, "f16", seed=n_seq)
    w.fill()
    _check(w, new, G)


@pytest.mark.parametrize("bits,D,page", [(8, 128, 64), (4, 64, 16), (4, 128, 32)])
@pytest.mark.parametrize("n_seq,chunk", [(3, 700), (130, 3000), (1024, 32768), (4200, 500)])
def test_one_prompt_beside_single_tokens_in_and_back(gpu, bits, D, page, n_seq, chunk):
    """A prompt beside single tokens and idle slots, written in two steps (the first ends inside
    a group) and read back: equal to the definition's bit for bit, whatever the lengths."""
    import torch
    H = 8 if n_seq == 1024 else 2
    rng = np.random.default_rng(n_seq)
    lens = [int(x) for x in rng.choice([0, 1, 1, 1, 17], n_seq)]
    lens[n_seq // 3], lens[0], lens[-1] = chunk, 0, 33
    w = World(gpu, lens, H, D, bits, page, "bf16", seed=n_seq)
    k, v = w.k.to(gpu), w.v.to(gpu)
    first = [n - 1 if n > 1 else 0 for n in lens]
    for new, have in ((first, first), ([n - f for n, f in zip(lens, first)], lens)):
        r = torch.from_numpy(w.rows(new, have)).to(gpu)
        w.cache.write(k[r], v[r], w.batch(new, have))
    got = w.cache.read(w.batch(lens))
    for a, x in zip(got, (w.k, w.v)):
        assert np.array_equal(_np(a), ref.value32(_np(x), bits))
    # the last 20 tokens at most of each alone, into rows that begin past the first
    tail = [min(n, 20) for n in lens]
    cu = np.concatenate([[0], np.cumsum(tail)]) + 5
    b = w.cache.batch(w.i32(w.table), w.i32(lens), w.i32(cu), int(cu[-1]) + 3, chunk, chunk)
    a, _ = w.cache.read(b)
    assert np.array_equal(_np(a)[5:-3], ref.value32(_np(w.k), bits)[w.rows(tail)])
    assert not a[:5].any() and not a[-3:].any()


def test_wide_bounds_in_and_back(gpu):
    """256 sequences whose bounds allow 131072 new tokens each, with some 640 in all."""
    rng = np.random.default_rng(1)
    lens = [int(x) for x in rng.integers(0, 6, 256)]
    w = World(gpu, lens, 8, 128, 8, 64, "bf16", seed=2)
    table = np.full((256, 131072 // 64), -1, np.int32)
    table[:, :w.table.shape[1]] = w.table
    b = w.cache.batch(w.i32(table), w.i32(lens), w.i32(np.concatenate([[0], np.cumsum(lens)])),
                      sum(lens), 131072, 131072)
    w.cache.write(w.k.to(gpu), w.v.to(gpu), b)
    k, v = w.cache.read(b)
    assert np.array_equal(_np(k), ref.value32(_np(w.k), 8))
    assert np.array_equal(_np(v), ref.value32(_np(w.v), 8))


def test_few_sequences_in_long_arrays(gpu):
    """Single tokens whose rows are the first of arrays of 2^18: the call is sized by the
    sequences, and the other rows keep what they had."""
    import torch
    w = World(gpu, [1200] * 6, 2, 256, 8, 64, "bf16", seed=3)
    w.fill()
    q = torch.randn(6, 32, 256, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    want = w.cache.attend(q, w.batch([1] * 6))
    T = 1 << 18
    long = torch.zeros(T, 32, 256, dtype=torch.bfloat16, device=gpu)
    long[3:9] = q
    cu = w.i32(np.arange(7) + 3)
    b = w.cache.batch(w.i32(w.table), w.i32(w.lens), cu, T, 1, 1200)
    out = torch.full_like(long, 5.0)
    w.cache.attend(long, b, out=out)
    assert torch.equal(out[3:9], want)
    assert (out[:3] == 5).all() and (out[9:] == 5).all()
    k = torch.ones(T, 2, 256, dtype=torch.bfloat16, device=gpu)
    w.cache.write(k, k, b)
    got = torch.zeros_like(k), torch.zeros_like(k)
    w.cache.read(b, k_out=got[0], v_out=got[1])
    for x in got:
        assert (x[3:9] == 1).all() and not x[:3].any() and not x[9:].any()
