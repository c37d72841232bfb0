"""The quantised key/value cache on the device at the edges of its ranges: scores
that are not finite, weights far below the largest."""
import numpy as np
import pytest

import kv_ref as ref

import jhq_gpu_amd as jg

from test_gpu_kv import World, _np

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 100, 1100, 3000])
@pytest.mark.parametrize("new", [1, 9, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kind", ["infinite", "overflow"])
def test_rows_whose_every_score_is_minus_infinity(gpu, n, new, D, kind):
    """An infinite query element against keys of the other sign, and a finite one whose
    scores pass float32's range: softmax is 0 / 0, which is not what a row gets that sees
    nothing.  The rows beside it stay within their own bounds."""
    import torch
    new = min(new, n)
    w = World(gpu, [n], 1, D, 8, 16, "bf16", seed=D + n)
    w.k[:, :, 0] = w.k[:, :, 0].abs() + 100  # a channel with a constant offset
    w.k[:, :, 1:] = w.k[:, :, 1:].clamp(-2, 2)
    w.fill()
    q = torch.randn(new, 4, D, generator=torch.Generator().manual_seed(n)).bfloat16()
    hit = (new // 2, 1)
    q[hit] = 0
    q[hit][0] = float("-inf") if kind == "infinite" else -3e38
    lse = torch.zeros(new, 4, device=gpu)
    out = _np(w.cache.attend(q.to(gpu), w.batch([new]), lse=lse))
    lse = lse.cpu().numpy()
    assert np.isnan(out[hit]).all() and np.isnan(lse[hit])
    k, v = w.held()
    q[hit] = 0
    o, l, tol, ltol = ref.attend(_np(q).astype(np.float64), k, v, D ** -0.5, unit=ref.UNIT["bf16"])
    others = np.ones((new, 4), bool)
    others[hit] = False
    assert (np.abs(out - o) <= tol)[others].all()
    assert (np.abs(lse - l) <= ltol)[others].all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n,new,H,G", [(900, 1, 1, 1), (1 << 20, 1, 1, 1), (131073, 40, 1, 1),
                                       (131073, 1024, 4, 16)])  # the last: no parts
@pytest.mark.parametrize("low", [25.1, 24.2, 28.3])
def test_many_small_weights_beside_a_large_one(gpu, bits, n, new, H, G, low):
    """One token of weight 1, all others 2^-low: together they are up to some percent of the
    output, and all of it in the element that the one token's value does not have.

    Bound: weights are rounded to 2^-11 of themselves or to 2^-34 of the largest, the result
    to 2^-11, logits (of magnitude low ln 2) are off by (D + 8) 2^-24 of it, and of the
    sums of weights and values, which are kept in 4 and in 2 places a row, an addition is off by
    2^-24 at most."""
    import torch
    D, page = 64, 1024
    c = jg.KVCache(-(-n // page), page, H, D, bits=bits, device=gpu)
    k = torch.zeros(n, H, D, dtype=torch.float16, device=gpu)
    v = torch.zeros_like(k)
    k[..., 1], v[..., 0] = 1, 1
    hot = n // 3
    k[hot, :, 0], k[hot, :, 1], v[hot, :, 0], v[hot, :, 1] = 1, 0, 0, 1
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    pages = torch.arange(c.num_pages, dtype=torch.int32, device=gpu)[None]
    c.write(k, v, c.batch(pages, i32([n]), i32([0, n]), n, n, n))
    q = torch.zeros(new, H * G, D, dtype=torch.float16, device=gpu)
    q[..., 0] = 1
    scale = low * np.log(2)
    out = _np(c.attend(q, c.batch(pages, i32([n]), i32([0, new]), new, new, n), scale=scale))
    w = 2.0 ** -low
    small = (np.arange(n - new, n)[:, None]) * w  # all that are seen but one
    want = np.concatenate([small / (1 + small), 1 / (1 + small)], 1)
    rel = (2.0 ** -11 + max(2.0 ** -11, 2.0 ** -34 / w) + 2 * scale * (D + 8) * 2.0 ** -24
           + (n / 4 + n / 2) * 2.0 ** -24)
    want = np.repeat(want[:, None], H * G, 1)
    err = np.abs(out[..., :2] - want)
    assert (err <= rel * want + 2.0 ** -25).all(), (err / want).max() / rel  # float16's smallest
    assert not out[..., 2:].any()


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32, 2 ** 32 + 16, 2 ** 70, np.int64(2 ** 32 + 16)])
def test_windows_past_32_bits(gpu, new, window):
    """They hide nothing, whatever their lower bits say; negative ones are refused likewise."""
    import torch
    w = World(gpu, [300], 2, 64, 8, 16, "bf16", seed=6)
    w.fill()
    q = torch.randn(new, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(gpu)
    b = w.batch([new])
    assert torch.equal(w.cache.attend(q, b, window=window), w.cache.attend(q, b))
    assert w.cache.work_bytes(b, 4, window) == w.cache.work_bytes(b, 4, 1 << 30)
    for bad in (-window, 16 - 2 ** 32):
        with pytest.raises(ValueError, match="window"):
            w.cache.attend(q, b, window=bad)
        with pytest.raises(ValueError, match="window"):
            w.cache.work_bytes(b, 4, bad)


@pytest.mark.parametrize("D", [64, 256])
def test_log_sum_exp_of_single_tokens(gpu, D):
    """Rows that see one token: the log-sum-exp is the score, within kv_ref's bound for small
    ones."""
    import torch
    w = World(gpu, [1] * 300, 2, D, 8, 16, "bf16", seed=D)
    w.fill()
    q = (torch.randn(300, 16, D, generator=torch.Generator().manual_seed(5)) * 1.5).bfloat16()
    lse = torch.zeros(300, 16, device=gpu)
    w.cache.attend(q.to(gpu), w.batch([1] * 300), scale=0.05 * D ** -0.5, lse=lse)
    lse = lse.cpu().numpy()
    k, v = w.held()
    qq = _np(q).astype(np.float64)
    for s in range(300):
        _, want, _, tol = ref.attend(qq[s:s + 1], k[s:s + 1], v[s:s + 1], 0.05 * D ** -0.5)
        assert (np.abs(lse[s] - want[0]) <= tol[0]).all(), s
