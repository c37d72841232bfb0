"""The quantised key/value cache on the device at the edges of its ranges: scores
that are not finite."""
import numpy as np
import pytest

import kv_ref as ref

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
