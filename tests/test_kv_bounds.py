"""The bounds that the device's attention is held to (kv_tight), on the CPU: a step of 64 tokens whose
values are missing, or counted twice, is outside of them wherever it stands."""
import numpy as np
import pytest

import kv_ref as ref
import kv_tight


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n,D", [(900, 64), (3000, 128), (3000, 256)])
def test_a_missing_or_doubled_step_is_out_of_bounds(n, D, bits):
    rng = np.random.default_rng(n + D)
    size = np.exp(rng.standard_normal((n, 1, 1)))
    k, v = (np.float16(rng.standard_normal((n, 1, D)) * s) for s in (size, size[::-1]))
    k = ref.value32(k, bits).astype(np.float64)
    codes, scale = ref.held(v, bits)
    v = codes.astype(np.float64) * scale
    q = np.float64(np.float16(rng.standard_normal((2, 2, D)) * 1.5))
    o, _, tol, _ = kv_tight.attend(q, k, v, codes, 0.05 * D ** -0.5, unit=ref.UNIT["bf16"])
    assert (tol <= ref.attend(q, k, v, 0.05 * D ** -0.5, unit=ref.UNIT["bf16"])[2]).all()
    for a in range(0, n, 64):
        for f in (0, 2):
            x = v.copy()
            x[a:a + 64] *= f
            wrong = ref.attend(q, k, x, 0.05 * D ** -0.5)[0]
            assert (np.abs(wrong - o) > tol).any(-1).all(), (a, f)
