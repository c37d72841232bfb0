"""examples/retrieve_attend.py: retrieval, cache and attention together; every output
against attention over the held values in float64 (kv_ref)."""
import importlib.util
import os

import numpy as np
import pytest

import kv_ref as ref

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("bits", [8, 4])
def test_retrieve_attend(gpu, bits):
    spec = importlib.util.spec_from_file_location(
        "retrieve_attend", os.path.join(ROOT, "examples", "retrieve_attend.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    r = ex.run(str(gpu), bits=bits, generate=3)
    assert (r["ids"] >= 0).all()
    for step in r["steps"]:
        at = 0
        for s, (a, n) in enumerate(zip(step["new"], step["length"])):
            k, v = (ref.value32(x[s][:n].float().numpy(), bits).astype(np.float64)
                    for x in (r["k"], r["v"]))
            q = step["q"][at:at + a].float().numpy().astype(np.float64)
            o, _, tol, _ = ref.attend(q, k, v, q.shape[2] ** -0.5, unit=ref.UNIT["bf16"])
            assert (np.abs(step["out"][at:at + a].float().numpy() - o) <= tol).all()
            at += a
