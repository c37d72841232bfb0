"""Pages, positions, cache and attention as a serving program runs them: answers are sampled side by side
from one prompt, tokens are dropped, sequences end and begin; every output against float64."""
import numpy as np
import pytest

import kv_ref as ref
import rotary_ref as rot

import jhq_gpu_amd as jg

pytestmark = pytest.mark.gpu


def _f64(t):
    return t.double().cpu().numpy()


class Server:
    """Sequences of rows, as the cache should hold them, beside the cache."""

    def __init__(self, gpu, bits, D, H, G, page, n_seq, dtype, rope, seed):
        import torch
        self.gpu, self.bits, self.D, self.H, self.G, self.rope = gpu, bits, D, H, G, rope
        self.dtype = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
        self.unit = ref.UNIT[dtype]
        self.cache = jg.KVCache(600, page, H, D, bits=bits, device=gpu)
        self.cache.data.fill_(0xff)
        self.pages = jg.KVPages(self.cache, n_seq, 4000)
        self.held = [[np.zeros((0, H, D)), np.zeros((0, H, D))] for _ in range(n_seq)]
        self.pos = [0] * n_seq  # tokens that a sequence has had: compaction keeps positions
        self.gen = torch.Generator().manual_seed(seed)

    def step(self, new, once):
        """A layer's step: q, k and v come out of one projection.  Returns how many groups share."""
        import torch
        T, H, G, D = sum(new), self.H, self.G, self.D
        x = torch.randn(T, H * G + 2 * H, D, generator=self.gen).to(self.dtype)
        fused = x.to(self.gpu)
        b = self.pages.extend(new)
        q, k, v = fused[:, :H * G], fused[:, H * G:H * G + H], fused[:, H * G + H:]
        pos = np.concatenate([np.arange(self.pos[s], self.pos[s] + a) for s, a in enumerate(new)])
        at = torch.from_numpy(pos.astype(np.int64)).to(self.gpu)
        moved = any(self.pages.length(s) != self.pos[s] + a for s, a in enumerate(new) if a)
        if moved:  # positions of their own where tokens have been dropped
            self.rope.apply(fused[:, :H * G + H], at, out=fused[:, :H * G + H])
            self.cache.write(k, v, b)
        else:
            self.cache.write(k, v, b, rotary=self.rope)
            self.rope.apply(q, b, out=q)
        prefix = self.pages.prefix()
        out = self.cache.attend(q, b, prefix=prefix, once=once)
        turned = _f64(q)
        want, tol = rot.turn(_f64(x[:, :H * G]), pos, self.rope.frequencies, self.rope.rot_dim,
                             self.rope.interleaved, self.rope.amplitude, False, self.unit)
        assert (np.abs(turned - want) <= tol).all()
        # what the cache holds of the new tokens is read back: codes may differ where a turned
        # key stands within float32's rounding of the middle between two
        kr, vr = self.cache.read(b)
        kw, ktol = rot.turn(_f64(x[:, H * G:H * G + H]), pos, self.rope.frequencies, self.rope.rot_dim,
                            self.rope.interleaved, self.rope.amplitude, False, self.unit if moved else 0.0)
        top = 127 if self.bits == 8 else 7
        step = np.abs(kw).max(-1, keepdims=True) / top
        assert (np.abs(_f64(kr) - kw) <= step * (0.5 + 2.0 ** -15) + 2 * ktol.max(-1, keepdims=True)).all()
        assert np.array_equal(vr.cpu().numpy(), ref.value32(x[:, H * G + H:].float().numpy(), self.bits))
        row = 0
        for s, a in enumerate(new):
            for z, y in enumerate((kr, vr)):
                self.held[s][z] = np.concatenate([self.held[s][z], _f64(y[row:row + a])])
            self.pos[s] += a
            if a:
                o, _, t, _ = ref.attend(turned[row:row + a], *self.held[s], D ** -0.5, unit=self.unit)
                assert (np.abs(_f64(out[row:row + a]) - o) <= t).all(), (s, a)
            row += a
        return 0 if prefix is None else int((prefix.kv_len > 0).sum())

    def fork(self, a, b):
        self.pages.fork(a, b)
        self.held[b], self.pos[b] = list(self.held[a]), self.pos[a]

    def compact(self, keep):
        self.pages.compact(keep)
        for s, at in keep.items():
            self.held[s] = [x[at] for x in self.held[s]]

    def free(self, s):
        self.pages.free(s)
        self.held[s] = [x[:0] for x in self.held[s]]
        self.pos[s] = 0


@pytest.mark.parametrize("once", [True, False])
@pytest.mark.parametrize("bits,D,H,G,page,dtype,kw", [
    (8, 128, 2, 4, 64, "bf16", dict()),
    (4, 64, 3, 2, 16, "f16", dict(interleaved=True, scaling=dict(kind="bands", factor=4, length=256))),
    (8, 256, 1, 8, 32, "bf16", dict(rot_dim=64, scaling=dict(kind="yarn", factor=8, length=128))),
])
def test_answers_side_by_side(gpu, bits, D, H, G, page, dtype, kw, once):
    rng = np.random.default_rng(D)
    w = Server(gpu, bits, D, H, G, page, 8, dtype, jg.Rotary(D, device=gpu, **kw), seed=D + bits)
    assert w.step([300, 0, 0, 0, 150, 0, 0, 0], once) == 0  # two prompts
    for s in (1, 2, 3):
        w.fork(0, s)
    w.fork(4, 5)
    for _ in range(3):
        assert w.step([1, 1, 1, 1, 1, 1, 0, 0], once) == 2
    assert w.step([2, 5, 1, 3, 0, 1, 0, 0], once) == 1  # proposed tokens, of different numbers
    w.free(2)
    keep = np.sort(rng.choice(w.pages.length(1), 180, replace=False))
    w.compact({1: keep, 5: np.arange(100, w.pages.length(5))})
    w.fork(3, 2)
    # a prompt beside single tokens; a question of some length beside them
    assert w.step([1, 1, 1, 1, 1, 1, 40, 0], once) >= 1
    assert w.step([1, 1, 17, 30, 1, 1, 1, 0], once) >= 1
    for s in range(8):
        w.free(s)
    assert w.pages.free_pages == 600
