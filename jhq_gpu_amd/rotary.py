"""Rotary positions on queries and keys (jhq_k_rotary of include/jhq.h; no counterpart in
the reference).

    rope = Rotary(128, base=500000.0)
    q = rope.apply(q, batch)                 # the batch's new tokens, before attend
    cache.write(k, v, batch, rotary=rope)    # keys turn on their way into the cache
"""
import ctypes
import math
import operator

import jhq_gpu_amd as _jg

from . import kv as _kv

__all__ = ["Rotary"]

_DTYPES, _POSITIONS = {}, {}  # element types, and the bytes of positions' types; filled with the first Rotary

_PER_TURN = 0x28BE60DB9391054A7F09D5F47D4D3770  # 2^128 / (2 pi)

_KINDS = {"linear": ("factor",), "ntk": ("factor",), "yarn": ("factor", "length", "fast", "slow"),
          "bands": ("factor", "length", "low", "high")}


def _scaled(rot_dim, base, scaling):
    """Radians a position of each pair, and the amplitude."""
    pairs = range(rot_dim // 2)
    if scaling is None:
        return [base ** (-2.0 * i / rot_dim) for i in pairs], 1.0
    s = dict(scaling)
    kind = s.pop("kind", None)
    if kind not in _KINDS:
        raise ValueError(f"scaling kind must be one of {', '.join(_KINDS)}, got {kind!r}")
    for name in s:
        if name not in _KINDS[kind]:
            raise ValueError(f"scaling {kind} has no {name}")
    for name in ("factor", "length"):
        if name in _KINDS[kind] and name not in s:
            raise ValueError(f"scaling {kind} needs {name}")
    s = {k: float(v) for k, v in s.items()}
    for name, v in s.items():
        if not (math.isfinite(v) and v > 0):
            raise ValueError(f"scaling {name} must be positive, got {v}")
    f = s["factor"]
    if kind == "ntk":
        if rot_dim == 2:
            raise ValueError("scaling ntk needs rot_dim > 2")
        base = base * f ** (rot_dim / (rot_dim - 2.0))
        if not math.isfinite(base):
            raise OverflowError
    w = [base ** (-2.0 * i / rot_dim) for i in pairs]
    if kind == "ntk":
        return w, 1.0
    if kind == "linear":
        return [x / f for x in w], 1.0
    if kind == "bands":
        # pairs that turn less than `low` times within `length` are slowed, those above
        # `high` not, the ones between in part
        low, high = s.get("low", 1.0), s.get("high", 4.0)
        if low >= high:
            raise ValueError(f"scaling low must be below high, got {low} and {high}")
        mix = [min(1.0, max(0.0, (s["length"] * x / (2 * math.pi) - low) / (high - low))) for x in w]
        return [x * (m + (1.0 - m) / f) for x, m in zip(w, mix)], 1.0
    # yarn: the same by a pair's number, between those that turn `fast` and `slow` times
    if base == 1.0:
        raise ValueError("scaling yarn needs a base other than 1")
    fast, slow = s.get("fast", 32.0), s.get("slow", 1.0)
    if fast <= slow:
        raise ValueError(f"scaling fast must be above slow, got {fast} and {slow}")

    def place(turns):
        return rot_dim * math.log(s["length"] / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo = max(math.floor(place(fast)), 0)
    hi = min(math.ceil(place(slow)), rot_dim - 1)
    mix = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in pairs]
    return ([x * (1.0 - m + m / f) for x, m in zip(w, mix)],
            0.1 * math.log(f) + 1.0 if f > 1.0 else 1.0)


class Rotary:
    """Turns pairs of a head's first rot_dim elements (default: all) by their
    token's position: pair i by base ** (-2 i / rot_dim) radians a position.  Pairs are
    (i, i + rot_dim / 2) or, interleaved, (2 i, 2 i + 1); head_dim is even, up to 1024.

    scaling stretches the frequencies for contexts longer than the model's:
      dict(kind="linear", factor=)              all of them by factor
      dict(kind="ntk", factor=)                 the base by factor ** (rot_dim / (rot_dim - 2))
      dict(kind="yarn", factor=, length=, fast=32, slow=1)   a ramp over the pairs between those
          that turn fast and slow times within length; amplitude 0.1 ln factor + 1
      dict(kind="bands", factor=, length=, low=1, high=4)    a ramp over the turns within length
    frequencies: rot_dim / 2 radians a position instead of base and scaling.
    amplitude: what turned pairs are multiplied by (default 1, yarn's its own).

    Frequencies are held as 64-bit parts of a turn, so that angles are as exact at
    position 2^30 as at 1."""

    def __init__(self, head_dim, rot_dim=None, base=10000.0, interleaved=False, scaling=None,
                 frequencies=None, amplitude=None, device="cuda"):
        head_dim = operator.index(head_dim)
        rot_dim = head_dim if rot_dim is None else operator.index(rot_dim)
        if head_dim < 2 or head_dim > 1024 or head_dim % 2:
            raise ValueError(f"head_dim must be even, 2 .. 1024, got {head_dim}")
        if rot_dim < 2 or rot_dim > head_dim or rot_dim % 2:
            raise ValueError(f"rot_dim must be even, 2 .. head_dim, got {rot_dim}")
        base = float(base)
        if not (math.isfinite(base) and base > 0):
            raise ValueError(f"base must be positive, got {base}")
        if frequencies is None:
            try:
                freq, amp = _scaled(rot_dim, base, scaling)
            except OverflowError:
                raise ValueError(f"frequencies of base {base} and scaling {scaling} pass float64's range") from None
        else:
            if scaling is not None:
                raise ValueError("frequencies are given: scaling does not apply")
            freq, amp = [float(x) for x in frequencies], 1.0
            if len(freq) != rot_dim // 2:
                raise ValueError(f"frequencies must be {rot_dim // 2}, got {len(freq)}")
        if not all(math.isfinite(x) for x in freq):
            raise ValueError("frequencies must be finite")
        amp = amp if amplitude is None else float(amplitude)
        if not math.isfinite(amp) or abs(amp) > 3.0e38:
            raise ValueError(f"amplitude must be a finite float32, got {amp}")
        torch = _kv._torch()
        if torch.device(device).type != "cuda":
            raise ValueError(f"the rotary must be on a GPU, not on {device}")
        self.head_dim, self.rot_dim, self.interleaved = head_dim, rot_dim, bool(interleaved)
        self.frequencies, self.amplitude = freq, amp
        self._turns = torch.tensor(turns(freq), dtype=torch.int64, device=device)
        self.device = self._turns.device
        self._index = self.device.index
        self._c = _jg._Rotary(head_dim, rot_dim, 1 if interleaved else 0, amp, self._turns.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._entry = _jg.lib().jhq_k_rotary
        self._current, self._device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        _DTYPES.update(_kv._DTYPES)
        _POSITIONS.update({torch.int32: 4, torch.int64: 8})

    def apply(self, x, positions, inverse=False, out=None, stream=None):
        """Turns x [n_tokens, heads, head_dim] (float32, bfloat16 or float16, any strides
        between rows) to `positions`: an int32 or int64 tensor [n_tokens], or a KVBatch,
        whose new tokens' positions they are (rows that no sequence has keep what out
        had, zero where out is None).  Computed in float32 and rounded once.  out: a tensor
        of x's shape and type, x itself among them; it must not share memory with x
        otherwise.  inverse turns back: the gradient's pass, which is the caller's to run, as
        autograd does not record the call (a result that it allocates requires no gradient)."""
        n, heads, xt, xh = self._rows(x, "x")
        dt = _DTYPES.get(x.dtype)
        if dt is None:
            dt = _kv._dtype(x.dtype, "x")
        if type(positions) is _kv.KVBatch:
            if positions._index != self._index:
                raise ValueError(f"the batch is on cuda:{positions._index}, the rotary on {self.device}")
            if positions.moved:
                raise ValueError(_kv._MOVED)
            if positions.n_tokens != n:
                raise ValueError(f"the batch has {positions.n_tokens} rows, x {n}")
            pp, size, ref = None, 0, positions._ref
        else:
            size, ref = _POSITIONS.get(positions.dtype), None
            if size is None or positions.dim() != 1 or positions.shape[0] != n \
                    or not positions.is_contiguous():
                raise ValueError(f"positions must be a contiguous int32 or int64 [{n}] tensor")
            if positions.get_device() != self._index:
                raise ValueError(f"positions are on {positions.device}, the rotary on {self.device}")
            pp = positions.data_ptr()
        if out is None:
            torch = _kv._torch()
            new = torch.empty if ref is None else torch.zeros
            with torch.cuda.stream(_kv._as_stream(stream, self.device)):
                out = new((n, heads, self.head_dim), dtype=x.dtype, device=self.device)
            ot, oh = heads * self.head_dim, self.head_dim
        elif out is x:
            ot, oh = xt, xh
        else:
            on, oheads, ot, oh = self._rows(out, "out")
            if on != n or oheads != heads or out.dtype != x.dtype:
                raise ValueError(f"out must be of x's shape and type, got {tuple(out.shape)} {out.dtype}")
        if n == 0 or heads == 0:
            return out
        if (ot == 0 and n > 1) or (oh == 0 and heads > 1):
            raise ValueError("out must not have rows that share memory")
        if self._device() != self._index:  # kernels are launched on the current device
            with _kv._torch().cuda.device(self._index):
                return self.apply(x, positions, inverse, out, stream)
        if stream is None:
            s = self._current(self._index)
        else:
            s = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
        rc = self._entry(self._ref, x.data_ptr(), xt, xh, n, heads, dt, pp, size, ref, 1 if inverse else 0,
                         out.data_ptr(), ot, oh, s)
        if rc:
            _jg._check(rc)
        return out

    def _rows(self, x, what):
        """Rows, heads and strides of a [n_tokens, heads, head_dim] tensor."""
        if x.dim() != 3 or x.shape[2] != self.head_dim:
            raise ValueError(f"{what} must be [n_tokens, heads, {self.head_dim}], got {tuple(x.shape)}")
        if x.get_device() != self._index:
            raise ValueError(f"{what} is on {x.device}, the rotary on {self.device}")
        n, heads, _ = x.shape
        tok, head, el = x.stride()
        if el != 1:
            raise ValueError(f"{what}: the elements of a row must be contiguous")
        return n, heads, tok, head


def turns(frequencies):
    """Radians a position as 2^-64ths of a turn modulo one turn, in int64."""
    out = []
    for x in frequencies:
        m, e = math.frexp(x)  # x = m 2^e, 53 bits of m
        n, down = int(m * (1 << 53)) * _PER_TURN, 64 + 53 - e
        n = (n + (1 << down - 1) >> down if down > 0 else n << -down) % (1 << 64)
        out.append(n - (1 << 64) if n >= 1 << 63 else n)
    return out
