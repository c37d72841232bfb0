"""Key/value cache of attention, held in 8 or 4 bits on the device (jhq_k_kv_*
of include/jhq.h; no counterpart in the reference).

A cache is a buffer of pages; which pages hold which sequence is the caller's
page table, and a ``KVBatch`` says what one call works on.  Everything is torch
device tensors, calls only enqueue work, on the current stream or the given one.
It is a store for serving: no gradient passes through write, read or attend, and
what they return never requires one, whatever the inputs do.

    cache = KVCache(num_pages=4096, page_size=64, kv_heads=8, head_dim=128, bits=8)
    batch = cache.batch(pages, kv_len, cu_q, n_tokens, max_q, max_kv)
    cache.write(k, v, batch)          # the batch's new tokens enter the cache
    out = cache.attend(q, batch)      # and attend to their sequences
"""
import ctypes
import math
import operator

import jhq_gpu_amd as _jg

__all__ = ["KVCache", "KVBatch"]

JHQ_BF16, JHQ_F16 = 3, 4


_MOVED = ("tokens of the batch's sequences have been moved (KVPages.compact), so that new ones' places are not their "
          "positions: turn them with Rotary.apply and a tensor of positions")

_DTYPES = {}  # torch type -> element type, filled when torch is first needed


def _torch():
    import torch
    if not _DTYPES:
        _DTYPES.update({torch.float32: _jg.JHQ_F32, torch.bfloat16: JHQ_BF16,
                        torch.float16: JHQ_F16})
    return torch


def _dtype(t, what):
    dt = _DTYPES.get(t)
    if dt is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t}")
    return dt


def _int32(v, what):
    """v as an int, refused where ctypes would cut it to its lower 32 bits."""
    v = int(v)
    if not -1 << 31 <= v < 1 << 31:
        raise ValueError(f"{what} is out of range: {v}")
    return v


def _window(window):
    """A window as the C entry points take it: an int, where one past 2^30, which hides
    nothing, is cut to it (ctypes would take it modulo 2^32)."""
    window = operator.index(window)
    if window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    return min(window, 1 << 30)


class KVBatch:
    """The sequences that a call works on (jhq_kv_batch).

    pages [n_seq, max_pages] int32, kv_len [n_seq] int32 and cu_q [n_seq + 1]
    int32 are device tensors that are read when the kernels run: they may be
    updated in place from one call to the next.  Sequence b has kv_len[b]
    tokens, token j in page pages[b, j // page_size]; its last
    cu_q[b+1] - cu_q[b] tokens are new, rows cu_q[b] .. of k, v and q.
    n_tokens rows in all; max_q and max_kv bound one sequence's new tokens and
    tokens.  Build it with KVCache.batch.

    moved: whether a sequence holds its tokens elsewhere than at their positions
    (KVPages.compact has moved them), so that nothing is turned to the batch's positions."""

    moved = False

    def __init__(self, device, page_size, pages, kv_len, cu_q, n_tokens, max_q, max_kv):
        torch = _torch()
        for name, t, nd in (("pages", pages, 2), ("kv_len", kv_len, 1), ("cu_q", cu_q, 1)):
            if t.dtype != torch.int32 or t.dim() != nd or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {nd}-d int32 tensor")
            if t.device != device:
                raise ValueError(f"{name} is on {t.device}, the cache on {device}")
        n = int(kv_len.shape[0])
        if pages.shape[0] != n or cu_q.shape[0] != n + 1:
            raise ValueError(f"pages {tuple(pages.shape)}, kv_len {tuple(kv_len.shape)} and cu_q "
                             f"{tuple(cu_q.shape)} do not describe the same sequences")
        for name, v in (("n_tokens", n_tokens), ("max_q", max_q), ("max_kv", max_kv)):
            if int(v) < 0 or int(v) > 1 << 30:
                raise ValueError(f"{name} must be 0 .. 2^30, got {v}")
        if int(max_kv) > int(pages.shape[1]) * page_size:
            raise ValueError(f"max_kv = {max_kv} tokens do not fit {int(pages.shape[1])} pages of "
                             f"{page_size}")
        self.pages, self.kv_len, self.cu_q = pages, kv_len, cu_q
        self._index = device.index
        self.n_tokens, self.max_q, self.max_kv = int(n_tokens), int(max_q), int(max_kv)
        self._c = _jg._KvBatch(n, int(pages.shape[1]), pages.data_ptr(), kv_len.data_ptr(),
                               cu_q.data_ptr(), self.n_tokens, self.max_q, self.max_kv)
        self._ref = ctypes.byref(self._c)


class KVCache:
    """A cache of num_pages pages of page_size tokens (a power of two,
    16 .. 1024), kv_heads key/value heads of head_dim (64, 128 or 256)
    elements, in 8 or 4 bits and a float32 scale per row.  `data` is its buffer
    (a uint8 tensor); its contents before the first write do not matter."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, bits=8, device="cuda"):
        # what is wrong within 32 bits the library refuses
        for name, v in (("num_pages", num_pages), ("page_size", page_size), ("kv_heads", kv_heads),
                        ("head_dim", head_dim), ("bits", bits)):
            _int32(v, name)
        self._c = _jg._KvParams(int(bits), int(kv_heads), int(head_dim), int(page_size),
                                int(num_pages))
        self._ref = ctypes.byref(self._c)
        L = _jg.lib()
        n = int(L.jhq_kv_bytes(self._ref))
        if n == 0:
            _jg._check(_jg.JHQ_EINVAL)
        torch = _torch()
        if torch.device(device).type != "cuda":
            raise ValueError(f"the cache must be on a GPU, not on {device}")
        self.data = torch.empty(n, dtype=torch.uint8, device=device)
        self.device = self.data.device
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.kv_heads, self.head_dim, self.bits = int(kv_heads), int(head_dim), int(bits)
        self._ptr = self.data.data_ptr()
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._index = self.device.index
        # plain numbers: a torch.cuda.Stream object costs two microseconds a call
        self._current, self._device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        self._write, self._read, self._attend = L.jhq_k_kv_write, L.jhq_k_kv_read, L.jhq_k_kv_attend
        self._write_rotary, self._attend_shared = L.jhq_k_kv_write_rotary, L.jhq_k_kv_attend_shared
        self._copy_pages, self._copy = L.jhq_k_kv_copy_pages, L.jhq_k_kv_copy

    def batch(self, pages, kv_len, cu_q, n_tokens, max_q, max_kv):
        """The sequences of a call (KVBatch)."""
        return KVBatch(self.device, self.page_size, pages, kv_len, cu_q, n_tokens, max_q, max_kv)

    def _call(self, entry, stream, batch, *args):
        if batch._index != self._index:
            raise ValueError(f"the batch is on cuda:{batch._index}, the cache on {self.device}")
        if self._device() != self._index:  # kernels are launched on the current device
            with _torch().cuda.device(self._index):
                return self._call(entry, stream, batch, *args)
        if stream is None:
            s = self._current(self._index)
        else:
            s = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
        rc = entry(self._ref, self._ptr, batch._ref, *args, s)
        if rc:
            _jg._check(rc)

    def _enqueue(self, entry, stream, *args):
        # not called by _call: 0.3 us of a single token's 10
        if self._device() != self._index:
            with _torch().cuda.device(self._index):
                return self._enqueue(entry, stream, *args)
        if stream is None:
            s = self._current(self._index)
        else:
            s = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
        rc = entry(*args, s)
        if rc:
            _jg._check(rc)

    def _rows(self, t, what, heads, batch):
        """Element type and strides of a [n_tokens, heads, head_dim] tensor."""
        if t.shape != (batch.n_tokens, heads, self.head_dim):
            raise ValueError(f"{what} must be [{batch.n_tokens}, {heads}, {self.head_dim}], got "
                             f"{tuple(t.shape)}")
        if t.get_device() != self._index:
            raise ValueError(f"{what} is on {t.device}, the cache on {self.device}")
        tok, head, el = t.stride()
        if el != 1:
            raise ValueError(f"{what}: the elements of a row must be contiguous")
        dt = _DTYPES.get(t.dtype)
        return _dtype(t.dtype, what) if dt is None else dt, tok, head

    def write(self, k, v, batch, stream=None, rotary=None):
        """Quantises the batch's new tokens into the cache: k, v [n_tokens,
        kv_heads, head_dim], float32, bfloat16 or float16, any strides between
        rows.  rotary: a Rotary that turns the keys to their tokens' positions on the
        way, in float32 (not where tokens of a sequence have been moved)."""
        dt, kt, kh = self._rows(k, "k", self.kv_heads, batch)
        dv, vt, vh = self._rows(v, "v", self.kv_heads, batch)
        if dt != dv:
            raise ValueError(f"k is {k.dtype}, v is {v.dtype}")
        if rotary is None:
            self._call(self._write, stream, batch, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, dt)
            return
        if rotary._index != self._index:
            raise ValueError(f"the rotary is on {rotary.device}, the cache on {self.device}")
        if batch.moved:
            raise ValueError(_MOVED)
        self._call(self._write_rotary, stream, batch, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, dt,
                   rotary._ref)

    def read(self, batch, dtype=None, k_out=None, v_out=None, stream=None):
        """The batch's new tokens as the cache holds them: k, v [n_tokens,
        kv_heads, head_dim] in `dtype` (default float32), or into k_out and
        v_out (contiguous, one type).  Rows that no sequence's tokens stand
        behind keep what they had (zero in new tensors)."""
        if (k_out is None) != (v_out is None):
            raise ValueError("k_out and v_out go together")
        if k_out is None:
            torch = _torch()
            shape = (batch.n_tokens, self.kv_heads, self.head_dim)
            dtype = torch.float32 if dtype is None else dtype
            _dtype(dtype, "dtype")
            with torch.cuda.stream(_as_stream(stream, self.device)):
                k_out = torch.zeros(shape, dtype=dtype, device=self.device)
                v_out = torch.zeros(shape, dtype=dtype, device=self.device)
        elif dtype is not None and dtype != k_out.dtype:
            raise ValueError(f"dtype is {dtype}, k_out is {k_out.dtype}")
        dt = self._rows(k_out, "k_out", self.kv_heads, batch)[0]
        if self._rows(v_out, "v_out", self.kv_heads, batch)[0] != dt:
            raise ValueError(f"k_out is {k_out.dtype}, v_out is {v_out.dtype}")
        if not (k_out.is_contiguous() and v_out.is_contiguous()):
            raise ValueError("k_out and v_out must be contiguous")
        self._call(self._read, stream, batch, k_out.data_ptr(), v_out.data_ptr(), dt)
        return k_out, v_out

    def copy_pages(self, src, dst, stream=None):
        """Copies whole pages: src, dst int32 device tensors [n].  No page may be written twice or
        both read and written in one call; pairs that name a page that the cache does
        not have are left out."""
        int32 = _torch().int32
        for name, t in (("src", src), ("dst", dst)):
            if t.dtype != int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous 1-d int32 tensor")
            if t.get_device() != self._index:
                raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if src.shape != dst.shape:
            raise ValueError(f"src has {src.shape[0]} pages, dst {dst.shape[0]}")
        self._enqueue(self._copy_pages, stream, self._ref, self._ptr, src.data_ptr(),
                      dst.data_ptr(), src.shape[0])

    def copy(self, slots, batch, source=None, stream=None):
        """Copies tokens as they are held: the batch's new token in row t becomes the token at
        slot slots[t] = page * page_size + place of `source`, a cache of the same bits,
        kv_heads and head_dim (default: this one).  slots: an int64 device tensor
        [n_tokens]; a slot that source does not have makes a token that reads back and counts
        as NaN.  Tokens that the call writes must not be among those that it reads."""
        source = self if source is None else source
        if slots.dtype != _torch().int64 or slots.shape != (batch.n_tokens,) or not slots.is_contiguous():
            raise ValueError(f"slots must be a contiguous int64 [{batch.n_tokens}] tensor")
        for name, i in (("slots are", slots.get_device()), ("the batch is", batch._index),
                        ("the source is", source._index)):
            if i != self._index:
                raise ValueError(f"{name} on cuda:{i}, the cache on {self.device}")
        self._enqueue(self._copy, stream, source._ref, source._ptr, slots.data_ptr(),
                      self._ref, self._ptr, batch._ref)

    def work_bytes(self, batch, q_heads, window=0, prefix=None, once=False):
        """Bytes of workspace that attend needs for this batch, prefix and once."""
        if prefix is not None:
            self._no_window(window)
            n = int(_jg.lib().jhq_kv_shared_work_bytes(self._ref, batch._ref, prefix._ref,
                                                       1 if once else 0, _int32(q_heads, "q_heads")))
        else:
            n = int(_jg.lib().jhq_kv_work_bytes(self._ref, batch._ref, _int32(q_heads, "q_heads"), _window(window)))
        if n < 0:
            _jg._check(_jg.JHQ_EINVAL)
        return n

    @staticmethod
    def _no_window(window):
        if window:
            raise ValueError("a window and a prefix do not go together")

    def attend(self, q, batch, scale=None, causal=True, window=0, out=None, lse=None, work=None,
               stream=None, prefix=None, once=False):
        """Attention of the batch's new tokens, which the cache already holds, to
        their sequences; q [n_tokens, q_heads, head_dim] bfloat16 or float16,
        any strides between rows; returns out, the same shape and type,
        contiguous.  scale defaults to head_dim ** -0.5.  lse: a float32
        [n_tokens, q_heads] tensor that gets the logarithms of the softmax sums.
        work: a uint8 tensor of work_bytes() bytes, this call's alone until it has
        run; without it the call takes one from torch's allocator.  Rows outside
        cu_q keep what they had (zero where out is None).

        prefix: a KVBatch that says which neighbouring sequences of the batch begin with the
        same tokens, so that these are read once for all of them; what comes out is the
        same.  Its sequences are the groups: rows cu_q[g] .. of the call are the new
        tokens of group g's sequences, kv_len[g] the tokens that they share (0: none), all before
        their new ones, pages[g] the pages of these (KVPages.prefix finds them).  No window then.
        Sequences that contradict their group may come out as NaN.  The bounds choose whether
        prefixes are read once (from some 35 MB saved on, with single tokens); once=True has them
        read once wherever a call can (n_tokens * q_heads below 2^31 / head_dim, and less than 2^30 steps of 64
        tokens by the bounds): past that every sequence reads them, with the same results."""
        window = _window(window)
        if prefix is not None:
            self._no_window(window)
            if prefix._index != self._index:
                raise ValueError(f"the prefix is on cuda:{prefix._index}, the cache on {self.device}")
            if prefix.n_tokens != batch.n_tokens:
                raise ValueError(f"the prefix has {prefix.n_tokens} rows, the batch {batch.n_tokens}")
        heads = q.shape[1] if q.dim() == 3 else 0
        dt, qt, qh = self._rows(q, "q", heads, batch)
        if dt == _jg.JHQ_F32:
            raise ValueError("q must be bfloat16 or float16")
        if out is None:
            torch = _torch()
            with torch.cuda.stream(_as_stream(stream, self.device)):
                out = torch.zeros((batch.n_tokens, heads, self.head_dim), dtype=q.dtype,
                                  device=self.device)
        else:
            if self._rows(out, "out", heads, batch)[0] != dt or not out.is_contiguous():
                raise ValueError("out must be contiguous and of q's type")
        lp = None
        if lse is not None:
            torch = _torch()
            if lse.dtype != torch.float32 or tuple(lse.shape) != (batch.n_tokens, heads) \
                    or not lse.is_contiguous() or lse.device != self.device:
                raise ValueError(f"lse must be a contiguous float32 [{batch.n_tokens}, {heads}] "
                                 f"tensor on {self.device}")
            lp = lse.data_ptr()
        if work is None:
            n = self.work_bytes(batch, heads, window, prefix, once) if heads else 0
            if n:
                torch = _torch()
                with torch.cuda.stream(_as_stream(stream, self.device)):
                    work = torch.empty(n, dtype=torch.uint8, device=self.device)
        elif work.element_size() != 1 or not work.is_contiguous() \
                or work.get_device() != self._index:
            raise ValueError(f"work must be a contiguous uint8 tensor on {self.device}")
        wp, wn = (work.data_ptr(), work.numel()) if work is not None else (None, 0)
        scale, causal = self._scale if scale is None else float(scale), 1 if causal else 0
        if prefix is None:
            self._call(self._attend, stream, batch, q.data_ptr(), qt, qh, heads, dt, scale, causal, window,
                       out.data_ptr(), lp, wp, wn)
        else:
            self._call(self._attend_shared, stream, batch, prefix._ref, 1 if once else 0, q.data_ptr(), qt, qh, heads, dt,
                       scale, causal, out.data_ptr(), lp, wp, wn)
        return out


def _as_stream(stream, device):
    torch = _torch()
    if stream is None:
        return torch.cuda.current_stream(device)
    return stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(int(stream), device=device)
