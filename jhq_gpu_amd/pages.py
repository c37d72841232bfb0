"""Who holds which page of a key/value cache: sequences that grow, fork, shrink, are compacted
and freed (no counterpart in the reference).

    pages = KVPages(cache, n_seq=64, max_tokens=32768)
    batch = pages.extend([len(prompt)] + [0] * 63)   # room for a prompt in sequence 0
    cache.write(k, v, batch)
    pages.fork(0, 1)                                 # sequence 1 begins with what 0 holds
    batch = pages.extend([1, 1] + [0] * 62)          # a token each, pages shared up to there
    cache.write(k, v, batch)
    out = cache.attend(q, batch, prefix=pages.prefix())
    pages.compact({0: kept_positions})               # tokens are dropped
    pages.free(1)
"""
import heapq
import operator

import numpy as np

from . import kv as _kv

__all__ = ["KVPages"]

_NONE = 1 << 62


class _Move:
    """What compact does with a sequence: the tokens `at` stay, moved together from page `stay` on, of which
    the first that moves is the one that becomes token `moved`."""

    def __init__(self, seq, at, stay, moved):
        self.seq, self.at, self.stay, self.moved = seq, at, stay, moved


class KVPages:
    """The pages of `cache` (which nothing else may give out) and the sequences 0 .. n_seq - 1 that
    hold them, of up to max_tokens tokens each.  Which page is whose is the host's
    knowledge; the cache's kernels see it as the arrays of the batches that extend returns.

    A page may be held by several sequences: it is then only read, and a sequence that is
    to write into it gets a copy first.  Pages are given out lowest number first.

    Calls enqueue work on the current stream, or `stream` (they are no part of a captured graph, which
    replays what extend wrote last); the device arrays are this
    object's own and are updated in place, so a batch is good until the next call that changes
    its sequences, and everything that uses them has to be ordered with that stream."""

    def __init__(self, cache, n_seq, max_tokens):
        n_seq, max_tokens = operator.index(n_seq), operator.index(max_tokens)
        if n_seq < 1 or max_tokens < 1 or max_tokens > 1 << 30:
            raise ValueError(f"n_seq must be at least 1 and max_tokens 1 .. 2^30, got {n_seq} and {max_tokens}")
        torch = _kv._torch()
        self.cache, self.n_seq, self.max_tokens = cache, n_seq, max_tokens
        self.page_size = cache.page_size
        self._width = -(-max_tokens // self.page_size)
        self._free = list(range(cache.num_pages))  # in order: a heap
        self._refs = np.zeros(cache.num_pages, np.int32)
        self._table = np.zeros((n_seq, self._width), np.int32)
        self._len = np.zeros(n_seq, np.int64)
        self._new = np.zeros(n_seq, np.int64)
        # the first token that compact has moved: from it on, places are not positions
        self._moved = np.full(n_seq, _NONE, np.int64)
        # lengths, first rows, page table: one array, so that one copy brings them
        head = 2 * n_seq + 1
        self._dev = torch.zeros(head + self._table.size, dtype=torch.int32, device=cache.device)
        self._kv_len, self._cu = self._dev[:n_seq], self._dev[n_seq:head]
        self._pages = self._dev[head:].view(n_seq, self._width)
        self._dirty = False  # the table is newer than the device's
        self._fresh = False  # nothing has changed since extend

    @property
    def free_pages(self):
        """Pages that no sequence holds."""
        return len(self._free)

    def length(self, seq):
        """Tokens of a sequence."""
        return int(self._len[self._seq(seq)])

    def pages_of(self, seq):
        """A sequence's pages, in order."""
        seq = self._seq(seq)
        return self._table[seq, :self._held(seq)].tolist()

    def extend(self, new, max_q=None, max_kv=None, stream=None):
        """Room for new[s] more tokens of each sequence s; returns the KVBatch that
        writes and attends with them.  Where a sequence goes on in a page that others hold
        too, it gets a copy of it.  max_q, max_kv: the batch's bounds, wider than its
        lengths (the default) where a captured call is replayed as they grow."""
        new = self._counts(new)
        P = self.page_size
        to = self._len + new
        if int(new.sum()) > 1 << 30:
            raise ValueError(f"{int(new.sum())} new tokens, 2^30 are the most")
        if (to > self.max_tokens).any():
            s = int(np.argmax(to > self.max_tokens))
            raise ValueError(f"sequence {s} would have {int(to[s])} tokens, {self.max_tokens} are the most")
        bounds = []
        for name, v, least, most in (("max_q", max_q, int(new.max()), 1 << 30),
                                     ("max_kv", max_kv, int(to.max()), self._width * P)):
            v = least if v is None else operator.index(v)
            if not least <= v <= most:
                raise ValueError(f"{name} must be {least} .. {most}, got {v}")
            bounds.append(v)
        grow = np.where(new > 0, -(-to // P) - -(-self._len // P), 0)
        split = []
        # a page that k sequences are about to write into is kept by the last of them
        refs = {}
        for s in np.nonzero((new > 0) & (self._len % P > 0))[0]:
            page = int(self._table[s, self._len[s] // P])
            left = refs.get(page, int(self._refs[page]))
            if left > 1:
                split.append(int(s))
                refs[page] = left - 1
        self._need(int(grow.sum()) + len(split))
        src, dst, taken = [], [], []
        for s in split:
            at = self._len[s] // P
            src.append(int(self._table[s, at]))
            dst.append(self._take())
            self._refs[src[-1]] -= 1
            self._table[s, at] = dst[-1]
        for s in np.nonzero(grow)[0]:
            held = self._held(s)
            for i in range(held, held + int(grow[s])):
                taken.append(self._take())
                self._table[s, i] = taken[-1]
        self._dirty |= bool(src) or bool(taken)
        try:
            with self._on(stream):
                if src:
                    pairs = self._to_device(np.array([src, dst], np.int32))
                    self.cache.copy_pages(pairs[0], pairs[1])
                self._upload(to, new)
            batch = self.cache.batch(self._pages, self._kv_len, self._cu, int(new.sum()), *bounds)
        except BaseException:
            # no memory, or a launch that failed: sequences and pages are as before, the device's arrays may not be
            for s, page in zip(split, src):
                self._table[s, self._len[s] // P] = page
                self._refs[page] += 1
            self._release(np.array(dst + taken, np.int64))
            self._dirty, self._fresh = True, False
            raise
        batch.moved = bool(((new > 0) & (self._moved < self._len)).any())
        self._len, self._new, self._fresh = to, new, True
        return batch

    def fork(self, src, dst):
        """Sequence dst, which is empty, begins with all tokens of src, in the same pages."""
        src, dst = self._seq(src), self._seq(dst)
        if src == dst or self._len[dst]:
            raise ValueError(f"sequence {dst} is not empty" if src != dst else
                             f"sequence {src} cannot fork into itself")
        held = self._held(src)
        self._table[dst, :held] = self._table[src, :held]
        np.add.at(self._refs, self._table[src, :held], 1)
        self._len[dst], self._moved[dst] = self._len[src], self._moved[src]
        self._dirty |= held > 0
        self._fresh = False

    def truncate(self, seq, n):
        """Keeps a sequence's first n tokens."""
        seq, n = self._seq(seq), operator.index(n)
        if n < 0 or n > self._len[seq]:
            raise ValueError(f"sequence {seq} has {int(self._len[seq])} tokens, not {n}")
        first, held = -(-n // self.page_size), self._held(seq)
        self._release(self._table[seq, first:held])
        self._len[seq] = n
        if n <= self._moved[seq]:
            self._moved[seq] = _NONE
        self._fresh = False

    def free(self, seq):
        """Gives a sequence's pages back: it is empty."""
        self.truncate(seq, 0)

    def compact(self, keep, stream=None):
        """keep: {sequence: ascending positions}.  Each of these sequences keeps those of its tokens,
        moved together; keys stay as they are, turned to the positions that they had, so tokens that
        come after are turned to positions of their own too: Rotary.apply with a tensor of them
        (it and write(rotary=) refuse a batch of such sequences, whose positions are not their places).
        Whole pages in front that keep all of their tokens stay; the others' tokens are
        copied into free pages.  Where there are not as many as they fill, pages that have
        become empty take what follows, in several copies: pages that keep nothing at once, and one free page is
        enough where nobody else holds the rest.  (Between two of them an error of the device loses what was
        moved; any other leaves everything as it was.)"""
        P, plan = self.page_size, []
        for s, at in keep.items():
            s, at = self._seq(s), np.asarray(at)
            if at.ndim != 1 or (at.size and at.dtype.kind not in "iu"):
                raise ValueError(f"sequence {s}: positions must be a 1-d array of integers")
            at = at.astype(np.int64)
            if at.size and (at[0] < 0 or at[-1] >= self._len[s] or (np.diff(at) <= 0).any()):
                raise ValueError(f"sequence {s}: positions must ascend within its {int(self._len[s])} tokens")
            moved = np.nonzero(at != np.arange(at.size))[0]
            # pages in front that stay: of a beginning, where no token moves, all that it fills
            plan.append(_Move(s, at, int(moved[0]) // P if moved.size else -(-at.size // P),
                              int(moved[0]) if moved.size else at.size))
        if len({m.seq for m in plan}) != len(plan):
            raise ValueError("a sequence is named twice")
        # everything that can fail comes before what changes this object
        free, refs = list(self._free), self._refs.copy()
        rounds = self._rounds(plan, free, refs)
        if rounds:
            with self._on(stream):
                for slots, batch in self._copies(rounds):
                    self.cache.copy(slots, batch)
        self._free, self._refs = free, refs
        for m in plan:
            self._table[m.seq, m.stay:m.stay + len(m.to)] = m.to
            # what was moved before, and what is now
            moved = min(int(np.searchsorted(m.at, self._moved[m.seq])), m.moved)
            self._moved[m.seq] = moved if moved < m.at.size else _NONE
            self._len[m.seq] = m.at.size
            self._fresh = False
        self._dirty |= bool(rounds)

    def _rounds(self, plan, free, refs):
        """Gives the moves pages out of `free` and gives back what they leave; returns the copies that this
        takes, one after the other: lists of (move, first new page, end).  A copy's pages are read by no
        move that is not done."""
        P = self.page_size
        need = sum(-(-m.at.size // P) - m.stay for m in plan)

        def release(pages):
            for page in pages.tolist():
                refs[page] -= 1
                if refs[page] == 0:
                    heapq.heappush(free, page)
        for m in plan:
            m.old = self._table[m.seq, m.stay:self._held(m.seq)]
            m.to, m.left = [], 0
        enough = need <= len(free)
        if not enough:  # what gives back most, for what it takes, first
            plan = sorted(plan, key=lambda m: -(-m.at.size // P) - m.stay - int((refs[m.old] == 1).sum()))
            for m in plan:
                # how many new pages are full when an old one is empty
                upto = np.searchsorted(m.at, (m.stay + np.arange(len(m.old) + 1)) * P)
                m.after = np.where(upto[1:] > upto[:-1], -(-upto[1:] // P) - m.stay, 0)
        rounds = []
        while True:
            if not enough:
                for m in plan:
                    done = m.after <= len(m.to)
                    release(m.old[done])
                    m.old, m.after = m.old[~done], m.after[~done]
            copies = []
            for m in plan:
                k, at = min(len(free), -(-m.at.size // P) - m.stay - len(m.to)), len(m.to)
                for _ in range(k):
                    m.to.append(heapq.heappop(free))
                    refs[m.to[-1]] = 1
                if k:
                    copies.append((m, at, at + k))
            if not copies:
                break
            rounds.append(copies)
        if sum(len(m.to) for m in plan) < need:
            raise RuntimeError(f"the cache is full: {need} pages are needed, {len(self._free)} are free")
        for m in plan:
            release(m.old)
        return rounds

    def _copies(self, rounds):
        """(slots, batch) of each round, all on the device before the first is copied.  A batch's sequences are
        what fills the new pages alone: where these stand in their sequence does not matter to a copy."""
        P, arrays, slots, cuts = self.page_size, [], [], []
        for copies in rounds:
            n, width = len(copies), max(b - a for _, a, b in copies)
            table, new = np.zeros((n, width), np.int64), np.zeros(n, np.int64)
            for i, (m, a, b) in enumerate(copies):
                at = m.at[(m.stay + a) * P:(m.stay + b) * P]
                slots.append(self._table[m.seq, at // P].astype(np.int64) * P + at % P)
                table[i, :b - a], new[i] = m.to[a:b], at.size
            arrays.append(np.concatenate([new, [0], np.cumsum(new), table.reshape(-1)]))
            cuts.append((n, width, int(new.sum()), int(new.max())))
        dev, slots = self._to_device(np.concatenate(arrays).astype(np.int32)), self._to_device(np.concatenate(slots))
        out = []
        for n, width, total, most in cuts:
            end = 2 * n + 1 + n * width
            out.append((slots[:total], self.cache.batch(dev[2 * n + 1:end].view(n, width), dev[:n],
                                                        dev[n:2 * n + 1], total, most, most)))
            dev, slots = dev[end:], slots[total:]
        return out

    def prefix(self, least=1, stream=None):
        """What attend takes as `prefix` beside the batch that extend returned last: neighbouring
        sequences (those that share pages are best given numbers in a row) whose tables begin with the
        same pages, least pages of them at the least, all before their new tokens.  None where no two
        do.  Its arrays are new ones, for this step: a captured call would replay those that it was captured
        with."""
        if not self._fresh:
            raise RuntimeError("sequences have changed since extend")
        P, groups = self.page_size, []
        least = max(1, operator.index(least))
        live = np.nonzero(self._new)[0]
        whole = (self._len - self._new)[live] // P
        # pages that a sequence begins with as the one before it does
        same = np.zeros(live.size, np.int64)
        if live.size > 1:
            width = int(whole.max())
            equal = self._table[live[1:], :width] == self._table[live[:-1], :width]
            same[1:] = np.where(equal.all(1), width, equal.argmin(1)) if width else 0
        for s, m, mine, rows in zip(live.tolist(), same.tolist(), whole.tolist(), self._new[live].tolist()):
            if groups:
                first, n, shared, total = groups[-1]
                m = min(m, shared, mine)
                # a sequence joins where that saves as many pages as it costs the others
                if m >= least and n * m >= (n - 1) * shared:
                    groups[-1] = (first, n + 1, m, total + rows)
                    continue
            groups.append((s, 1, mine, rows))
        if not any(n > 1 for _, n, _, _ in groups):
            return None
        shared = np.array([m if n > 1 else 0 for _, n, m, _ in groups], np.int64)
        total = np.array([t for _, _, _, t in groups], np.int64)
        width, n = max(1, int(shared.max())), len(groups)
        table = self._table[[f for f, _, _, _ in groups], :width]
        arrays = np.concatenate([shared * P, [0], np.cumsum(total), table.reshape(-1)])
        with self._on(stream):
            dev = self._to_device(arrays.astype(np.int32))
        return self.cache.batch(dev[2 * n + 1:].view(n, width), dev[:n], dev[n:2 * n + 1],
                                int(total.sum()), int(total.max()), int(shared.max()) * P)

    def everything(self, stream=None):
        """The batch whose new tokens are all tokens of all sequences, one after the other: what
        reads them back."""
        arrays = np.concatenate([self._len, [0], np.cumsum(self._len), self._table.reshape(-1)])
        if int(self._len.sum()) > 1 << 30:
            raise ValueError(f"the sequences hold {int(self._len.sum())} tokens, 2^30 are the most")
        n = self.n_seq
        with self._on(stream):
            dev = self._to_device(arrays.astype(np.int32))
        batch = self.cache.batch(dev[2 * n + 1:].view(n, self._width), dev[:n], dev[n:2 * n + 1],
                                 int(self._len.sum()), int(self._len.max()), int(self._len.max()))
        batch.moved = bool((self._moved < self._len).any())
        return batch

    # ---- inside ----

    def _seq(self, s):
        s = operator.index(s)
        if not 0 <= s < self.n_seq:
            raise ValueError(f"there is no sequence {s}")
        return s

    def _counts(self, new):
        new = np.asarray(new)
        if new.shape != (self.n_seq,) or new.dtype.kind not in "iu" or (new < 0).any() \
                or (new > self.max_tokens).any():
            raise ValueError(f"new must be {self.n_seq} numbers of tokens, 0 .. {self.max_tokens}")
        return new.astype(np.int64)

    def _held(self, s):
        return int(-(-self._len[s] // self.page_size))

    def _need(self, n):
        if n > len(self._free):
            raise RuntimeError(f"the cache is full: {n} pages are needed, {len(self._free)} are free")

    def _take(self):
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _release(self, pages):
        for page in pages.tolist():
            self._refs[page] -= 1
            if self._refs[page] == 0:
                heapq.heappush(self._free, page)

    def _on(self, stream):
        return _stream_of(stream, self.cache.device)

    def _host(self, a):
        """The array in pinned memory, which torch keeps until copies from it have run."""
        torch = _kv._torch()
        t = torch.from_numpy(np.ascontiguousarray(a))
        if self.cache.device.type != "cuda":
            return t
        return torch.empty(t.shape, dtype=t.dtype, pin_memory=True).copy_(t)

    def _to_device(self, a):
        return self._host(a).to(self.cache.device, non_blocking=True)

    def _upload(self, lens, new):
        head = np.concatenate([lens, [0], np.cumsum(new)]).astype(np.int32)
        a = np.concatenate([head, self._table.reshape(-1)]) if self._dirty else head
        self._dev[:a.size].copy_(self._host(a), non_blocking=True)
        self._dirty = False


def _stream_of(stream, device):
    import contextlib
    if stream is None or device.type != "cuda":
        return contextlib.nullcontext()
    return _kv._torch().cuda.stream(_kv._as_stream(stream, device))
