"""Cases of the key/value cache operators: a paged cache of attention keys and
values held in 8 or 4 bits.

* ``store``   one step's new tokens are quantised into the cache's pages and a
  range of tokens is read back as 16- or 32-bit values (what a program does
  that hands the cache, or part of it, to something else);
* ``attend``  the new tokens of a batch of sequences attend to everything that
  the cache holds of their sequence, themselves included: one token each, a few
  or a long chunk of a prompt.

A row x (one token's key or value in one head, D elements) is stored as
codes rne(top * x / max|x|), top = 127 in 8 bits and 7 in 4 bits, and the scale
max|x| / top in float32; a row whose largest magnitude is below 2**-60 is
stored as zeros.  New token i of a sequence with q new tokens among its n
stands at position n - q + i and sees the positions up to its own (all n
where ``causal`` is false), the last ``window`` of them where window > 0.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
FLOOR = 2.0 ** -60
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# The largest listed case's operations and bytes (prompt_long, cache_out_4):
# no drawn case costs more.
MOST_FLOPS = 4.3e12
MOST_BYTES = 8.7e8


def _store(name, **kw):
    c = dict(name=name, kind="store", bits=8, kv_heads=8, head_dim=128, page=64, dtype="bf16",
             out="bf16", seqs=1, new_lo=1, new_hi=1, old_lo=0, old_hi=0, whole=False, lens=1)
    c.update(kw)
    return c


def _attend(name, **kw):
    c = dict(name=name, kind="attend", bits=8, heads=32, kv_heads=8, head_dim=128, page=64,
             dtype="bf16", seqs=1, new_lo=1, new_hi=1, old_lo=0, old_hi=0, causal=True, window=0,
             lens=1)
    c.update(kw)
    return c


def listed():
    return [
        # one decoding step of a serving batch: a token each of 64 sequences goes
        # into the cache and comes back as the cache holds it
        _store("token_in_8", seqs=64, old_lo=100, old_hi=4000),
        # prompts of ragged lengths enter the cache; all of it is read back
        _store("prompts_in_8", seqs=9, new_lo=1, new_hi=4001, page=16, whole=True, lens=2),
        # a long cache handed on in full after one more chunk, in 4 bits
        _store("cache_out_4", bits=4, seqs=2, new_lo=8192, new_hi=8192, old_lo=150000,
               old_hi=150001, head_dim=64, dtype="f16", out="f16", whole=True, lens=3),
        # one sequence's next token over a short context: latency
        _attend("token_short", heads=16, kv_heads=2, old_lo=776, old_hi=776),
        # a serving batch's next tokens, contexts from short to long
        _attend("token_batch", seqs=64, old_lo=300, old_hi=9000, lens=4),
        # few sequences of very long contexts, 4 bits, eight query heads to a key head
        _attend("token_long_4", bits=4, heads=64, seqs=4, dtype="f16", old_lo=130001,
                old_hi=131071, lens=5),
        # a few proposed tokens a sequence are checked at once, every head its own keys
        _attend("few_each", heads=16, kv_heads=16, head_dim=64, page=32, seqs=24, new_lo=2,
                new_hi=7, old_lo=50, old_hi=5000, lens=6),
        # a prompt attends to itself (an odd length, no older tokens)
        _attend("prompt_self", new_lo=2999, new_hi=2999, page=16),
        # chunks of prompts of ragged lengths beside sequences that decode, a
        # sliding window, 256-wide heads
        _attend("mixed_window_256", heads=8, kv_heads=4, head_dim=256, dtype="f16", seqs=12,
                new_lo=1, new_hi=1500, old_lo=0, old_hi=6000, window=1024, lens=7),
        # queries that see all of the passages that a search returned (no causal
        # mask), 4 bits
        _attend("passages_4", bits=4, heads=12, kv_heads=12, head_dim=64, seqs=10, new_lo=100,
                new_hi=700, old_lo=500, old_hi=3500, causal=False, lens=8),
        # a long prompt's last chunk over all that came before
        _attend("prompt_long", new_lo=8192, new_hi=8192, old_lo=28001, old_hi=28001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        bits = rng.choice((8, 8, 4))
        D = rng.choice((64, 128, 128, 256))
        H = rng.choice((1, 2, 4, 8, 8, 12, 16))
        page = rng.choice((16, 32, 64, 64, 128, 256))
        dtype = rng.choice(("bf16", "bf16", "f16"))
        shape = rng.choice(("token", "token", "few", "chunk", "chunk"))
        seqs = _log(rng, 1, {"token": 96, "few": 48, "chunk": 12}[shape])
        new_hi = {"token": 1, "few": rng.randint(2, 16), "chunk": _log(rng, 30, 8192)}[shape]
        new_lo = rng.choice((new_hi, max(1, new_hi // 4)))
        old_hi = _log(rng, 10, 131071 if seqs <= 4 else 12000)
        old_lo = rng.choice((old_hi, old_hi // 2, old_hi // 20))
        c = dict(bits=bits, kv_heads=H, head_dim=D, page=page, dtype=dtype, seqs=seqs,
                 new_lo=new_lo, new_hi=new_hi, old_lo=old_lo, old_hi=old_hi,
                 lens=rng.randint(0, 1 << 30))
        if rng.random() < 0.3:
            c.update(kind="store", whole=rng.random() < 0.5, out=rng.choice((dtype, dtype, "f32")))
        else:
            c.update(kind="attend", heads=H * rng.choice((1, 2, 4, 4, 7, 8)),
                     causal=rng.random() < 0.85, window=0)
            if c["causal"] and rng.random() < 0.25:
                c["window"] = _log(rng, 16, 4096)
            if c["heads"] > 64:
                continue
        w = work(c)
        # the tokens of the whole cache bound what has to be prepared
        held = sum(_lens(c)[1]) * H * D
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and held <= 5.4e8:
            return c


# ---- sizes ------------------------------------------------------------------

def _lens(c):
    """New tokens and all tokens of each sequence (in a batch of three or more
    the last sequence but one has none at all, as a slot that is idle)."""
    rng = random.Random(c["lens"])
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    old = [rng.randint(c["old_lo"], c["old_hi"]) for _ in range(c["seqs"])]
    if c["seqs"] >= 3:
        new[-2] = old[-2] = 0
    return new, [a + b for a, b in zip(new, old)]


def _pairs(c, q, n):
    """Visible (new token, token) pairs of a sequence, and the tokens that any
    of its new tokens sees."""
    if q == 0:
        return 0, 0
    if not c["causal"]:
        return q * n, n
    p = np.arange(n - q, n, dtype=np.int64)
    lo = np.maximum(0, p - c["window"] + 1) if c["window"] else np.zeros_like(p)
    return int((p + 1 - lo).sum()), int(n - lo[0])


def work(case):
    c = case
    H, D = c["kv_heads"], c["head_dim"]
    new, full = _lens(c)
    T = sum(new)
    held = 2 * H * (D * c["bits"] // 8 + 4)  # bytes of a token in the cache
    e = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "store":
        R = sum(full) if c["whole"] else T
        eo = 4 if c["out"] == "f32" else 2
        # codes written by this pass are outputs; tokens read back are inputs
        return {"bytes": 2 * T * H * D * e + T * held + R * held + 2 * R * H * D * eo,
                "flops": 4 * T * H * D + 2 * R * H * D}
    pairs = seen = 0
    for q, n in zip(new, full):
        a, b = _pairs(c, q, n)
        pairs += a
        seen += b
    return {"bytes": 2 * T * c["heads"] * D * e + seen * held, "flops": 4 * pairs * c["heads"] * D}


# ---- inputs -----------------------------------------------------------------

def _inputs(c, seed):
    """Keys and values of all tokens, sequence after sequence, and the new
    tokens' queries.  Keys have a few strong channels and values differ in size
    from token to token, as a model's do; the first tokens of a sequence draw
    much of the attention and have small values."""
    new, full = _lens(c)
    H, D, t = c["kv_heads"], c["head_dim"], TYPES[c["dtype"]]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 2 + 1)
    n = sum(full)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    chan = torch.exp(0.5 * normal(H, D))
    size = torch.exp(0.4 * normal(n, 1, 1)).to(t)
    k = torch.empty(n, H, D, device=DEV, dtype=t)
    v = torch.empty(n, H, D, device=DEV, dtype=t)
    step = max(1, (1 << 26) // (H * D))
    for i in range(0, n, step):
        m = min(step, n - i)
        k[i:i + m] = normal(m, H, D) * chan
        v[i:i + m] = normal(m, H, D) * size[i:i + m].float()
    starts = np.concatenate([[0], np.cumsum(full)[:-1]])
    for s, f in zip(starts, full):
        v[s:s + min(2, f)] *= 0.05
    q = None
    if c["kind"] == "attend":
        G = c["heads"] // H
        q = normal(sum(new), H, G, D) / chan[:, None, :] * torch.exp(0.5 * normal(1, H, G, 1))
        q = q.reshape(sum(new), c["heads"], D).to(t)
    return new, full, k, v, q


def _new_rows(new, full):
    """Rows of the new tokens among all tokens."""
    at, rows = 0, []
    for a, f in zip(new, full):
        rows.append(np.arange(at + f - a, at + f))
        at += f
    return torch.from_numpy(np.concatenate(rows)).to(DEV)


def _i32(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device=DEV)


def _cu(n):
    return np.concatenate([[0], np.cumsum(n)])


def _quantise(x, bits):
    """float32 codes and scales [.., 1] of rows x."""
    x = x.float()
    top = 127.0 if bits == 8 else 7.0
    amax = x.abs().amax(-1, keepdim=True)
    live = amax >= FLOOR
    code = torch.round(x * top / torch.where(live, amax, torch.ones_like(amax)))
    return torch.where(live, code, torch.zeros_like(code)), torch.where(
        live, amax / top, torch.zeros_like(amax))


def _slots(table, page, lo, hi):
    pos = torch.arange(lo, hi, device=DEV)
    return table[pos // page].long() * page + pos % page


def prepare(case, seed):
    c = case
    new, full, k, v, q = _inputs(c, seed)
    H, D, page = c["kv_heads"], c["head_dim"], c["page"]
    per = [-(-f // page) for f in full]
    pages = sum(per) + 3
    # pages as a serving program's allocator leaves them: in no order
    order = np.random.default_rng(seed).permutation(pages)
    table = np.zeros((len(full), max(max(per), 1)), np.int32)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at:at + p]
        at += p
    st = dict(case=c, new=new, full=full, table=_i32(table), kv_len=_i32(full))
    # the new tokens' queries, keys and values come out of one projection
    rows = _new_rows(new, full)
    T, Hq = sum(new), c.get("heads", 0)
    fused = torch.empty(T, Hq + 2 * H, D, device=DEV, dtype=k.dtype)
    fused[:, Hq:Hq + H] = k[rows]
    fused[:, Hq + H:] = v[rows]
    if q is not None:
        fused[:, :Hq] = q
    st["q"], st["k"], st["v"] = fused[:, :Hq], fused[:, Hq:Hq + H], fused[:, Hq + H:]
    old = [f - a for a, f in zip(new, full)]
    whole = c["kind"] == "attend" or c["whole"]
    st["from"] = [0] * len(new) if whole else old
    if own:
        import jhq_gpu_amd as jg
        cache = jg.KVCache(pages, page, H, D, bits=c["bits"], device=DEV)
        step = cache.batch(st["table"], st["kv_len"], _i32(_cu(new)), sum(new), max(new),
                           max(full))
        everything = cache.batch(st["table"], st["kv_len"], _i32(_cu(full)), sum(full),
                                 max(full), max(full))
        cache.write(k, v, everything)
        st.update(cache=cache, step=step, back=everything if whole else step)
        if q is not None:
            st["out"] = torch.empty(T, Hq, D, device=DEV, dtype=k.dtype)
            st["work"] = torch.empty(cache.work_bytes(step, Hq, c["window"]), device=DEV,
                                     dtype=torch.uint8)
        else:
            R = sum(f - a for a, f in zip(st["from"], full))
            st["k_out"] = torch.empty(R, H, D, device=DEV, dtype=TYPES[c["out"]])
            st["v_out"] = torch.empty(R, H, D, device=DEV, dtype=TYPES[c["out"]])
        return st
    st.update(kc=torch.zeros(pages * page, H, D, device=DEV, dtype=torch.int8),
              vc=torch.zeros(pages * page, H, D, device=DEV, dtype=torch.int8),
              ks=torch.zeros(pages * page, H, 1, device=DEV),
              vs=torch.zeros(pages * page, H, 1, device=DEV))
    at = 0
    for b, f in enumerate(full):
        if f:
            _put(st, b, 0, f, k[at:at + f], v[at:at + f])
        at += f
    return st


# ---- the plain forms --------------------------------------------------------

def _put(st, b, lo, hi, k, v):
    c = st["case"]
    slot = _slots(st["table"][b], c["page"], lo, hi)
    step = max(1, (1 << 27) // (c["kv_heads"] * c["head_dim"]))
    for i in range(0, hi - lo, step):
        s = slot[i:i + step]
        for x, codes, scales in ((k, st["kc"], st["ks"]), (v, st["vc"], st["vs"])):
            code, scale = _quantise(x[i:i + step], c["bits"])
            codes[s] = code.to(torch.int8)
            scales[s] = scale


def _run_store(st):
    c = st["case"]
    at = 0
    for b, (a, f) in enumerate(zip(st["new"], st["full"])):
        if a:
            _put(st, b, f - a, f, st["k"][at:at + a], st["v"][at:at + a])
        at += a
    slot = torch.cat([_slots(st["table"][b], c["page"], lo, f)
                      for b, (lo, f) in enumerate(zip(st["from"], st["full"]))])
    t = TYPES[c["out"]]
    return [torch.cat([(codes[s].float() * scales[s]).to(t) for s in slot.split(1 << 17)])
            for codes, scales in ((st["kc"], st["ks"]), (st["vc"], st["vs"]))]


def _mask(c, lo, hi, n, q):
    """Whether the new tokens lo .. hi-1 of q see the tokens 0 .. n-1."""
    p = torch.arange(n - q + lo, n - q + hi, device=DEV)[:, None]
    j = torch.arange(n, device=DEV)[None, :]
    if not c["causal"]:
        return torch.ones(hi - lo, n, device=DEV, dtype=torch.bool)
    m = j <= p
    if c["window"]:
        m &= j > p - c["window"]
    return m


def _run_attend(st):
    c = st["case"]
    H, D = c["kv_heads"], c["head_dim"]
    G = c["heads"] // H
    scale = 1.0 / math.sqrt(D)
    out = torch.zeros(sum(st["new"]), c["heads"], D, device=DEV, dtype=st["q"].dtype)
    at = 0
    for b, (a, f) in enumerate(zip(st["new"], st["full"])):
        if a == 0:
            continue
        slot = _slots(st["table"][b], c["page"], 0, f)
        q = st["q"][at:at + a].float().reshape(a, H, G, D)
        # as many key heads at once as the score matrix allows
        hs = max(1, min(H, (1 << 29) // (a * G * f)))
        rows = max(1, min(a, (1 << 30) // (hs * G * f)))
        for h in range(0, H, hs):
            kx, vx = [(codes[slot, h:h + hs].float() * scales[slot, h:h + hs]).transpose(0, 1)
                      .contiguous() for codes, scales in ((st["kc"], st["ks"]),
                                                          (st["vc"], st["vs"]))]
            kt = kx.transpose(1, 2).contiguous()
            for r in range(0, a, rows):
                e = min(a, r + rows)
                qr = q[r:e, h:h + hs].permute(1, 0, 2, 3).reshape(-1, (e - r) * G, D)
                s = torch.matmul(qr, kt) * scale
                s = s.reshape(-1, e - r, G, f)
                s = s.masked_fill(~_mask(c, r, e, f, a)[None, :, None, :], -math.inf)
                p = torch.exp(s - s.amax(-1, keepdim=True))
                p = p / p.sum(-1, keepdim=True)
                o = torch.matmul(p.reshape(-1, (e - r) * G, f), vx)
                o = o.reshape(-1, e - r, G, D).permute(1, 0, 2, 3).reshape(e - r, -1, D)
                out[at + r:at + e, h * G:(h + hs) * G] = o.to(out.dtype)
        at += a
    return out


def run(state):
    st = state
    if own:
        if st["case"]["kind"] == "store":
            st["cache"].write(st["k"], st["v"], st["step"])
            return list(st["cache"].read(st["back"], k_out=st["k_out"], v_out=st["v_out"]))
        c = st["case"]
        return st["cache"].attend(st["q"], st["step"], causal=c["causal"], window=c["window"],
                                  out=st["out"], work=st["work"])
    return _run_store(st) if st["case"]["kind"] == "store" else _run_attend(st)


# ---- 64 bits ----------------------------------------------------------------

def _value64(x, bits):
    """What the cache holds of rows x, in float64."""
    x = x.double()
    top = 2 ** (bits - 1) - 1
    big = x.abs().max(-1, keepdim=True).values
    safe = big.clamp_min(FLOOR)
    val = (x * top / safe).round() * (safe / top)
    return torch.where(big < FLOOR, 0.0 * x, val)


def exact(case, seed):
    c = case
    new, full, k, v, q = _inputs(c, seed)
    H, D, bits = c["kv_heads"], c["head_dim"], c["bits"]
    if c["kind"] == "store":
        if not c["whole"]:
            rows = _new_rows(new, full)
            k, v = k[rows], v[rows]
        return [_value64(k, bits).cpu(), _value64(v, bits).cpu()]
    G = c["heads"] // H
    out = torch.zeros(sum(new), c["heads"], D, dtype=torch.float64, device=DEV)
    row = tok = 0
    for a, f in zip(new, full):
        for h in range(H if a else 0):
            kh = _value64(k[tok:tok + f, h], bits)
            vh = _value64(v[tok:tok + f, h], bits)
            pos = torch.arange(f - a, f, device=DEV)
            col = torch.arange(f, device=DEV)
            hidden = torch.zeros(a, f, dtype=torch.bool, device=DEV)
            if c["causal"]:
                hidden |= col[None] > pos[:, None]
                if c["window"]:
                    hidden |= col[None] <= pos[:, None] - c["window"]
            for g in range(G):
                s = q[row:row + a, h * G + g].double() @ kh.t() / math.sqrt(D)
                s[hidden] = -math.inf
                out[row:row + a, h * G + g] = torch.softmax(s, -1) @ vh
        row += a
        tok += f
    return out.cpu()
