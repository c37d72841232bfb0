"""Cases of the operators around the key/value cache: positions on queries and
keys, pages that are copied and compacted, and sequences that share a prefix.

* ``rotary``   queries and keys are turned to their positions (or turned back,
  which is the gradient's pass).  With r of a head's elements in pairs, (i, i +
  r/2) in halves or (2i, 2i + 1) interleaved, pair i of a token at position p
  turns by p f_i, f_i = base^(-2i/r), the frequencies scaled where contexts are
  longer than the model's; the other elements stay;
* ``fork``     whole pages are copied (what sequences that were forked need
  before they write into a page that they share), and read back;
* ``compact``  the tokens of sequences that are kept move together, codes and
  scales as they are, and are read back;
* ``shared``   the new tokens of sequences in groups attend to their group's
  prefix, which the cache holds once, and to their sequence's own tokens;
* ``step``     one step of a model's layer over such sequences: the new tokens'
  queries and keys are turned to their positions, keys and values enter the
  cache, the queries attend.

A row x (one token's key or value in one head) is held as codes rne(top * x /
max|x|), top = 127 in 8 bits and 7 in 4 bits, and the scale max|x| / top.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
FLOOR = 2.0 ** -60
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}

# The largest listed cases' operations and bytes (shared_questions, evict_long_4): no drawn
# case costs more.
MOST_FLOPS = 9.0e11
MOST_BYTES = 6.8e8


def _rope(name, **kw):
    c = dict(name=name, kind="rotary", heads=40, head_dim=128, rot=128, interleaved=False,
             base=10000.0, scaling="", factor=1.0, length=4096, dtype="bf16", inverse=False,
             given=False, seqs=1, new_lo=1, new_hi=1, old_lo=0, old_hi=0, lens=1)
    c.update(kw)
    return c


def _fork(name, **kw):
    c = dict(name=name, kind="fork", bits=8, kv_heads=8, head_dim=128, page=64, dtype="bf16",
             copies=16, parents=4, lens=1)
    c.update(kw)
    return c


def _compact(name, **kw):
    c = dict(name=name, kind="compact", bits=8, kv_heads=8, head_dim=128, page=64, dtype="bf16",
             seqs=1, old_lo=1, old_hi=1, keep=0.5, run=1, lens=1)
    c.update(kw)
    return c


def _shared(name, **kw):
    c = dict(name=name, kind="shared", bits=8, heads=32, kv_heads=8, head_dim=128, page=64,
             dtype="bf16", groups=1, seqs=8, prefix_lo=1000, prefix_hi=1000, new_lo=1, new_hi=1,
             old_lo=0, old_hi=100, causal=True, lens=1)
    c.update(kw)
    return c


def listed():
    return [
        # one sequence's next token, queries and keys of one projection: latency
        _rope("rope_token", heads=18, old_lo=776, old_hi=776),
        # the next tokens of a serving batch
        _rope("rope_batch", seqs=64, old_lo=300, old_hi=9000, lens=2),
        # prompts of ragged lengths, pairs side by side
        _rope("rope_prompts", seqs=7, new_hi=4001, interleaved=True, dtype="f16", base=500000.0,
              scaling="bands", factor=8.0, length=8192, lens=3),
        # the gradient's pass in training: float32, a quarter of a wide head, far
        # positions of a stretched context
        _rope("rope_part_back", heads=12, head_dim=256, rot=64, dtype="f32", scaling="yarn",
              factor=16.0, new_lo=8191, new_hi=8191, old_lo=57000, old_hi=57000, inverse=True,
              given=True),
        # answers sampled side by side: each gets a tail page of its own
        _fork("fork_tails", copies=63, parents=9),
        # a serving batch drops half of what it holds, token by token
        _compact("evict_batch", seqs=16, old_lo=500, old_hi=6000, lens=4),
        # passages leave two long contexts, in 4 bits
        _compact("evict_long_4", bits=4, head_dim=64, dtype="f16", seqs=2, old_lo=150000,
                 old_hi=150001, keep=0.7, run=150, lens=5),
        # a few answers to one prompt, short: latency
        _shared("shared_short", heads=16, kv_heads=2, seqs=8, old_lo=1, old_hi=200),
        # a serving batch behind one long system prompt
        _shared("shared_batch", seqs=64, prefix_lo=16003, prefix_hi=16003, old_lo=50, old_hi=1500,
                lens=6),
        # proposed tokens of groups with prefixes of their own, 4 bits, every head its own keys
        _shared("shared_groups_4", bits=4, heads=16, kv_heads=16, head_dim=64, page=32, dtype="f16",
                groups=4, seqs=40, prefix_lo=2000, prefix_hi=30000, new_lo=2, new_hi=5, old_lo=10,
                old_hi=900, lens=7),
        # questions over the passages that a search returned for all of them
        _shared("shared_questions", seqs=24, dtype="f16", prefix_lo=12000, prefix_hi=12000,
                new_lo=40, new_hi=300, old_lo=0, old_hi=64, lens=8),
        # a layer's step: positions, cache and attention, wide heads of which half turns
        _shared("step_256", kind="step", heads=16, kv_heads=4, head_dim=256, rot=128,
                interleaved=False, base=10000.0, scaling="linear", factor=4.0, length=4096, seqs=48,
                groups=3, prefix_lo=4000, prefix_hi=9000, old_lo=20, old_hi=700, lens=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _turn_of(rng, D):
    rot = rng.choice((D, D, D // 2, D // 4))
    scaling = rng.choice(("", "", "linear", "ntk", "yarn", "bands"))
    return dict(rot=rot, interleaved=rng.random() < 0.4, base=rng.choice((10000.0, 500000.0, 1e6)),
                scaling=scaling, factor=rng.choice((2.0, 4.0, 8.0, 16.0)) if scaling else 1.0,
                length=rng.choice((4096, 8192, 32768)))


def _draw(rng):
    kind = rng.choice(("rotary", "rotary", "fork", "compact", "shared", "shared", "shared", "step"))
    c = dict(kind=kind, lens=rng.randint(0, 1 << 30))
    if kind == "rotary":
        D = rng.choice((64, 64, 80, 96, 128, 128, 128, 192, 256))
        few = rng.random() < 0.5
        hi = 1 if few else _log(rng, 2, 16384)
        c.update(_turn_of(rng, D), heads=_log(rng, 1, 80), head_dim=D,
                 dtype=rng.choice(("bf16", "bf16", "f16", "f32")), inverse=rng.random() < 0.3,
                 given=rng.random() < 0.4, seqs=_log(rng, 1, 256 if few else 12), new_hi=hi,
                 new_lo=rng.choice((hi, max(1, hi // 5))), old_hi=_log(rng, 1, 1 << 20))
        c["old_lo"] = rng.choice((c["old_hi"], c["old_hi"] // 10))
        return c
    c.update(bits=rng.choice((8, 8, 4)), head_dim=rng.choice((64, 128, 128, 256)),
             kv_heads=rng.choice((1, 2, 4, 8, 8, 16)), page=rng.choice((16, 32, 64, 64, 128, 256)),
             dtype=rng.choice(("bf16", "bf16", "f16")))
    if kind == "fork":
        c.update(copies=_log(rng, 1, 2000), parents=_log(rng, 1, 60))
    elif kind == "compact":
        hi = _log(rng, 20, 150000)
        c.update(seqs=_log(rng, 1, 32), old_hi=hi, old_lo=rng.choice((hi, hi // 4)),
                 keep=rng.uniform(0.1, 0.95), run=rng.choice((1, 1, 4, 40, 300)))
    else:
        chunk = rng.random()
        hi = 1 if chunk < 0.5 else rng.randint(2, 8) if chunk < 0.75 else _log(rng, 10, 600)
        seqs = _log(rng, 2, 96 if hi <= 8 else 24)
        ph = _log(rng, 200, 100000 if seqs <= 8 else 24000)
        c.update(heads=c["kv_heads"] * rng.choice((1, 2, 4, 4, 7, 8)), seqs=seqs,
                 groups=min(seqs, rng.choice((1, 1, 1, 2, 3, 5))), prefix_hi=ph,
                 prefix_lo=rng.choice((ph, ph // 5)), new_hi=hi, new_lo=rng.choice((hi, (hi + 3) // 4)),
                 old_hi=_log(rng, 1, 3000), causal=rng.random() < 0.85)
        c["old_lo"] = rng.choice((0, c["old_hi"] // 2, c["old_hi"]))
        if kind == "step":
            c.update(_turn_of(rng, c["head_dim"]))
    return c


def draw(rng):
    while True:
        c = _draw(rng)
        if c.get("heads", 1) > 80:
            continue
        w = work(c)
        if c["kind"] != "rotary" and _held(c) * c["kv_heads"] * c["head_dim"] > 3.0e8:
            continue  # tokens of the whole cache bound what has to be prepared
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return c


# ---- sizes ------------------------------------------------------------------

def _ragged(c):
    """New tokens and all tokens of each sequence (of three or more the last but one
    is idle, with no token at all)."""
    rng = random.Random(c["lens"])
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    old = [rng.randint(c["old_lo"], c["old_hi"]) for _ in range(c["seqs"])]
    if c["seqs"] >= 3:
        new[-2] = old[-2] = 0
    return new, [a + b for a, b in zip(new, old)]


def _kept(c):
    """Tokens of each sequence, and the positions that are kept of them: runs of
    about `run` tokens."""
    rng = np.random.default_rng(c["lens"])
    lens = [int(x) for x in rng.integers(c["old_lo"], c["old_hi"] + 1, c["seqs"])]
    keep = []
    for n in lens:
        runs = rng.random(n // c["run"] + 2) < c["keep"]
        runs[0] = True  # what a context begins with stays
        at = (np.arange(n) + int(rng.integers(0, c["run"]))) // c["run"]
        keep.append(np.nonzero(runs[at])[0])
    return lens, keep


def _groups(c):
    """Of each group: its prefix's tokens, and each sequence's (new, own) tokens, own
    with the new ones."""
    rng = random.Random(c["lens"])
    cut = sorted(rng.sample(range(1, c["seqs"]), c["groups"] - 1))
    out = []
    for lo, hi in zip([0] + cut, cut + [c["seqs"]]):
        p = rng.randint(c["prefix_lo"], c["prefix_hi"])
        seqs = []
        for _ in range(lo, hi):
            a = rng.randint(c["new_lo"], c["new_hi"])
            seqs.append((a, a + rng.randint(c["old_lo"], c["old_hi"])))
        out.append((p, seqs))
    return out


def _held(c):
    """Tokens that the cache holds."""
    if c["kind"] == "fork":
        return (c["copies"] + c["parents"]) * c["page"]
    if c["kind"] == "compact":
        lens, keep = _kept(c)
        return sum(lens) + sum(len(k) for k in keep)
    return sum(p + sum(n for _, n in s) for p, s in _groups(c))


def work(case):
    c = case
    if c["kind"] == "rotary":
        rows = sum(_ragged(c)[0]) * c["heads"]
        return {"bytes": 2 * rows * c["head_dim"] * BYTES[c["dtype"]], "flops": rows * c["rot"] * 3}
    H, D, e = c["kv_heads"], c["head_dim"], BYTES[c["dtype"]]
    held = 2 * H * (D * c["bits"] // 8 + 4)  # bytes of a token in the cache
    if c["kind"] in ("fork", "compact"):
        R = c["copies"] * c["page"] if c["kind"] == "fork" else sum(len(k) for k in _kept(c)[1])
        # tokens read and written where they are held, and their values
        return {"bytes": 2 * R * held + 2 * R * H * D * e, "flops": 2 * R * H * D}
    groups = _groups(c)
    T = sum(a for _, s in groups for a, _ in s)
    pairs = 0
    for p, seqs in groups:
        for a, n in seqs:
            pairs += a * (p + n) - (a * (a - 1) // 2 if c["causal"] else 0)
    bytes_ = 2 * T * c["heads"] * D * e + _held(c) * held
    flops = 4 * pairs * c["heads"] * D
    if c["kind"] == "step":
        # the turned queries are an output beside attention's, new keys and values come in
        bytes_ += T * c["heads"] * D * e + 2 * T * H * D * e
        flops += 3 * T * (c["heads"] + H) * c["rot"]
    return {"bytes": bytes_, "flops": flops}


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 2 + 1)
    return g


def _i32(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device=DEV)


def _cu(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int64)


def _rope_inputs(c, seed):
    new, full = _ragged(c)
    g = _gen(seed)
    x = torch.randn(sum(new), c["heads"], c["head_dim"], device=DEV, generator=g)
    x *= torch.exp(0.5 * torch.randn(1, c["heads"], c["head_dim"], device=DEV, generator=g))
    pos = np.concatenate([np.arange(f - a, f) for a, f in zip(new, full)])
    return new, full, x.to(TYPES[c["dtype"]]), torch.from_numpy(pos).to(DEV)


def _rows(c, n, g):
    """Keys and values of n tokens: keys have a few strong channels, values differ in
    size from token to token, as a model's do."""
    H, D, t = c["kv_heads"], c["head_dim"], TYPES[c["dtype"]]
    chan = torch.exp(0.5 * torch.randn(H, D, device=DEV, generator=g))
    size = torch.exp(0.4 * torch.randn(n, 1, 1, device=DEV, generator=g))
    k = torch.empty(n, H, D, device=DEV, dtype=t)
    v = torch.empty(n, H, D, device=DEV, dtype=t)
    step = max(1, (1 << 26) // (H * D))
    for i in range(0, n, step):
        m = min(step, n - i)
        k[i:i + m] = torch.randn(m, H, D, device=DEV, generator=g) * chan
        v[i:i + m] = torch.randn(m, H, D, device=DEV, generator=g) * size[i:i + m]
    return k, v, chan


def _shared_inputs(c, seed):
    """Keys and values, group after group: the prefix's tokens, then each sequence's
    own; the new tokens' queries.  The first tokens of a prefix draw much of the
    attention and have small values."""
    groups, g = _groups(c), _gen(seed)
    k, v, chan = _rows(c, _held(c), g)
    at = 0
    for p, seqs in groups:
        v[at:at + min(2, p)] *= 0.05
        at += p + sum(n for _, n in seqs)
    T = sum(a for _, s in groups for a, _ in s)
    H, D = c["kv_heads"], c["head_dim"]
    G = c["heads"] // H
    q = torch.randn(T, H, G, D, device=DEV, generator=g) / chan[:, None, :]
    q = q * torch.exp(0.5 * torch.randn(1, H, G, 1, device=DEV, generator=g))
    return groups, k, v, q.reshape(T, c["heads"], D).to(TYPES[c["dtype"]])


def _frequencies(c):
    """Radians a position, float64, and what the turned pairs are multiplied by."""
    r, f = c["rot"], c["factor"]
    i = np.arange(r // 2, dtype=np.float64)
    base = c["base"] * (f ** (r / (r - 2.0)) if c["scaling"] == "ntk" else 1.0)
    w = base ** (-2.0 * i / r)
    if c["scaling"] == "linear":
        return w / f, 1.0
    if c["scaling"] == "bands":
        turns = c["length"] * w / (2 * math.pi)  # within the model's own context
        mix = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
        return w * (mix + (1.0 - mix) / f), 1.0
    if c["scaling"] == "yarn":
        def place(turns):
            return r * math.log(c["length"] / (turns * 2 * math.pi)) / (2 * math.log(c["base"]))
        lo, hi = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), r - 1)
        mix = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return w * (1.0 - mix + mix / f), 0.1 * math.log(f) + 1.0
    return w, 1.0


def _rotary(c):
    import jhq_gpu_amd as jg
    how = {"linear": dict(kind="linear", factor=c["factor"]),
           "ntk": dict(kind="ntk", factor=c["factor"]),
           "yarn": dict(kind="yarn", factor=c["factor"], length=c["length"]),
           "bands": dict(kind="bands", factor=c["factor"], length=c["length"])}
    return jg.Rotary(c["head_dim"], rot_dim=c["rot"], base=c["base"], interleaved=c["interleaved"],
                     scaling=how.get(c["scaling"]), device=DEV)


def prepare(case, seed):
    return {"rotary": _prepare_rotary, "fork": _prepare_moved, "compact": _prepare_moved,
            "shared": _prepare_shared, "step": _prepare_shared}[case["kind"]](case, seed)


def _prepare_rotary(c, seed):
    new, full, x, pos = _rope_inputs(c, seed)
    # queries and keys lie in one projection, values behind them
    T, h, D = x.shape
    fused = torch.empty(T, h + 2, D, device=DEV, dtype=x.dtype)
    fused[:, :h] = x
    st = dict(case=c, x=fused[:, :h], pos=pos)
    if own:
        import jhq_gpu_amd as jg
        st.update(rotary=_rotary(c), out=torch.empty(T, h, D, device=DEV, dtype=x.dtype))
        if not c["given"]:
            cache = jg.KVCache(1, 1024, 1, 64, device=DEV)
            table = np.zeros((len(new), -(-max(full) // 1024)), np.int32)
            st["pos"] = cache.batch(_i32(table), _i32(full), _i32(_cu(new)), T, max(new), max(full))
        return st
    w, st["size"] = _frequencies(c)
    st["freq"] = torch.from_numpy(w).to(DEV)
    return st


def _table(per, spare, seed):
    """Pages of each sequence as a serving program's allocator leaves them: in no
    order; and the number of pages."""
    pages = sum(per) + spare
    order = np.random.default_rng(seed).permutation(pages)
    table = np.zeros((len(per), max(max(per), 1)), np.int32)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at:at + p]
        at += p
    return table, pages


def _store(c, pages):
    """The plain forms' cache: codes and scales of every slot."""
    n, H, D = pages * c["page"], c["kv_heads"], c["head_dim"]
    return dict(kc=torch.zeros(n, H, D, device=DEV, dtype=torch.int8),
                vc=torch.zeros(n, H, D, device=DEV, dtype=torch.int8),
                ks=torch.zeros(n, H, 1, device=DEV), vs=torch.zeros(n, H, 1, device=DEV))


def _prepare_moved(c, seed):
    page, H, D, t = c["page"], c["kv_heads"], c["head_dim"], TYPES[c["dtype"]]
    if c["kind"] == "fork":
        # the parents' pages, and the children's places for a copy of one each
        rng = np.random.default_rng(c["lens"])
        lens, to = [page] * c["parents"], [page] * c["copies"]
        src = rng.integers(0, c["parents"], c["copies"])
    else:
        lens, keep = _kept(c)
        to = [len(k) for k in keep]
    k, v, _ = _rows(c, sum(lens), _gen(seed))
    table, pages = _table([-(-n // page) for n in lens + to], 3, seed)
    old, new = table[:len(lens)], np.ascontiguousarray(table[len(lens):])
    st = dict(case=c, to=to, table=_i32(table))
    if c["kind"] == "fork":
        st["src"], st["dst"] = _i32(old[src, 0]), _i32(new[:, 0])
    else:
        at = [old[b, j // page].astype(np.int64) * page + j % page for b, j in enumerate(keep)]
        st["slots"] = torch.from_numpy(np.concatenate(at)).to(DEV)
    if own:
        import jhq_gpu_amd as jg
        cache = jg.KVCache(pages, page, H, D, bits=c["bits"], device=DEV)
        cache.write(k, v, cache.batch(_i32(old), _i32(lens), _i32(_cu(lens)), sum(lens), max(lens),
                                      max(lens)))
        st.update(cache=cache, moved=cache.batch(_i32(new), _i32(to), _i32(_cu(to)), sum(to),
                                                 max(to), max(to)),
                  k_out=torch.empty(sum(to), H, D, device=DEV, dtype=t),
                  v_out=torch.empty(sum(to), H, D, device=DEV, dtype=t))
        return st
    st.update(_store(c, pages))
    at = 0
    for b, n in enumerate(lens):
        _put(st, _slots(st["table"][b], page, 0, n), k[at:at + n], v[at:at + n])
        at += n
    st["new"] = torch.cat([_slots(st["table"][len(lens) + b], page, 0, n) for b, n in enumerate(to)])
    return st


def _prepare_shared(c, seed):
    groups, k, v, q = _shared_inputs(c, seed)
    page, H, D = c["page"], c["kv_heads"], c["head_dim"]
    # whole pages of a prefix are held once; what it has in its last page, every
    # sequence holds for itself, before its own tokens
    per, lead = [], []
    for p, seqs in groups:
        per.append(-(-p // page))
        per += [-(-(p % page + n) // page) for _, n in seqs]
    tab, pages = _table(per, 3, seed)
    rows, lens, new, of, prefix, at = [], [], [], [], [], 0
    for g, (p, seqs) in enumerate(groups):
        prefix.append(tab[at, :-(-p // page)])
        for i, (a, n) in enumerate(seqs):
            rows.append(np.concatenate([tab[at, :p // page], tab[at + 1 + i, :per[at + 1 + i]]]))
            lens.append(p + n)
            new.append(a)
            of.append(g)
        at += 1 + len(seqs)
    table = np.zeros((len(rows), max(len(r) for r in rows)), np.int32)
    for b, r in enumerate(rows):
        table[b, :len(r)] = r
    ptable = np.zeros((len(groups), max(max(len(r) for r in prefix), 1)), np.int32)
    for g, r in enumerate(prefix):
        ptable[g, :len(r)] = r
    st = dict(case=c, groups=groups, lens=lens, new=new, of=of, table=_i32(table), ptable=_i32(ptable))
    # every token where it lies among k and v
    parts, writes, at = [], [], 0
    for g, (p, seqs) in enumerate(groups):
        writes.append((None, g, 0, p, torch.arange(at, at + p, device=DEV)))
        head = at + p // page * page
        nxt = at + p
        for _, n in seqs:
            b = len(parts)
            parts.append((nxt, n))
            mine = torch.cat([torch.arange(head, at + p, device=DEV),
                              torch.arange(nxt, nxt + n, device=DEV)])
            writes.append((b, g, p // page * page, p + n, mine))
            nxt += n
        at = nxt
    # the new tokens' queries, keys and values come out of one projection
    T, Hq = sum(new), c["heads"]
    fresh = torch.cat([torch.arange(lo + n - a, lo + n, device=DEV) for (lo, n), a in zip(parts, new)])
    fused = torch.empty(T, Hq + 2 * H, D, device=DEV, dtype=k.dtype)
    fused[:, :Hq], fused[:, Hq:Hq + H], fused[:, Hq + H:] = q, k[fresh], v[fresh]
    st["q"], st["k"], st["v"] = fused[:, :Hq], fused[:, Hq:Hq + H], fused[:, Hq + H:]
    if own:
        import jhq_gpu_amd as jg
        cache = jg.KVCache(pages, page, H, D, bits=c["bits"], device=DEV)
        for b, g, lo, hi, mine in writes:
            if hi > lo:
                t = st["ptable"][g:g + 1] if b is None else st["table"][b:b + 1]
                cache.write(k[mine], v[mine], cache.batch(t.contiguous(), _i32([hi]), _i32([0, hi - lo]),
                                                          hi - lo, hi - lo, hi))
        step = cache.batch(st["table"], _i32(lens), _i32(_cu(new)), T, max(new), max(lens))
        cu, most = _cu(new), _cu([len(s) for _, s in groups])
        rows = [int(cu[b] - cu[a]) for a, b in zip(most[:-1], most[1:])]
        prefix = cache.batch(st["ptable"], _i32([p for p, _ in groups]), _i32(_cu(rows)), T, max(rows),
                             max(p for p, _ in groups))
        st.update(cache=cache, step=step, prefix=prefix,
                  out=torch.empty(T, Hq, D, device=DEV, dtype=k.dtype),
                  work=torch.empty(cache.work_bytes(step, Hq, prefix=prefix), device=DEV,
                                   dtype=torch.uint8))
        if c["kind"] == "step":
            st.update(rotary=_rotary(c), turned=torch.empty(T, Hq, D, device=DEV, dtype=k.dtype))
        return st
    st.update(_store(c, pages))
    for b, g, lo, hi, mine in writes:
        t = st["ptable"][g] if b is None else st["table"][b]
        _put(st, _slots(t, page, lo, hi), k[mine], v[mine])
    if c["kind"] == "step":
        w, st["size"] = _frequencies(c)
        st["freq"] = torch.from_numpy(w).to(DEV)
        st["pos"] = torch.cat([torch.arange(n - a, n, device=DEV) for a, n in zip(new, lens)])
    return st


# ---- the plain forms --------------------------------------------------------

def _slots(table, page, lo, hi):
    pos = torch.arange(lo, hi, device=DEV)
    return table[pos // page].long() * page + pos % page


def _put(st, slots, k, v):
    c = st["case"]
    top = 127.0 if c["bits"] == 8 else 7.0
    step = max(1, (1 << 27) // (c["kv_heads"] * c["head_dim"]))
    for i in range(0, slots.numel(), step):
        s = slots[i:i + step]
        for x, codes, scales in ((k, st["kc"], st["ks"]), (v, st["vc"], st["vs"])):
            f = x[i:i + step].float()
            amax = f.abs().amax(-1, keepdim=True)
            live = amax >= FLOOR
            code = torch.round(f * top / torch.where(live, amax, torch.ones_like(amax)))
            codes[s] = torch.where(live, code, torch.zeros_like(code)).to(torch.int8)
            scales[s] = torch.where(live, amax / top, torch.zeros_like(amax))


def _turn(st, x):
    """Rows x [T, heads, D] turned to their positions, in float32."""
    c = st["case"]
    r = c["rot"]
    angle = (st["pos"].double()[:, None] * st["freq"])[:, None, :]
    cos, sin = (torch.cos(angle) * st["size"]).float(), (torch.sin(angle) * st["size"]).float()
    if c.get("inverse"):
        sin = -sin
    f = x.float()
    y = f.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = f[..., a] * cos - f[..., b] * sin
    y[..., b] = f[..., b] * cos + f[..., a] * sin
    return y


def _values(st, slots):
    t = TYPES[st["case"]["dtype"]]
    return [torch.cat([(codes[s].float() * scales[s]).to(t) for s in slots.split(1 << 17)])
            for codes, scales in ((st["kc"], st["ks"]), (st["vc"], st["vs"]))]


def _run_moved(st):
    c = st["case"]
    src = st.get("slots")
    if c["kind"] == "fork":
        in_page = torch.arange(c["page"], device=DEV)
        src = (st["src"].long()[:, None] * c["page"] + in_page).reshape(-1)
    for x in ("kc", "vc", "ks", "vs"):
        st[x][st["new"]] = st[x][src]
    return _values(st, st["new"])


def _attend(st, q):
    c = st["case"]
    H, D = c["kv_heads"], c["head_dim"]
    G = c["heads"] // H
    scale = 1.0 / math.sqrt(D)
    out = torch.zeros(sum(st["new"]), c["heads"], D, device=DEV, dtype=q.dtype)
    at = 0
    for b, (a, f) in enumerate(zip(st["new"], st["lens"])):
        p = st["groups"][st["of"][b]][0]
        slot = torch.cat([_slots(st["ptable"][st["of"][b]], c["page"], 0, p),
                          _slots(st["table"][b], c["page"], p, f)])
        qb = q[at:at + a].float().reshape(a, H, G, D)
        hidden = torch.zeros(a, f, dtype=torch.bool, device=DEV)
        if c["causal"]:
            hidden = torch.arange(f, device=DEV)[None] > torch.arange(f - a, f, device=DEV)[:, None]
        # as many key heads at once as the score matrix allows
        hs = max(1, min(H, (1 << 29) // (a * G * f)))
        for h in range(0, H, hs):
            kx, vx = [(codes[slot, h:h + hs].float() * scales[slot, h:h + hs]).transpose(0, 1)
                      .contiguous() for codes, scales in ((st["kc"], st["ks"]),
                                                          (st["vc"], st["vs"]))]
            qr = qb[:, h:h + hs].permute(1, 0, 2, 3).reshape(-1, a * G, D)
            s = torch.matmul(qr, kx.transpose(1, 2).contiguous()) * scale
            s = s.reshape(-1, a, G, f).masked_fill(hidden[None, :, None, :], -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            e = e / e.sum(-1, keepdim=True)
            o = torch.matmul(e.reshape(-1, a * G, f), vx).reshape(-1, a, G, D)
            out[at:at + a, h * G:(h + hs) * G] = o.permute(1, 0, 2, 3).reshape(a, -1, D).to(out.dtype)
        at += a
    return out


def run(state):
    st = state
    c = st["case"]
    if own:
        if c["kind"] == "rotary":
            return st["rotary"].apply(st["x"], st["pos"], inverse=c["inverse"], out=st["out"])
        if c["kind"] in ("fork", "compact"):
            if c["kind"] == "fork":
                st["cache"].copy_pages(st["src"], st["dst"])
            else:
                st["cache"].copy(st["slots"], st["moved"])
            return list(st["cache"].read(st["moved"], k_out=st["k_out"], v_out=st["v_out"]))
        q = st["q"]
        if c["kind"] == "step":
            q = st["rotary"].apply(q, st["step"], out=st["turned"])
            st["cache"].write(st["k"], st["v"], st["step"], rotary=st["rotary"])
        out = st["cache"].attend(q, st["step"], causal=c["causal"], prefix=st["prefix"], out=st["out"],
                                 work=st["work"])
        return [q, out] if c["kind"] == "step" else out
    if c["kind"] == "rotary":
        return _turn(st, st["x"]).to(st["x"].dtype)
    if c["kind"] in ("fork", "compact"):
        return _run_moved(st)
    if c["kind"] == "shared":
        return _attend(st, st["q"])
    q = _turn(st, st["q"]).to(st["q"].dtype)
    fresh = torch.cat([_slots(st["table"][b], c["page"], f - a, f)
                       for b, (a, f) in enumerate(zip(st["new"], st["lens"]))])
    _put(st, fresh, _turn(st, st["k"]), st["v"])
    return [q, _attend(st, q)]


# ---- 64 bits ----------------------------------------------------------------

def _value64(x, bits):
    """What the cache holds of rows x, in float64."""
    x = x.double()
    top = 2 ** (bits - 1) - 1
    big = x.abs().max(-1, keepdim=True).values
    safe = big.clamp_min(FLOOR)
    return torch.where(big < FLOOR, 0.0 * x, (x * top / safe).round() * (safe / top))


def _turn64(c, x, pos):
    """Pairs as complex numbers times size * exp(i p f)."""
    r, f = c["rot"], c["factor"]
    j = torch.arange(0, r, 2, dtype=torch.float64, device=DEV)
    base, size = c["base"], 1.0
    if c["scaling"] == "ntk":
        base = base * f ** (r / (r - 2.0))
    freq = torch.exp(-j / r * math.log(base))
    slow = freq / f
    if c["scaling"] == "linear":
        freq = slow
    elif c["scaling"] == "bands":
        waves = 2 * math.pi / freq
        mix = (c["length"] / waves - 1.0) / (4.0 - 1.0)
        mid = (1 - mix) * slow + mix * freq
        freq = torch.where(waves > c["length"], slow, torch.where(waves < c["length"] / 4.0, freq, mid))
    elif c["scaling"] == "yarn":
        edge = [r * math.log(c["length"] / (n * 2 * math.pi)) / (2 * math.log(c["base"]))
                for n in (32.0, 1.0)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
        ramp = ((j / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        freq = slow * ramp + freq * (1 - ramp)
        size = 1.0 + 0.1 * math.log(f)
    angle = pos.double()[:, None, None] * freq
    if c.get("inverse"):
        angle = -angle
    turn = torch.polar(torch.full_like(angle, size), angle)
    y = x.double().clone()
    head = y[..., :r]
    pair = head.unflatten(-1, (r // 2, 2)) if c["interleaved"] else \
        head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    y[..., :r] = (z if c["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    return y


def exact(case, seed):
    c = case
    if c["kind"] == "rotary":
        _, _, x, pos = _rope_inputs(c, seed)
        return _turn64(c, x, pos).cpu()
    if c["kind"] in ("fork", "compact"):
        if c["kind"] == "fork":
            src = np.random.default_rng(c["lens"]).integers(0, c["parents"], c["copies"])
            at = (src[:, None] * c["page"] + np.arange(c["page"])).reshape(-1)
            n = c["parents"] * c["page"]
        else:
            lens, keep = _kept(c)
            at = np.concatenate([s + j for s, j in zip(_cu(lens), keep)])
            n = sum(lens)
        k, v, _ = _rows(c, n, _gen(seed))
        at = torch.from_numpy(at).to(DEV)
        return [_value64(x[at], c["bits"]).cpu() for x in (k, v)]
    groups, k, v, q = _shared_inputs(c, seed)
    H, D, bits = c["kv_heads"], c["head_dim"], c["bits"]
    G = c["heads"] // H
    turned = None
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    if c["kind"] == "step":
        pos = torch.cat([torch.arange(p + n - a, p + n, device=DEV) for p, s in groups for a, n in s])
        turned = _turn64(c, q, pos)
        q = turned.to(q.dtype)  # attention starts from the queries that came out
    row = tok = 0
    for p, seqs in groups:
        nxt = tok + p
        for a, n in seqs:
            f = p + n
            at = torch.cat([torch.arange(tok, tok + p, device=DEV), torch.arange(nxt, nxt + n, device=DEV)])
            ks, vs = k[at].double(), v[at].double()
            if c["kind"] == "step":
                ks[f - a:] = _turn64(c, ks[f - a:], torch.arange(f - a, f, device=DEV))
            later = torch.arange(f, device=DEV)[None] > torch.arange(f - a, f, device=DEV)[:, None]
            for h in range(H):
                kh, vh = _value64(ks[:, h], bits), _value64(vs[:, h], bits)
                for i in range(h * G, h * G + G):
                    s = q[row:row + a, i].double() @ kh.t() / math.sqrt(D)
                    if c["causal"]:
                        s[later] = -math.inf
                    out[row:row + a, i] = torch.softmax(s, -1) @ vh
            row += a
            nxt += n
        tok = nxt
    return out.cpu() if turned is None else [turned.cpu(), out.cpu()]
