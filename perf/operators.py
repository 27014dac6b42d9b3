"""The operators around the paged key/value cache, measured: rotary positions
written into the pages, attention over the pages of a ragged batch (sliding
window and sinks, shared prefixes), and the moves of pages.

With `own` false `run()` computes them in elementary torch operations on the
same pages; with `own` true it makes the calls of tang_amd.capi.  `prepare()`
gives both sides the same inputs and the same pages: the cache hands out its
lowest free page first, so the page tables follow from the order in which
sequences grow.  Where `own` is true it puts them into the library's objects
(the cache with its sequences, the begun batch, buffers), which a program has
in hand before the call.
"""
import math
import random

import torch

own = False

# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # One new token of one chat: its step begins, then q, k and v of four
        # layers are rotated and stored. The smallest call: latency.
        dict(name="append_token", kind="append", B=1, heads=32, kv_heads=8, hd=128, page=16, lo=4000, hi=4000, q_lo=1, q_hi=1, layers=4,
             x="f32", cache="f16", layout="interleaved", rot=128, scaling="none"),
        # A decode step of 61 sequences of very different lengths, bf16
        # throughout, half of each head rotated in the half layout.
        dict(name="append_batch", kind="append", B=61, heads=16, kv_heads=8, hd=64, page=32, lo=20, hi=20000, q_lo=1, q_hi=1, layers=4,
             x="bf16", cache="bf16", layout="half", rot=32, scaling="ramp"),
        # Five prompts of 16000 tokens in all, positions scaled for long contexts.
        dict(name="append_prompt", kind="append", B=5, heads=32, kv_heads=8, hd=128, page=16, lo=0, hi=700, q_lo=900, q_hi=8000, layers=1,
             x="f32", cache="f16", layout="half", rot=128, scaling="bands"),
        # One new token over an 8K context, four layers: latency, and the
        # split of one long row.
        dict(name="attn_token", kind="attn", B=1, heads=32, kv_heads=8, hd=128, page=16, lo=8191, hi=8191, q_lo=1, q_hi=1, prefix=0, window=0,
             sinks=0, layers=4, q="f32", cache="f16"),
        # A decode step of 48 sequences from 100 to 16000 positions: the
        # cache's bandwidth, with ragged lengths.
        dict(name="attn_batch", kind="attn", B=48, heads=32, kv_heads=8, hd=128, page=16, lo=100, hi=16000, q_lo=1, q_hi=1, prefix=0, window=0,
             sinks=0, layers=1, q="bf16", cache="bf16"),
        # Decode of long streams with a window of 1000 positions and four sinks.
        dict(name="attn_window_batch", kind="attn", B=24, heads=16, kv_heads=2, hd=64, page=32, lo=500, hi=30000, q_lo=1, q_hi=1, prefix=0,
             window=1000, sinks=4, layers=2, q="f32", cache="f16"),
        # A whole prompt of 8192 tokens, bf16: matrix work.
        dict(name="attn_prompt", kind="attn", B=1, heads=32, kv_heads=8, hd=128, page=16, lo=0, hi=0, q_lo=8192, q_hi=8192, prefix=0, window=0,
             sinks=0, layers=1, q="bf16", cache="bf16"),
        # Prompt chunks of six sequences of odd lengths behind what they have
        # cached, window and sinks, f32 queries.
        dict(name="attn_window_chunks", kind="attn", B=6, heads=16, kv_heads=8, hd=128, page=16, lo=33, hi=2500, q_lo=17, q_hi=1500, prefix=0,
             window=1024, sinks=4, layers=1, q="f32", cache="f16"),
        # 64 answers to one long document: decode with 8192 shared positions.
        dict(name="prefix_batch", kind="attn", B=64, heads=32, kv_heads=8, hd=128, page=16, lo=30, hi=400, q_lo=1, q_hi=1, prefix=8192, window=0,
             sinks=0, layers=2, q="f32", cache="f16"),
        # Eight samples of one short prompt.
        dict(name="prefix_small", kind="attn", B=8, heads=16, kv_heads=4, hd=64, page=16, lo=5, hi=60, q_lo=1, q_hi=1, prefix=992, window=0,
             sinks=0, layers=2, q="bf16", cache="bf16"),
        # Eight continuations of a prompt begin: each gets its own copy of the
        # last page, in eight layers, and goes again.
        dict(name="pages_fork", kind="fork", n=8, kv_heads=8, hd=128, page=16, length=1000, layers=8, cache="f16"),
        # A long sequence keeps some of its positions (the others are behind
        # the window or were rejected), other pages went before: its rows are
        # gathered, then the pages close the gap.
        dict(name="pages_compact", kind="compact", kv_heads=8, hd=128, page=16, length=20000, keep=9001, hole=700, layers=8, cache="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attn", "attn", "attn", "chunks", "chunks", "prefix", "prefix", "fork", "compact"])
    kv_heads = rng.choice([1, 2, 4, 8])
    hd, page = rng.choice([64, 128, 128, 256, 80, 96]), rng.choice([16, 16, 32, 64])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    q, cache = rng.choice([("f32", "f16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
    if kind == "append":
        prompts = rng.random() < 0.4
        B = _log_int(rng, 1, 8 if prompts else 128)
        lo, hi = rng.randrange(0, 300), _log_int(rng, 300, 20000)
        rot = hd if rng.random() < 0.5 else 2 * rng.randrange(4, hd // 2)
        return dict(kind=kind, B=B, heads=heads, kv_heads=kv_heads, hd=hd, page=page, lo=lo, hi=hi, q_lo=rng.randrange(5, 400) if prompts else 1,
                    q_hi=rng.randrange(400, 2000) if prompts else 1, layers=1 if prompts else rng.randrange(1, 5), x=q, cache=cache,
                    layout=rng.choice(["half", "interleaved"]), rot=rot, scaling=rng.choice(["none", "linear", "base", "bands", "ramp"]))
    window = rng.choice([0, 0, rng.randrange(100, 4000)])
    sinks = rng.choice([0, 4, rng.randrange(1, 40)]) if window else 0
    if kind in ("attn", "prefix"):
        B = _log_int(rng, 1 if kind == "attn" else 2, 64)
        prefix = page * rng.randrange(1, 8000 // page) if kind == "prefix" else 0
        hi = _log_int(rng, 40, 2000 if prefix else 12000)
        return dict(kind="attn", B=B, heads=heads, kv_heads=kv_heads, hd=hd, page=page, lo=rng.randrange(0, 40), hi=hi, q_lo=1,
                    q_hi=rng.choice([1, 1, rng.randrange(2, 6)]), prefix=prefix, window=window, sinks=sinks, layers=rng.randrange(1, 4), q=q, cache=cache)
    if kind == "chunks":
        return dict(kind="attn", B=rng.randrange(1, 6), heads=heads, kv_heads=kv_heads, hd=hd, page=page, lo=rng.randrange(0, 200),
                    hi=rng.randrange(200, 3000), q_lo=rng.randrange(1, 60), q_hi=_log_int(rng, 60, 2000), prefix=0, window=window, sinks=sinks,
                    layers=1, q=q, cache=cache)
    layers = rng.randrange(1, 9)
    if kind == "fork":
        n = page * rng.randrange(1, 100)
        return dict(kind=kind, n=_log_int(rng, 1, 64), kv_heads=kv_heads, hd=hd, page=page, length=n + rng.randrange(1, page), layers=layers, cache=cache)
    n = _log_int(rng, 300, 16000)
    keep = rng.randrange(1, n)
    return dict(kind=kind, kv_heads=kv_heads, hd=hd, page=page, length=n, keep=keep, hole=rng.randrange(1, 800), layers=layers, cache=cache)


# ---------------------------------------------------------------------------
# Shapes: they follow from the case alone
# ---------------------------------------------------------------------------

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _spread(lo, hi, n, rng):
    """n lengths over [lo, hi], even in their logarithm, in any order."""
    v = [int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * (i + 0.5) / n))) - 1 for i in range(n)]
    rng.shuffle(v)
    return v


def _lengths(c):
    """Positions that each sequence has cached of its own, and its new ones."""
    rng = random.Random(c["B"] * 7919 + c["hi"])
    return _spread(c["lo"], c["hi"], c["B"], rng), _spread(c["q_lo"], c["q_hi"], c["B"], rng)


class _Pages:
    """The tables of sequences that grow in turns, lowest free page first (none goes)."""

    def __init__(self, page, used=0):
        self.page, self.used, self.table, self.steps = page, used, [], []

    def grow(self, i, length):
        need = -(-length // self.page)
        while len(self.table[i]) < need:
            self.table[i].append(self.used)
            self.used += 1
        self.steps.append((i, length))


def _tables(c, prefix):
    """The batch's sequences: shared pages first, then grown a few pages at a
    time in turns, then by their new positions in the batch's order."""
    starts, news = _lengths(c)
    P = _Pages(c["page"])
    shared = list(range(prefix // c["page"]))
    P.used = len(shared)
    P.table = [list(shared) for _ in starts]
    at, turn = [0] * len(starts), 5 * c["page"]
    while any(a < s for a, s in zip(at, starts)):
        for i, s in enumerate(starts):
            if at[i] < s:
                at[i] = min(s, at[i] + turn)
                P.grow(i, prefix + at[i])
        turn = min(turn * 2, 1024 * c["page"])
    steps = list(P.steps)
    for i, (s, n) in enumerate(zip(starts, news)):
        P.grow(i, prefix + s + n)
    return [prefix + s for s in starts], news, P.table, P.used, steps


def _freqs(c, device):
    """Frequencies of the pairs and the factor of the tables, in 64 bits."""
    rot, base, kind = c["rot"], 10000.0, c["scaling"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    if kind == "base":
        base = base * 4.0 ** (rot / (rot - 2))
    f = base ** (-2.0 * i / rot)
    if kind == "linear":
        return f / 4.0, 1.0
    if kind == "bands":  # short waves as they are, long ones stretched, a ramp between
        waves = 8192.0 * f / (2 * math.pi)
        keep = ((waves - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return keep * f + (1 - keep) * f / 8.0, 1.0
    if kind == "ramp":  # a ramp over the pairs' indices, and warmer tables
        at = lambda turns: rot * math.log(4096.0 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return (1 - ramp) * f + ramp * f / 16.0, 0.1 * math.log(16.0) + 1.0
    return f, 1.0


#: The same scalings as the library takes them.
_SCALINGS = {"none": {}, "linear": dict(kind="linear", factor=4.0), "base": dict(kind="base", factor=4.0),
             "bands": dict(kind="bands", factor=8.0, original_len=8192, low=1.0, high=4.0),
             "ramp": dict(kind="ramp", factor=16.0, original_len=4096, low=1.0, high=32.0)}


# ---------------------------------------------------------------------------
# The library's objects
# ---------------------------------------------------------------------------

_dev = None


def _device():
    from tang_amd import capi
    global _dev
    if _dev is None:
        _dev = capi.HipComputeDevice(0)
    return _dev


class _Span:
    def __init__(self, ptr, typestr, shape, keep):
        self.keep = keep
        self.__cuda_array_interface__ = dict(shape=shape, typestr=typestr, data=(ptr, False), version=2, strides=None)


def _at(ptr, dt, shape, keep):
    """A tensor over device memory that `keep` holds."""
    t = torch.as_tensor(_Span(ptr, {"f32": "<f4", "f16": "<f2", "bf16": "<i2"}[dt], shape, keep), device="cuda")
    return t.view(torch.bfloat16) if dt == "bf16" else t


class _Buf:
    """A library buffer and the tensor over its memory, with t's values."""

    def __init__(self, t):
        from tang_amd import capi
        dt = {v: k for k, v in _DT.items()}[t.dtype]
        self.buf = _device().alloc(t.numel(), {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[dt])
        self.t = _at(self.buf.device_ptr(), dt, tuple(t.shape), self.buf)
        self.t.copy_(t)


def _cache(c, pages, seqs, length, pool):
    """A cache whose pages hold what `pool` does (and whose memory it then is)."""
    from tang_amd import capi
    dt = {"f16": capi.F16, "bf16": capi.BF16}[c["cache"]]
    cache = _device().kv_cache(c["layers"], c["kv_heads"], c["hd"], c["page"], pages, seqs, length, dt)
    view = _at(cache.page_pointers(0)[0], c["cache"], tuple(pool.shape), cache)
    view.copy_(pool)
    return cache, view


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, dt, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(_DT[dt])


def _pool(c, g, pages):
    """[layer][K, V][page][kv head][position][dim]; all pages hold what some sequence left there."""
    return _normal(g, c["cache"], c["layers"], 2, pages, c["kv_heads"], c["page"], c["hd"])


class _State:
    pass


def _rows(c, starts, news, table):
    """Of every new row: its sequence, position, page and place in the page."""
    seq = [i for i, n in enumerate(news) for _ in range(n)]
    pos = [s + j for s, n in zip(starts, news) for j in range(n)]
    t = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    return t(seq), t(pos), t([table[i][p // c["page"]] for i, p in zip(seq, pos)]), t([p % c["page"] for p in pos])


def _prepare_append(c, seed):
    g, S = _gen(seed), _State()
    starts, news, table, pages, steps = _tables(c, 0)
    R, top = sum(news), max(s + n for s, n in zip(starts, news))
    S.pool = _pool(c, g, pages)
    S.q = [_normal(g, c["x"], R, c["heads"], c["hd"]) for _ in range(c["layers"])]
    S.k, S.v = ([_normal(g, c["x"], R, c["kv_heads"], c["hd"]) for _ in range(c["layers"])] for _ in range(2))
    if own:
        from tang_amd import capi
        cs, sn = capi.rope_tables_scaled(c["rot"], top, 10000.0, **_SCALINGS[c["scaling"]])
        S.cos, S.sin = _device().upload(cs), _device().upload(sn)
        S.cache, S.pool = _cache(c, pages, c["B"], top, S.pool)
        S.seqs = S.cache.seq_create(c["B"])
        for i, n in steps:
            S.cache.seq_resize(S.seqs[i], n)
        S.batch, S.news, S.none = S.cache.batch(c["B"], R, c["heads"]), news, [0] * c["B"]
        S.out = [_Buf(torch.zeros_like(q)) for q in S.q]
        S.q, S.k, S.v = ([_Buf(t) for t in v] for v in (S.q, S.k, S.v))
        S.layout = {"interleaved": capi.ROPE_INTERLEAVED, "half": capi.ROPE_HALF}[c["layout"]]
        return S
    f, m = _freqs(c, "cuda")
    angle = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * f
    S.cos, S.sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    _, S.pos, S.page, S.place = _rows(c, starts, news, table)
    return S


def _prepare_attn(c, seed):
    g, S = _gen(seed), _State()
    starts, news, table, pages, steps = _tables(c, c["prefix"])
    R, top = sum(news), max(s + n for s, n in zip(starts, news))
    S.pool = _pool(c, g, pages)
    S.q = [_normal(g, c["q"], R, c["heads"], c["hd"]) for _ in range(c["layers"])]
    if own:
        S.cache, S.pool = _cache(c, pages, c["B"] + 1, top, S.pool)
        if c["prefix"]:
            first = S.cache.seq_create(1)[0]
            S.cache.seq_resize(first, c["prefix"])
            S.seqs = S.cache.seq_fork(first, c["B"])
        else:
            S.seqs = S.cache.seq_create(c["B"])
        for i, n in steps:
            S.cache.seq_resize(S.seqs[i], n)
        S.batch = S.cache.batch(c["B"], R, c["heads"])
        S.batch.begin(S.seqs, news)
        S.out = [_Buf(torch.zeros_like(q)) for q in S.q]
        S.q = [_Buf(q) for q in S.q]
        return S
    # the rows as a block [sequence][new position], row R behind the others standing for none
    B, M, P = c["B"], max(news), max(len(t) for t in table)
    seq, pos, _, _ = _rows(c, starts, news, table)
    place = torch.tensor([j for n in news for j in range(n)], dtype=torch.int64, device="cuda")
    S.block = torch.full((B, M), R, dtype=torch.int64, device="cuda")
    S.block[seq, place] = torch.arange(R, device="cuda")
    S.pos = torch.zeros(B, M, dtype=torch.int64, device="cuda")
    S.pos[seq, place] = pos
    S.row = (seq, place)
    S.table = torch.tensor([t + [0] * (P - len(t)) for t in table], dtype=torch.int64, device="cuda")
    return S


def _prepare_fork(c, seed):
    g, S = _gen(seed), _State()
    have = -(-c["length"] // c["page"])
    S.pool = _pool(c, g, have + c["n"])
    if own:
        S.cache, S.pool = _cache(c, have + c["n"], c["n"] + 1, c["length"] + 1, S.pool)
        S.parent = S.cache.seq_create(1)[0]
        S.cache.seq_resize(S.parent, c["length"])
        S.batch, S.ones = S.cache.batch(c["n"], c["n"], c["kv_heads"]), [1] * c["n"]
        return S
    S.src = torch.full((c["n"],), have - 1, dtype=torch.int64, device="cuda")
    S.dst = torch.arange(have, have + c["n"], device="cuda")
    return S


def _compact_plan(c):
    """Positions that stay, and the moves of pages that close the gap."""
    rng = random.Random(c["length"] * 31 + c["keep"])
    kept = sorted(rng.sample(range(c["length"]), c["keep"]))
    have, need = -(-c["length"] // c["page"]), -(-c["keep"] // c["page"])
    first = have + c["hole"]
    live = have + need
    movers = [p for p in range(first, first + need) if p >= live]
    holes = [p for p in range(have, first) if p < live]
    return kept, have, need, first, movers, holes


def _prepare_compact(c, seed):
    g, S = _gen(seed), _State()
    kept, have, need, first, movers, holes = _compact_plan(c)
    S.pool = _pool(c, g, first + need)
    if own:
        import numpy as np
        S.cache, S.pool = _cache(c, first + need, 3, max(c["length"], c["hole"] * c["page"]), S.pool)
        S.parent = S.cache.seq_create(1)[0]
        S.cache.seq_resize(S.parent, c["length"])
        S.kept, S.hole = np.array(kept, np.uint32), c["hole"] * c["page"]
        return S
    t = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    at, to = t(kept), torch.arange(c["keep"], device="cuda")
    S.from_page, S.from_place = at // c["page"], at % c["page"]
    S.to_page, S.to_place = first + to // c["page"], to % c["page"]
    S.movers, S.holes = t(movers), t(holes)
    return S


_PREPARE = {"append": _prepare_append, "attn": _prepare_attn, "fork": _prepare_fork, "compact": _prepare_compact}


def prepare(case, seed):
    S = _PREPARE[case["kind"]](case, seed)
    S.case = case
    if own:
        torch.cuda.synchronize()  # the library works on a stream of its own
    return S


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _rotate(x, cos, sin, rot, layout):
    x = x.float()
    r, rest = x[..., :rot], x[..., rot:]
    if layout == "interleaved":
        a, b = r[..., 0::2], r[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)
    a, b = r[..., :rot // 2], r[..., rot // 2:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)


def _plain_append(S, c, layer):
    cos, sin = S.cos[S.pos][:, None], S.sin[S.pos][:, None]
    S.pool[layer, 0][S.page, :, S.place] = _rotate(S.k[layer], cos, sin, c["rot"], c["layout"]).to(S.pool.dtype)
    S.pool[layer, 1][S.page, :, S.place] = S.v[layer].to(S.pool.dtype)
    return _rotate(S.q[layer], cos, sin, c["rot"], c["layout"]).to(S.q[layer].dtype)


def _plain_attn(S, c, layer):
    q = S.q[layer]
    B, P, H, KH, D = S.table.shape[0], S.table.shape[1], c["heads"], c["kv_heads"], c["hd"]
    G, M, L = H // KH, S.block.shape[1], P * c["page"]
    k, v = (S.pool[layer, w][S.table].transpose(1, 2).reshape(B * KH, L, D).float() for w in (0, 1))
    x = torch.cat((q, torch.zeros_like(q[:1])))[S.block].float()  # [B, M, H, D]
    x = x.reshape(B, M, KH, G, D).permute(0, 2, 3, 1, 4).reshape(B * KH, G * M, D)
    s = torch.bmm(x, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(D)).view(B, KH, G, M, L)
    key, pos = torch.arange(L, device="cuda"), S.pos[:, :, None]
    seen = key <= pos
    if c["window"]:
        seen &= (key > pos - c["window"]) | (key < c["sinks"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1).reshape(B * KH, G * M, 1)
    o = torch.bmm(s.view(B * KH, G * M, L), v).div_(total)
    o = o.view(B, KH, G, M, D).permute(0, 3, 1, 2, 4).reshape(B, M, H, D)
    return o[S.row].to(q.dtype)


def _run_append(S, c):
    if own:
        S.batch.begin(S.seqs, S.news)
        [S.batch.append(l, S.q[l].buf, S.k[l].buf, S.v[l].buf, S.out[l].buf, S.cos, S.sin, c["rot"], S.layout) for l in range(c["layers"])]
        S.batch.trim(S.none)  # the next pass stores the same positions again
        return [o.t for o in S.out], S.pool
    return [_plain_append(S, c, l) for l in range(c["layers"])], S.pool


def _run_attn(S, c):
    if own:
        [S.batch.attention(l, S.q[l].buf, S.out[l].buf, window=c["window"], sinks=c["sinks"]) for l in range(c["layers"])]
        return [o.t for o in S.out]
    return [_plain_attn(S, c, l) for l in range(c["layers"])]


def _run_fork(S, c):
    if own:
        children = S.cache.seq_fork(S.parent, c["n"])
        S.batch.begin(children, S.ones)
        S.cache.seq_free(children)
        return S.pool
    S.pool[:, :, S.dst] = S.pool[:, :, S.src]
    return S.pool


def _run_compact(S, c):
    if own:
        gap = S.cache.seq_create(1)
        S.cache.seq_resize(gap[0], S.hole)
        child = S.cache.seq_fork(S.parent, 1)
        S.cache.seq_select(child[0], S.kept)
        S.cache.seq_free(gap)
        S.cache.compact()
        S.cache.seq_free(child)
        return S.pool
    S.pool[:, :, S.to_page, :, S.to_place] = S.pool[:, :, S.from_page, :, S.from_place]
    S.pool[:, :, S.holes] = S.pool[:, :, S.movers]
    return S.pool


_RUN = {"append": _run_append, "attn": _run_attn, "fork": _run_fork, "compact": _run_compact}


def run(state):
    return _RUN[state.case["kind"]](state, state.case)


# ---------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ---------------------------------------------------------------------------


def _exact_append(c, seed):
    g = _gen(seed)
    starts, news, table, pages, _ = _tables(c, 0)
    R = sum(news)
    pool = _pool(c, g, pages).double()
    q = [_normal(g, c["x"], R, c["heads"], c["hd"]).double() for _ in range(c["layers"])]
    k, v = ([_normal(g, c["x"], R, c["kv_heads"], c["hd"]).double() for _ in range(c["layers"])] for _ in range(2))
    f, m = _freqs(c, "cuda")
    half = c["rot"] // 2
    first = torch.arange(half, device="cuda") * (2 if c["layout"] == "interleaved" else 1)
    second = first + (1 if c["layout"] == "interleaved" else half)
    for l in range(c["layers"]):
        at = 0
        for s, n, t in zip(starts, news, table):
            pos = torch.arange(s, s + n, dtype=torch.float64, device="cuda")
            turn = torch.polar(torch.full((n, half), m, dtype=torch.float64, device="cuda"), pos[:, None] * f)
            for x in (q[l], k[l]):  # a pair is a complex number that is turned
                z = torch.complex(x[at:at + n, :, first], x[at:at + n, :, second]) * turn[:, None]
                x[at:at + n, :, first], x[at:at + n, :, second] = z.real, z.imag
            for j in range(0, n):
                p = s + j
                pool[l, 0, t[p // c["page"]], :, p % c["page"]] = k[l][at + j]
                pool[l, 1, t[p // c["page"]], :, p % c["page"]] = v[l][at + j]
            at += n
    return q, pool


def _exact_attn(c, seed):
    g = _gen(seed)
    starts, news, table, pages, _ = _tables(c, c["prefix"])
    R, D = sum(news), c["hd"]
    pool = _pool(c, g, pages)
    G = c["heads"] // c["kv_heads"]
    outs = []
    for l in range(c["layers"]):
        q = _normal(g, c["q"], R, c["heads"], D).double()
        out = torch.empty_like(q)
        at = 0
        for s, n, t in zip(starts, news, table):
            t = torch.tensor(t, device="cuda")
            # [kv head][position][dim] of this sequence
            k, v = (pool[l, w].index_select(0, t).double().permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, D)[:, :s + n].contiguous() for w in (0, 1))
            for a in range(0, n, 512):
                b = min(n, a + 512)
                i = torch.arange(s + a, s + b, device="cuda")[:, None]
                j = torch.arange(s + b, device="cuda")[None]
                hidden = j > i
                if c["window"]:
                    hidden = hidden | ((i - j >= c["window"]) & (j >= c["sinks"]))
                for h in range(c["heads"]):
                    w = q[at + a:at + b, h] @ k[h // G, :s + b].t().contiguous() / D ** 0.5
                    w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                    out[at + a:at + b, h] = w @ v[h // G, :s + b]
            at += n
        outs.append(out)
    return outs


def _exact_fork(c, seed):
    have = -(-c["length"] // c["page"])
    pool = _pool(c, _gen(seed), have + c["n"]).double()
    for i in range(c["n"]):
        pool[:, :, have + i] = pool[:, :, have - 1]
    return pool


def _exact_compact(c, seed):
    kept, have, need, first, movers, holes = _compact_plan(c)
    pool = _pool(c, _gen(seed), first + need).double()
    L, _, _, KH, page, D = pool.shape
    line = pool.permute(0, 1, 3, 2, 4, 5).reshape(L, 2, KH, -1, D)  # every place of every page in one line (a copy)
    line[:, :, :, first * page:first * page + len(kept)] = line[:, :, :, torch.tensor(kept, device="cuda")]
    pool = line.view(L, 2, KH, -1, page, D).permute(0, 1, 3, 2, 4, 5).contiguous()
    for a, b in zip(movers, holes):
        pool[:, :, b] = pool[:, :, a]
    return pool


_EXACT = {"append": _exact_append, "attn": _exact_attn, "fork": _exact_fork, "compact": _exact_compact}


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def _visible(c, p):
    return p + 1 if not c["window"] else min(p + 1, c["window"] + min(c["sinks"], max(0, p + 1 - c["window"])))


def _work_attn(c):
    starts, news, _, _, _ = _tables(c, c["prefix"])
    pairs = rows = 0
    first = None  # the lowest position behind the sinks that some row sees in the shared pages
    for s, n in zip(starts, news):
        pairs += sum(_visible(c, p) for p in range(s, s + n))
        low = max(0, s + 1 - c["window"]) if c["window"] else 0
        first = low if first is None else min(first, low)
        mine = max(low, c["prefix"])
        rows += s + n - mine + max(0, min(c["sinks"], mine) - c["prefix"])
    if c["prefix"]:
        first = min(first, c["prefix"])
        rows += c["prefix"] - first + min(c["sinks"], first)
    R, width = sum(news), c["heads"] * c["hd"]
    return dict(bytes=c["layers"] * (rows * c["kv_heads"] * c["hd"] * 2 * _SIZE[c["cache"]] + 2 * R * width * _SIZE[c["q"]]),
                flops=c["layers"] * 4 * width * pairs)


def work(case):
    c = case
    if c["kind"] == "attn":
        return _work_attn(c)
    if c["kind"] == "append":
        R = sum(_lengths(c)[1])
        q, kv = c["heads"] * c["hd"], 2 * c["kv_heads"] * c["hd"]
        return dict(bytes=c["layers"] * R * (2 * q * _SIZE[c["x"]] + kv * (_SIZE[c["x"]] + _SIZE[c["cache"]])),
                    flops=c["layers"] * R * 3 * c["rot"] * (c["heads"] + c["kv_heads"]))
    row = 2 * c["layers"] * c["kv_heads"] * c["hd"] * _SIZE[c["cache"]]
    if c["kind"] == "fork":  # the last page's rows: read once, written for each
        return dict(bytes=row * (c["length"] % c["page"]) * (1 + c["n"]), flops=0)
    _, _, _, _, movers, _ = _compact_plan(c)
    return dict(bytes=2 * row * (c["keep"] + len(movers) * c["page"]), flops=0)
