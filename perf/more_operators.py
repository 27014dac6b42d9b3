"""What a serving step computes around the paged cache, measured: products of
8-bit integers with a scale for each token and each channel, norms of the query
and key heads in the same pass as their rotation (into rows, or into the pages
of the cache), and the choice of tokens from given random numbers.

With `own` false `run()` computes them in elementary torch operations; with
`own` true it makes the calls of tang_amd.capi.  `prepare()` gives both sides
the same inputs; where `own` is true it puts them into the library's objects
(buffers, packed weights, the cache with its begun batch), which a program has
in hand before the call.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6

# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # One token through one square projection: the smallest product, f32 in
        # and out; latency and the weights' bandwidth.
        dict(name="i8_token", kind="i8", m=1, k=4096, n=4096, x="f32", y="f32", bias=False),
        # A decode step of 61 sequences through an up projection.
        dict(name="i8_batch", kind="i8", m=61, k=4096, n=11008, x="bf16", y="bf16", bias=False),
        # A ragged batch of prompt chunks, no size a multiple of anything, with a bias.
        dict(name="i8_odd", kind="i8", m=509, k=2047, n=5631, x="f32", y="f32", bias=True),
        # A long prompt through an up projection: matrix work.
        dict(name="i8_prompt", kind="i8", m=8192, k=4096, n=11008, x="bf16", y="bf16", bias=False),
        # The heads of one token: latency.
        dict(name="heads_token", kind="heads", rows=1, heads=32, kv_heads=8, hd=128, rot=128, layout="half", x="f32", w="f32", packed=False,
             scattered=False),
        # The packed q, k, v rows of 16000 prompt tokens, each with its own position.
        dict(name="heads_prompt", kind="heads", rows=16000, heads=32, kv_heads=8, hd=128, rot=128, layout="half", x="bf16", w="bf16",
             packed=True, scattered=True),
        # A decode step of 61 sequences: packed rows of four layers into the
        # pages, half of each head rotated.
        dict(name="pages_batch", kind="pages", B=61, lo=20, hi=20000, q_lo=1, q_hi=1, heads=16, kv_heads=8, hd=64, page=32, layers=4, rot=32,
             layout="interleaved", x="bf16", w="bf16", cache="bf16", packed=True),
        # Five prompts of some 16000 tokens in all, f32 rows into an f16 cache.
        dict(name="pages_prompt", kind="pages", B=5, lo=0, hi=700, q_lo=900, q_hi=8000, heads=32, kv_heads=8, hd=128, page=16, layers=1, rot=128,
             layout="half", x="f32", w="f32", cache="f16", packed=False),
        # One chat's next token: latency.
        dict(name="sample_token", kind="sample", rows=1, vocab=32000, x="f32", mode="all", masked=0.0),
        # 48 requests, each with its own settings (some greedy, some without
        # filters), rows that start on no 16-byte border, half the tokens masked in some.
        dict(name="sample_batch", kind="sample", rows=48, vocab=50001, x="f32", mode="mixed", masked=0.5),
        # 16 rows drawn from everything: temperature alone.
        dict(name="sample_open", kind="sample", rows=16, vocab=100000, x="f32", mode="open", masked=0.0),
        # 256 samples over a large vocabulary, logits in 16 bits (many ties).
        dict(name="sample_large", kind="sample", rows=256, vocab=131072, x="bf16", mode="nucleus", masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["i8", "i8", "i8", "heads", "pages", "sample", "sample", "sample"])
    x = rng.choice(["f32", "bf16", "f16"])
    if kind == "i8":
        m, k, n = _log_int(rng, 1, 8192), _log_int(rng, 100, 12000), _log_int(rng, 100, 16000)
        if rng.random() < 0.5:
            k, n = k // 64 * 64 or 64, n // 16 * 16 or 16
        while m * k * n > 8192 * 4096 * 11008:
            m = (m + 1) // 2
        return dict(kind=kind, m=m, k=k, n=n, x=x, y=rng.choice([x, "f32"]), bias=rng.random() < 0.4)
    if kind == "sample":
        rows, vocab = _log_int(rng, 1, 256), _log_int(rng, 1000, 200000)
        while rows * vocab > 256 * 131072:
            rows = (rows + 1) // 2
        return dict(kind=kind, rows=rows, vocab=vocab, x=x, mode=rng.choice(["all", "mixed", "mixed", "open", "nucleus"]),
                    masked=rng.choice([0.0, 0.0, 0.3, 0.9]))
    kv_heads, hd = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256, 80, 96])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    c = dict(kind=kind, heads=heads, kv_heads=kv_heads, hd=hd, rot=hd if rng.random() < 0.5 else 2 * rng.randrange(4, hd // 2),
             layout=rng.choice(["half", "interleaved"]), x=x, w=rng.choice(["f32", "bf16"]), packed=rng.random() < 0.5)
    if kind == "heads":
        rows = _log_int(rng, 1, 16000)
        while rows * heads * hd > 16000 * 40 * 128:
            rows = (rows + 1) // 2
        return dict(c, rows=rows, scattered=rng.random() < 0.5)
    prompts = rng.random() < 0.4
    return dict(c, B=_log_int(rng, 1, 8 if prompts else 128), lo=rng.randrange(0, 300), hi=_log_int(rng, 300, 20000),
                q_lo=rng.randrange(5, 400) if prompts else 1, q_hi=rng.randrange(400, 2000) if prompts else 1, page=rng.choice([16, 16, 32, 64]),
                layers=1 if prompts else rng.randrange(1, 5), cache=rng.choice(["f16", "bf16"]))


# ---------------------------------------------------------------------------
# The library's objects
# ---------------------------------------------------------------------------

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_TYPESTR = {torch.float32: "<f4", torch.float16: "<f2", torch.bfloat16: "<i2", torch.int32: "<i4", torch.int8: "|i1"}

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


def _at(ptr, dtype, shape, keep):
    """A tensor over device memory that `keep` holds."""
    t = torch.as_tensor(_Span(ptr, _TYPESTR[dtype], shape, keep), device="cuda")
    return t.view(torch.bfloat16) if dtype == torch.bfloat16 else t


class _Buf:
    """A library buffer and the tensor over its memory, with t's values."""

    def __init__(self, t):
        from tang_amd import capi
        kinds = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16, torch.int32: capi.I32, torch.int8: capi.I8}
        self.buf = _device().alloc(t.numel(), kinds[t.dtype])
        self.t = _at(self.buf.device_ptr(), t.dtype, tuple(t.shape), self.buf)
        self.t.copy_(t)


def _buf_u32(t):
    from tang_amd import capi
    b = _device().alloc(t.numel(), capi.U32)
    _at(b.device_ptr(), torch.int32, tuple(t.shape), b).copy_(t)
    return b


def _new(dt, *shape):
    return _Buf(torch.zeros(shape, dtype=_DT[dt], device="cuda"))


class _State:
    pass


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, dt, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(_DT[dt])


# ---------------------------------------------------------------------------
# Products in 8-bit integers
# ---------------------------------------------------------------------------


def _i8_inputs(c, seed):
    """Activations with a few channels of large values, as linears see them, and
    weights with a scale for each channel."""
    g = _gen(seed)
    x = torch.randn(c["m"], c["k"], generator=g, device="cuda")
    loud = torch.randint(0, c["k"], (max(1, c["k"] // 500),), generator=g, device="cuda")
    x[:, loud] *= 12.0
    w = torch.randint(-127, 128, (c["n"], c["k"]), generator=g, device="cuda", dtype=torch.int8)
    t = torch.rand(c["n"], generator=g, device="cuda") * 0.002 + 0.0005
    b = torch.randn(c["n"], generator=g, device="cuda") if c["bias"] else None
    return x.to(_DT[c["x"]]), w, t, b


def _prepare_i8(c, seed):
    S = _State()
    S.x, S.w, S.t, S.b = _i8_inputs(c, seed)
    if own:
        from tang_amd import capi
        kp = -(-c["k"] // 64) * 64
        rows = torch.zeros(c["n"], kp, dtype=torch.int8, device="cuda")
        rows[:, :c["k"]] = S.w
        w, t = _Buf(rows), _Buf(S.t)
        torch.cuda.synchronize()
        S.w = _device().q8_pack_rows(w.buf, t.buf, c["n"], c["k"])
        S.x, S.b = _Buf(S.x), None if S.b is None else _Buf(S.b)
        S.q, S.s = _device().alloc(c["m"] * kp, capi.I8), _device().alloc(c["m"], capi.F32)
        S.y = _new(c["y"], c["m"], c["n"])
    return S


def _run_i8(S, c):
    if own:
        _device().quantize_rows(S.x.buf, c["m"], c["k"], S.q, S.s)
        _device().gemm_i8(S.q, S.s, c["m"], S.w, S.y.buf, None if S.b is None else S.b.buf)
        return S.y.t
    x = S.x.float()
    s = x.abs().amax(1, keepdim=True) / 127.0
    q = (x.double() / s.double()).round_().clamp_(-127, 127).float()  # 64 bits: next to a half, 32 may round the other way
    y = torch.matmul(q, S.w.float().t()) * s * S.t
    return (y if S.b is None else y + S.b).to(_DT[c["y"]])


def _exact_i8(c, seed):
    x, w, t, b = _i8_inputs(c, seed)
    x = x.double()
    s = (x.abs().amax(1) / 127).float().double()  # the scale is held in 32 bits
    whole = torch.floor(x / s[:, None])
    part = x - whole * s[:, None]  # exact
    up = (2 * part > s[:, None]) | ((2 * part == s[:, None]) & (whole % 2 != 0))
    q = torch.where(up, whole + 1, whole)
    w = w.double().t().contiguous()
    y = torch.cat([(q[i:i + 1024] @ w) * s[i:i + 1024, None] * t.double() for i in range(0, c["m"], 1024)])
    return y if b is None else y + b.double()


def _work_i8(c):
    return dict(bytes=c["m"] * c["k"] * _SIZE[c["x"]] + c["n"] * (c["k"] + 4 + 4 * c["bias"]) + c["m"] * c["n"] * _SIZE[c["y"]],
                flops=2 * c["m"] * c["n"] * c["k"])


# ---------------------------------------------------------------------------
# Norms of heads with the rotation, into rows or into the cache's pages
# ---------------------------------------------------------------------------


def _freqs(c):
    return 10000.0 ** (-2.0 * torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda") / c["rot"])


def _head_weights(c, g):
    return [(1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda")).to(_DT[c["w"]]) for _ in range(2)]


def _qkv(c, g, R):
    """Rows of q, k and v, or (packed) the rows of one product that hold all three."""
    H, K, D = c["heads"], c["kv_heads"], c["hd"]
    if c["packed"]:
        return [_normal(g, c["x"], R, H + 2 * K, D) * 3]
    return [_normal(g, c["x"], R, n, D) * 3 for n in (H, K, K)]


def _split(c, rows):
    H, K = c["heads"], c["kv_heads"]
    return (rows[0][:, :H], rows[0][:, H:H + K], rows[0][:, H + K:]) if c["packed"] else rows


def _turned_norm(x, w, cos, sin, c):
    """Each head over its root mean square, times w, its pairs turned; in 32 bits."""
    x, rot = x.float(), c["rot"]
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    r, rest = x[..., :rot], x[..., rot:]
    if c["layout"] == "interleaved":
        a, b = r[..., 0::2], r[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)
    a, b = r[..., :rot // 2], r[..., rot // 2:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)


def _turned_norm64(x, w, pos, c):
    """The same from the definition: a pair is a complex number that is turned."""
    x = x.double()
    x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["hd"] + EPS) * w.double()
    half = c["rot"] // 2
    first = torch.arange(half, device="cuda") * (2 if c["layout"] == "interleaved" else 1)
    second = first + (1 if c["layout"] == "interleaved" else half)
    turn = torch.polar(torch.ones(len(pos), half, dtype=torch.float64, device="cuda"), pos.double()[:, None] * _freqs(c))
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _heads_inputs(c, seed):
    g = _gen(seed)
    rows = _qkv(c, g, c["rows"])
    w = _head_weights(c, g)
    if c["scattered"]:
        pos = torch.randint(0, 16384, (c["rows"],), generator=g, device="cuda")
    else:
        pos = torch.arange(c["rows"], device="cuda") + int(torch.randint(0, 384, (1,), generator=g, device="cuda"))
    return rows, w, pos


def _own_tables(S, c, top):
    from tang_amd import capi
    cs, sn = capi.rope_tables_scaled(c["rot"], top, 10000.0)
    S.cos, S.sin = _device().upload(cs), _device().upload(sn)
    S.layout = {"interleaved": capi.ROPE_INTERLEAVED, "half": capi.ROPE_HALF}[c["layout"]]


def _prepare_heads(c, seed):
    S = _State()
    rows, S.w, pos = _heads_inputs(c, seed)
    if own:
        _own_tables(S, c, 16384)
        S.rows, S.w = [_Buf(t) for t in rows], [_Buf(t) for t in S.w]
        S.start, S.pos = (0, _buf_u32(pos)) if c["scattered"] else (int(pos[0]), None)
        S.out = [_new(c["x"], c["rows"], n, c["hd"]) for n in (c["heads"], c["kv_heads"])]
        return S
    S.rows = rows
    angle = torch.arange(16384, dtype=torch.float64, device="cuda")[:, None] * _freqs(c)
    S.cos, S.sin, S.pos = angle.cos().float(), angle.sin().float(), pos
    return S


def _run_heads(S, c):
    if own:
        k = None if c["packed"] else S.rows[1].buf
        stride = (c["heads"] + 2 * c["kv_heads"]) * c["hd"] if c["packed"] else 0
        _device().qk_norm_rope(S.rows[0].buf, k, S.w[0].buf, S.w[1].buf, EPS, S.cos, S.sin, c["rows"], c["heads"], c["kv_heads"], c["hd"], c["rot"],
                               S.layout, start_pos=S.start, positions=S.pos, q_stride=stride, q_out=S.out[0].buf, k_out=S.out[1].buf)
        return [o.t for o in S.out]
    q, k, _ = _split(c, S.rows)
    cos, sin = S.cos[S.pos][:, None], S.sin[S.pos][:, None]
    return [_turned_norm(x, w, cos, sin, c).to(_DT[c["x"]]) for x, w in ((q, S.w[0]), (k, S.w[1]))]


def _exact_heads(c, seed):
    rows, w, pos = _heads_inputs(c, seed)
    q, k, _ = _split(c, rows)
    return [_turned_norm64(q, w[0], pos, c), _turned_norm64(k, w[1], pos, c)]


def _work_heads(c):
    n = c["rows"] * (c["heads"] + c["kv_heads"])
    return dict(bytes=2 * n * c["hd"] * _SIZE[c["x"]], flops=n * (4 * c["hd"] + 3 * c["rot"]))


def _spread(lo, hi, n, rng):
    """n lengths over [lo, hi], even in their logarithm, in any order."""
    v = [int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * (i + 0.5) / n))) - 1 for i in range(n)]
    rng.shuffle(v)
    return v


def _pages_plan(c):
    """Positions that each sequence has, its new ones, and its pages: those that
    it has, then those of the step, the cache's lowest free page first."""
    rng = random.Random(c["B"] * 7919 + c["hi"])
    starts, news = _spread(c["lo"], c["hi"], c["B"], rng), _spread(c["q_lo"], c["q_hi"], c["B"], rng)
    news = [max(1, n) for n in news]
    table, used = [], 0
    for s in starts:
        n = -(-s // c["page"])
        table.append(list(range(used, used + n)))
        used += n
    for t, s, n in zip(table, starts, news):
        more = -(-(s + n) // c["page"]) - len(t)
        t += range(used, used + more)
        used += more
    return starts, news, table, used


def _pages_inputs(c, seed):
    g = _gen(seed)
    starts, news, table, pages = _pages_plan(c)
    pool = _normal(g, c["cache"], c["layers"], 2, pages, c["kv_heads"], c["page"], c["hd"])
    rows = [_qkv(c, g, sum(news)) for _ in range(c["layers"])]
    w = [_head_weights(c, g) for _ in range(c["layers"])]
    return pool, rows, w, starts, news, table, pages


def _prepare_pages(c, seed):
    S = _State()
    S.pool, S.rows, S.w, starts, news, table, pages = _pages_inputs(c, seed)
    top = max(s + n for s, n in zip(starts, news))
    if own:
        from tang_amd import capi
        _own_tables(S, c, top)
        S.cache = _device().kv_cache(c["layers"], c["kv_heads"], c["hd"], c["page"], pages, c["B"], top, {"f16": capi.F16, "bf16": capi.BF16}[c["cache"]])
        view = _at(S.cache.page_pointers(0)[0], _DT[c["cache"]], tuple(S.pool.shape), S.cache)
        view.copy_(S.pool)
        S.pool, S.seqs = view, S.cache.seq_create(c["B"])
        for i, s in enumerate(starts):
            S.cache.seq_resize(S.seqs[i], s)
        S.batch = S.cache.batch(c["B"], sum(news), c["heads"])
        S.batch.begin(S.seqs, news)
        S.rows = [[_Buf(t) for t in rows] for rows in S.rows]
        S.w = [[_Buf(t) for t in w] for w in S.w]
        S.out = [_new(c["x"], sum(news), c["heads"], c["hd"]) for _ in range(c["layers"])]
        return S
    pos = [s + j for s, n in zip(starts, news) for j in range(n)]
    seq = [i for i, n in enumerate(news) for _ in range(n)]
    S.page = torch.tensor([table[i][p // c["page"]] for i, p in zip(seq, pos)], device="cuda")
    S.pos = torch.tensor(pos, device="cuda")
    S.place = S.pos % c["page"]
    angle = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * _freqs(c)
    S.cos, S.sin = angle.cos().float(), angle.sin().float()
    return S


def _plain_pages(S, c, layer):
    q, k, v = _split(c, S.rows[layer])
    cos, sin = S.cos[S.pos][:, None], S.sin[S.pos][:, None]
    S.pool[layer, 0][S.page, :, S.place] = _turned_norm(k, S.w[layer][1], cos, sin, c).to(S.pool.dtype)
    S.pool[layer, 1][S.page, :, S.place] = v.to(S.pool.dtype)
    return _turned_norm(q, S.w[layer][0], cos, sin, c).to(_DT[c["x"]])


def _run_pages(S, c):
    if own:
        for l, (rows, w) in enumerate(zip(S.rows, S.w)):
            q, k, v = [t.buf for t in rows] if len(rows) == 3 else (rows[0].buf, None, None)
            S.batch.append_norm(l, q, k, v, S.out[l].buf, w[0].buf, w[1].buf, EPS, S.cos, S.sin, c["rot"], S.layout)
        return [o.t for o in S.out], S.pool
    return [_plain_pages(S, c, l) for l in range(c["layers"])], S.pool


def _exact_pages(c, seed):
    pool, rows, w, starts, news, table, _ = _pages_inputs(c, seed)
    pool, outs = pool.double(), []
    for l in range(c["layers"]):
        q, k, v = _split(c, rows[l])
        out, at = [], 0
        for s, n, t in zip(starts, news, table):
            pos = torch.arange(s, s + n, device="cuda")
            out.append(_turned_norm64(q[at:at + n], w[l][0], pos, c))
            ks, page = _turned_norm64(k[at:at + n], w[l][1], pos, c), torch.tensor(t, device="cuda")[pos // c["page"]]
            pool[l, 0, page, :, pos % c["page"]] = ks
            pool[l, 1, page, :, pos % c["page"]] = v[at:at + n].double()
            at += n
        outs.append(torch.cat(out))
    return outs, pool


def _work_pages(c):
    R = sum(_pages_plan(c)[1])
    q, kv = c["heads"] * c["hd"], 2 * c["kv_heads"] * c["hd"]
    return dict(bytes=c["layers"] * R * (2 * q * _SIZE[c["x"]] + kv * (_SIZE[c["x"]] + _SIZE[c["cache"]])),
                flops=c["layers"] * R * (c["heads"] + c["kv_heads"]) * (4 * c["hd"] + 3 * c["rot"]))


# ---------------------------------------------------------------------------
# The choice of tokens
# ---------------------------------------------------------------------------


def _sample_inputs(c, seed):
    """Logits with a broad floor and a few tokens that stand out, and each row's
    settings: temperature (0: greedy), top_k (0: off), top_p (1: off), min_p (0: off)."""
    g, R, V = _gen(seed), c["rows"], c["vocab"]
    x = torch.randn(R, V, generator=g, device="cuda") * 2.0
    peaks = torch.randint(0, V, (R, min(V, 64)), generator=g, device="cuda")
    x.scatter_add_(1, peaks, torch.rand(R, peaks.shape[1], generator=g, device="cuda") * 10)
    if c["masked"]:  # tokens that a grammar forbids, in every second row
        gone = torch.rand(R, V, generator=g, device="cuda") < c["masked"]
        gone[1::2] = False
        x.masked_fill_(gone, -math.inf)
    u = torch.rand(R, generator=g, device="cuda")
    rng = np.random.default_rng(int(seed) + 17)
    temp, k, p, low = rng.uniform(0.3, 1.5, R), np.zeros(R, np.int64), np.ones(R), np.zeros(R)
    if c["mode"] in ("all", "mixed"):
        k, p, low = rng.integers(1, 200, R), rng.uniform(0.5, 1.0, R), rng.uniform(0.0, 0.05, R)
    if c["mode"] == "nucleus":
        p, low = rng.uniform(0.8, 1.0, R), np.where(rng.random(R) < 0.5, 0.0, rng.uniform(0.001, 0.1, R))
    if c["mode"] == "mixed":
        temp, k = np.where(rng.random(R) < 0.2, 0.0, temp), np.where(rng.random(R) < 0.4, 0, k)
        p, low = np.where(rng.random(R) < 0.4, 1.0, p), np.where(rng.random(R) < 0.4, 0.0, low)
    as32 = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    return x.to(_DT[c["x"]]), u, as32(temp), torch.tensor(k, dtype=torch.int32, device="cuda"), as32(p), as32(low)


def _prepare_sample(c, seed):
    S = _State()
    S.x, S.u, S.temp, S.k, S.p, S.low = _sample_inputs(c, seed)
    if own:
        from tang_amd import capi
        S.x, S.u, S.temp, S.p, S.low = (_Buf(t) for t in (S.x, S.u, S.temp, S.p, S.low))
        S.k = _buf_u32(S.k)
        S.token_buf, S.prob = _device().alloc(c["rows"], capi.U32), _new("f32", c["rows"])
        S.token = _at(S.token_buf.device_ptr(), torch.int32, (c["rows"],), S.token_buf)
    return S


def _run_sample(S, c):
    if own:
        _device().sample_rows(S.x.buf, c["rows"], c["vocab"], S.u.buf, temperature=S.temp.buf, top_k=S.k, top_p=S.p.buf, min_p=S.low.buf,
                              tokens=S.token_buf, prob=S.prob.buf)
        return S.token, S.prob.t
    V = c["vocab"]
    x, u, p, low = S.x.double(), S.u.double()[:, None], S.p.double()[:, None], S.low.double()[:, None]  # 64 bits: a border decides a token
    index = torch.arange(V, device="cuda")
    top = x.amax(1, keepdim=True)
    first = torch.where(x == top, index, V).amin(1)
    temp = torch.where(S.temp > 0, S.temp, torch.ones_like(S.temp)).double()[:, None]
    w = torch.exp((x - top) / temp)
    down, order = torch.sort(x, dim=1, descending=True, stable=True)
    wd = w.gather(1, order)
    k = torch.where((S.k > 0) & (S.k < V), S.k, V).long()[:, None]
    wd = torch.where(down >= down.gather(1, k - 1), wd, 0.0)
    before = wd.cumsum(1) - wd
    keep = (p >= 1) | (before < p * wd.sum(1, keepdim=True))
    wd = torch.where(keep & (wd >= low), wd, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, wd)
    total = w.sum(1, keepdim=True)
    past = (w.cumsum(1) <= u * total) | (w == 0)
    last = torch.where(w > 0, index, -1).amax(1)
    token = torch.where(past, V, index).amin(1)
    token = torch.where(token == V, last, token)
    greedy = S.temp <= 0
    token = torch.where(greedy, first, token)
    prob = torch.where(greedy, 1.0, w.gather(1, token[:, None])[:, 0] / total[:, 0])
    return token.int(), prob.float()


def _exact_sample(c, seed):
    x, u, temp, k, p, low = (t.double().cpu().numpy() for t in _sample_inputs(c, seed))
    tokens, probs = np.empty(c["rows"], np.int32), np.ones(c["rows"])
    for r in range(c["rows"]):
        row = x[r]
        if temp[r] <= 0:
            tokens[r] = np.flatnonzero(row == row.max())[0]
            continue
        seen = np.flatnonzero(row > -math.inf)
        seen = seen[np.lexsort((seen, -row[seen]))]  # by descending logit, equal ones by index
        if 0 < k[r] < len(seen):
            seen = seen[row[seen] >= row[seen[int(k[r]) - 1]]]
        w = np.exp((row[seen] - row[seen[0]]) / temp[r])
        if p[r] < 1:
            n = int(np.searchsorted(np.cumsum(w), p[r] * w.sum())) + 1
            seen, w = seen[:n], w[:n]
        seen, w = seen[w >= low[r]], w[w >= low[r]]
        w = w[np.argsort(seen)]
        seen = np.sort(seen)
        at = min(int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")), len(seen) - 1)
        tokens[r], probs[r] = seen[at], w[at] / w.sum()
    return torch.from_numpy(tokens), torch.from_numpy(probs)


def _work_sample(c):
    return dict(bytes=c["rows"] * (c["vocab"] * _SIZE[c["x"]] + 28), flops=c["rows"] * c["vocab"] * 4)


# ---------------------------------------------------------------------------

_KINDS = {
    "i8": (_prepare_i8, _run_i8, _exact_i8, _work_i8),
    "heads": (_prepare_heads, _run_heads, _exact_heads, _work_heads),
    "pages": (_prepare_pages, _run_pages, _exact_pages, _work_pages),
    "sample": (_prepare_sample, _run_sample, _exact_sample, _work_sample),
}


def prepare(case, seed):
    S = _KINDS[case["kind"]][0](case, seed)
    S.case = case
    if own:
        torch.cuda.synchronize()  # the library works on a stream of its own
    return S


def run(state):
    return _KINDS[state.case["kind"]][1](state, state.case)


def exact(case, seed):
    return _KINDS[case["kind"]][2](case, seed)


def work(case):
    return _KINDS[case["kind"]][3](case)
