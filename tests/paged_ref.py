"""Plain 64-bit statements of what the paged cache's operators compute."""
import numpy as np

import oracle
from tang_amd import capi

EPS = {capi.F32: 2.0 ** -24, capi.F16: 2.0 ** -11, capi.BF16: 2.0 ** -8}  # half a step, relative
LEAST = {capi.F32: 2.0 ** -150, capi.F16: 2.0 ** -25, capi.BF16: 2.0 ** -134}  # half of the smallest step


def to_bits(x, dt):
    """f32 values as the host array of a buffer of type dt (one rounding)."""
    x = np.ascontiguousarray(x, np.float32)
    if dt == capi.F32:
        return x
    with np.errstate(over="ignore"):
        return oracle.f32_to_bf16(x.reshape(-1)).reshape(x.shape) if dt == capi.BF16 else x.astype(np.float16).view(np.uint16)


def from_bits(b, dt):
    """The values of such an array, exactly, as f32."""
    if dt == capi.F32:
        return np.asarray(b, np.float32)
    b = np.ascontiguousarray(b, np.uint16)
    return (b.astype(np.uint32) << 16).view(np.float32) if dt == capi.BF16 else b.view(np.float16).astype(np.float32)


def rounded(x, dt):
    return from_bits(to_bits(x, dt), dt)


def rotate(x, cos, sin, pos, rot, half):
    """x [rows][heads][hd] f32, tables [n][rot/2]: in f32, products and sums rounded one by one."""
    y = np.array(x, np.float32)
    if rot == 0:
        return y
    c, s = cos[pos][:, None], sin[pos][:, None]
    i = np.arange(rot // 2)
    u, w = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    a, b = x[..., u].astype(np.float32), x[..., w].astype(np.float32)
    y[..., u] = a * c - b * s
    y[..., w] = (b * c + a * s) if half else (a * s + b * c)
    return y


def seen(pos, n, window, sinks):
    """[rows][n]: which keys the rows at these positions see."""
    j, p = np.arange(n)[None, :], np.asarray(pos)[:, None]
    ok = j <= p
    return ok & ((j > p - window) | (j < sinks)) if window else ok


def attention(q, k, v, pos, window=0, sinks=0, scale=None):
    """q [rows][H][D] at positions pos of one sequence with k, v [n][KH][D]."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    H, KH, D = q.shape[1], k.shape[1], q.shape[2]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    ok = seen(pos, k.shape[0], window, sinks)
    out = np.empty_like(q)
    for h in range(H):
        s = np.where(ok, (q[:, h] @ k[:, h // (H // KH)].T) * scale, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = (p / p.sum(-1, keepdims=True)) @ v[:, h // (H // KH)]
    return out


def attention_bound(q, k, v, pos, qdt, cdt, odt, window=0, sinks=0, scale=None):
    """How far a result may be from attention(): every rounding counted at its worst.

    With A the largest sum of |q k| times the scale, and u = 2^-23 the step that an
    MFMA may truncate by: a score is off by (4 + parts * D / 16 + 8) u A (the
    query's parts, the MFMAs in a chain and the alignment inside one, the product
    with the scale, the exponent's argument), a probability by that and 2^-22 of itself. Sums over n
    keys, in blocks of 32 or 64 that meet in plain additions: (n / 32 + 24) u. The quotient doubles both.
    Queries and results of the cache's type: a probability is rounded to it (half a step). The result's own rounding comes last."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    H, KH, D, n = q.shape[1], k.shape[1], q.shape[2], k.shape[0]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    A = max((np.abs(q[:, h]) @ np.abs(k[:, h // (H // KH)]).T).max() for h in range(H))
    A *= scale
    u, parts = 2.0 ** -23, 1 if qdt == cdt == odt else 3
    e = (4 + parts * D / 16 + 8) * u * A + 2.0 ** -22 + (n / 32 + 24) * u
    top = np.abs(v).max()
    # (of n weights, those below the type's normal range are off by half its smallest step)
    once = (EPS[cdt] + n * LEAST[cdt]) * top if qdt == cdt == odt else 0.0
    return 2.0 * e * top + once + max(EPS[odt] * top, LEAST[odt])


def attention_bounds(q, k, v, pos, qdt, cdt, odt, window=0, sinks=0, scale=None, tiles=True):
    """The same element by element [rows][H][D], from the weights w_j and values v_j that a result o = sum_j w_j v_j has.

    A weight is off by e_j = (4 + parts D / 16 + 8) u A_j + 2^-22 of itself (as in attention_bound, A_j = scale sum |q k_j|), which moves the
    quotient by at most sum_j w_j e_j (|v_j| + |o|), and to first order: twice that covers the rest. Sums over n keys, an MFMA of 16 keys at
    a time that truncates: (n / 16 + 24) u of sum_j w_j |v_j|, for the dividend and the divisor.
    Queries and results of the cache's type: weights go in with two parts of it (EPS^2 is left), with one where the rows make up tiles: each is
    off by d_j, |d_j| <= EPS w_j, and as the divisor has the same weights the quotient moves by sum_j d_j (v_j - o): at most
    EPS sum_j w_j |v_j - o|, and, the roundings being independent of each other, beyond 7.5 EPS sqrt(sum_j w_j^2 (v_j - o)^2) with a
    probability of 2 exp(-7.5^2 / 2) = 1e-12 an element (Hoeffding). A weight in f16 is one of 2^9 times the largest or more, so those
    below the normal range are off by LEAST 2^-9 of the largest. The result's own rounding comes last."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    H, KH, D = q.shape[1], k.shape[1], q.shape[2]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    ok, own = seen(pos, k.shape[0], window, sinks), qdt == cdt == odt
    u, parts = 2.0 ** -23, 1 if own else 3
    out = np.empty_like(q)
    for h in range(H):
        kk, vv = k[:, h // (H // KH)], v[:, h // (H // KH)]
        s = np.where(ok, (q[:, h] @ kk.T) * scale, -np.inf)
        w = np.exp(s - s.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        o, mean = w @ vv, w @ np.abs(vv)
        we = w * ((12 + parts * D / 16) * u * scale * (np.abs(q[:, h]) @ np.abs(kk).T) + 2.0 ** -22)
        n = ok.sum(-1, keepdims=True)
        b = 2.0 * (we @ np.abs(vv) + we.sum(-1, keepdims=True) * np.abs(o)) + 2.0 * (n / 16 + 24) * u * mean
        if own:
            b += EPS[cdt] ** 2 * (mean + np.abs(o))
        if own and tiles:
            w2 = w * w
            l2 = np.sqrt(np.maximum(w2 @ (vv * vv) - 2 * o * (w2 @ vv) + o * o * w2.sum(-1, keepdims=True), 0.0))
            b += np.minimum(EPS[cdt] * (mean + np.abs(o)), 7.5 * EPS[cdt] * l2)
            if cdt == capi.F16:
                b += n * LEAST[cdt] * 2.0 ** -9 * w.max(-1, keepdims=True) * (np.abs(vv).max() + np.abs(o))
        out[:, h] = b * (1 + EPS[odt]) + np.maximum(EPS[odt] * np.abs(o), LEAST[odt])
    return out
