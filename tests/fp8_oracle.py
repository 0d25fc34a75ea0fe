"""8-bit floating point matrices with a scale for each block of 128, routing of
tokens to experts and the experts' products in numpy, 64 bits, from their
definitions (include/miaie.h): what the tests compare with."""
import numpy as np

from mx_oracle import bf16, bf16_bits, from_bf16_bits  # noqa: F401

# the 127 magnitudes of E4M3, by code
CODES = np.arange(127)
GRID = np.where(CODES >= 8, (8 + CODES % 8) * 2.0**(CODES // 8 - 10), CODES * 2.0**-9)


def up(n, unit=128):
    return -(-n // unit) * unit


def encode(a):
    """Codes of values (|a| <= 448 but for a rounding), to nearest, halves to the even code."""
    m = np.abs(a)
    i = np.clip(np.searchsorted(GRID, m, side="right") - 1, 0, 125)
    lo, hi = GRID[i], GRID[i + 1]
    mid = (lo + hi) / 2
    code = np.where((m > mid) | ((m == mid) & (i % 2 == 1)), i + 1, i)
    return (code | np.signbit(a).astype(np.int64) << 7).astype(np.uint8)


def decode(q):
    q = np.asarray(q)
    g = np.append(GRID, np.nan)
    return np.where(q >= 128, -1.0, 1.0) * g[q & 127]


def pack(X, block=1):
    """(Q, S) of X packed along its rows; blocks with an infinity or NaN have scale NaN and codes 0."""
    X = np.asarray(X, np.float64)
    R, C = X.shape
    x = np.zeros((up(R, block), up(C)))
    x[:R, :C] = X
    x = x.reshape(-1, block, up(C) // 128, 128)
    bad = ~np.isfinite(x).all((1, 3))
    amax = np.abs(np.where(bad[:, None, :, None], 0, x)).max((1, 3))
    m, e = np.frexp(amax)  # 448 = 0.875 2^9
    S = np.ldexp(1.0, np.maximum(np.where(amax > 0, e - 9 + (m > 0.875), -126), -126))
    Q = encode(np.where(bad[:, None, :, None], 0, x) / S[:, None, :, None]).reshape(-1, up(C))[:R]
    Q[:, C:] = 0
    return Q, np.ascontiguousarray(np.where(bad, np.nan, S).T.astype(np.float32))


def spread(S, R, K, block):
    """The scale of each element."""
    return np.asarray(S, np.float64).T.repeat(block, 0)[:R].repeat(128, 1)[:, :K]


def values(Q, S, R, K, block=1):
    return decode(Q)[:R, :K] * spread(S, R, K, block)


def rounded(X, block=1):
    return values(*pack(X, block), *X.shape, block)


def product_bound(A, B):
    """Most that an fp32 product may be off.  The matrix instruction adds the
    products of eight neighbouring k at 2^-13 of the power of two below the largest
    of them, what is smaller being cut off (seen on the device: a product of 2^-13 of
    the largest is kept, one of 2^-14 is not), so seven of them may each lose as
    much; the largest is at most the largest |a| times the largest |b|.  The sums of
    eight are added one by one at worst, each addition off by at most a unit in the
    last place of a partial sum; two scales and their use are three roundings, and
    the blocks' sums and their joining from several waves one for each addition."""
    K = A.shape[1]
    a, b = (np.pad(np.abs(m), ((0, 0), (0, -K % 8))).reshape(len(m), -1, 8).max(-1) for m in (A, B))
    return 7 * 2.0**-13 * (a @ b.T) + 2.0**-23 * (16 + 3 + K / 128 + 16) * (np.abs(A) @ np.abs(B).T)


# ---------------------------------------------------------------- routing
def scores(logits, scoring):
    l = np.asarray(logits, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        if scoring == "sigmoid":
            return 1 / (1 + np.exp(-l))
        top = l.max(-1, keepdims=True)
        e = np.exp(l - np.where(np.isneginf(top), 0, top))
        return e / np.where(np.isneginf(top), 1, e.sum(-1, keepdims=True))


def route(logits, bias, k, scoring, groups=1, kept=1, group_top=1, renormalize=True, scale=1.0):
    """(idx, w) a token at a time (finite logits and -infinity)."""
    T, E = logits.shape
    s = scores(logits, scoring)
    idx, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        c = {e: s[t, e] + (0 if bias is None else float(bias[e])) for e in range(E) if logits[t, e] != -np.inf}
        c = {e: v for e, v in c.items() if v != -np.inf}
        size = E // groups
        of = {}
        for e, v in c.items():
            of.setdefault(e // size, []).append(v)
        of = {g: sum(sorted(v, reverse=True)[:group_top]) for g, v in of.items()}
        keep = sorted(of, key=lambda g: (-of[g], g))[:kept] if groups > 1 else list(of)
        best = sorted((e for e in c if e // size in keep), key=lambda e: (-c[e], e))[:k]
        idx[t, :len(best)] = best
        w[t, :len(best)] = s[t, best]
        w[t] = scale * (w[t] / (w[t].sum() + 1e-20) if renormalize else w[t])
    return idx, w


def weights(logits, idx, scoring, renormalize, scale):
    """w of a given choice (entries outside [0, E): none)."""
    T, E = logits.shape
    s = scores(logits, scoring)
    some = (idx >= 0) & (idx < E)
    w = np.where(some, np.take_along_axis(s, np.where(some, idx, 0), 1), 0.0)
    return scale * (w / (w.sum(-1, keepdims=True) + 1e-20) if renormalize else w)


def route_grad(logits, idx, dw, scoring, renormalize, scale):
    T, E = logits.shape
    p = scores(logits, scoring)
    some = (idx >= 0) & (idx < E)
    at = np.where(some, idx, 0)
    chosen = np.where(some, np.take_along_axis(p, at, 1), 0.0)
    d = np.where(some, dw, 0.0)
    if renormalize:
        total = chosen.sum(-1, keepdims=True) + 1e-20
        d = (d - (d * chosen).sum(-1, keepdims=True) / total) / total
    d = scale * np.where(some, d, 0.0)
    ds = np.zeros((T, E))
    for j in range(idx.shape[1]):
        np.add.at(ds, (np.arange(T), at[:, j]), d[:, j])
    if scoring == "sigmoid":
        return ds * p * (1 - p)
    return p * (ds - (ds * p).sum(-1, keepdims=True))


def route_grad_terms(logits, idx, dw, scoring, renormalize, scale):
    """Sums of the magnitudes of the terms that route_grad adds and takes from each other."""
    T, E = logits.shape
    p = scores(logits, scoring)
    some = (idx >= 0) & (idx < E)
    at = np.where(some, idx, 0)
    chosen = np.where(some, np.take_along_axis(p, at, 1), 0.0)
    d = np.where(some, np.abs(dw), 0.0)
    if renormalize:
        total = chosen.sum(-1, keepdims=True) + 1e-20
        d = (d + (d * chosen).sum(-1, keepdims=True) / total) / total
    ds = np.zeros((T, E))
    for j in range(idx.shape[1]):
        np.add.at(ds, (np.arange(T), at[:, j]), scale * np.where(some, d, 0.0)[:, j])
    if scoring == "sigmoid":
        return ds * p * (1 - p)
    return p * (ds + (ds * p).sum(-1, keepdims=True))


# ---------------------------------------------------------------- slots
def slot_rows(T, k, E):
    n = T * k
    used = min(E, n)
    return 128 * (used + (n - used) // 128)


def order(idx, E):
    """dict of the parts of the order, and the whole array (parts that are not written hold -7)."""
    T, k = idx.shape
    R = slot_rows(T, k, E)
    start, count = np.zeros(E + 1, np.int32), np.zeros(E, np.int32)
    slot, pair, expert = np.full((T, k), -1, np.int32), np.full(R, -7, np.int32), np.full(R // 128, -1, np.int32)
    at = 0
    for e in range(E):
        start[e] = at
        hits = np.flatnonzero(idx.ravel() == e)
        count[e] = len(hits)
        slot.ravel()[hits] = at + np.arange(len(hits))
        end = at + up(len(hits))
        pair[at:end] = -1
        pair[at:at + len(hits)] = hits
        expert[at // 128:end // 128] = e
        at = end
    start[E] = at
    head = np.full(up(2 * E + 1, 16), -7, np.int32)
    head[:E + 1], head[E + 1:2 * E + 1] = start, count
    body = np.full(up(T * k, 16), -7, np.int32)
    body[:T * k] = slot.ravel()
    return {"start": start, "count": count, "slot": slot, "pair": pair, "expert": expert,
            "all": np.concatenate((head, body, pair, expert)), "used": at, "rows": R}


def used_slots(o):
    """[(expert, slots)] of the experts that have some."""
    return [(e, np.arange(o["start"][e], o["start"][e] + n)) for e, n in enumerate(o["count"]) if n]


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g))


def swiglu(GU):
    g, u = np.split(GU, 2, -1)
    return silu(g) * u


def swiglu_grad(GU, dH):
    g, u = np.split(GU, 2, -1)
    s = 1 / (1 + np.exp(-g))
    return np.concatenate((dH * u * s * (1 + g * (1 - s)), dH * g * s), -1)


def over_slots(o, X, w=None):
    """Rows of X by slot (zero in padding), times w."""
    k = o["slot"].shape[1]
    out = np.zeros((o["rows"], X.shape[1]))
    some = np.flatnonzero(o["pair"] >= 0)
    pair = o["pair"][some]
    out[some] = X[pair // k] * (1 if w is None else w.ravel()[pair][:, None])
    return out


def combine(o, Y, w=None):
    T, k = o["slot"].shape
    out = np.zeros((T, Y.shape[1]))
    for j in range(k):
        some = o["slot"][:, j] >= 0
        out[some] += Y[o["slot"][some, j]] * (1 if w is None else w[some, j][:, None])
    return out
