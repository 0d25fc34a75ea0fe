"""MXFP4 matrices and the norms around a block in numpy, 64 bits, from their
definitions (include/miaie.h): what the GPU tests compare with.

A packed matrix is (Q, S) in the library's layout; values() gives the float64
matrix it stands for."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def bf16(x):
    """float values rounded to bf16 (nearest even), as float32; NaN stays NaN."""
    x = np.asarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32)
    return np.where(np.isnan(x), np.float32(np.nan), r.view(np.float32))


def bf16_bits(x):
    return (bf16(x).view(np.uint32) >> 16).astype(np.uint16)


def from_bf16_bits(u):
    return (np.asarray(u, np.uint16).astype(np.uint32) << 16).view(np.float32)


def pack(X):
    """(Q, S) of X (float64 or float32) packed along its rows."""
    X = np.asarray(X, np.float64)
    R, C = X.shape
    G = (C + 511) // 512
    x = np.zeros((R, 512 * G))
    x[:, :C] = X
    x = x.reshape(R, 16 * G, 32)
    bad = ~np.isfinite(x).all(-1)
    amax = np.abs(np.where(bad[..., None], 0, x)).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(amax > 0, np.frexp(amax)[1] - 3, -127)  # floor(log2) - 2
    e = np.maximum(e, -127)
    a = np.abs(x) / np.exp2(e.astype(np.float64))[..., None]
    code = np.zeros(a.shape, np.uint8)
    for i in range(7):  # a value halfway between two neighbours goes to the even code
        mid = (GRID[i] + GRID[i + 1]) / 2
        code[(a >= mid) if i % 2 else (a > mid)] = i + 1
    code |= np.signbit(x).astype(np.uint8) << 3
    S = np.where(bad, 255, e + 127).astype(np.uint8)
    pairs = code.reshape(R, -1, 2)
    Q = (pairs[..., 0] | pairs[..., 1] << 4)[:, :(C + 255) // 256 * 128]
    return np.ascontiguousarray(Q), np.ascontiguousarray(S.reshape(R, G, 4, 4).transpose(1, 0, 3, 2))


def block_scales(S):
    """[R][blocks] scale bytes of S."""
    G, R = S.shape[:2]
    return S.transpose(1, 0, 3, 2).reshape(R, 16 * G)


def values(Q, S, C):
    code = np.stack((Q & 15, Q >> 4), -1).reshape(Q.shape[0], -1)[:, :C]
    v = np.where(code >= 8, -1.0, 1.0) * GRID[code & 7]
    s = np.repeat(block_scales(S), 32, axis=1)[:, :C]
    return np.where(s == 255, np.nan, v * np.exp2(s.astype(np.float64) - 127))


def product_bound(A, B):
    """Most that an fp32 sum of the products may be off: every 128 columns the
    sums of four blocks (exact) and the accumulator are added, each addition
    off by at most half a unit of a partial sum, which is at most sum |a b|;
    joining partial sums of the k axis adds fewer.  (One more unit each for a
    matrix instruction that truncates.)"""
    K = A.shape[1]
    return 2.0**-23 * (K / 32 + 4) * (np.abs(A) @ np.abs(B).T)


# ---------------------------------------------------------------- norms
def gate_of(gate, rows, gate_rows):
    return 1.0 if gate is None else gate[np.arange(rows) // gate_rows]


def norm_block(x, b, gate, w_after, w_before, gate_rows, alpha, eps, store=lambda v: v):
    """(out, y, rstd) in 64 bits; `store` rounds out as the stream's type does."""
    r, ra, rb, y = x, None, None, None
    if b is not None:
        ra = 1 / np.sqrt((b * b).mean(1) + eps)
        r = store(alpha * x + gate_of(gate, len(x), gate_rows) * w_after * b * ra[:, None])
    if w_before is not None:
        rb = 1 / np.sqrt((r * r).mean(1) + eps)
        y = w_before * r * rb[:, None]
    return r, y, ra, rb


def norm_block_grad(r, b, gate, w_after, w_before, ra, rb, dout, dy, gate_rows, alpha):
    """Gradients in 64 bits: dict of dx, db, dgate, dw_after, dw_before."""
    g, rows = {}, len(r)
    dr = np.zeros_like(r) if dout is None else dout
    if dy is not None:
        m, t = r * rb[:, None], dy * w_before
        g["dw_before"] = (dy * m).sum(0)
        dr = dr + rb[:, None] * (t - m * (t * m).mean(1, keepdims=True))
    g["dx"] = dr * (1.0 if b is None else alpha)
    if b is not None:
        n, gg = b * ra[:, None], gate_of(gate, rows, gate_rows)
        g["dw_after"] = (dr * gg * n).sum(0)
        if gate is not None:
            p = dr * w_after * n
            g["dgate"] = np.stack([p[i:i + gate_rows].sum(0) for i in range(0, rows, gate_rows)])
        u = dr * gg * w_after
        g["db"] = ra[:, None] * (u - n * (u * n).mean(1, keepdims=True))
    return g
