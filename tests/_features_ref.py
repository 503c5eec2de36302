"""The feature operators in 64 bits (numpy), with the bounds that the tests hold the kernels to.

Every bound is arithmetic: u = 2^-24 is half a step of a 32-bit number, ``half_step`` that of the
result's type; sums of m terms in any order are off by at most (m - 1) u times the sum of the
terms' magnitudes, sums whose longest chain of additions has H links by H u times that.
First-order bounds are multiplied by 1.01 for the higher orders.
"""
import numpy as np
import torch

U = 2.0 ** -24
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(exact, err32, dtype):
    """Bound of a value known to err32 in 32 bits and rounded once to dtype; the last term is half
    the step of the type's smallest numbers."""
    e = 1.01 * err32
    if dtype != torch.float32:
        e = e + half_step(dtype) * (np.abs(exact) + e)
    fi = torch.finfo(dtype)
    return e + fi.smallest_normal * fi.eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


# --------------------------------------------------------------------------- embedding
def embed(tokens, table, scale, empty):
    """(values, bound / half step part in 32 bits)"""
    rows = table.shape[0]
    ok = (tokens >= 0) & (tokens < rows)
    if empty is not None:
        ok &= tokens != empty
    out = np.where(ok[..., None], table[np.where(ok, tokens, 0)] * np.float64(np.float32(scale)), np.nan)
    if empty is not None:
        out[tokens == empty] = 0.0
    return out, U * np.abs(out)


def embed_grad(tokens, dy, rows, scale, empty):
    flat, dy = tokens.reshape(-1), dy.reshape(-1, dy.shape[-1])
    ok = (flat >= 0) & (flat < rows)
    if empty is not None:
        ok &= flat != empty
    g, mag = np.zeros((rows, dy.shape[1])), np.zeros((rows, dy.shape[1]))
    np.add.at(g, flat[ok], dy[ok])
    np.add.at(mag, flat[ok], np.abs(dy[ok]))
    m = np.bincount(flat[ok], minlength=rows)[:, None]
    s = np.float64(np.float32(scale))
    return g * s, abs(s) * U * (np.maximum(m - 1, 0) + 1) * mag


# --------------------------------------------------------------------------- layer norm
def layer_norm(x, w, b, eps):
    """x [rows,D] -> dict of values and 32-bit bounds, also of xhat for the gradient"""
    rows, D = x.shape
    H = D / 32 + 64  # a thread adds up at most every 32nd value; then warps and threads are added
    w = np.ones(D) if w is None else w
    b = np.zeros(D) if b is None else b
    mean = x.mean(1, keepdims=True)
    xc = x - mean
    var = (xc * xc).mean(1, keepdims=True)
    sd = np.sqrt(var + eps)
    xhat = xc / sd
    # x - x0, its mean, and their difference
    dist = np.abs(x - x[:, :1])
    d_c = U * (dist + np.abs(xc)) + U * (H + 3) * dist.mean(1, keepdims=True)
    # the sum of squares, /D, + eps, sqrt, 1/: relative to var + eps
    r = (2 * np.abs(xc) * d_c).mean(1, keepdims=True) / (2 * sd * sd) + U * (H + 6)
    e_xhat = d_c / sd + np.abs(xhat) * (r + U)
    y = xhat * w + b
    return {"y": y, "e_y": np.abs(w) * e_xhat + U * np.abs(y), "xhat": xhat, "e_xhat": e_xhat, "sd": sd, "r": r, "w": w,
            "H": H}


def layer_norm_grad(f, dy):
    xhat, sd, e, r, H, w = f["xhat"], f["sd"], f["e_xhat"], f["r"], f["H"], f["w"]
    rows = dy.shape[0]
    g = dy * w
    m1, m2 = g.mean(1, keepdims=True), (g * xhat).mean(1, keepdims=True)
    core = g - m1 - xhat * m2
    dx = core / sd
    e1 = U * (H + 3) * np.abs(g).mean(1, keepdims=True)
    e2 = U * (H + 4) * np.abs(g * xhat).mean(1, keepdims=True) + (np.abs(g) * e).mean(1, keepdims=True)
    e_core = (U * (2 * np.abs(g) + np.abs(m1) + 3 * np.abs(xhat * m2) + np.abs(core)) + e1 + np.abs(xhat) * e2
              + np.abs(m2) * e)
    res = {"dx": dx, "e_dx": e_core / sd + np.abs(dx) * (r + 2 * U)}
    res["dw"], res["db"] = (dy * xhat).sum(0), dy.sum(0)
    res["e_dw"] = U * (rows + 1) * np.abs(dy * xhat).sum(0) + (np.abs(dy) * e).sum(0)
    res["e_db"] = U * rows * np.abs(dy).sum(0)
    return res


# --------------------------------------------------------------------------- dropout
M = (0xD2511F53, 0xCD9E8D57)
W = (0x9E3779B9, 0xBB67AE85)
LOW = 0xFFFFFFFF


def philox(counter, key, rounds=7):
    """One block in Python integers: counter of four words, key of two."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * M[0], c[2] * M[1]
        c = [(b >> 32) ^ c[1] ^ k[0], b & LOW, (a >> 32) ^ c[3] ^ k[1], a & LOW]
        k = [(k[0] + W[0]) & LOW, (k[1] + W[1]) & LOW]
    return c


def words(first, count, seed, offset):
    """Random words of the values first .. first + count - 1 (first a multiple of 4), vectorised."""
    blocks = (count + 3) // 4
    q = np.arange(blocks, dtype=np.uint64) + np.uint64(first // 4)
    c = [q & np.uint64(LOW), q >> np.uint64(32), np.full(blocks, offset & LOW, np.uint64),
         np.full(blocks, (offset >> 32) & LOW, np.uint64)]
    k = [seed & LOW, (seed >> 32) & LOW]
    for _ in range(7):
        a, b = c[0] * np.uint64(M[0]), c[2] * np.uint64(M[1])
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & np.uint64(LOW),
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & np.uint64(LOW)]
        k = [(k[0] + W[0]) & LOW, (k[1] + W[1]) & LOW]
    return np.stack(c, 1).reshape(-1)[:count]


def dropout(x, p, seed, offset, first=0):
    """(values, 32-bit bound) of the flat x, whose first value is the tensor's value `first`"""
    if p == 1.0:
        return np.zeros_like(x), np.zeros_like(x)
    keep = words(first, x.size, seed, offset) >= np.uint64(int(p * 2.0 ** 32))
    y = np.where(keep, x / (1.0 - p), 0.0)
    return y, 2 * U * np.abs(y)


# --------------------------------------------------------------------------- comparison
def assert_within(got, exact, err32, what=""):
    """got: a tensor; every element within the bound of its type, NaN exactly where it should be."""
    dtype, g = got.dtype, f64(got).reshape(exact.shape)
    bad_nan = np.isnan(g) != np.isnan(exact)
    assert not bad_nan.any(), f"{what}: {int(bad_nan.sum())} NaN too many or too few"
    bound = rounded(exact, err32, dtype)
    off = np.where(np.isnan(exact), 0.0, np.abs(g - exact))
    ratio = np.where(np.isnan(exact), 0.0, off / bound)
    worst = float(ratio.max()) if ratio.size else 0.0
    assert worst <= 1.0, (f"{what}: {worst:.3g} times the bound at {np.unravel_index(int(ratio.argmax()), ratio.shape)}"
                          f" ({int((ratio > 1).sum())} of {ratio.size} values)")
    return worst
