"""AdamW from its formulas, in numpy: float64 where the result is a number, float32 operation by operation where a code is
decided on it (the roundings are part of the definition of the 8-bit moments, include/ddcn_hip.h)."""
import numpy as np

BLOCK = 256
F = np.float32


def starts_of(sizes):
    out, total = [], 0
    for n in sizes:
        out.append(total)
        total += -(-n // BLOCK) * BLOCK
    return out, total


def noise(place, seed):
    """The two 16-bit numbers of an element as fractions of one."""
    m = np.uint64(0xFFFFFFFF)
    h = (place.astype(np.uint64) * np.uint64(0x9E3779B1) + np.uint64(seed & 0xFFFFFFFF) * np.uint64(0x1F83D9AB)
         + np.uint64(0x5BE0CD19)) & m
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x6A09E667)) & m
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0x510E527F)) & m
    h = h ^ (h >> np.uint64(15))
    return (h & np.uint64(0xFFFF)).astype(F) * F(2.0 ** -16), (h >> np.uint64(16)).astype(F) * F(2.0 ** -16)


def encode(x, u, top):
    """(codes, scale) of one block of values >= 0 (float32)."""
    most = np.float32(np.max(x))
    if not np.isfinite(most):
        return np.zeros(x.shape, np.int64), F(np.nan)
    if most < F(2.0 ** -100):
        return np.zeros(x.shape, np.int64), F(0)
    scale = F(most / F(top * top))
    root = np.sqrt((x * F(F(1) / scale)).astype(F)).astype(F)
    return np.minimum(np.floor((root + u).astype(F)), top).astype(np.int64), scale


def decode_m(q, scale):
    q = q.astype(np.int64)
    with np.errstate(invalid="ignore"):
        return (F(scale) * (q * np.abs(q)).astype(F)).astype(F)


def decode_r(q, scale):
    q = q.astype(np.int64)
    with np.errstate(invalid="ignore"):
        return (F(scale) * (q * q).astype(F)).astype(F)


def coefficient(norm, max_norm):
    return F(min(F(1), F(F(max_norm) / F(F(norm) + F(1e-6)))))


def moments32(g, m, v, b1, b2, c=F(1)):
    """(m, v) in float32, one rounding an operation."""
    g = (g.astype(F) * c).astype(F)
    m = ((F(b1) * m).astype(F) + (F(1.0 - b1) * g).astype(F)).astype(F)
    v = ((F(b2) * v).astype(F) + ((F(1.0 - b2) * g).astype(F) * g).astype(F)).astype(F)
    return m, v


def step64(p, g, m, v, t, lr, betas, eps, wd, c=1.0):
    """float64: (p, m, v, allowed): the new values, and how far a float32 evaluation of p may be off: every operation of
    the formula is off by half a step of float32 (2^-24), of the sums' larger terms where they cancel.  p (1 - lr wd):
    the constant and the product, then the subtraction; the update: g c, its product, the two terms and their sum in m;
    as many in v, halved by the root; root, its product, the sum with eps, the quotient, step size and its product -- 16
    in all, of the update with |b1 m| + |(1 - b1) g| in the place of m."""
    b1, b2 = betas
    p, g, m, v = (np.asarray(a, np.float64) for a in (p, g, m, v))
    g = g * c
    big = np.abs(b1 * m) + np.abs((1 - b1) * g)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    scale = lr / (1 - b1 ** t) / (np.sqrt(v) / np.sqrt(1 - b2 ** t) + eps)
    new = p * (1 - lr * wd) - scale * m
    return new, m, v, 2.0 ** -24 * (4 * np.abs(p) + 16 * scale * big)
