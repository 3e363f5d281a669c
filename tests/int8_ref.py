"""Products in 8-bit integers from their formulas, in numpy: codes from float32 operations (part of the definition,
include/ddcn_hip.h), sums in int64, the rest in float64."""
import numpy as np

F = np.float32


def quantize(x):
    """(codes int64 [rows, k], scale float32 [rows]) of the rows of x (float32)."""
    x = np.ascontiguousarray(x, F)
    top = np.max(np.abs(x), axis=1)                      # NaN where the row holds one
    fine = np.isfinite(top)
    m = np.maximum(np.where(fine, top, 1), F(2.0 ** -96)).astype(F)
    scale = np.where(fine, (m / F(127)).astype(F), F(np.nan)).astype(F)
    factor = (F(127) / m).astype(F)
    with np.errstate(invalid="ignore"):
        q = np.rint((x * factor[:, None]).astype(F))
    return np.where(fine[:, None], q, 0).astype(np.int64), scale


def product(x, wq, ws, bias=None, relu=False):
    """(y float64 [tokens, channels], allowed): allowed is what float32 may be off by: the sum's conversion, the two
    products of scales and sum and the addition are half a step (2^-24) each, of |sum s s| or |y|."""
    q, sx = quantize(x)
    y = (q @ wq.astype(np.int64).T).astype(np.float64) * sx[:, None].astype(np.float64) * ws[None].astype(np.float64)
    tol = 2.0 ** -24 * 3 * np.abs(y)
    if bias is not None:
        y = y + bias[None].astype(np.float64)
    tol = tol + 2.0 ** -24 * (np.abs(y) + tol)
    return np.where(y < 0, 0.0, y) if relu else y, tol
