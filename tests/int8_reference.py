"""The 8-bit integer products in 64 bits, and the few f32 roundings that the definition names."""
import numpy as np


def codes(x, axis):
    """(codes as f64 whole numbers, f32 maxima, NaN where a vector is not finite) of the vectors of x along
    axis: round half to even of 127 x / max|x|, the quotient a real number (f64 forms it well enough: x has
    at most 24 bits)."""
    x = np.asarray(x).astype(np.float64)
    with np.errstate(all="ignore"):
        most = np.abs(x).max(axis=axis, keepdims=True)
        plain = np.isfinite(most) & (most > 0)
        c = np.where(plain, np.rint(x * 127 / np.where(plain, most, 1)), 0.0)
        most = np.where(np.isfinite(most), most, np.nan).astype(np.float32)
    return np.where(np.isfinite(c), c, 0.0), np.squeeze(most, axis)


def product(a, w):
    """a [M, K] by w [K, N]: exact sums, then f32(sum) * sa * sw with sa = max / 127 in f32 where both scales
    lie in [2^-60, 2^60] or are 0, the same in f64 elsewhere; rounded to a's type.  Bit for bit what the
    product returns (f64 sums of whole numbers below 2^53 are exact)."""
    ca, ma = codes(a, 1)
    cw, mw = codes(w, 0)
    with np.errstate(all="ignore"):
        total = ca @ cw
        sa, sw = ma / np.float32(127), mw / np.float32(127)
        odd = [~((s == 0) | np.isnan(s) | ((s >= 2.0 ** -60) & (s <= 2.0 ** 60))) for s in (sa, sw)]
        c = total.astype(np.float32) * sa[:, None] * sw[None, :]
        for r in np.nonzero(odd[0])[0]:
            c[r] = (total[r] * (float(ma[r]) / 127) * (mw.astype(np.float64) / 127)).astype(np.float32)
        for n in np.nonzero(odd[1])[0]:
            c[:, n] = (total[:, n] * (ma.astype(np.float64) / 127) * (float(mw[n]) / 127)).astype(np.float32)
        return c.astype(a.dtype)


def group_rows(ids, experts):
    """offsets, order, position of a stable sort by id; ids outside the experts last."""
    ids = np.asarray(ids, dtype=np.int64).reshape(-1)
    key = np.where((ids >= 0) & (ids < experts), ids, experts)
    order = np.argsort(key, kind="stable")
    position = np.empty_like(order)
    position[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=experts + 1)[:experts])])
    return offsets.astype(np.int32), order.astype(np.int32), position.astype(np.int32)


def same_bits(a, b):
    """Equal bit for bit, any NaN being equal to any other."""
    a, b = np.asarray(a), np.asarray(b)
    if a.shape != b.shape or a.dtype != b.dtype:
        return False
    u = np.uint16 if a.dtype == np.float16 else np.uint32
    nan = np.isnan(a) & np.isnan(b)
    return bool(np.all(nan | (a.view(u) == b.view(u))))
