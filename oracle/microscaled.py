"""64-bit restatement (numpy) of the microscaled formats and of the operators on them.

Written from the definition: a block's scale is 2^(floor(log2(max |x|)) - emax), an element is the
nearest of all values its type has, ties to the even code.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32


def _grid(bits: int) -> np.ndarray:
    """Magnitudes of the element type in code order."""
    if bits == 4:
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    e, m = np.divmod(np.arange(127), 8)                    # e4m3: 127 finite magnitudes
    return np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))


def quantize(x: np.ndarray, bits: int):
    """(codes as signed magnitude indices, signs, scale bytes) of rows x [R, C]."""
    b = np.asarray(x, dtype=np.float64).reshape(x.shape[0], -1, BLOCK)
    with np.errstate(all="ignore"):
        big = np.abs(b).max(-1)
        bad = ~np.isfinite(b).all(-1)
        expo = np.frexp(np.where(bad, 1.0, big))[1] - 1                # floor(log2)
        s = np.where(big == 0, -127, np.maximum(expo - (2 if bits == 4 else 8), -127))
        y = np.where(bad[..., None], 0.0, b) / (2.0 ** s.astype(np.float64))[..., None]
    g = _grid(bits)
    mag = np.minimum(np.abs(y), g[-1])
    lo = np.clip(np.searchsorted(g, mag, side="right") - 1, 0, len(g) - 1)
    hi = np.minimum(lo + 1, len(g) - 1)
    below, above = mag - g[lo], g[hi] - mag
    code = np.where((above < below) | ((above == below) & (lo % 2 == 1)), hi, lo)
    scale = np.where(bad, 255, s + 127)
    return code.reshape(x.shape), np.signbit(y).reshape(x.shape), scale.astype(np.uint8)


def values(x: np.ndarray, bits: int) -> np.ndarray:
    """What the rows stand for once quantised; NaN in the blocks that hold none."""
    code, neg, scale = quantize(x, bits)
    v = np.where(neg, -1.0, 1.0) * _grid(bits)[code]
    s = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
    return (v.reshape(*scale.shape, BLOCK) * s[..., None]).reshape(x.shape)


def linear(a: np.ndarray, w: np.ndarray, bias=None):
    """(a w^T + bias of the quantised values, the same sum of magnitudes)."""
    qa, qw = values(a, 4), values(w, 4)
    out, mag = qa @ qw.T, np.abs(qa) @ np.abs(qw).T
    return (out, mag) if bias is None else (out + bias, mag + np.abs(bias))


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """One query per head, q [H, d] over k, v [n, Hk, d] (values, not codes): (out, sum of p |v|,
    largest score error unit sum_d |q k| scale).  No keys give zeros."""
    h, d = q.shape
    if k.shape[0] == 0:
        return np.zeros((h, d)), np.zeros((h, d)), np.zeros(h)
    grp = h // k.shape[1]
    out, mag, unit = np.empty((h, d)), np.empty((h, d)), np.empty(h)
    for i in range(h):
        kk, vv = k[:, i // grp], v[:, i // grp]
        s = kk @ q[i] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i], mag[i] = p @ vv, p @ np.abs(vv)
        unit[i] = (np.abs(kk) @ np.abs(q[i])).max() * abs(scale)
    return out, mag, unit
