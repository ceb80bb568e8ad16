"""A paged cache of keys and values in few bits, in 64 bits and bytes, straight from its definition (include/axhip.h)."""
import numpy as np

from attn_oracle import Rules, attention

F16, I8, MX4 = 0, 1, 2
LADDER = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def row_bytes(kind, dk):
    return (dk * (16, 8, 4)[kind] // 8 + 15) // 16 * 16


def ladder_code(y):
    """The code of the nearest of LADDER to y >= 0: of two as near the one whose last bit is zero; the last one beyond it."""
    above = np.clip(np.searchsorted(LADDER, y), 1, 7)
    low, high = LADDER[above - 1], LADDER[above]
    return np.where((y - low > high - y) | ((y - low == high - y) & (above % 2 == 0)), above, above - 1)


def quantised(kind, x):
    """x [rows, heads, dk] fp32 -> (payload bytes [rows, heads, row bytes], scale bytes [rows, heads, 4], what they stand for in 64 bits)"""
    x = np.asarray(x, np.float32)
    rows, heads, dk = x.shape
    out = np.zeros((rows, heads, row_bytes(kind, dk)), np.uint8)
    if rows == 0:
        return out, np.zeros((0, heads, 4), np.uint8), x.astype(np.float64)
    if kind == MX4:
        groups = (dk + 31) // 32
        y = np.zeros((rows, heads, groups * 32), np.float64)
        y[..., :dk] = x
        y = y.reshape(rows, heads, groups, 32)
        finite = np.isfinite(y).all(-1, keepdims=True)
        y = np.where(finite, y, 0)
        e = np.maximum(np.frexp(np.abs(y).max(-1, keepdims=True))[1] - 1 - 2, -127)
        e = np.where(np.abs(y).max(-1, keepdims=True) == 0, -127, e)
        code = ladder_code(np.abs(y) * 2.0 ** -e)
        value = np.where(finite, np.where(np.signbit(y), -1.0, 1.0) * LADDER[code] * 2.0 ** e, np.nan).reshape(rows, heads, -1)[..., :dk]
        code = (code + 8 * np.signbit(y)).astype(np.uint8).reshape(rows, heads, -1)
        out[..., :groups * 16] = code[..., 0::2] + 16 * code[..., 1::2]
        scales = np.zeros((rows, heads, 4), np.uint8)
        scales[..., :groups] = np.where(finite, e + 127, 255)[..., 0]
        return out, scales, value
    finite = np.isfinite(x).all(-1, keepdims=True)
    y = np.where(finite, x, np.float32(0)).astype(np.float64)
    top = np.abs(y).max(-1, keepdims=True)
    if kind == F16:
        s = 2.0 ** np.maximum(np.where(top > 0, np.frexp(top)[1] - 1 - 14, -1000), -100)
        n = (y / s).astype(np.float16)
        out[..., :2 * dk] = n.view(np.uint8)
    else:
        s = np.maximum(top.astype(np.float32) / np.float32(127), np.float32(2.0 ** -100)).astype(np.float64)
        n = np.clip(np.rint(y / s), -127, 127).astype(np.int8)
        out[..., :dk] = n.view(np.uint8)
    s = np.where(finite, s, np.nan)
    return out, np.ascontiguousarray(s[..., 0].astype(np.float32)).view(np.uint8).reshape(rows, heads, 4), n.astype(np.float64) * s


class PagedRules(Rules):
    """What the queries of one sequence, its last ones, see: `there` [length] says which keys have a page."""

    def __init__(self, there, cap=0.0, slopes=None, window=0, sinks=0):
        super().__init__(cap=cap, slopes=slopes)
        self.there, self.window, self.sinks = there, window, sinks

    def sees(self, b, Sq, Sk):
        p = Sk - Sq + np.arange(Sq)
        j = np.arange(Sk)
        m = (j <= p[:, None]) & self.there[:Sk]
        if self.window:
            m &= (p[:, None] - j < self.window) | (j < self.sinks)
        return m, p


def paged_attention(q, k, v, there, scale, cap=0.0, slopes=None, window=0, sinks=0):
    """One sequence: q [n, H, dk] its last rows, k and v [length, Hkv, dk] what the cache holds (64 bits) -> attention()'s dict, o and lse by rows"""
    n = len(q)
    if len(k) == 0:
        none = {"o": np.zeros(q.shape), "lse": np.full(q.shape[:2], -np.inf)}
        return dict(none, tol_o=np.zeros(q.shape), tol_lse=np.zeros(q.shape[:2]))
    w = attention(q[None], k[None], v[None], scale, PagedRules(there, cap, slopes, window, sinks))
    return {"o": w["o"][0], "lse": w["lse"][0].T, "tol_o": w["tol_o"][0], "tol_lse": w["tol_lse"][0].T}
