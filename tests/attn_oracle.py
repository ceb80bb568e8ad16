"""Rotary positions, norms of heads and attention under score rules in 64 bits, straight from their definitions (include/axhip.h), with their gradients;
and how far fp32 kernels may be from them.

A bound counts half steps of fp32, U = 2^-24.  A product of two operands is off by at most 8 U of its size (each operand rounded to 23 bits, 2 U each,
and what a product of two terms leaves out, 4 U); a sum of n products by n U of the sum of sizes; exp2 of a number x in log2 units by
2 |x| U ln 2 + 4 U, where the rounding of x itself counts.  A probability below 2^-126, the smallest float that the exponential gives, comes out as zero: off
by TINY = 2^-126 whatever its size, so every pair adds TINY times the size of what its probability multiplies."""
import numpy as np

U = 2.0 ** -24
TINY = 2.0 ** -126
LOG2E = 1.4426950408889634


# ---- rows of heads ---------------------------------------------------------------------------------------------------

def rotate(x, pos, freq, rot, amplitude, layout, back=False):
    """x [rows, heads, dk]"""
    a = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)
    c, s = amplitude * np.cos(a), amplitude * np.sin(a) * (-1 if back else 1)
    out = np.array(x, np.float64)
    i = np.arange(rot // 2)
    p, q = (2 * i, 2 * i + 1) if layout == 0 else (i, i + rot // 2)
    out[..., p], out[..., q] = x[..., p] * c - x[..., q] * s, x[..., q] * c + x[..., p] * s
    return out


def pair_size(x, rot, amplitude, layout):
    """For every value the size of what its rotation adds up: amplitude (|x| + |y|) of its pair, |x| where it is not turned."""
    x = np.abs(np.asarray(x, np.float64))
    out = np.array(x)
    i = np.arange(rot // 2)
    p, q = (2 * i, 2 * i + 1) if layout == 0 else (i, i + rot // 2)
    out[..., p] = out[..., q] = abs(amplitude) * (x[..., p] + x[..., q])
    return out


def inv_rms(x, eps):
    return 1 / np.sqrt((x.astype(np.float64) ** 2).mean(-1) + eps)


def norm_grad(dn, x, r, gamma):
    """(dx, dn * xhat) of y = gamma x r(x), r = 1 / sqrt(mean x^2 + eps) given; all [rows, heads, dk] but r [rows, heads]."""
    hat = x * r[..., None]
    g = dn * gamma
    return r[..., None] * (g - hat * (g * hat).mean(-1, keepdims=True)), dn * hat


# ---- attention -------------------------------------------------------------------------------------------------------

class Rules:
    """Host arrays or None, as axhip_attn_rules."""

    def __init__(self, cap=0.0, causal=0, slopes=None, prefix=None, start=None, lens=None, doc_q=None, doc_k=None):
        self.cap, self.causal, self.slopes, self.prefix, self.start, self.lens, self.doc_q, self.doc_k = cap, causal, slopes, prefix, start, lens, doc_q, doc_k

    ARRAYS = ("slopes", "prefix", "start", "lens", "doc_q", "doc_k")

    def sees(self, b, Sq, Sk):
        """[Sq, Sk] and the positions [Sq]"""
        n = Sk if self.lens is None else min(max(int(self.lens[b]), 0), Sk)
        p = (Sk - Sq if self.start is None else int(self.start[b])) + np.arange(Sq)
        j = np.arange(Sk)
        m = np.broadcast_to(j < n, (Sq, Sk)).copy()
        if self.causal:
            m &= (j <= p[:, None]) | (j < (0 if self.prefix is None else int(self.prefix[b])))
            m &= p[:, None] < n
        if self.doc_q is not None:
            m &= (self.doc_q[b][:, None] == self.doc_k[b]) & (self.doc_q[b][:, None] >= 0)
        return m, p

    def scores(self, raw, h, p, Sk):
        """(scores, their derivative by raw)"""
        slope = np.ones_like(raw)
        x = raw
        if self.cap:
            t = np.tanh(raw / self.cap)
            x, slope = self.cap * t, 1 / np.cosh(np.clip(raw / self.cap, -300, 300)) ** 2
        if self.slopes is not None:
            x = x - float(self.slopes[h]) * np.abs(p[:, None] - np.arange(Sk))
        return x, slope


def attention(q, k, v, scale, rules, d_o=None):
    """q [B, Sq, H, dk], k and v [B, Sk, Hkv, dk] -> dict of results and, for each, its bound ("tol_...").  What a query does not see is left out of
    every sum, whatever it holds."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    B, Sq, H, dk = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    out = {"o": np.zeros((B, Sq, H, dk)), "lse": np.full((B, H, Sq), -np.inf)}
    out.update({"tol_o": np.zeros(out["o"].shape), "tol_lse": np.zeros(out["lse"].shape)})
    if d_o is not None:
        d_o = np.asarray(d_o, np.float64)
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            out[n], out["tol_" + n] = np.zeros(x.shape), np.zeros(x.shape)
    for b in range(B):
        m, p = rules.sees(b, Sq, Sk)
        kk_any = m.any(0)
        for h in range(H):
            g = h * Hkv // H
            qq = np.where(m.any(1)[:, None], q[b, :, h], 0)
            kk, vv = np.where(kk_any[:, None], k[b, :, g], 0), np.where(kk_any[:, None], v[b, :, g], 0)
            with np.errstate(all="ignore"):
                raw = qq @ kk.T * scale
                size = np.abs(qq) @ np.abs(kk).T * abs(scale)
            x, slope = rules.scores(raw, h, p, Sk)
            # a pair that is not seen may hold infinities of rows that others see
            x, size, slope = np.where(m, x, -np.inf), np.where(m, size, 0), np.where(m, slope, 0)
            top = x.max(-1, keepdims=True, initial=-np.inf)
            live = np.isfinite(top[:, 0])
            with np.errstate(all="ignore"):
                e = np.where(m, np.exp(x - top), 0)
                total = e.sum(-1, keepdims=True)
                P = np.where(m & live[:, None], e / total, 0)
                lse = np.where(live, (top + np.log(total))[:, 0], -np.inf)
            out["lse"][b, h] = lse
            o = P @ vv
            out["o"][b, :, h] = o
            # errors of a score (natural units), of the exponential, of a probability relative to itself
            biggest = np.where(m, np.abs(np.where(m, x, 0)), 0).max(-1, initial=0)
            dx = U * ((dk + 12) * size.max(-1, initial=0) + 3 * biggest)
            rel = 2 * dx + U * (4 * LOG2E * biggest + Sk / 8 + 24)
            out["tol_o"][b, :, h] = rel[:, None] * (P @ np.abs(vv)) + TINY * np.abs(vv).sum(0) + 1e-38
            out["tol_lse"][b, h] = np.where(live, dx + U * (4 * np.abs(np.where(live, lse, 0)) + 4 * biggest + Sk / 8 + 24), 0)
            if d_o is None:
                continue
            do = np.where(live[:, None], d_o[b, :, h], 0)
            dp, dp_size = do @ vv.T, np.abs(do) @ np.abs(vv).T
            delta, delta_size = (do * o).sum(-1, keepdims=True), (np.abs(do) * np.abs(o)).sum(-1, keepdims=True)
            ds = P * (dp - delta) * slope
            # log-sum-exp comes rounded to fp32
            relp = (rel + 2 * U * np.abs(np.where(live, lse, 0)))[:, None]
            err = TINY * (dp_size + delta_size) + relp * np.abs(ds) + P * slope * U * ((dk + 12) * dp_size + (dk + 12) * delta_size) + P * relp * delta_size * slope
            if rules.cap:                        # the slope's own error: as the score's, over the cap, twice
                err += P * np.abs(dp - delta) * (2 * dx[:, None] / rules.cap + 16 * U)
            n = Sq * (H // Hkv)
            out["dq"][b, :, h] = ds @ kk * scale
            out["tol_dq"][b, :, h] = abs(scale) * (err @ np.abs(kk) + U * (Sk / 8 + 24) * (np.abs(ds) @ np.abs(kk))) + 1e-38
            out["dk"][b, :, g] += ds.T @ qq * scale
            out["tol_dk"][b, :, g] += abs(scale) * (err.T @ np.abs(qq) + U * (n / 8 + 24) * (np.abs(ds).T @ np.abs(qq))) + 1e-38
            out["dv"][b, :, g] += P.T @ do
            out["tol_dv"][b, :, g] += (P * relp).T @ np.abs(do) + TINY * np.abs(do).sum(0) + U * (n / 8 + 24) * (P.T @ np.abs(do)) + 1e-38
    return out
