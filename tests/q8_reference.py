"""Rows in eight bits, the norm and the products on them, restated in numpy: what is defined operation by operation is computed so (f32, or f64 where the
definition says f64), the gated product in f64."""
import numpy as np

from kv4_reference import bf16_bits, bf16_round, from_bits  # noqa: F401  (used by the tests that import this file)

F = np.float32


def hold(x):
    """Codes (i8) and scales (f32) of rows x (f32)."""
    x = np.asarray(x, F)
    most = np.abs(x).max(-1) if x.shape[-1] else np.zeros(x.shape[:-1], F)      # (NaN where the row has one)
    fine = np.isfinite(most)
    held = fine & (np.where(fine, most, 0) >= F(2.0**-119))
    safe = np.where(held, most, F(1))
    codes = np.rint(np.where(held[..., None], x, F(0)) * (F(127) / safe)[..., None])
    return codes.astype(np.int8), np.where(held, safe / F(127), np.where(fine, F(0), F(np.nan))).astype(F)


def rmsnorm(x, weight, eps, residual=None, residual_bf16=True):
    """(y in f32, h): every operation rounded as documented."""
    h = np.asarray(x, F)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        if residual is not None:
            h = h + np.asarray(residual, F)
            if residual_bf16:
                h = bf16_round(h)
        s = (h.astype(np.float64)**2).sum(-1, keepdims=True)
        r = (1 / np.sqrt(s / h.shape[-1] + np.float64(F(eps)))).astype(F)
        return (h * r) * np.asarray(weight, F), h


def product(a, a_scales, w, w_scales, bias=None):
    """f32 rows: the exact sum, rounded, times both scales, plus the bias."""
    sums = np.asarray(a, np.float64) @ np.asarray(w, np.float64).T              # whole numbers below 2^53: exact in any order
    with np.errstate(invalid="ignore", over="ignore"):
        y = (sums.astype(F) * np.asarray(a_scales, F)[:, None]) * np.asarray(w_scales, F)
        return y if bias is None else y + np.asarray(bias, F)


def gated(a, a_scales, gate, gate_scales, up, up_scales, act):
    """(y, bound) in f64: act(g) u, and how far an f32 computation may be off.

    With u = 2^-24: g and u carry three roundings each (the sum's, two products').  act(g)'s relative change is at most (1 + 1.702 |g|) times g's.  The sigmoid's power of two has
    an argument of up to 2.46 |g| with three roundings (its constants', two products'): 7.4 |g| u in the argument, ln 2 of that in the result; the hardware's power of two and
    reciprocal with its Newton step add 4 u and 2 u, the products behind them 2 u.  In sum (14 + 11 |g|) u; and where the sigmoid leaves the normal range of f32, zero."""
    exact = lambda q, s: (np.asarray(a, np.float64) @ np.asarray(q, np.float64).T) * np.asarray(a_scales, np.float64)[:, None] * np.asarray(s, np.float64)  # noqa: E731
    g, u = exact(gate, gate_scales), exact(up, up_scales)
    if act == "relu":
        y = np.maximum(g, 0) * u
    else:
        with np.errstate(over="ignore"):
            y = g / (1 + np.exp(-g * (1.702 if act == "gelu" else 1.0))) * u
    return y, (14 + 11 * np.abs(g)) * 2.0**-24 * np.abs(y) + 2.0**-118 * np.abs(u) + 2.0**-140
