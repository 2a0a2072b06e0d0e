"""Inputs and bounds for the attention over the four-bit cache that a wrong result cannot meet.

The bound of a number of the result follows the roundings that each kernel makes, with u = 2^-8 (half a step of bf16, relative to the value):

* both: the result is rounded to bf16, u |y|.
* few rows: keys and values are exact.  Each weight times its value's step is rounded to bf16 and meets code - 8: u sum p step |c - 8|.  A score is
  a (q . (128 + c)) + b sum(q), a = scale step, b = scale (low - 128 step), in f32: a, b, the product and the sum are rounded, four times 2^-24 of the two terms at most, and the
  sums over the head lose nothing where q's numbers are 0 or one power of two (sums of whole numbers below 2^24), else (dim + 4) 2^-23 of sum |q| in each term.
* many rows: keys and values are step * code + low rounded once to bf16, at most bf16's largest number; the reference takes them as they are then.  Each weight is rounded: u sum p |v|.
  A score's f32 sum is off by (dim + 4) 2^-23 of scale sum |q k|.
* A score off by e_j moves the normalised weight p_j to p_j' with |p_j' - p_j| <= p_j (exp(e_j + E) - 1), exp(E) = sum p exp(e), and as both sum to one the result moves by no more
  than sum p_j (exp(e_j + E) - 1) |v_j - y|.
* both: f32 sums of weights and products, at most tokens / 16 + 200 additions in a row where work is shared among lanes, each off by 2^-23 of the sum; powers of two within 2^-21.
"""
import numpy as np

import kv4_reference as ref

U = 2.0**-8
BF16_MAX = float(ref.from_bits(np.array([0x7F7F]))[0])


def bf16_once(x):
    """f64 rounded to the nearest bf16 (ties to even) in one step, as f64."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        unit = np.maximum(np.frexp(x)[1] - 8, -133)
        r = np.ldexp(np.rint(np.ldexp(x, -unit)), unit)
        r = np.where(np.abs(r) > BF16_MAX, np.copysign(np.inf, x), r)
    return np.where(np.isfinite(x), r, x)


def is_few(rows, group):
    """Whether a sequence of so many rows is the few-rows kernel's."""
    return group <= 16 and rows * group <= 16


def visible(tokens, n, window):
    j = np.arange(n)
    seen = j <= tokens[:, None]
    return seen & (j > tokens[:, None] - window) if window else seen


class Exact:
    """One sequence's attention in 64 bits: q [rows, heads, dim] (f64 of bf16 numbers) at `tokens`, keys and values f32 [len, kv_heads, dim] as they were appended.
    ``y`` and ``bound`` [rows, heads, dim]; ``without(gone)`` and ``masked(seen)`` are results of what a wrong kernel might do."""

    def __init__(self, q, k, v, tokens, scale, window, whole_q=False):
        rows, heads, dim = q.shape
        kv_heads = k.shape[1]
        self.q, self.scale, self.heads, self.group, self.few = q, scale, heads, heads // kv_heads, is_few(rows, heads // kv_heads)
        self.held = [ref.held(x) for x in (k, v)]
        if not self.few:
            self.held = [np.clip(bf16_once(x), -BF16_MAX, BF16_MAX) for x in self.held]
        self.seen = visible(np.asarray(tokens), k.shape[0], window)
        _, k_step, k_low = (x[..., None] if x.ndim == 2 else x for x in ref.quantise(k))
        v_codes, v_step, _ = ref.quantise(v)
        k_step, k_low = k_step.astype(np.float64)[..., 0], k_low.astype(np.float64)[..., 0]
        self.y, self.bound = np.zeros(q.shape), np.zeros(q.shape)
        adds = (k.shape[0] / 16 + 200) * 2.0**-23 + 2.0**-21
        for h in range(heads):
            g = h // self.group
            kk, vv = self.held[0][:, g], self.held[1][:, g]
            p = self._weights(h, self.seen)
            y = p @ vv
            size = np.abs(q[:, h]).sum(-1)[:, None]
            if self.few:
                a, b = np.abs(k_step[:, g]), np.abs(k_low[:, g] - 128 * k_step[:, g])
                terms = scale * ((143 * a + b) * size)
                e = terms * (2.0**-22 if whole_q else 2.0**-22 + (dim + 4) * 2.0**-23)
                cut = p @ (np.abs(v_step[:, g])[:, None] * np.abs(v_codes[:, g].astype(np.float64) - 8))
                parts = p @ (np.abs(v_step[:, g, None] * (v_codes[:, g] - 8.0)) + np.abs(vv))
            else:
                e = (dim + 4) * 2.0**-23 * scale * (np.abs(q[:, h]) @ np.abs(kk).T)
                cut = parts = p @ np.abs(vv)
            e = np.where(self.seen, np.broadcast_to(e, p.shape), 0.0)
            both = np.log(np.maximum((p * np.exp(e)).sum(-1, keepdims=True), 1.0))
            factor = p * np.expm1(e + both)
            moved = np.stack([(factor[r][:, None] * np.abs(vv - y[r])).sum(0) for r in range(rows)])
            self.y[:, h], self.bound[:, h] = y, U * np.abs(y) + U * cut + moved + adds * parts

    def _weights(self, h, seen):
        x = np.where(seen, self.q[:, h] @ self.held[0][:, h // self.group].T * self.scale, -np.inf)
        top = x.max(-1, keepdims=True)
        p = np.exp(x - np.where(np.isfinite(top), top, 0.0))
        return p / np.maximum(p.sum(-1, keepdims=True), 1e-300)

    def masked(self, seen):
        """The result under another mask [rows, len]."""
        return np.stack([self._weights(h, seen) @ self.held[1][:, h // self.group] for h in range(self.heads)], 1)

    def over(self, y):
        """How far the worst number of each row is over its bound, [rows]; positive: refused."""
        with np.errstate(all="ignore"):
            d = np.abs(y - self.y) - self.bound
        return np.where(np.isnan(d), np.inf, d).max((1, 2))


def hot_run_case(rng, n, heads, dim, scale, classes):
    """Keys and values of a sequence whose every run of 64 tokens has one token that matters, and only to queries of its class: run c to class c % classes, the direction of
    that number.  Losing a run changes the rows of its class by a share that no rounding reaches."""
    k, v = (rng.standard_normal((n, heads, dim)).astype(np.float32) * s for s in (np.float32(0.3), np.float32(1.0)))
    runs = np.arange(-(-n // 64))
    at = np.minimum(runs * 64 + rng.integers(0, 64, len(runs)), n - 1)
    k[at, :, runs % classes] += np.float32(12.0 / scale)
    return k, v, at


def hot_edge_case(rng, n, heads, dim, scale):
    """Keys and values where every token matters to queries of its own direction, token % dim."""
    k, v = (rng.standard_normal((n, heads, dim)).astype(np.float32) * s for s in (np.float32(0.3), np.float32(1.0)))
    k[np.arange(n), :, np.arange(n) % dim] += np.float32(12.0 / scale)
    return k, v


def edge_queries(tokens, heads, dim, window):
    """Queries of rows at `tokens` that look at the tokens on both sides of what they see."""
    q = np.zeros((len(tokens), heads, dim))
    for r, p in enumerate(tokens):
        for j in (p, p + 1) + ((p - window, p - window + 1) if window else ()):
            if j >= 0:
                q[r, :, j % dim] = 1.0
    return q


# lens of one sequence: n, rows, heads, group, dim, page
LONG = [(20011, 1, 1, 1, 64, 64), (20011, 1, 1, 8, 128, 64), (20011, 4, 1, 4, 128, 64), (20011, 2, 2, 5, 64, 16), (20011, 1, 1, 16, 128, 32), (20011, 20, 1, 4, 128, 64),
        (20011, 130, 1, 2, 64, 64), (9000, 1, 2, 17, 64, 32), (40000, 1, 1, 4, 128, 64), (33333, 5, 1, 8, 128, 64)]
# n, rows, heads, group, dim, page, window
EDGES = [(2000, 1, 1, 8, 128, 16, 0), (1000, 3, 1, 6, 128, 64, 0), (513, 40, 2, 5, 128, 64, 0), (1999, 1, 4, 1, 64, 64, 777), (400, 257, 1, 3, 128, 16, 0), (700, 1, 1, 16, 128, 32, 0),
         (300, 200, 1, 4, 128, 32, 64), (520, 300, 1, 1, 128, 64, 129), (1500, 5, 2, 3, 64, 32, 1000), (1500, 16, 1, 1, 128, 64, 200), (1300, 100, 1, 7, 64, 16, 500), (129, 2, 2, 8, 64, 64, 1)]
# n, rows, heads, group, dim, page, sharp, scale: random scores
RANDOM = [(150, 1, 1, 4, 128, 32, 40.0, None), (150, 6, 1, 1, 128, 32, 40.0, None), (150, 50, 1, 4, 128, 32, 40.0, None), (150, 1, 1, 4, 64, 32, 1.5, 3.0), (150, 50, 1, 4, 64, 32, 1.5, 3.0),
          (3000, 1, 2, 4, 128, 64, 1.5, None), (3000, 30, 2, 2, 64, 16, 1.5, None), (3000, 12, 1, 1, 64, 32, 1.5, None)]


def long_case(n, rows, heads, group, dim, page):
    """(k, v, at, queries of each call [rows, heads * group, dim], scale): the calls' columns share the classes out among them."""
    rng = np.random.default_rng(n + 7 * rows + dim + group)
    scale, cols = dim**-0.5, rows * group
    calls = -(-16 // cols)
    classes = min(calls * cols, dim)
    k, v, at = hot_run_case(rng, n, heads, dim, scale, classes)
    qs = []
    for m in range(calls):
        q = np.zeros((rows, heads, group, dim))
        for r in range(rows):
            for g in range(group):
                q[r, :, g, (m * cols + r * group + g) % classes] = 1.0
        qs.append(q.reshape(rows, heads * group, dim))
    return k, v, at, qs, scale


def edge_case(n, rows, heads, group, dim, page, window):
    rng = np.random.default_rng(n + 7 * rows + dim + group + window)
    scale, tokens = dim**-0.5, np.arange(n - rows, n)
    k, v = hot_edge_case(rng, n, heads, dim, scale)
    return k, v, edge_queries(tokens, heads * group, dim, window), scale


def random_case(n, rows, heads, group, dim, page, sharp, scale):
    rng = np.random.default_rng(n + 7 * rows + dim + group)
    k = (rng.standard_normal((n, heads, dim)) + rng.standard_normal((1, heads, dim)) * 0.5).astype(np.float32)
    v = (rng.standard_normal((n, heads, dim)) + rng.standard_normal((1, heads, dim))).astype(np.float32)
    q = ref.bf16_round((rng.standard_normal((rows, heads * group, dim)) * sharp).astype(np.float32)).astype(np.float64)
    return k, v, q, scale or dim**-0.5
