"""Plain restatement of the four-bit key/value cache and of the attention over it: the cache's rule in f32 steps (numpy, every
operation rounded as the header says), everything after it in 64 bits."""
import numpy as np

U = 2.0**-8                     # half a step of bf16, relative to the value


def bf16_round(x):
    """f32 rounded to the nearest bf16 (ties to even), as f32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def bf16_bits(x):
    return (bf16_round(x).view(np.uint32) >> 16).astype(np.uint16)


def from_bits(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def _down(x):
    bits = np.ascontiguousarray(x, np.float32).view(np.int32).astype(np.int64)
    cut = bits & ~0xFFFF
    cut = np.where((bits != cut) & (bits < 0), cut + 0x10000, cut)
    return cut.astype(np.int32).view(np.float32)


def quantise(x):
    """codes u8, step f32, low f32 of rows of f32 [..., dim]."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(x).all(-1, keepdims=True)
        y = np.where(bad, np.float32(0), x)
        low = _down(y.min(-1, keepdims=True))
        spread = y.max(-1, keepdims=True) - low
        bad |= ~np.isfinite(spread)
        step = -_down(-(spread / np.float32(15)))
        step = np.where(step < np.float32(2.0**-126), np.float32(0), step)
        codes = np.where(step > 0, np.clip(np.rint((y - low) / np.where(step > 0, step, 1)), 0, 15), 0)
    nan = np.float32(np.nan)
    return np.where(bad, 0, codes).astype(np.uint8), np.where(bad, nan, step)[..., 0], np.where(bad, nan, low)[..., 0]


def held(x):
    """What the cache holds of rows of f32, in 64 bits."""
    codes, step, low = quantise(x)
    return step[..., None].astype(np.float64) * codes + low[..., None].astype(np.float64)


def block_bytes(k, v):
    """The bytes of blocks that hold these keys and values, f32 [..., page, dim] -> u8 [..., page * (dim + 8)]."""
    codes_out, params_out = [], []
    for x in (k, v):
        codes, step, low = quantise(x)
        c = codes.reshape(*codes.shape[:-1], -1, 8)
        words = np.zeros(c.shape[:-1], np.uint32)
        for e in range(8):
            words |= c[..., e].astype(np.uint32) << np.uint32(4 * (e // 2 + 4 * (e % 2)))
        codes_out.append(words.reshape(*codes.shape[:-2], -1).view(np.uint8))
        p = np.stack([np.where(np.isnan(step), np.uint16(0x7FC0), bf16_bits(step)), np.where(np.isnan(low), np.uint16(0x7FC0), bf16_bits(low))], -1)
        params_out.append(np.ascontiguousarray(p.reshape(*p.shape[:-2], -1)).view(np.uint8))
    return np.concatenate(codes_out + params_out, -1)


def rotate(x, cs, interleaved):
    """Rows [rows, heads, dim] f32 turned by cs [rows, pairs, 2], every operation rounded to f32."""
    x = np.array(x, np.float32)
    pairs = cs.shape[1]
    first = np.arange(pairs) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., first], x[..., second]
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    return x


def attention(q, k, v, tokens, scale, window):
    """Rows q [rows, heads, dim] at `tokens` over keys and values [len, kv_heads, dim], all f64.  Returns y and, for the bounds of the tests,
    sum p |v| and the largest sum |q k| scale of what each row sees, [rows, heads, dim] and [rows, heads]."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    y, weight, reach = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    j = np.arange(k.shape[0])
    for r in range(rows):
        seen = j[(j <= tokens[r]) & ((j > tokens[r] - window) if window else True)]
        if len(seen) == 0:
            continue
        for h in range(heads):
            kk, vv = k[seen, h // group], v[seen, h // group]
            x = kk @ q[r, h] * scale
            with np.errstate(all="ignore"):
                p = np.exp(x - x.max())
                p /= p.sum()
                y[r, h], weight[r, h] = p @ vv, p @ np.abs(vv)
                reach[r, h] = (np.abs(kk) @ np.abs(q[r, h])).max() * scale
    return y, weight, reach


class Cache:
    """A cache with sequences in it: f32 keys and values of every token, their pages in the pool in a shuffled order."""

    def __init__(self, rng, lens, heads, dim, page, spare=3, extra_columns=1, scale=1.0):
        self.lens, self.heads, self.dim, self.page = list(lens), heads, dim, page
        counts = [-(-n // page) for n in lens]
        self.n_pages = sum(counts) + spare
        self.stride = max(counts + [1]) + extra_columns
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.stride), -1, np.int32)      # an entry that nothing may look at
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.k = [(rng.standard_normal((n, heads, dim)) * scale + rng.standard_normal((1, heads, dim)) * 0.5).astype(np.float32) for n in lens]
        self.v = [rng.standard_normal((n, heads, dim)).astype(np.float32) for n in lens]

    def pool(self, fill=0xFF):
        """The bytes of the pool; where no token is, `fill` (0xFF: parameters that are NaN)."""
        block = self.page * (self.dim + 8)
        out = np.full((self.n_pages, self.heads, block), fill, np.uint8)
        half = self.page * self.dim // 2
        for b, n in enumerate(self.lens):
            for c in range(-(-n // self.page)):
                have = min(self.page, n - c * self.page)
                k, v = (np.zeros((self.heads, self.page, self.dim), np.float32) for _ in range(2))
                k[:, :have] = self.k[b][c * self.page:c * self.page + have].transpose(1, 0, 2)
                v[:, :have] = self.v[b][c * self.page:c * self.page + have].transpose(1, 0, 2)
                new = block_bytes(k, v)
                to = out[self.table[b, c]]
                for start, row in ((0, self.dim // 2), (half, self.dim // 2), (2 * half, 4), (2 * half + 4 * self.page, 4)):
                    to[:, start:start + have * row] = new[:, start:start + have * row]
        return out
