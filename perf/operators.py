"""Performance cases of the operators between the projections of a step and its output projection: a paged key/value cache held
in four bits, the append that fills it (with the position rotation on the way), the attention that reads it, and its read-out.

``listed()`` names the cases, ``draw(rng)`` makes further ones of the same ranges, ``prepare(case, seed)`` is what a program holds
before the call, ``run(state)`` is one pass, ``work(case)`` the bytes and operations that the pass cannot do without, and
``exact(case, seed)`` the same results in 64 bits.  With ``own`` false, ``run`` computes the operators in elementary torch
operations; with ``own`` true it calls the framework.

The kinds of pass (``case["kind"]``):

* ``append``   the new rows' keys and values are rotated, cut to four bits and put into the cache, the queries are rotated; then the
               appended rows are read back, so that what is held comes out as the values it stands for.
* ``restore``  the rows of whole sequences are read out of the cache as bf16 (a sequence that leaves for another place).
* ``attend``   attention of each sequence's new rows over its cache: one row a sequence (token generation), a few (verification of
               proposed tokens), or a prompt, in one piece or as a chunk behind what is cached already, or all of these mixed.

The cache: pages of ``page`` tokens; a page holds one block for each key/value head: codes of the keys [page][dim / 2], codes of
the values, then for each key and for each value row its (step, low) in bf16.  Code e of a row lies in 32-bit word e / 8, at nibble
(e % 8) / 2 + 4 (e % 2), and stands for step * code + low.
"""
from __future__ import annotations

import math

import torch

own = False

SHIFTS = [4 * ((e >> 1) + 4 * (e & 1)) for e in range(8)]


def listed():
    return [
        # one sequence's next token, queries, keys and values as the W4A16 products leave them: latency counts
        {"name": "append_one_token", "kind": "append", "seqs": 1, "rows": 1, "len": 300, "ragged": False, "heads": 8, "group": 4, "dim": 128,
         "page": 64, "type": "f32", "axes": 1, "rot": 128, "interleaved": False},
        # the next tokens of a batch of 256
        {"name": "append_256_tokens", "kind": "append", "seqs": 256, "rows": 1, "len": 2048, "ragged": True, "heads": 8, "group": 4, "dim": 128,
         "page": 32, "type": "f32", "axes": 1, "rot": 128, "interleaved": False},
        # a prompt of text and video frames: bf16 rows, three position axes
        {"name": "append_prompt_3_axes", "kind": "append", "seqs": 1, "rows": 8192, "len": 8192, "ragged": False, "heads": 8, "group": 4, "dim": 128,
         "page": 64, "type": "bf16", "axes": 3, "rot": 128, "interleaved": False},
        # a short sequence read out, small heads
        {"name": "restore_37_rows", "kind": "restore", "seqs": 1, "rows": 37, "len": 37, "ragged": False, "heads": 4, "group": 1, "dim": 64, "page": 16},
        # sixteen sequences read out whole
        {"name": "restore_16_sequences", "kind": "restore", "seqs": 16, "rows": 4000, "len": 4000, "ragged": True, "heads": 8, "group": 1, "dim": 128, "page": 64},
        # the smallest step: one token over a short context
        {"name": "decode_one_short", "kind": "attend", "seqs": 1, "rows": 1, "len": 77, "ragged": False, "heads": 8, "group": 4, "dim": 128, "page": 16, "window": 0},
        # a full batch of token generation, contexts of all lengths, one slot empty
        {"name": "decode_batch_128", "kind": "attend", "seqs": 128, "rows": 1, "len": 8192, "ragged": True, "heads": 8, "group": 8, "dim": 128, "page": 64, "window": 0},
        # one token over one long context: the work has to be split along it
        {"name": "decode_long_131072", "kind": "attend", "seqs": 1, "rows": 1, "len": 131072, "ragged": False, "heads": 8, "group": 8, "dim": 128, "page": 64, "window": 0},
        # five proposed tokens a sequence, a head for every query head, a sliding window
        {"name": "verify_5_window", "kind": "attend", "seqs": 32, "rows": 5, "len": 2500, "ragged": True, "heads": 16, "group": 1, "dim": 64, "page": 32, "window": 1000},
        # a chunk of a prompt behind what is cached already
        {"name": "chunk_2048_on_8192", "kind": "attend", "seqs": 1, "rows": 2048, "len": 10240, "ragged": False, "heads": 8, "group": 4, "dim": 128, "page": 64, "window": 0},
        # single tokens and chunks of all sizes in one batch, a group of seven
        {"name": "mixed_batch_24", "kind": "attend", "seqs": 24, "rows": 701, "len": 4096, "ragged": True, "heads": 4, "group": 7, "dim": 64, "page": 16, "window": 0},
        # a prompt in one piece
        {"name": "prompt_8192", "kind": "attend", "seqs": 1, "rows": 8192, "len": 8192, "ragged": False, "heads": 8, "group": 4, "dim": 128, "page": 64, "window": 0},
    ]


# --------------------------------------------------------------------------- further cases of the same ranges

def _log(rng, lo, hi):
    return int(min(max(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))), lo), hi))


def draw(rng):
    kind = rng.choice(["append", "append", "restore", "attend", "attend", "attend", "attend"])
    dim, page, heads = rng.choice([64, 128]), rng.choice([16, 32, 64]), rng.choice([1, 2, 4, 8, 8, 12, 16])
    if kind == "append":
        group, rows = rng.choice([1, 2, 4, 7, 8]), rng.choice([1, 1, _log(rng, 2, 8192)])
        seqs = _log(rng, 1, 256 if rows == 1 else max(1, 8192 // rows))
        most = 8192 * 48 * 128 // (dim * heads * (group + 2))            # rows that cost what the listed prompt costs
        rows, seqs = max(1, min(rows, most)), max(1, min(seqs, most // max(1, min(rows, most))))
        return {"kind": kind, "seqs": seqs, "rows": rows, "len": rows + _log(rng, 1, 4096) - 1, "ragged": rng.random() < 0.5, "heads": heads,
                "group": group, "dim": dim, "page": page, "type": rng.choice(["f32", "bf16"]), "axes": rng.choice([1, 3]),
                "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.3}
    if kind == "restore":
        rows = _log(rng, 1, 32768)
        seqs = max(1, min(64, 16 * 4000 * 8 * 128 // (rows * heads * dim)))
        return {"kind": kind, "seqs": rng.randint(1, seqs), "rows": rows, "len": rows, "ragged": rng.random() < 0.5, "heads": heads, "group": 1,
                "dim": dim, "page": page}
    group, window = rng.choice([1, 2, 3, 4, 7, 8, 16]), rng.choice([0, 0, 0, 128, 1000, 4096])
    if rng.random() < 0.6:                                               # token generation and verification
        rows = rng.choice([1, 1, 1, 2, 3, 5, 8])
        length = rows + _log(rng, 1, 131072) - 1
        most = 10**9 // (length * heads * (dim + 8))                     # bytes of cache that cost no more than the largest batch
        return {"kind": kind, "seqs": _log(rng, 1, max(1, min(256, most))), "rows": rows, "len": length, "ragged": rng.random() < 0.7, "heads": heads,
                "group": group, "dim": dim, "page": page, "window": window}
    rows = _log(rng, 17, 8192)
    length = rows + rng.choice([0, _log(rng, 1, 32768)])
    while 4 * dim * heads * group * rows * length > 11e11 // 2:          # no more than half of the square of the listed prompt
        rows, length = max(1, rows // 2), max(rows // 2, length // 2)
    most = int(11e11 // 2 / (4 * dim * heads * group * rows * length))
    return {"kind": kind, "seqs": _log(rng, 1, max(1, min(32, most))), "rows": rows, "len": length, "ragged": rng.random() < 0.5, "heads": heads,
            "group": group, "dim": dim, "page": page, "window": window}


# --------------------------------------------------------------------------- shapes of a batch

def _uneven(b):
    """A fraction in (0, 1], another for each sequence, spread over the range."""
    return 1.0 - (0.6180339887 * b) % 1.0


def _rows(case):
    """New rows of each sequence."""
    n, seqs = case["rows"], case["seqs"]
    if not case["ragged"] or n <= 8:
        return [n] * seqs
    if case["kind"] != "attend":
        return [max(1, int(n * _uneven(b))) for b in range(seqs)]
    return [n if b == 0 else max(1, int(n * _uneven(b) ** 3)) for b in range(seqs)]


def _lens(case):
    """Tokens of each sequence, the new rows among them; the sixth slot of a large batch of single tokens is empty."""
    rows, n = _rows(case), case["len"]
    if case["kind"] == "restore":
        return rows
    if not case["ragged"]:
        return [n] * case["seqs"]
    lens = [max(rows[b], int(n * (0.25 + 0.75 * _uneven(b)))) for b in range(case["seqs"])]
    if case["kind"] == "attend" and case["seqs"] > 16 and case["rows"] == 1:
        lens[5] = 0
    return lens


# --------------------------------------------------------------------------- inputs

def _bf16_down(x):
    """The largest bf16 not above x (f32), as f32."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    return torch.where((bits != cut) & (bits < 0), cut + 65536, cut).view(torch.float32)


def _quantise(x):
    """Codes, step and low of rows of f32: the operator's definition, each operation rounded to f32."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    low = _bf16_down(low)
    step = -_bf16_down(-((high - low) / torch.full_like(low, 15.0)))     # (a plain 15.0 would be multiplied by its rounded inverse)
    step = torch.where(step < 2.0**-126, torch.zeros_like(step), step)
    codes = torch.where(step > 0, torch.round((x - low) / step).clamp(0, 15), torch.zeros_like(x))
    return codes, step, low


def _block(k, v):
    """The bytes of blocks that hold these rows: k, v f32 [..., page, dim]."""
    parts, params = [], []
    for x in (k, v):
        codes, step, low = _quantise(x)
        words = codes.to(torch.int64).unflatten(-1, (-1, 8))
        words = torch.stack([words[..., e] << SHIFTS[e] for e in range(8)], -1).sum(-1)
        parts.append(torch.where(words >= 2**31, words - 2**32, words).to(torch.int32).flatten(-2).view(torch.uint8))
        params.append(torch.cat([step, low], -1).to(torch.bfloat16).flatten(-2).view(torch.uint8))
    return torch.cat(parts + params, -1)


def _table(case):
    """cos and sin of every position and pair, f32 [positions][pairs][2]."""
    pairs, n = case["rot"] // 2, max(_lens(case)) + 64
    rate = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
    angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * rate
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def _axis_pairs(case):
    pairs = case["rot"] // 2
    return [pairs] if case["axes"] == 1 else [pairs - 2 * (3 * pairs // 8), 3 * pairs // 8, 3 * pairs // 8]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    heads, dim, page, group = case["heads"], case["dim"], case["page"], case["group"]
    rows, lens = _rows(case), _lens(case)
    pages = [max(1, -(-n // page)) for n in lens]
    total, stride = sum(pages), max(pages)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    first = torch.tensor([sum(pages[:b]) for b in range(len(pages))], device="cuda")
    count = torch.tensor(pages, device="cuda")
    column = torch.arange(stride, device="cuda")
    table = torch.where(column < count[:, None], order[(first[:, None] + column).clamp(max=total - 1)], 0).to(torch.int32).contiguous()
    s = {"case": dict(case), "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "n_rows": sum(rows), "most": max(rows),
         "uniform": min(rows) == max(rows),
         "start": torch.tensor([sum(rows[:b]) for b in range(len(rows) + 1)], dtype=torch.int32, device="cuda")}
    n = s["n_rows"]
    if case["kind"] == "append":
        wide = (group + 2) * heads * dim                                 # one row of a product that gives q, k and v side by side
        s["qkv"] = (normal(n, wide) * 1.5).to(torch.float32 if case["type"] == "f32" else torch.bfloat16)
        s["rope"] = _table(case)
        s["pool"] = torch.zeros(total, heads, page * (dim + 8), dtype=torch.uint8, device="cuda")
        s["q_out"] = torch.empty(n, group * heads, dim, dtype=torch.bfloat16, device="cuda")
        if case["axes"] == 3:                                            # frames of 24 x 32 places behind each other
            at = torch.arange(n, device="cuda") % max(lens)
            s["positions"] = torch.stack([at // 768, at // 32 % 24 + at // 768, at % 32 + at // 768]).to(torch.int32).contiguous()
    else:
        bias = normal(2, heads, 1, dim) * 0.5
        s["pool"] = torch.cat([_block(normal(len(p), heads, page, dim) + bias[0], normal(len(p), heads, page, dim))
                               for p in torch.arange(total).split(2048)]).contiguous()
    if case["kind"] == "attend":
        s["q"] = (normal(n, heads * group, dim) * 1.5).to(torch.bfloat16)
        s["y"] = torch.empty_like(s["q"])
    else:
        s["k_out"] = torch.empty(n, heads, dim, dtype=torch.bfloat16, device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    return s


# --------------------------------------------------------------------------- one pass

_runtime = None


def _calls(s):
    """The framework's records for a state: made with its first pass and kept, as a program keeps them."""
    global _runtime
    import importlib
    t0 = importlib.import_module("rust-gpu_b200")
    if _runtime is None:
        _runtime = t0.GpuRuntime(0)
    torch.cuda.current_stream().synchronize()    # the runtime's stream does not wait for torch's, on which the inputs were made (nor torch's for results: readers wait for the device)
    rt, case = _runtime, s["case"]
    heads, dim, group = case["heads"], case["dim"], case["group"]
    batch = rt.kv4_batch(s["pool"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(), n_pages=s["pool"].shape[0], page_size=case["page"],
                         n_kv_heads=heads, head_dim=dim, n_seqs=case["seqs"], table_stride=s["table"].shape[1], n_rows=s["n_rows"],
                         max_rows=s["most"], row_start=0 if s["uniform"] else s["start"].data_ptr())
    if case["kind"] == "attend":
        return [(rt.kv4_attention, batch, rt.kv4_attention_args(s["q"].data_ptr(), s["y"].data_ptr(), n_q_heads=heads * group, scale=dim**-0.5,
                                                                window=case["window"]))]
    calls = [(rt.kv4_dequant, batch, rt.kv4_dequant_args(s["k_out"].data_ptr(), s["v_out"].data_ptr()))]
    if case["kind"] == "append":
        q, size, wide = s["qkv"].data_ptr(), s["qkv"].element_size(), s["qkv"].shape[1]
        k = q + group * heads * dim * size
        args = rt.kv4_append_args(k, k + heads * dim * size, k_stride=wide, v_stride=wide, in_f32=case["type"] == "f32", q=q, q_stride=wide,
                                  q_out=s["q_out"].data_ptr(), n_q_heads=group * heads, rope=s["rope"].data_ptr(), n_positions=s["rope"].shape[0],
                                  rot_dim=case["rot"], interleaved=case["interleaved"], axis_pairs=_axis_pairs(case),
                                  positions=s["positions"].data_ptr() if case["axes"] == 3 else 0)
        calls.insert(0, (rt.kv4_append, batch, args))
    return calls


def _row_positions(s):
    """For each row its sequence and its position there."""
    at = torch.arange(s["n_rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["start"], at, right=True) - 1
    return seq, s["lens"][seq].long() - s["start"][seq + 1].long() + at


def _rotate(x, s, seq_positions):
    """x f32 [rows, heads, dim], each pair turned by its angle."""
    case = s["case"]
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        cs = s["rope"][seq_positions]
    else:
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(_axis_pairs(case), device="cuda"), output_size=pairs)
        cs = s["rope"][s["positions"][axis].long().T, torch.arange(pairs, device="cuda")]
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if case["interleaved"] else (turned[..., :pairs], turned[..., pairs:])
    a, b = a * c - b * n, b * c + a * n
    turned = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _values(blocks, page, dim):
    """Keys and values f32 [..., page, dim] of blocks of bytes."""
    half = page * dim // 2
    out = []
    for codes, params in ((blocks[..., :half], blocks[..., 2 * half:2 * half + 4 * page]), (blocks[..., half:2 * half], blocks[..., 2 * half + 4 * page:])):
        words = codes.contiguous().view(torch.int32).unflatten(-1, (page, dim // 8))
        codes = torch.stack([(words >> shift) & 15 for shift in SHIFTS], -1).flatten(-2).float()
        step, low = params.contiguous().view(torch.bfloat16).unflatten(-1, (page, 2)).float().unbind(-1)
        out.append(codes * step[..., None] + low[..., None])
    return out


def run(s):
    case = s["case"]
    if own:
        if "calls" not in s:
            s["calls"] = _calls(s)
        for call, batch, args in s["calls"]:
            call(batch, args)
        return s["y"] if case["kind"] == "attend" else [s["q_out"], s["k_out"], s["v_out"]] if case["kind"] == "append" else [s["k_out"], s["v_out"]]
    heads, dim, group, page = case["heads"], case["dim"], case["group"], case["page"]
    seq, at = _row_positions(s)
    if case["kind"] == "append":
        q, k, v = s["qkv"].float().unflatten(-1, (-1, dim)).split([group * heads, heads, heads], 1)
        held = [step * codes + low for codes, step, low in (_quantise(_rotate(k, s, at)), _quantise(v))]
        return [_rotate(q, s, at).to(torch.bfloat16)] + [x.to(torch.bfloat16) for x in held]
    if case["kind"] == "restore":
        held, slot = s["table"][seq, at // page].long(), at % page
        return [x[held, :, slot].to(torch.bfloat16) for x in _values(s["pool"], page, dim)]
    # attention, every sequence filled up to the most rows and the longest context
    seqs, most = case["seqs"], s["most"]
    k, v = _values(s["pool"][s["table"].long()], page, dim)              # [seqs, pages, heads, page, dim]
    k, v = (x.transpose(1, 2).flatten(2, 3) for x in (k, v))
    i = torch.arange(most, device="cuda")
    n = (s["start"][1:] - s["start"][:-1]).long()
    row = torch.where(i < n[:, None], s["start"][:-1, None].long() + i, s["n_rows"])
    q = torch.cat([s["q"], s["q"].new_zeros(1, heads * group, dim)])[row].float().unflatten(2, (heads, group))
    q = q.transpose(1, 2).flatten(2, 3) * dim**-0.5                      # [seqs, heads, rows x group, dim]
    p = (s["lens"].long() - n)[:, None] + i                              # position of each row
    j = torch.arange(k.shape[2], device="cuda")
    seen = j <= p[..., None]
    if case["window"]:
        seen &= j > p[..., None] - case["window"]
    hidden = ~seen.repeat_interleave(group, 1)[:, None]
    x = (q @ k.transpose(-1, -2)).masked_fill_(hidden, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    y = (x @ v) / x.sum(-1, keepdim=True).clamp_(min=1e-30)
    y = y.unflatten(2, (most, group)).transpose(1, 2).flatten(2, 3)      # [seqs, rows, heads x group, dim]
    out = s["q"].new_zeros(s["n_rows"] + 1, heads * group, dim)
    out[row.flatten()] = y.flatten(0, 1).to(torch.bfloat16)
    return out[:-1]


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    heads, dim, group = case["heads"], case["dim"], case["group"]
    rows, lens = _rows(case), _lens(case)
    n = sum(rows)
    back = n * heads * (dim + 8 + 4 * dim)                               # read-out: codes and parameters in, keys and values out
    if case["kind"] == "restore":
        return {"bytes": back, "flops": 4 * n * heads * dim}
    if case["kind"] == "append":
        size = 4 if case["type"] == "f32" else 2
        come = n * heads * dim * (group + 2) * size + n * heads * (2 * dim * group + dim + 8) + min(n, max(lens)) * case["rot"] * 4
        return {"bytes": come + back, "flops": n * heads * dim * (3 * (group + 1) + 8)}
    seen, read = 0, 0
    for r, length in zip(rows, lens):
        w = case["window"] or length
        first = length - r                                               # position of the first row
        if length == 0:
            continue
        full = max(0, min(r, length - max(first, w - 1)))                # rows that see a whole window
        part = r - full                                                  # rows at positions first .. first + part - 1, below the window
        seen += full * w + part * (first + 1) + part * (part - 1) // 2
        read += length - max(0, first + 1 - w)
    return {"bytes": read * heads * (dim + 8) + 4 * n * heads * group * dim, "flops": 4 * dim * heads * group * seen}


# --------------------------------------------------------------------------- the same results in 64 bits

def _round_to(x, up):
    """f64 to the next bf16 not below (up) or not above, as f64."""
    near = x.to(torch.bfloat16)
    for _ in range(2):                                                   # the nearest may be on the wrong side, by one place
        wrong = near.double() < x if up else near.double() > x
        away = (near > 0) == up
        moved = torch.where(near == 0, torch.full_like(near, 2.0**-133 if up else -(2.0**-133)),
                            (near.view(torch.int16) + torch.where(away, 1, -1).to(torch.int16)).view(torch.bfloat16))
        near = torch.where(wrong, moved, near)
    return near.double()


def _held64(x):
    low = _round_to(x.min(-1, keepdim=True).values, False)
    step = _round_to((x.max(-1, keepdim=True).values - low) / 15, True)
    return low + step * ((x - low) / step).round().clamp(0, 15)


def _rows64(s, b, which):
    """The keys (0) or values (1) of sequence b in f64, [heads, tokens, dim]."""
    case = s["case"]
    page, dim = case["page"], case["dim"]
    n = int(s["lens"][b])
    blocks = s["pool"][s["table"][b, :-(-n // page)].long()]             # [pages, heads, bytes]
    e = torch.arange(dim, device="cuda")
    nibble = (e % 8) // 2 + 4 * (e % 2)
    codes = blocks[..., which * page * dim // 2:(which + 1) * page * dim // 2].unflatten(-1, (page, dim // 2))
    codes = (codes[..., e // 8 * 4 + nibble // 2].long() >> (4 * (nibble % 2))) & 15
    params = blocks[..., page * dim + which * 4 * page:page * dim + (which + 1) * 4 * page].contiguous().view(torch.bfloat16).unflatten(-1, (page, 2)).double()
    x = codes.double() * params[..., 0:1] + params[..., 1:2]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    heads, dim, group = case["heads"], case["dim"], case["group"]
    rows, lens = _rows(case), _lens(case)
    if case["kind"] == "append":
        at = torch.cat([torch.arange(length - r, length, device="cuda") for r, length in zip(rows, lens)])
        pairs = case["rot"] // 2
        where = at[:, None].expand(-1, pairs)
        if case["axes"] == 3:
            sections = _axis_pairs(case)
            where = torch.cat([s["positions"][a][:, None].expand(-1, sections[a]) for a in range(3)], 1).long()
        angle = s["rope"].double()[where, torch.arange(pairs, device="cuda")]
        turn = torch.complex(angle[..., 0], angle[..., 1])[:, None]
        x = s["qkv"].double().unflatten(-1, (-1, dim))
        qk, v = x[:, :(group + 1) * heads].clone(), x[:, (group + 1) * heads:]
        first = torch.arange(pairs, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else pairs)
        z = torch.complex(qk[..., first], qk[..., second]) * turn
        qk[..., first], qk[..., second] = z.real, z.imag
        return [qk[:, :group * heads], _held64(qk[:, group * heads:]), _held64(v)]
    if case["kind"] == "restore":
        return [torch.cat([_rows64(s, b, which).transpose(0, 1) for b in range(case["seqs"])]) for which in (0, 1)]
    out = torch.zeros(s["n_rows"], heads * group, dim, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (r, length) in enumerate(zip(rows, lens)):
        if length:
            k, v = _rows64(s, b, 0), _rows64(s, b, 1)
            p = torch.arange(length - r, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")
            seen = j <= p
            if case["window"]:
                seen = seen & (j > p - case["window"])
            for h in range(heads * group):
                x = s["q"][begin:begin + r, h].double() @ k[h // group].T / math.sqrt(dim)
                out[begin:begin + r, h] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v[h // group]
        begin += r
    return out
