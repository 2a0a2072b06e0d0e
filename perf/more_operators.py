"""Performance cases of the products in eight bits and of the calls around them: rows made eight bits with a scale for each, the
root-mean-square norm that adds the residual and leaves rows in eight bits, the product of eight-bit rows with eight-bit weights (a scale for
each token and channel), and the gated pair of products of a feed-forward block.

``listed()`` names the cases, ``draw(rng)`` makes further ones of the same ranges, ``prepare(case, seed)`` is what a program holds
before the call, ``run(state)`` is one pass, ``work(case)`` the bytes and operations that the pass cannot do without, and
``exact(case, seed)`` the same results in 64 bits.  With ``own`` false, ``run`` computes the operators in elementary torch
operations; with ``own`` true it calls the framework.

The kinds of pass (``case["kind"]``):

* ``quant``  rows (bf16 or f32) are held in eight bits, then read back as bf16, so that what is held comes out as the values it stands for.
* ``norm``   a branch's rows are added to the residual, which is kept, the sum is normalised, weighted and held in eight bits; read back likewise.
* ``gemm``   y = (codes of a) (codes of w)^T, times the token's and the channel's scale, plus a bias.
* ``gated``  y = act(a gate^T) * (a up^T), both products as above.

A row x is held as scale = max|x| / 127 and codes rint(x * (127 / max|x|)).
"""
from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # a decode batch's gated rows on their way to the down projection
        {"name": "quant_16x11008", "kind": "quant", "rows": 16, "dim": 11008, "type": "bf16"},
        # a prompt's gated rows, or a weight matrix when it is loaded
        {"name": "quant_8192x14336", "kind": "quant", "rows": 8192, "dim": 14336, "type": "bf16"},
        # the norm between two blocks of one sequence's next token, the branch in f32 as a product leaves it: latency counts
        {"name": "norm_one_token", "kind": "norm", "rows": 1, "dim": 4096, "type": "f32", "residual": "bf16"},
        # the same for a prompt
        {"name": "norm_prompt_8192", "kind": "norm", "rows": 8192, "dim": 4096, "type": "bf16", "residual": "bf16"},
        # one token through a projection: the weights are read once
        {"name": "gemm_one_token", "kind": "gemm", "m": 1, "n": 11008, "k": 4096, "type": "f32", "bias": False},
        # a small decode batch through a down projection
        {"name": "gemm_16_down", "kind": "gemm", "m": 16, "n": 4096, "k": 11008, "type": "bf16", "bias": False},
        # a batch of 128 tokens
        {"name": "gemm_128_square", "kind": "gemm", "m": 128, "n": 4096, "k": 4096, "type": "f32", "bias": True},
        # nothing a multiple of anything: rows of another stride than their length, a ragged edge on every side
        {"name": "gemm_ragged", "kind": "gemm", "m": 777, "n": 1111, "k": 1357, "type": "f32", "bias": True},
        # a prompt through a projection
        {"name": "gemm_prompt_8192", "kind": "gemm", "m": 8192, "n": 14336, "k": 4096, "type": "bf16", "bias": False},
        # one token through the gated pair
        {"name": "gated_one_token", "kind": "gated", "m": 1, "n": 11008, "k": 4096, "type": "bf16", "act": "silu"},
        # a batch of an odd number of tokens
        {"name": "gated_100_tokens", "kind": "gated", "m": 100, "n": 14336, "k": 4096, "type": "bf16", "act": "gelu"},
        # a prompt through the gated pair
        {"name": "gated_prompt_4096", "kind": "gated", "m": 4096, "n": 11008, "k": 4096, "type": "bf16", "act": "silu"},
    ]


# --------------------------------------------------------------------------- further cases of the same ranges

def _log(rng, lo, hi):
    return int(min(max(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))), lo), hi))


def _size(rng, lo, hi):
    """A size between lo and hi: any, or one in whole units of 128, as weights mostly are."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.4 else min(max(128, (n + 64) // 128 * 128), hi // 128 * 128)


def draw(rng):
    kind = rng.choice(["quant", "norm", "gemm", "gemm", "gemm", "gated", "gated"])
    if kind == "quant":
        dim = _size(rng, 64, 28672)
        return {"kind": kind, "rows": _log(rng, 1, min(32768, 8192 * 14336 // dim)), "dim": dim, "type": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "norm":
        dim = _size(rng, 64, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(32768, 8192 * 4096 // dim)), "dim": dim, "type": rng.choice(["bf16", "f32"]),
                "residual": rng.choice(["bf16", "bf16", "f32", "none"])}
    m = _log(rng, 1, 16) if rng.random() < 0.4 else _log(rng, 17, 8192)
    most = 8192 * 14336 * 4096 if kind == "gemm" else 4096 * 11008 * 4096
    n, k = _size(rng, 256, 16384), _size(rng, 256, 14336)
    while m * n * k > most:
        m = (m + 1) // 2
    case = {"kind": kind, "m": m, "n": n, "k": k, "type": rng.choice(["f32", "bf16"])}
    return case | ({"bias": rng.random() < 0.3} if kind == "gemm" else {"act": rng.choice(["silu", "silu", "gelu", "relu"])})


# --------------------------------------------------------------------------- inputs

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def _hold(x):
    """Codes (i8) and scales of rows of f32: the operator's definition, each operation rounded to f32."""
    most = x.abs().amax(-1, keepdim=True)
    full = torch.full_like(most, 127.0)
    held = most >= 2.0**-119
    codes = torch.where(held, torch.round(x * torch.where(held, full / most, 0.0)), 0.0)
    return codes.to(torch.int8), torch.where(held, most / full, 0.0).squeeze(-1)     # (a plain 127.0 would be multiplied by its rounded inverse)


def _stride(n):
    """Bytes from one row of codes to the next: rows start on 16-byte boundaries."""
    return (n + 15) // 16 * 16


def _held_rows(x):
    """Rows as they are held: i8 [rows][stride] and f32 [rows]."""
    codes, scales = _hold(x)
    out = torch.zeros(x.shape[0], _stride(x.shape[1]), dtype=torch.int8, device="cuda")
    out[:, :x.shape[1]] = codes
    return out, scales.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    s = {"case": dict(case)}
    if case["kind"] in ("quant", "norm"):
        rows, dim, wide = case["rows"], case["dim"], (case["dim"] + 7) // 8 * 8
        # tokens of different size, a few channels far above the others
        x = normal(rows, wide) * normal(rows, 1).mul_(0.5).exp_()
        x[:, ::97] *= 8
        s["x"] = x.to(TYPES[case["type"]])
        if case["kind"] == "norm":
            s["weight"] = (1 + 0.2 * normal(dim)).to(torch.bfloat16)
            if case["residual"] != "none":
                s["residual"] = (normal(rows, wide) * 3).to(TYPES[case["residual"]])
                s["sum"] = torch.zeros_like(s["residual"])
        s["q"] = torch.zeros(rows, _stride(dim), dtype=torch.int8, device="cuda")
        s["scales"] = torch.zeros(rows, device="cuda")
        s["y"] = torch.zeros(rows, wide, dtype=torch.bfloat16, device="cuda")
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["a"], s["a_scales"] = _held_rows(normal(m, k) * normal(m, 1).mul_(0.5).exp_())
    for name in ("w",) if case["kind"] == "gemm" else ("gate", "up"):
        s[name], s[name + "_scales"] = _held_rows(normal(n, k) * k**-0.5 * normal(n, 1).mul_(0.2).exp_())
    if case.get("bias"):
        s["bias"] = normal(n)
    s["y"] = torch.zeros(m, n, dtype=TYPES[case["type"]], device="cuda")
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
    at = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"] in ("quant", "norm"):
        size = dict(n_rows=case["rows"], dim=case["dim"])
        wide = s["x"].shape[1]
        back = rt.q8_dequant_args(at["q"], at["scales"], at["y"], **size, y_stride=wide)
        if case["kind"] == "quant":
            first = rt.q8_quant, rt.q8_quant_args(at["x"], at["q"], at["scales"], **size, x_f32=case["type"] == "f32", x_stride=wide)
        else:
            more = {} if case["residual"] == "none" else dict(residual=at["residual"], residual_out=at["sum"], residual_f32=case["residual"] == "f32",
                                                              residual_stride=wide, residual_out_stride=wide)
            first = rt.q8_rmsnorm, rt.q8_rmsnorm_args(at["x"], at["weight"], **size, eps=EPS, x_f32=case["type"] == "f32", x_stride=wide, q=at["q"],
                                                      scales=at["scales"], **more)
        return [first, (rt.q8_dequant, back)]
    size = dict(m=case["m"], n=case["n"], k=case["k"], out_bf16=case["type"] == "bf16")
    if case["kind"] == "gemm":
        return [(rt.q8_gemm, rt.q8_gemm_args(at["a"], at["a_scales"], at["w"], at["w_scales"], at["y"], **size, bias=at.get("bias", 0)))]
    return [(rt.q8_gated, rt.q8_gated_args(at["a"], at["a_scales"], at["gate"], at["gate_scales"], at["up"], at["up_scales"], at["y"], **size,
                                           activation=case["act"]))]


def _outputs(s, y, total):
    dim = s["case"].get("dim")
    out = {"y": y if dim is None else y[:, :dim]}
    if total is not None:
        out["sum"] = total[:, :dim]
    return out


def _act(x, name):
    return x * torch.sigmoid(x) if name == "silu" else x * torch.sigmoid(1.702 * x) if name == "gelu" else x.clamp(min=0)


def run(s):
    case = s["case"]
    if own:
        if "calls" not in s:
            s["calls"] = _calls(s)
        for call, args in s["calls"]:
            call(args)
        return _outputs(s, s["y"], s.get("sum"))
    if case["kind"] in ("quant", "norm"):
        dim = case["dim"]
        x, total = s["x"][:, :dim].float(), None
        if case["kind"] == "norm":
            if "residual" in s:
                total = (x + s["residual"][:, :dim].float()).to(s["residual"].dtype)
                x = total.float()
            x = x * (1 / (x.double().square().sum(-1, keepdim=True) / dim + EPS).sqrt()).float() * s["weight"].float()
        codes, scales = _hold(x)
        return _outputs(s, (codes.float() * scales[:, None]).to(torch.bfloat16), total)
    k, y = case["k"], []
    a = s["a"][:, :k].float()
    for name in ("w",) if case["kind"] == "gemm" else ("gate", "up"):
        y.append((a @ s[name][:, :k].float().T).mul_(s["a_scales"][:, None]).mul_(s[name + "_scales"]))
    if case["kind"] == "gated":
        y = _act(y[0], case["act"]) * y[1]
    else:
        y = y[0] + s["bias"] if case["bias"] else y[0]
    return _outputs(s, y.to(TYPES[case["type"]]), None)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = {"f32": 4, "bf16": 2, "none": 0}
    if case["kind"] in ("quant", "norm"):
        n = case["rows"] * case["dim"]
        back, flops = n + 4 * case["rows"] + 2 * n, 4 * n                # codes, scales and the values they stand for
        if case["kind"] == "norm":
            back, flops = back + 2 * n * size[case["residual"]] + 2 * case["dim"], flops + 5 * n
        return {"bytes": n * size[case["type"]] + back, "flops": flops}
    m, n, k = case["m"], case["n"], case["k"]
    pairs = 2 if case["kind"] == "gated" else 1
    more = 4 * n if case.get("bias") else 0
    return {"bytes": m * k + 4 * m + pairs * (n * k + 4 * n) + m * n * size[case["type"]] + more, "flops": 2 * pairs * m * n * k}


# --------------------------------------------------------------------------- the same results in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("quant", "norm"):
        x = s["x"][:, :case["dim"]].double()
        out = {}
        if case["kind"] == "norm":
            if "residual" in s:
                x = x + s["residual"][:, :case["dim"]].double()
                out["sum"] = x
                x = x.to(s["residual"].dtype).double()               # what is kept is what is normalised
            x = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * s["weight"].double()
        step = x.abs().max(1, keepdim=True).values / 127
        out["y"] = torch.where(step > 0, torch.round(x / step) * step, 0.0)
        return out
    k = case["k"]

    def product(name):
        w = s[name][:, :k].double() * s[name + "_scales"].double()[:, None]
        return (s["a"][:, :k].double() * s["a_scales"].double()[:, None]) @ w.T

    if case["kind"] == "gemm":
        y = product("w")
        return {"y": y + s["bias"].double() if case["bias"] else y}
    g = product("gate")
    if case["act"] == "relu":
        g = torch.maximum(g, torch.zeros_like(g))
    else:
        g = g / (1 + torch.exp(-g * (1.702 if case["act"] == "gelu" else 1.0)))
    return {"y": g * product("up")}
