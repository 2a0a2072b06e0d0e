"""Products in eight bits and the calls around them, without a GPU: the records, the arithmetic's restatement, and every refusal that the host makes."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import q8_reference as ref


def test_struct_sizes_match_the_header(t0, tmp_path):
    names = {"quant": t0.Q8QuantArgs, "dequant": t0.Q8DequantArgs, "rmsnorm": t0.Q8RmsnormArgs, "gemm": t0.Q8GemmArgs, "gated": t0.Q8GatedArgs}
    lines, want = [], []
    for name, record in names.items():
        lines.append(f'printf("%zu\\n", sizeof(t0_q8_{name}_args));')
        want.append(ctypes.sizeof(record))
        for field, *_ in record._fields_:
            lines.append(f'printf("%zu\\n", offsetof(t0_q8_{name}_args, {field}));')
            want.append(getattr(record, field).offset)
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "t0b200.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.dirname(t0.HEADER_PATH), str(src), "-o", str(exe)], check=True)
    assert [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()] == want


def test_what_is_held_is_near_what_was_given():
    # half a step, and the roundings of scale, factor and product (three of 2^-24, of up to 127 steps)
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 1000)) * np.exp(rng.uniform(-40, 40, (64, 1)))).astype(np.float32)
    codes, scales = ref.hold(x)
    assert np.abs(codes).max() == 127
    off = np.abs(codes.astype(np.float64) * scales[:, None] - x)
    assert (off <= (0.5 + 127 * 4 * 2.0**-24) * scales[:, None].astype(np.float64)).all()


def refused(t0, entry, args):
    """(code, message) of a call without a runtime: a call whose arguments are in order ends at that."""
    L = t0.lib()
    rc = getattr(L, entry)(None, ctypes.byref(args))
    return t0.ERR_NAMES[rc], L.t0_last_error().decode()


A, B, C, D, E, G, H = (0x100000 * (i + 1) for i in range(7))
QUANT = dict(x=A, q=B, scales=C, n_rows=3, dim=64)
DEQUANT = dict(q=A, scales=B, y=C, n_rows=3, dim=64)
NORM = dict(x=A, weight=B, q=C, scales=D, n_rows=3, dim=64, eps=1e-5)
SUM = dict(NORM, residual=E, residual_out=G, y=H)
GEMM = dict(a=A, a_scales=B, w=C, w_scales=D, y=E, m=3, n=5, k=64)
GATED = dict(a=A, a_scales=B, gate=C, gate_scales=D, up=E, up_scales=G, y=H, m=3, n=5, k=64)


def call(t0, name, kw):
    return refused(t0, "t0_q8_" + name, getattr(t0.GpuRuntime, f"q8_{name}_args")(**kw))


FINE = [
    ("quant", QUANT), ("quant", dict(QUANT, n_rows=0, x=0)), ("quant", dict(QUANT, dim=63, x_stride=64)), ("quant", dict(QUANT, dim=32768, x_f32=True, n_rows=1)),
    ("quant", dict(QUANT, dim=1, x_stride=8, q_stride=16)),
    ("dequant", DEQUANT), ("dequant", dict(DEQUANT, dim=131071, y_stride=131072, n_rows=1)), ("dequant", dict(DEQUANT, dim=13, out_f32=True, y_stride=16)),
    ("rmsnorm", NORM), ("rmsnorm", SUM), ("rmsnorm", dict(NORM, q=0, scales=0, y=H)), ("rmsnorm", dict(SUM, residual_out=E)), ("rmsnorm", dict(SUM, residual_out=A)),
    ("rmsnorm", dict(SUM, residual_out=0)), ("rmsnorm", dict(NORM, eps=0.0)), ("rmsnorm", dict(NORM, n_rows=0)),
    ("gemm", GEMM), ("gemm", dict(GEMM, m=0)), ("gemm", dict(GEMM, n=0)), ("gemm", dict(GEMM, k=131071, m=1, n=1)), ("gemm", dict(GEMM, y=E + 4, y_stride=7, bias=G)),
    ("gemm", dict(GEMM, y=E + 2, out_bf16=True)), ("gemm", dict(GEMM, k=63)), ("gemm", dict(GEMM, a_stride=80, w_stride=96)),
    ("gated", GATED), ("gated", dict(GATED, activation="relu")), ("gated", dict(GATED, activation="gelu", out_bf16=False)), ("gated", dict(GATED, up=C + 5 * 64)),
    ("gated", dict(GATED, m=0)),
]


@pytest.mark.parametrize("name, kw", FINE)
def test_calls_in_order_get_as_far_as_the_runtime(t0, name, kw):
    assert call(t0, name, kw) == ("INVALID", "null runtime")


BAD = [
    ("quant", QUANT, dict(x=0), "INVALID", "null"), ("quant", QUANT, dict(q=0), "INVALID", "null"), ("quant", QUANT, dict(scales=0), "INVALID", "null"),
    ("quant", QUANT, dict(dim=0), "INVALID", "dim=0"), ("quant", QUANT, dict(dim=32769, x_stride=32776), "UNSUPPORTED", "dim=32769"),
    ("quant", QUANT, dict(n_rows=0x80000000), "INVALID", "n_rows"), ("quant", QUANT, dict(x=A + 8), "INVALID", "16-byte"), ("quant", QUANT, dict(dim=63), "INVALID", "16-byte"),
    ("quant", QUANT, dict(x_stride=63), "INVALID", "stride"), ("quant", QUANT, dict(x_stride=68), "INVALID", "16-byte"), ("quant", QUANT, dict(q=B + 8), "INVALID", "16-byte"),
    ("quant", QUANT, dict(scales=C + 2), "INVALID", "4-byte"), ("quant", QUANT, dict(q_stride=72), "INVALID", "stride of 72"), ("quant", QUANT, dict(q_stride=48), "INVALID", "stride of 48"),
    ("quant", QUANT, dict(q=A + 2 * 128), "INVALID", "overlap"), ("quant", QUANT, dict(scales=A + 4), "INVALID", "overlap"), ("quant", QUANT, dict(scales=B + 3 * 64 - 4), "INVALID", "overlap"),
    ("dequant", DEQUANT, dict(q=0), "INVALID", "null"), ("dequant", DEQUANT, dict(scales=0), "INVALID", "null"), ("dequant", DEQUANT, dict(y=0), "INVALID", "null"),
    ("dequant", DEQUANT, dict(dim=131072), "UNSUPPORTED", "dim=131072"), ("dequant", DEQUANT, dict(y=C + 4), "INVALID", "16-byte"), ("dequant", DEQUANT, dict(y_stride=60), "INVALID", "stride"),
    ("dequant", DEQUANT, dict(y=A), "INVALID", "overlaps"), ("dequant", DEQUANT, dict(y=B - 128), "INVALID", "overlaps"), ("dequant", DEQUANT, dict(dim=0), "INVALID", "dim=0"),
    ("rmsnorm", NORM, dict(x=0), "INVALID", "null"), ("rmsnorm", NORM, dict(weight=0), "INVALID", "null"), ("rmsnorm", NORM, dict(q=0), "INVALID", "null"),
    ("rmsnorm", NORM, dict(scales=0), "INVALID", "null"), ("rmsnorm", NORM, dict(q=0, scales=0), "INVALID", "neither"), ("rmsnorm", NORM, dict(residual_out=G), "INVALID", "without a residual"),
    ("rmsnorm", NORM, dict(eps=-1e-6), "INVALID", "eps"), ("rmsnorm", NORM, dict(eps=float("nan")), "INVALID", "eps"), ("rmsnorm", NORM, dict(eps=float("inf")), "INVALID", "eps"),
    ("rmsnorm", NORM, dict(weight=B + 8), "INVALID", "weight"), ("rmsnorm", NORM, dict(x=A + 2), "INVALID", "x: rows"), ("rmsnorm", SUM, dict(residual=E + 2), "INVALID", "residual: rows"),
    ("rmsnorm", SUM, dict(residual_out=G + 2), "INVALID", "residual_out: rows"), ("rmsnorm", SUM, dict(y=H + 2), "INVALID", "y: rows"), ("rmsnorm", SUM, dict(residual_stride=66), "INVALID", "residual"),
    ("rmsnorm", NORM, dict(dim=32769, x_stride=32776), "UNSUPPORTED", "dim"), ("rmsnorm", NORM, dict(dim=0), "INVALID", "dim"),
    ("rmsnorm", SUM, dict(residual_out=E + 128), "INVALID", "overlaps what is read"), ("rmsnorm", SUM, dict(residual_out=A, x_f32=True), "INVALID", "overlaps what is read"),
    ("rmsnorm", SUM, dict(residual_out=E, residual_out_stride=72), "INVALID", "overlaps what is read"), ("rmsnorm", SUM, dict(residual_out=B), "INVALID", "overlaps what is read"),
    ("rmsnorm", SUM, dict(y=A), "INVALID", "overlaps what is read"), ("rmsnorm", SUM, dict(q=B), "INVALID", "overlaps what is read"), ("rmsnorm", SUM, dict(scales=E), "INVALID", "overlaps what is read"),
    ("rmsnorm", SUM, dict(y=G), "INVALID", "written overlap"), ("rmsnorm", SUM, dict(y=C), "INVALID", "written overlap"), ("rmsnorm", SUM, dict(scales=C + 64), "INVALID", "written overlap"),
    ("gemm", GEMM, dict(a=0), "INVALID", "null"), ("gemm", GEMM, dict(a_scales=0), "INVALID", "null"), ("gemm", GEMM, dict(w=0), "INVALID", "null"), ("gemm", GEMM, dict(w_scales=0), "INVALID", "null"),
    ("gemm", GEMM, dict(y=0), "INVALID", "null"), ("gemm", GEMM, dict(k=0), "INVALID", "k must"), ("gemm", GEMM, dict(k=131072), "UNSUPPORTED", "k=131072"),
    ("gemm", GEMM, dict(m=0x40000001), "INVALID", "m="), ("gemm", GEMM, dict(n=0x40000001), "INVALID", "n="), ("gemm", GEMM, dict(a=A + 8), "INVALID", "16-byte"),
    ("gemm", GEMM, dict(w=C + 1), "INVALID", "16-byte"), ("gemm", GEMM, dict(a_scales=B + 1), "INVALID", "4-byte"), ("gemm", GEMM, dict(w_scales=D + 2), "INVALID", "4-byte"),
    ("gemm", GEMM, dict(a_stride=72), "INVALID", "a: a stride"), ("gemm", GEMM, dict(w_stride=48), "INVALID", "w: a stride"), ("gemm", GEMM, dict(y=E + 2), "INVALID", "aligned"),
    ("gemm", GEMM, dict(y=E + 1, out_bf16=True), "INVALID", "aligned"), ("gemm", GEMM, dict(y_stride=4), "INVALID", "stride of 4"), ("gemm", GEMM, dict(bias=G + 2), "INVALID", "bias"),
    ("gemm", GEMM, dict(y=A + 64), "INVALID", "y overlaps a"), ("gemm", GEMM, dict(y=B), "INVALID", "y overlaps a"), ("gemm", GEMM, dict(y=C + 4 * 64), "INVALID", "y overlaps w"),
    ("gemm", GEMM, dict(y=D + 4), "INVALID", "y overlaps w"), ("gemm", GEMM, dict(bias=E + 20), "INVALID", "bias"),
    ("gated", GATED, dict(gate=0), "INVALID", "null"), ("gated", GATED, dict(up=0), "INVALID", "null"), ("gated", GATED, dict(up_scales=0), "INVALID", "null"),
    ("gated", GATED, dict(up=E + 8), "INVALID", "up: codes"), ("gated", GATED, dict(activation="abs"), "INVALID", "activation"), ("gated", GATED, dict(y=E), "INVALID", "overlaps up"),
    ("gated", GATED, dict(y=C + 64), "INVALID", "overlaps gate"), ("gated", GATED, dict(y=G), "INVALID", "overlaps up"), ("gated", GATED, dict(k=0), "INVALID", "k must"),
    ("gated", GATED, dict(k=140000), "UNSUPPORTED", "k=140000"),
]


@pytest.mark.parametrize("name, kw, change, code, text", BAD)
def test_bad_calls_are_refused(t0, name, kw, change, code, text):
    got, message = call(t0, name, dict(kw, **change))
    assert got == code and text in message, message


def test_null_records_are_refused(t0):
    L = t0.lib()
    for name in ("quant", "dequant", "rmsnorm", "gemm", "gated"):
        assert getattr(L, "t0_q8_" + name)(None, None) == 1 and b"null arguments" in L.t0_last_error()
