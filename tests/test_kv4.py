"""The four-bit key/value cache, without a GPU: the records, the sizes and every refusal that the host makes."""
import ctypes

import numpy as np
import pytest

import kv4_reference as ref


def test_struct_sizes_match_the_header(t0, tmp_path):
    import os
    import subprocess
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "t0b200.h"\nint main(void){printf("%zu %zu %zu %zu\\n",sizeof(t0_kv4_batch),sizeof(t0_kv4_append_args),'
                   'sizeof(t0_kv4_dequant_args),sizeof(t0_kv4_attention_args));return 0;}\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.dirname(t0.HEADER_PATH), str(src), "-o", str(exe)], check=True)
    sizes = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(x) for x in (t0.Kv4Batch, t0.Kv4AppendArgs, t0.Kv4DequantArgs, t0.Kv4AttentionArgs)]


def test_page_bytes(t0):
    assert t0.kv4_page_bytes(16, 1, 64) == 16 * 72
    assert t0.kv4_page_bytes(64, 8, 128) == 64 * 136 * 8
    assert [t0.kv4_page_bytes(*a) for a in ((8, 1, 64), (128, 1, 64), (48, 1, 128), (16, 1, 32), (16, 1, 96), (16, 1, 256))] == [0] * 6


BATCH = dict(n_pages=8, page_size=16, n_kv_heads=2, head_dim=64, n_seqs=2, table_stride=4, n_rows=2, max_rows=1, row_start=0)


def batch(t0, pages=0x1000, page_table=0x2000, seq_lens=0x3000, **kw):
    return t0.GpuRuntime.kv4_batch(pages, page_table, seq_lens, **{**BATCH, **kw})


def refused(t0, entry, b, args):
    """(code, message) of a call without a runtime: a call whose arguments are in order ends at that."""
    L = t0.lib()
    rc = getattr(L, entry)(None, ctypes.byref(b), ctypes.byref(args))
    return t0.ERR_NAMES[rc], L.t0_last_error().decode()


def entries(t0):
    R = t0.GpuRuntime
    return {"t0_kv4_append": R.kv4_append_args(0x10000, 0x20000), "t0_kv4_dequant": R.kv4_dequant_args(0x10000, 0x20000),
            "t0_kv4_attention": R.kv4_attention_args(0x10000, 0x20000, n_q_heads=4, scale=0.125)}


BAD_BATCHES = [
    (dict(page_size=8), "UNSUPPORTED", "page_size=8"), (dict(page_size=128), "UNSUPPORTED", "page_size=128"), (dict(page_size=0), "UNSUPPORTED", "page_size=0"),
    (dict(head_dim=96), "UNSUPPORTED", "head_dim=96"), (dict(head_dim=256), "UNSUPPORTED", "head_dim=256"), (dict(head_dim=0), "UNSUPPORTED", "head_dim=0"),
    (dict(n_kv_heads=0), "INVALID", "n_kv_heads=0"), (dict(pages=0), "INVALID", "null"), (dict(page_table=0), "INVALID", "null"),
    (dict(seq_lens=0), "INVALID", "null"), (dict(pages=0x1008), "INVALID", "16-byte"), (dict(page_table=0x2002), "INVALID", "4-byte"),
    (dict(seq_lens=0x3001), "INVALID", "4-byte"), (dict(row_start=0x4002), "INVALID", "4-byte"), (dict(n_pages=0), "INVALID", "n_pages"),
    (dict(table_stride=0), "INVALID", "table_stride"), (dict(table_stride=1 << 28), "INVALID", "table_stride"), (dict(max_rows=0), "INVALID", "max_rows"),
    (dict(max_rows=3), "INVALID", "max_rows=3"), (dict(n_rows=3), "INVALID", "without row_start"), (dict(n_seqs=1 << 21, n_rows=1 << 21), "INVALID", "sequences"),
    (dict(n_rows=1 << 25, row_start=0x4000), "INVALID", "rows"),
]


@pytest.mark.parametrize("change, code, text", BAD_BATCHES)
def test_bad_batches_are_refused_by_every_entry(t0, change, code, text):
    for entry, args in entries(t0).items():
        got, message = refused(t0, entry, batch(t0, **change), args)
        assert got == code and text in message, (entry, got, message)


def test_calls_in_order_get_as_far_as_the_runtime(t0):
    for entry, args in entries(t0).items():
        for b in (batch(t0), batch(t0, n_seqs=0, n_rows=0), batch(t0, n_rows=0), batch(t0, n_rows=7, max_rows=3, row_start=0x4000)):
            assert refused(t0, entry, b, args) == ("INVALID", "null runtime"), entry


def test_null_records_are_refused(t0):
    L = t0.lib()
    for entry, args in entries(t0).items():
        assert getattr(L, entry)(None, None, ctypes.byref(args)) == 1 and b"null batch" in L.t0_last_error()
        assert getattr(L, entry)(None, ctypes.byref(batch(t0)), None) == 1 and b"null arguments" in L.t0_last_error()


QUERY = dict(q=0x30000, q_out=0x40000, n_q_heads=4)
ROPE = dict(rope=0x50000, n_positions=32, rot_dim=64)


@pytest.mark.parametrize("change, text", [
    (dict(k=0), "null"), (dict(v=0), "null"), (dict(k=0x10008), "k: rows"), (dict(v=0x20004, in_f32=True), "v: rows"), (dict(k_stride=64), "k: a stride"),
    (dict(v_stride=132), "v: rows"), (dict(k_stride=130, in_f32=True), "k: rows"), (dict(QUERY, q_out=0), "q_out"), (dict(QUERY, n_q_heads=0), "n_q_heads"),
    (dict(QUERY, q=0x30002), "q: rows"), (dict(QUERY, q_out=0x40008), "q_out: rows"), (dict(QUERY, q_stride=128), "q: a stride"),
    (dict(QUERY, q_out=0x30000, in_f32=True), "overlaps"), (dict(QUERY, q_out=0x30010), "overlaps"), (dict(QUERY, q_out=0x10000), "overlaps"),
    (dict(QUERY, q_out=0x30000, q_stride=512), "overlaps"), (dict(ROPE, rope=0x50008), "aligned"), (dict(ROPE, positions=0x60002), "aligned"),
    (dict(ROPE, rot_dim=0), "rot_dim"), (dict(ROPE, rot_dim=24), "rot_dim=24"), (dict(ROPE, rot_dim=80), "rot_dim=80"), (dict(ROPE, n_positions=0), "n_positions"),
    (dict(ROPE, axis_pairs=[16]), "one axis"), (dict(ROPE, axis_pairs=[16, 16]), "positions"), (dict(ROPE, axis_pairs=[16, 8], positions=0x60000), "the axes have 24"),
    (dict(ROPE, axis_pairs=[2**32 - 16, 32, 16], positions=0x60000), "the axes have"),
])
def test_append_refusals(t0, change, text):
    change = dict(change)
    args = t0.GpuRuntime.kv4_append_args(change.pop("k", 0x10000), change.pop("v", 0x20000), **change)
    code, message = refused(t0, "t0_kv4_append", batch(t0), args)
    assert code == "INVALID" and text in message, message


def test_append_calls_in_order(t0):
    R = t0.GpuRuntime
    wide = dict(q=0x30000, q_stride=512, k_stride=512, v_stride=512, n_q_heads=4)       # q, k and v as columns of one array
    for kw in (dict(), QUERY, ROPE, dict(QUERY, **ROPE), dict(QUERY, q_out=0x30000), dict(ROPE, axis_pairs=[8, 12, 12], positions=0x60000),
               dict(ROPE, rot_dim=16, axis_pairs=[8], positions=0x60000), dict(ROPE, axis_pairs=[32, 0], positions=0x60000)):
        assert refused(t0, "t0_kv4_append", batch(t0), R.kv4_append_args(0x10000, 0x20000, **kw))[1] == "null runtime", kw
    assert refused(t0, "t0_kv4_append", batch(t0), R.kv4_append_args(0x30000 + 512, 0x30000 + 768, q_out=0x30000, q_out_stride=512, **wide))[1] == "null runtime"
    with pytest.raises(ValueError):
        R.kv4_append_args(0x10000, 0x20000, axis_pairs=[8, 8, 8, 8])


@pytest.mark.parametrize("change, code, text", [
    (dict(k_out=0, v_out=0), "INVALID", "null"), (dict(k_out=0x10008), "INVALID", "k_out: rows"), (dict(v_out_stride=127), "INVALID", "v_out: a stride"),
    (dict(v_out_stride=132), "INVALID", "v_out: rows"), (dict(v_out=0x10000), "INVALID", "overlap"), (dict(v_out=0x10100, k_out_stride=144, v_out_stride=136), "INVALID", "overlap"),
])
def test_dequant_refusals(t0, change, code, text):
    args = t0.GpuRuntime.kv4_dequant_args(change.get("k_out", 0x10000), change.get("v_out", 0x20000), k_out_stride=change.get("k_out_stride", 0),
                                          v_out_stride=change.get("v_out_stride", 0))
    got, message = refused(t0, "t0_kv4_dequant", batch(t0), args)
    assert got == code and text in message, message


def test_dequant_calls_in_order(t0):
    for k, v, stride in ((0, 0x20000, 0), (0x10000, 0, 0), (0x10000, 0x10100, 256)):
        args = t0.GpuRuntime.kv4_dequant_args(k, v, k_out_stride=stride, v_out_stride=stride)
        assert refused(t0, "t0_kv4_dequant", batch(t0), args)[1] == "null runtime"


@pytest.mark.parametrize("change, text", [
    (dict(q=0), "null"), (dict(y=0), "null"), (dict(n_q_heads=0), "n_q_heads"), (dict(n_q_heads=3), "multiple"), (dict(n_q_heads=130), "64 times"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"),
    (dict(window=1 << 31), "window"), (dict(q=0x10004), "q: rows"), (dict(y_stride=260), "y: rows"), (dict(q_stride=248), "q: a stride"), (dict(y=0x10100), "overlaps"),
    (dict(y=0x10000, y_stride=264), "overlaps"),
])
def test_attention_refusals(t0, change, text):
    kw = dict(dict(n_q_heads=4, scale=0.125), **change)
    args = t0.GpuRuntime.kv4_attention_args(kw.pop("q", 0x10000), kw.pop("y", 0x20000), **kw)
    code, message = refused(t0, "t0_kv4_attention", batch(t0), args)
    assert code == "INVALID" and text in message, message


@pytest.mark.parametrize("change", [
    dict(n_seqs=1 << 18, n_rows=1 << 18, table_stride=1 << 16, page_size=16),                        # units of few rows: 2^18 x 2^14 x 2
    dict(n_seqs=1, n_rows=1 << 24, max_rows=1 << 24, table_stride=1 << 16, page_size=16, row_start=0x4000),   # of many: 2^17 tiles x 2^13 x 2
])
def test_attention_too_long_for_one_call(t0, change):
    args = t0.GpuRuntime.kv4_attention_args(0x10000, 1 << 44, n_q_heads=4, scale=0.125)
    code, message = refused(t0, "t0_kv4_attention", batch(t0, **change), args)
    assert code == "UNSUPPORTED" and "too much for one call" in message, message
    change.update(table_stride=64)
    assert refused(t0, "t0_kv4_attention", batch(t0, **change), args)[1] == "null runtime"


def test_the_reference_holds_what_it_is_given(t0):
    # the restatement the GPU tests compare with: its codes stand for the numbers to half a step, and its blocks decode to its values
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((3, 16, 64)) * 10.0 ** rng.integers(-3, 4, (3, 16, 1))).astype(np.float32)
    codes, step, low = ref.quantise(x)
    assert np.all(np.abs(ref.held(x) - x) <= step[..., None] * (0.5 + 1e-5))
    assert np.array_equal(ref.bf16_round(step), step) and np.array_equal(ref.bf16_round(low), low) and codes.max() == 15 and codes.min() == 0
    block = ref.block_bytes(x, x[::-1])
    assert block.shape == (3, 16 * 72)
    e = np.arange(64)
    nibble = e % 8 // 2 + 4 * (e % 2)
    rows = block[0, 16 * 32:2 * 16 * 32].reshape(16, 32)                   # the values' codes
    assert np.array_equal((rows[:, e // 8 * 4 + nibble // 2] >> (4 * (nibble % 2))) & 15, ref.quantise(x[2])[0])
    constant, mixed = np.full((1, 64), -7.3, np.float32), np.ones((1, 64), np.float32)
    mixed[0, 5] = np.inf
    assert np.allclose(ref.held(constant), -7.3, rtol=ref.U) and np.all(np.isnan(ref.held(mixed)))
