"""Calls on the four-bit key/value cache whose results would be written over the cache: refused by the host."""
import pytest

from test_kv4 import BATCH, batch, refused

PAGES, SIZE = 0x100000, 8 * 2304                    # the eight pages of BATCH


@pytest.mark.parametrize("at, inside", [(PAGES, True), (PAGES + SIZE - 16, True), (PAGES - 16, True), (PAGES + SIZE, False), (PAGES - 2 * 256, False), (PAGES - 2 * 256 + 16, True)])
def test_rows_in_the_cache(t0, at, inside):
    # two rows of 256 bytes: read out, or the attention of two heads; queries likewise
    R = t0.GpuRuntime
    assert t0.kv4_page_bytes(BATCH["page_size"], BATCH["n_kv_heads"], BATCH["head_dim"]) * BATCH["n_pages"] == SIZE
    b = batch(t0, pages=PAGES)
    for entry, args, name in (("t0_kv4_dequant", R.kv4_dequant_args(at, 0), "k_out"), ("t0_kv4_dequant", R.kv4_dequant_args(0, at), "v_out"),
                              ("t0_kv4_attention", R.kv4_attention_args(0x10000, at, n_q_heads=2, scale=0.1), "y"),
                              ("t0_kv4_append", R.kv4_append_args(0x10000, 0x20000, q=0x30000, q_out=at, n_q_heads=2), "q_out")):
        code, message = refused(t0, entry, b, args)
        assert code == "INVALID" and message == (f"{name} overlaps the cache" if inside else "null runtime"), (entry, message)


def test_rows_around_the_cache(t0):
    # rows on both sides of it, by their stride
    args = t0.GpuRuntime.kv4_attention_args(0x10000, PAGES - 512, n_q_heads=2, scale=0.1, y_stride=SIZE)
    assert refused(t0, "t0_kv4_attention", batch(t0, pages=PAGES), args) == ("INVALID", "y overlaps the cache")
