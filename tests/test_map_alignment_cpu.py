"""Maps, lengths and scales of the attention and FP8 cache entry points are read as 4-byte words: others are refused before
any CUDA call."""
import ctypes

import pytest

import test_attention_cpu
import test_kv_cache_fp8_cpu as cache

ODD = ctypes.c_void_p(0x1002)


@pytest.mark.parametrize("name", ["page_table", "q_start", "kv_len"])
def test_attention_maps(clef_lib, name):
    assert test_attention_cpu.attention(clef_lib, **{name: ODD}) == -1
    assert b"4-byte aligned" in clef_lib.clef_last_error()


@pytest.mark.parametrize("name", ["k_scales", "v_scales"])
def test_attention_scales(clef_lib, name):
    fp8 = {"cache_dtype": 2, "k_scales": test_attention_cpu.P, "v_scales": test_attention_cpu.P, name: ODD}
    assert test_attention_cpu.attention(clef_lib, **fp8) == -1
    assert b"4-byte aligned" in clef_lib.clef_last_error()


@pytest.mark.parametrize("name", cache.WRITES)
@pytest.mark.parametrize("arg", ["seq_start", "pos_base", "pos_map", "cache_map", "cache_len"])
def test_write_maps(clef_lib, name, arg):
    assert cache.status(clef_lib, name, **{arg: ODD}) == -1
    assert b"4-byte aligned" in clef_lib.clef_last_error()


def test_read_map(clef_lib):
    assert cache.status(clef_lib, "clef_kv_read_fp8", row_map=ODD) == -1
    assert b"map 4-byte" in clef_lib.clef_last_error()
