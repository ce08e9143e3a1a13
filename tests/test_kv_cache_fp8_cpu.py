"""The FP8 KV cache entry points and clef_add_rms_norm_fp8_bf16 refuse bad arguments before touching CUDA."""
import ctypes

import pytest

P, Q, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000), ctypes.c_void_p(0x1004)
CACHE = dict(cache_k=P, cache_v=P, k_scales=P, v_scales=P)
MAPS = dict(seq_start=None, pos_base=None, pos_map=None, cache_map=None, cache_len=None, cache_rows=64, dtype=0)
GOOD = {
    "clef_rope_kv_write_fp8": dict(stream=None, **CACHE, k=P, v=P, cos=P, sin=P, tokens=4, kv_heads=2, head_dim=128, rotary_dim=64, **MAPS),
    "clef_rope_qkv_write_fp8": dict(stream=None, q_out=P, q=Q, q_heads=16, **CACHE, k=P, v=P, kv_heads=2, cos=P, sin=P, tokens=4,
                                    head_dim=128, rotary_dim=64, **MAPS),
    "clef_qk_norm_rope_kv_write_fp8": dict(stream=None, **CACHE, k=P, v=P, weight=P, cos=P, sin=P, tokens=4, kv_heads=2, head_dim=128,
                                           rotary_dim=64, eps=1e-6, **MAPS),
    "clef_kv_read_fp8": dict(stream=None, k_out=P, v_out=P, **CACHE, row_map=None, rows=4, cache_rows=64, kv_heads=2, head_dim=128, dtype=0),
    "clef_add_rms_norm_fp8_bf16": dict(stream=None, sum_out=P, a=P, b=P, weight=P, q_out=P, q_scales=P, bf_out=None, rows=4, cols=2048,
                                       eps=1e-6, dtype=0),
}
WRITES = [n for n in GOOD if "write" in n]


def status(lib, name, **other):
    assert set(other) <= set(GOOD[name])
    return getattr(lib, name)(*{**GOOD[name], **other}.values())


@pytest.mark.parametrize("name", WRITES)
@pytest.mark.parametrize("other,want", [
    (dict(dtype=2), -1), (dict(cache_k=None), -1), (dict(k_scales=None), -1), (dict(v=None), -1), (dict(cos=None), -1),
    (dict(tokens=-1), -1), (dict(kv_heads=0), -1), (dict(head_dim=100), -1), (dict(rotary_dim=24), -1), (dict(rotary_dim=144), -1),
    (dict(head_dim=264), -3), (dict(tokens=1 << 29), -3), (dict(cache_rows=-1), -1), (dict(k=ODD), -1), (dict(cache_v=ODD), -1),
])
def test_writes(clef_lib, name, other, want):
    assert status(clef_lib, name, **other) == want
    assert name.encode() in clef_lib.clef_last_error()


def test_write_particulars(clef_lib):
    assert status(clef_lib, "clef_rope_qkv_write_fp8", q_out=Q) == -1
    assert status(clef_lib, "clef_rope_qkv_write_fp8", q_heads=0) == -1
    assert status(clef_lib, "clef_qk_norm_rope_kv_write_fp8", weight=None) == -1
    for name in WRITES:
        assert status(clef_lib, name, tokens=0) == 0


@pytest.mark.parametrize("other,want", [
    (dict(dtype=2), -1), (dict(v_out=None), -1), (dict(v_scales=None), -1), (dict(rows=-1), -1), (dict(head_dim=12), -1),
    (dict(k_out=ODD), -1), (dict(rows=1 << 30), -3), (dict(rows=0), 0),
])
def test_read(clef_lib, other, want):
    assert status(clef_lib, "clef_kv_read_fp8", **other) == want


@pytest.mark.parametrize("other,want", [
    (dict(dtype=2), -1), (dict(sum_out=None), -1), (dict(b=None), -1), (dict(weight=None), -1), (dict(rows=-1), -1), (dict(cols=12), -1),
    (dict(cols=0), -1), (dict(cols=16392), -3), (dict(a=ODD), -1), (dict(q_out=ODD), -1), (dict(bf_out=ODD), -1), (dict(rows=0), 0),
])
def test_add_norm(clef_lib, other, want):
    assert status(clef_lib, "clef_add_rms_norm_fp8_bf16", **other) == want
