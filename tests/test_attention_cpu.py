"""clef_paged_attention refuses bad arguments before touching CUDA, and its workspace size is a function of the shapes."""
import ctypes

import pytest

import aiis_clef_b200 as clef

P = ctypes.c_void_p(0x1000)   # never dereferenced: every call below is refused on its arguments
Q = ctypes.c_void_p(0x2000)
GOOD = dict(stream=None, out=P, q=Q, cache_k=P, cache_v=P, k_scales=None, v_scales=None, page_table=P, q_start=P, kv_len=P,
            n_seqs=2, total_q=5, q_heads=16, kv_heads=2, head_dim=128, page_size=16, table_width=8, cache_pages=64, scale=0.1,
            workspace=P, workspace_bytes=1 << 40, cache_dtype=0, dtype=0)


def attention(lib, **other):
    return lib.clef_paged_attention(*{**GOOD, **other}.values())


@pytest.mark.parametrize("other,status,word", [
    (dict(dtype=2), -1, b"dtype"), (dict(cache_dtype=1), -1, b"cache_dtype"), (dict(cache_dtype=2), -1, b"null"),
    (dict(out=None), -1, b"null"), (dict(page_table=None), -1, b"null"), (dict(workspace=None), -1, b"null"),
    (dict(out=Q), -1, b"alias"), (dict(q=ctypes.c_void_p(0x2004)), -1, b"aligned"),
    (dict(workspace=ctypes.c_void_p(0x1008)), -1, b"aligned"), (dict(workspace_bytes=64), -1, b"workspace"),
    (dict(n_seqs=-1), -1, b"n_seqs"), (dict(total_q=-1), -1, b"total_q"), (dict(q_heads=15), -1, b"multiple"),
    (dict(kv_heads=0), -1, b"kv_heads"), (dict(head_dim=96), -1, b"head_dim"), (dict(q_heads=130), -3, b"per kv head"),
    (dict(page_size=0), -1, b"page_size"), (dict(table_width=0), -1, b"table_width"), (dict(cache_pages=-1), -1, b"cache_pages"),
    (dict(table_width=1 << 26), -3, b"pages"), (dict(cache_pages=1 << 28), -3, b"pages"), (dict(total_q=1 << 28), -3, b"total_q"),
])
def test_refusals(clef_lib, other, status, word):
    assert attention(clef_lib, **other) == status
    assert word in clef_lib.clef_last_error()


def test_nothing_to_do_needs_no_device(clef_lib):
    assert attention(clef_lib, n_seqs=0, out=None) == 0
    assert attention(clef_lib, total_q=0, workspace=None) == 0


def test_workspace_size(clef_lib):
    size = clef.paged_attention_workspace
    assert size(0, 0, 16, 2, 128) == 0
    assert 0 < size(1, 1, 16, 2, 128) <= size(1, 1, 16, 2, 256)
    assert size(64, 64, 16, 2, 128) == size(1, 1, 16, 2, 128)
    assert size(64, 8192, 16, 2, 128) < 1 << 28
    with pytest.raises(clef.ClefError, match="head_dim"):
        size(1, 1, 16, 2, 80)
    assert clef_lib.clef_paged_attention_workspace(1, 1, 16, 2, 128, None) == -1
