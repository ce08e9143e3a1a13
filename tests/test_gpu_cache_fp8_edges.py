"""The FP8 cache's writers at their edges: padding tokens whose positions lie outside the tables, tables too short for the
positions a call stands for, passes so large that a warp takes two groups of head rows. Bytes are compared as in
test_gpu_kv_cache_fp8.py."""
import pytest
import torch

import aiis_clef_b200 as clef
from gpu_util import Guarded, call, ptr, stream
from test_gpu_kv_cache_fp8 import EPS, Cache, gen, recipe, tables

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
IDS = ["bf16", "f32"]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("dim,rotary", [(64, 32), (128, 64), (256, 256)])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_padding_tokens_at_any_position(cuda_dev, norm, dim, rotary, dtype):
    """Where only k and v are written a padding token's position is not looked up at all."""
    g = gen(dim)
    tokens, kvh, table = 21, 2, 40
    k, v = (torch.randn(tokens, kvh, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.randn(dim, generator=g, device="cuda") * 0.1
    cos, sin = tables(table, rotary)
    pos = torch.randperm(table, generator=g, device="cuda")[:tokens].to(torch.int32)
    where = torch.randperm(tokens, generator=g, device="cuda").to(torch.int32)
    for token, at in ((0, -1), (4, 1 << 30), (5, -(1 << 31)), (11, table), (20, (1 << 31) - 1)):
        where[token], pos[token] = -1, at
    keep = torch.tensor([t for t in range(tokens) if t not in (0, 4, 5, 11, 20)], device="cuda")
    cache = Cache(tokens, kvh, dim)
    code = 0 if dtype == torch.bfloat16 else 1
    rest = (None, None, ptr(pos), ptr(where), None, tokens, code)
    if norm:
        call("clef_qk_norm_rope_kv_write_fp8", stream(), *cache.pointers(), ptr(k), ptr(v), ptr(w), ptr(cos), ptr(sin), tokens, kvh, dim,
             rotary, EPS, *rest)
        want, _ = cuda_dev.qk_norm_rope_dev(k[keep].float().view(-1, dim), w, cos, sin, keep.numel() * kvh, kvh, dim, rotary, EPS,
                                            pos_map=pos[keep])
    else:
        call("clef_rope_kv_write_fp8", stream(), *cache.pointers(), ptr(k), ptr(v), ptr(cos), ptr(sin), tokens, kvh, dim, rotary, *rest)
        want = cuda_dev.rope_apply_dev(k[keep].float(), cos, sin, keep.numel(), kvh, dim, rotary, pos_map=pos[keep])
    torch.cuda.synchronize()
    cache.check(where[keep].long(), want.view(-1, kvh, dim), v[keep].float())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_padding_tokens_beside_q(cuda_dev, dtype):
    """With q, a padding token's row is rotated by its position, a negative one taken as 0."""
    g = gen(17)
    tokens, qh, kvh, dim, rotary = 19, 6, 2, 128, 64
    q, k, v = (torch.randn(tokens, h, dim, generator=g, device="cuda").to(dtype) for h in (qh, kvh, kvh))
    cos, sin = tables(30, rotary)
    pos = torch.randperm(30, generator=g, device="cuda")[:tokens].to(torch.int32)
    where = torch.randperm(tokens, generator=g, device="cuda").to(torch.int32)
    where[2], where[7], where[18] = -1, -1, 1 << 30      # 7 keeps a position of the tables
    pos[2], pos[18] = -1, -(1 << 31)
    keep = torch.tensor([t for t in range(tokens) if t not in (2, 7, 18)], device="cuda")
    cache, q_out = Cache(tokens, kvh, dim), Guarded(q.numel() * q.element_size())
    call("clef_rope_qkv_write_fp8", stream(), q_out.ptr, ptr(q), qh, *cache.pointers(), ptr(k), ptr(v), kvh, ptr(cos), ptr(sin), tokens, dim,
         rotary, None, None, ptr(pos), ptr(where), None, tokens, 0 if dtype == torch.bfloat16 else 1)
    torch.cuda.synchronize()
    q_out.check_guards("q_out")
    at = pos.clamp(min=0)
    assert torch.equal(q_out.payload().view(dtype).view(q.shape), cuda_dev.rope_apply_dev(q, cos, sin, tokens, qh, dim, rotary, pos_map=at))
    turned = cuda_dev.rope_apply_dev(k.float(), cos, sin, tokens, kvh, dim, rotary, pos_map=at)
    cache.check(where[keep].long(), turned[keep], v[keep].float())


def test_tables_too_short_for_the_default_positions_are_refused(cuda_dev):
    tokens, kvh, dim, rotary = 9, 2, 64, 32
    c = torch.zeros(16, kvh, dim, dtype=torch.uint8, device="cuda")
    cache = (c, c.clone(), torch.zeros(16, kvh, device="cuda"), torch.zeros(16, kvh, device="cuda"))
    x, q = torch.randn(tokens, kvh, dim, device="cuda"), torch.randn(tokens, 4, dim, device="cuda")
    w = torch.zeros(dim, device="cuda")
    short, full = tables(tokens - 1, rotary), tables(tokens, rotary)
    base = torch.tensor([-1], dtype=torch.int32, device="cuda")
    start = torch.tensor([0] * 5 + [5] * 4, dtype=torch.int32, device="cuda")
    for t, refused in ((short, True), (full, False)):
        for go in (lambda: cuda_dev.rope_kv_write_fp8_dev(*cache, x, x, *t, tokens, kvh, dim, rotary),
                   lambda: cuda_dev.rope_qkv_write_fp8_dev(q, *cache, x, x, *t, tokens, 4, kvh, dim, rotary),
                   lambda: cuda_dev.qk_norm_rope_kv_write_fp8_dev(*cache, x, x, w, *t, tokens, kvh, dim, rotary, EPS)):
            if refused:
                with pytest.raises(clef.ClefError, match="cos must"):
                    go()
            else:
                go()
    cuda_dev.rope_kv_write_fp8_dev(*cache, x, x, *short, tokens, kvh, dim, rotary, seq_start=start)     # 0 .. 4 and 0 .. 3
    with pytest.raises(clef.ClefError, match="cos must"):
        cuda_dev.rope_kv_write_fp8_dev(*cache, x, x, short[0][:0], short[1][:0], tokens, kvh, dim, rotary, pos_base=base)
    torch.cuda.synchronize()
    code, scale = recipe(x.float())
    assert torch.equal(cache[1][:tokens], code) and torch.equal(cache[3][:tokens], scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tokens,qh,kvh,dim,rotary", [(9001, 3, 1, 64, 32), (9001, 5, 2, 48, 16), (3001, 6, 2, 128, 64), (3001, 5, 2, 96, 96),
                                                      (1501, 5, 1, 256, 64), (1203, 4, 3, 192, 0), (3203, 1, 1, 256, 256)])
def test_full_passes(cuda_dev, tokens, qh, kvh, dim, rotary, dtype):
    """Passes of so many head rows that a warp takes two groups of them (4,736 warps and more on 148 SMs): head counts that leave the
    last group of a token short, and groups that hold rows of q and of k, or of k and of v."""
    g = gen(tokens + dim)
    q, k, v = (torch.randn(tokens, h, dim, generator=g, device="cuda").to(dtype) for h in (qh, kvh, kvh))
    per_warp = 32 // (4 if dim <= 64 else 8 if dim <= 128 else 16)
    assert tokens * (qh + 2 * kvh) // per_warp >= torch.cuda.get_device_properties(0).multi_processor_count * 32
    cos, sin = tables(tokens, max(rotary, 2))
    pos = torch.randperm(tokens, generator=g, device="cuda").to(torch.int32)
    where = torch.randperm(tokens + 7, generator=g, device="cuda")[:tokens].to(torch.int32)
    skipped = torch.arange(0, tokens, 97, device="cuda")
    where[skipped] = -1
    keep = torch.ones(tokens, dtype=torch.bool, device="cuda")
    keep[skipped] = False
    cache, q_out = Cache(tokens + 7, kvh, dim), Guarded(q.numel() * q.element_size())
    call("clef_rope_qkv_write_fp8", stream(), q_out.ptr, ptr(q), qh, *cache.pointers(), ptr(k), ptr(v), kvh, ptr(cos), ptr(sin), tokens, dim,
         rotary, None, None, ptr(pos), ptr(where), None, tokens + 7, 0 if dtype == torch.bfloat16 else 1)
    torch.cuda.synchronize()
    q_out.check_guards("q_out")
    want_q = cuda_dev.rope_apply_dev(q, cos, sin, tokens, qh, dim, rotary, pos_map=pos) if rotary else q
    turned = cuda_dev.rope_apply_dev(k.float(), cos, sin, tokens, kvh, dim, rotary, pos_map=pos) if rotary else k.float()
    assert torch.equal(q_out.payload().view(dtype).view(q.shape), want_q)
    cache.check(where[keep].long(), turned[keep], v[keep].float())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tokens,kvh,dim,rotary", [(20001, 1, 64, 64), (9001, 3, 128, 32), (9001, 1, 256, 64)])
def test_full_passes_without_q(cuda_dev, tokens, kvh, dim, rotary, dtype):
    g = gen(tokens + dim)
    k, v = (torch.randn(tokens, kvh, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    per_warp = 32 // (4 if dim <= 64 else 8 if dim <= 128 else 16)
    assert tokens * 2 * kvh // per_warp >= torch.cuda.get_device_properties(0).multi_processor_count * 32
    cos, sin = tables(tokens, rotary)
    cache = Cache(tokens, kvh, dim)
    call("clef_rope_kv_write_fp8", stream(), *cache.pointers(), ptr(k), ptr(v), ptr(cos), ptr(sin), tokens, kvh, dim, rotary, None, None, None,
         None, None, tokens, 0 if dtype == torch.bfloat16 else 1)
    torch.cuda.synchronize()
    cache.check(torch.arange(tokens, device="cuda"), cuda_dev.rope_apply_dev(k.float(), cos, sin, tokens, kvh, dim, rotary), v.float())
