"""The FP8 KV cache: the three writing entry points against clef_rope / clef_qk_norm_rope in f32 followed by the recipe (byte
for byte) and against the definition in 64 bits, and reading back (exact up to the one rounding of the output type)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import aiis_clef_b200 as clef
from gpu_util import Guarded, call, ptr, stream

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
EPS = 1e-6


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tables(rows, rotary):
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] / 1e7 ** (
        torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / max(rotary, 1))
    angle = torch.cat([angle, angle], 1)
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def recipe(x):
    """(codes, scales) of f32 head rows, in f32 steps."""
    amax = x.abs().amax(-1)
    # (a quotient of two tensors: torch turns one by a number into a product with its reciprocal, which rounds twice)
    scale = torch.where(amax >= 2.0 ** -100, amax / torch.full_like(amax, 448.0), torch.zeros_like(amax))
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    return (x * inv[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


class Cache:
    def __init__(self, rows, heads, dim):
        self.rows, self.heads, self.dim = rows, heads, dim
        self.k, self.v = Guarded(rows * heads * dim), Guarded(rows * heads * dim)
        self.ks, self.vs = Guarded(rows * heads * 4), Guarded(rows * heads * 4)

    def pointers(self):
        return self.k.ptr, self.v.ptr, self.ks.ptr, self.vs.ptr

    def tensors(self):
        shape = (self.rows, self.heads, self.dim)
        return (self.k.payload().view(shape), self.v.payload().view(shape), self.ks.payload().view(torch.float32).view(shape[:2]),
                self.vs.payload().view(torch.float32).view(shape[:2]))

    def check(self, where, want_k, want_v):
        """Rows `where` hold the recipe of the two f32 tensors, every other byte is untouched."""
        for g, name in ((self.k, "k"), (self.v, "v"), (self.ks, "k scales"), (self.vs, "v scales")):
            g.check_guards(name)
        k, v, ks, vs = self.tensors()
        rest = torch.ones(self.rows, dtype=torch.bool, device="cuda")
        rest[where] = False
        for got, scales, want in ((k, ks, want_k), (v, vs, want_v)):
            code, scale = recipe(want)
            assert torch.equal(scales[where].view(torch.int32), scale.view(torch.int32))
            assert torch.equal(got[where], code)
            assert (got[rest] == 0xA5).all() and (scales[rest].contiguous().view(torch.uint8) == 0xA5).all()


SHAPES = [(1, 16, 2, 128, 64), (61, 16, 2, 256, 64), (130, 4, 4, 64, 64), (33, 6, 2, 128, 128), (7, 3, 1, 96, 32), (50, 2, 2, 192, 0),
          (515, 16, 2, 128, 64), (9, 5, 5, 8, 0), (12, 1, 1, 80, 16), (20, 2, 1, 256, 256)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("tokens,qh,kvh,dim,rotary", SHAPES)
def test_rope_qkv_write(cuda_dev, tokens, qh, kvh, dim, rotary, dtype):
    g = gen(tokens + dim)
    q, k, v = (torch.randn(tokens, h, dim, generator=g, device="cuda").to(dtype) for h in (qh, kvh, kvh))
    cos, sin = tables(tokens + 40, max(rotary, 2))
    pos = torch.randperm(tokens + 40, generator=g, device="cuda")[:tokens].to(torch.int32)
    rows = tokens + 11
    where = torch.randperm(rows, generator=g, device="cuda")[:tokens].to(torch.int32)
    cache = Cache(rows, kvh, dim)
    q_out = Guarded(q.numel() * q.element_size())
    code = 0 if dtype == torch.bfloat16 else 1
    call("clef_rope_qkv_write_fp8", stream(), q_out.ptr, ptr(q), qh, *cache.pointers(), ptr(k), ptr(v), kvh, ptr(cos), ptr(sin), tokens,
         dim, rotary, None, None, ptr(pos), ptr(where), None, rows, code)
    torch.cuda.synchronize()
    q_out.check_guards("q_out")
    turned = cuda_dev.rope_apply_dev(k.float(), cos, sin, tokens, kvh, dim, rotary, pos_map=pos) if rotary else k.float()
    want_q = cuda_dev.rope_apply_dev(q, cos, sin, tokens, qh, dim, rotary, pos_map=pos) if rotary else q
    assert torch.equal(q_out.payload().view(dtype).view(q.shape), want_q)
    cache.check(where.long(), turned, v.float())
    # the k / v form without q writes the same bytes
    again = Cache(rows, kvh, dim)
    call("clef_rope_kv_write_fp8", stream(), *again.pointers(), ptr(k), ptr(v), ptr(cos), ptr(sin), tokens, kvh, dim, rotary, None, None,
         ptr(pos), ptr(where), None, rows, code)
    torch.cuda.synchronize()
    for a, b in zip((cache.k, cache.v, cache.ks, cache.vs), (again.k, again.v, again.ks, again.vs)):
        b.check_guards("cache")
        assert torch.equal(a.payload(), b.payload())


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("tokens,kvh,dim,rotary", [(61, 2, 128, 64), (5, 4, 256, 64), (33, 1, 64, 32), (10, 3, 96, 32), (300, 2, 256, 256)])
def test_qk_norm_rope_kv_write(cuda_dev, tokens, kvh, dim, rotary, dtype):
    g = gen(tokens * dim)
    k, v = (torch.randn(tokens, kvh, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.randn(dim, generator=g, device="cuda") * 0.1
    cos, sin = tables(tokens + 9, rotary)
    pos = torch.randperm(tokens + 9, generator=g, device="cuda")[:tokens].to(torch.int32)
    cache = Cache(tokens + 5, kvh, dim)
    length = torch.tensor([3], dtype=torch.int32, device="cuda")
    call("clef_qk_norm_rope_kv_write_fp8", stream(), *cache.pointers(), ptr(k), ptr(v), ptr(w), ptr(cos), ptr(sin), tokens, kvh, dim, rotary,
         EPS, None, None, ptr(pos), None, ptr(length), tokens + 5, 0 if dtype == torch.bfloat16 else 1)
    torch.cuda.synchronize()
    want, _ = cuda_dev.qk_norm_rope_dev(k.float().view(-1, dim), w, cos, sin, tokens * kvh, kvh, dim, rotary, EPS, pos_map=pos)
    cache.check(torch.arange(3, 3 + tokens, device="cuda"), want.view(tokens, kvh, dim), v.float())


def test_stored_values_against_64_bits(cuda_dev):
    """code * scale is within half an E4M3 step of the exact rotated value: 2^-4 of it, or half the subnormal step 2^-10 of the
    scale, and 2^-21 of the scale's 448 for the f32 rotation and quotient."""
    g = gen(3)
    tokens, kvh, dim, rotary = 777, 2, 128, 64
    k, v = (torch.randn(tokens, kvh, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    cos, sin = tables(tokens, rotary)
    c = torch.zeros(tokens, kvh, dim, dtype=torch.uint8, device="cuda")
    cache = (c, c.clone(), torch.zeros(tokens, kvh, device="cuda"), torch.zeros(tokens, kvh, device="cuda"))
    cuda_dev.rope_kv_write_fp8_dev(*cache, k, v, cos, sin, tokens, kvh, dim, rotary)
    z = torch.complex(k[..., :32].double(), k[..., 32:64].double()) * torch.complex(cos[:, :32].double(), sin[:, :32].double())[:, None]
    exact = torch.cat([z.real, z.imag, k[..., 64:].double()], -1)
    for code, scale, want in ((cache[0], cache[2], exact), (cache[1], cache[3], v.double())):
        s = scale.double()[..., None]
        got = code.view(torch.float8_e4m3fn).double() * s
        assert ((got - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) + s * 448 * 2.0 ** -21).all()
        assert torch.allclose(s[..., 0], want.abs().amax(-1) / 448, rtol=2.0 ** -21, atol=0)


def test_padding_tokens_and_default_rows(cuda_dev):
    """Rows outside the cache are skipped; seq_start and pos_base positions; no map writes at token + cache_len."""
    g = gen(4)
    tokens, kvh, dim, rotary = 20, 2, 128, 64
    k, v = (torch.randn(tokens, kvh, dim, generator=g, device="cuda") for _ in range(2))
    cos, sin = tables(64, rotary)
    seq_start = torch.tensor([0] * 8 + [8] * 12, dtype=torch.int32, device="cuda")
    base = torch.tensor([5], dtype=torch.int32, device="cuda")
    where = torch.arange(tokens, dtype=torch.int32, device="cuda")
    where[3], where[9], where[10] = -1, 1 << 30, -(1 << 31)
    want = cuda_dev.rope_apply_dev(k, cos, sin, tokens, kvh, dim, rotary, seq_start=seq_start, pos_base=base)
    cache = Cache(tokens, kvh, dim)
    call("clef_rope_kv_write_fp8", stream(), *cache.pointers(), ptr(k), ptr(v), ptr(cos), ptr(sin), tokens, kvh, dim, rotary, ptr(seq_start),
         ptr(base), None, ptr(where), None, tokens, 1)
    torch.cuda.synchronize()
    keep = torch.tensor([t for t in range(tokens) if t not in (3, 9, 10)], device="cuda")
    cache.check(keep, want[keep], v[keep])
    short = Cache(12, kvh, dim)       # the last eight tokens fall behind the cache
    call("clef_rope_kv_write_fp8", stream(), *short.pointers(), ptr(k), ptr(v), ptr(cos), ptr(sin), tokens, kvh, dim, rotary, ptr(seq_start),
         ptr(base), None, None, None, 12, 1)
    torch.cuda.synchronize()
    short.check(torch.arange(12, device="cuda"), want[:12], v[:12])


def test_special_head_rows(cuda_dev):
    """Zeros, tiny maxima, the largest finite values, infinities and NaN."""
    dim = 128
    x = torch.randn(8, 1, dim, generator=gen(5), device="cuda")
    x[0] = 0.0
    x[1] = -0.0
    x[2] *= 1e-35
    x[3, 0, :] = 0.0
    x[3, 0, 5] = -3.0e38
    x[4, 0, 17] = math.inf
    x[5, 0, 100] = math.nan
    x[6] *= 1e-29
    cos, sin = tables(8, 32)
    c = torch.full((8, 1, dim), 0xA5, dtype=torch.uint8, device="cuda")
    cache = (c, c.clone(), torch.full((8, 1), 9.0, device="cuda"), torch.full((8, 1), 9.0, device="cuda"))
    cuda_dev.rope_kv_write_fp8_dev(*cache, x, x, cos, sin, 8, 1, dim, 0)
    for code, scale in (cache[0::2], cache[1::2]):
        assert (scale[:3] == 0).all() and (code[:3] & 0x7F == 0).all()
        assert torch.isnan(scale[4:6]).all() and (code[4:6] == 0).all()
        want, s = recipe(x[[3, 6, 7]])
        assert torch.equal(code[[3, 6, 7]], want) and torch.equal(scale[[3, 6, 7]], s)
    k, v = cuda_dev.kv_read_fp8_dev(*cache, 8, 1, dim)
    assert torch.isnan(k[4:6]).all() and torch.isnan(v[4:6]).all() and (k[:3] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,kvh,dim", [(1, 1, 8), (777, 2, 256), (300, 3, 96), (64, 8, 128), (5000, 2, 64)])
def test_kv_read(cuda_dev, rows, kvh, dim, dtype):
    g = gen(rows)
    total = rows + 7
    codes = torch.randint(0, 256, (2, total, kvh, dim), generator=g, device="cuda", dtype=torch.int32)
    codes = torch.where(codes & 0x7F == 0x7F, codes - 1, codes).to(torch.uint8)
    scales = torch.rand(2, total, kvh, generator=g, device="cuda")
    at = torch.randint(0, total, (rows,), generator=g, device="cuda", dtype=torch.int32)     # repeats among them
    if rows > 4:
        at[2], at[3] = -1, total
    k, v = Guarded(rows * kvh * dim * dtype.itemsize), Guarded(rows * kvh * dim * dtype.itemsize)
    for m in (at, None):
        call("clef_kv_read_fp8", stream(), k.ptr, v.ptr, ptr(codes[0]), ptr(codes[1]), ptr(scales[0]), ptr(scales[1]), ptr(m), rows, total, kvh,
             dim, 0 if dtype == torch.bfloat16 else 1)
        torch.cuda.synchronize()
        index = torch.arange(rows, device="cuda") if m is None else m.long()
        there = (index >= 0) & (index < total)
        for got, c, s in ((k, codes[0], scales[0]), (v, codes[1], scales[1])):
            got.check_guards("rows")
            i = index.clamp(0, total - 1)
            want = c[i].view(torch.float8_e4m3fn).float() * s[i][..., None]
            want = torch.where(there[:, None, None], want, torch.zeros_like(want)).to(dtype)
            assert torch.equal(got.payload().view(dtype).view(rows, kvh, dim), want)


def test_write_and_read_captured(cuda_dev):
    g = gen(8)
    tokens, kvh, dim = 33, 2, 128
    k, v = (torch.randn(tokens, kvh, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    cos, sin = tables(tokens, 64)
    c = torch.zeros(tokens, kvh, dim, dtype=torch.uint8, device="cuda")
    cache = (c, c.clone(), torch.zeros(tokens, kvh, device="cuda"), torch.zeros(tokens, kvh, device="cuda"))

    def go():
        cuda_dev.rope_kv_write_fp8_dev(*cache, k, v, cos, sin, tokens, kvh, dim, 64)
        return cuda_dev.kv_read_fp8_dev(*cache, tokens, kvh, dim)

    want = [t.clone() for t in go()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = go()
    for t in cache:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_past_32_bit_offsets(cuda_dev):
    rows, kvh, dim = 2_200_000, 8, 128        # 2.25e9 codes per cache
    k = torch.zeros(rows, kvh, dim, dtype=torch.uint8, device="cuda")
    cache = (k, torch.zeros_like(k), torch.zeros(rows, kvh, device="cuda"), torch.zeros(rows, kvh, device="cuda"))
    x = torch.randn(2, kvh, dim, generator=gen(9), device="cuda").bfloat16()
    cos, sin = tables(4, 64)
    where = torch.tensor([rows - 1, 0], dtype=torch.int32, device="cuda")
    cuda_dev.rope_kv_write_fp8_dev(*cache, x, x, cos, sin, 2, kvh, dim, 0, cache_map=where)
    got, _ = cuda_dev.kv_read_fp8_dev(*cache, 2, kvh, dim, row_map=where, dtype=torch.float32)
    code, scale = recipe(x.float())
    assert torch.equal(got, code.view(torch.float8_e4m3fn).float() * scale[..., None])
    assert not cache[0][1:rows - 1].any()


def fp8_cache(rows, kvh, dim):
    c = torch.zeros(rows, kvh, dim, dtype=torch.uint8, device="cuda")
    return [c, torch.zeros_like(c), torch.zeros(rows, kvh, device="cuda"), torch.zeros(rows, kvh, device="cuda")]


def test_calls_without_a_token(cuda_dev):
    cache = fp8_cache(8, 2, 64)
    x, q = torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 4, 64, device="cuda")
    cos, sin = tables(4, 32)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    cuda_dev.rope_kv_write_fp8_dev(*cache, x, x, cos, sin, 0, 2, 64, 32, cache_map=none)
    assert cuda_dev.rope_qkv_write_fp8_dev(q, *cache, x, x, cos, sin, 0, 4, 2, 64, 32).shape == q.shape
    cuda_dev.qk_norm_rope_kv_write_fp8_dev(*cache, x, x, torch.zeros(64, device="cuda"), cos, sin, 0, 2, 64, 32, EPS)
    k, v = cuda_dev.kv_read_fp8_dev(*cache, 0, 2, 64, row_map=none)
    assert k.shape == v.shape == (0, 2, 64)
    torch.cuda.synchronize()
    assert not any(t.any() for t in cache)


def test_reading_past_the_cache_without_a_map(cuda_dev):
    cache = fp8_cache(5, 2, 64)
    cache[0].fill_(0x38), cache[1].fill_(0x40), cache[2].fill_(1.0), cache[3].fill_(0.5)
    k, v = cuda_dev.kv_read_fp8_dev(*cache, 9, 2, 64)
    assert (k[:5] == 1).all() and (v[:5] == 1).all() and not k[5:].any() and not v[5:].any()


def test_a_row_read_many_times(cuda_dev):
    cache = fp8_cache(70, 3, 96)
    x, y = (torch.randn(70, 3, 96, generator=gen(11), device="cuda") for _ in range(2))
    cos, sin = tables(80, 32)
    cuda_dev.rope_kv_write_fp8_dev(*cache, x, y, cos, sin, 70, 3, 96, 0)
    at = torch.full((501,), 69, dtype=torch.int32, device="cuda")
    k, v = cuda_dev.kv_read_fp8_dev(*cache, 501, 3, 96, row_map=at, dtype=torch.float32)
    for got, want in ((k, x), (v, y)):
        code, scale = recipe(want[69])
        assert torch.equal(got, (code.view(torch.float8_e4m3fn).float() * scale[:, None]).expand(501, 3, 96))


def test_on_another_stream_behind_its_work(cuda_dev):
    """Written on a stream that has first to finish filling the inputs, read on the same one."""
    tokens, kvh, dim = 4000, 2, 128
    cache = fp8_cache(tokens, kvh, dim)
    cos, sin = tables(tokens, 64)
    x = torch.randn(tokens, kvh, dim, generator=gen(12), device="cuda").bfloat16()
    k = torch.zeros_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            k.copy_(-x)
        k.copy_(x)
        cuda_dev.rope_kv_write_fp8_dev(*cache, k, k, cos, sin, tokens, kvh, dim, 0)
        got, _ = cuda_dev.kv_read_fp8_dev(*cache, tokens, kvh, dim, dtype=torch.float32)
    side.synchronize()
    code, scale = recipe(x.float())
    assert torch.equal(got, code.view(torch.float8_e4m3fn).float() * scale[..., None])


def test_the_binding_refuses_what_does_not_fit(cuda_dev):
    cache = fp8_cache(16, 2, 64)
    k, q = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, 8, 64, device="cuda")
    cos, sin = tables(8, 32)
    at = torch.arange(4, dtype=torch.int32, device="cuda")
    w = torch.zeros(64, device="cuda")

    def refused(match, call, *args, **kw):
        with pytest.raises(clef.ClefError, match=match):
            call(*args, **kw)

    write, read = cuda_dev.rope_kv_write_fp8_dev, cuda_dev.kv_read_fp8_dev
    refused("k must", write, *cache, k[:3], k, cos, sin, 4, 2, 64, 32)
    refused("v must be .*float32", write, *cache, k, k.bfloat16(), cos, sin, 4, 2, 64, 32)
    refused("cos must", write, *cache, k, k, cos.bfloat16(), sin, 4, 2, 64, 32)
    refused("sin must", write, *cache, k, k, cos, sin.cpu(), 4, 2, 64, 32)
    refused("cache_map must be .*int32", write, *cache, k, k, cos, sin, 4, 2, 64, 32, cache_map=at.long())
    refused("pos_map must", write, *cache, k, k, cos, sin, 4, 2, 64, 32, pos_map=at[:3])
    refused("E4M3", write, cache[0].float(), *cache[1:], k, k, cos, sin, 4, 2, 64, 32)
    refused("k_scales must", write, cache[0], cache[1], cache[2][:8], cache[3], k, k, cos, sin, 4, 2, 64, 32)
    refused("q must be .*float32", cuda_dev.rope_qkv_write_fp8_dev, q.bfloat16(), *cache, k, k, cos, sin, 4, 8, 2, 64, 32)
    refused("weight must", cuda_dev.qk_norm_rope_kv_write_fp8_dev, *cache, k, k, w[:32], cos, sin, 4, 2, 64, 32, EPS)
    refused("row_map must", read, *cache, 4, 2, 64, row_map=at.cpu())
    refused("float32", read, *cache, 4, 2, 64, dtype=torch.float16)
    a = torch.zeros(4, 64, device="cuda")
    refused("b must be .*float32", cuda_dev.add_rms_norm_fp8_bf16_dev, a, a.bfloat16(), w, 4, 64, EPS)
    refused("weight must", cuda_dev.add_rms_norm_fp8_bf16_dev, a, a, w.bfloat16(), 4, 64, EPS)
    refused("sum_out must", cuda_dev.add_rms_norm_fp8_bf16_dev, a, a, w, 4, 64, EPS, sum_out=a[:2])
    assert [t.shape for t in cuda_dev.add_rms_norm_fp8_bf16_dev(a[:0], a[:0], w, 0, 64, EPS)] == [(0, 64), (0, 64), (0,), (0, 64)]
