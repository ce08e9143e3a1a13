"""clef_add_rms_norm_fp8_bf16: byte for byte clef_add followed by clef_rms_norm_fp8_bf16, over every kernel variant, with the
sum in place of an input, on special rows; and against the definition in 64 bits. And the new operators as a layer uses them:
FP8 cache write, attention over it, gating, residual and norm."""
import math

import pytest
import torch

import aiis_clef_b200 as clef
from gpu_util import Guarded, call, ptr, stream

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
EPS = 1e-6


def inputs(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a, b = (torch.randn(rows, cols, generator=g, device="cuda") for _ in range(2))
    a[:, :3] *= 20.0
    w = torch.randn(cols, generator=g, device="cuda") * 0.1
    return a.to(dtype), b.to(dtype), w


def chain(dev, a, b, w, rows, cols):
    total = dev.add_dev(a, b, rows * cols).view(rows, cols)
    return (total, *dev.rms_norm_fp8_bf16_dev(total, w, rows, cols, EPS))


def same(x, y):
    return torch.equal(x.view(torch.uint8) if x.dtype != torch.uint8 else x, y.view(torch.uint8) if y.dtype != torch.uint8 else y)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 2048), (778, 2048), (1, 4096), (301, 4096), (3, 8), (65, 1000), (9, 512), (40, 1792), (17, 2056),
                                       (6, 6144), (5, 8200), (2, 16384), (2500, 2048), (1300, 4096)])
def test_equals_the_chain(cuda_dev, rows, cols, dtype):
    a, b, w = inputs(rows, cols, dtype, rows + cols)
    if rows > 8:
        a[2], b[2] = 0, 0
        b[3] = -a[3]
        a[4, 5] = math.inf
        a[5, 7] = math.nan
        a[6], b[6] = a[6] * 1e-30, b[6] * 1e-30
        a[7, 1], b[7, 1] = 3e38, 3e38
    want = chain(cuda_dev, a, b, w, rows, cols)
    n = rows * cols
    outs = [Guarded(n * a.element_size()), Guarded(n), Guarded(rows * 2), Guarded(n * 2)]
    call("clef_add_rms_norm_fp8_bf16", stream(), outs[0].ptr, ptr(a), ptr(b), ptr(w), outs[1].ptr, outs[2].ptr, outs[3].ptr, rows, cols, EPS,
         0 if dtype == torch.bfloat16 else 1)
    torch.cuda.synchronize()
    for got, t, name in zip(outs, want, ("sum", "codes", "scales", "copy")):
        got.check_guards(name)
        assert same(got.payload(), t.contiguous().view(-1)), name
    # the sum over an input, no bf16 copy
    for over in (a, b):
        x, y = a.clone(), b.clone()
        target = x if over is a else y
        q, s = torch.empty(n, dtype=torch.uint8, device="cuda"), torch.empty(rows, dtype=torch.int16, device="cuda")
        call("clef_add_rms_norm_fp8_bf16", stream(), ptr(target), ptr(x), ptr(y), ptr(w), ptr(q), ptr(s), None, rows, cols, EPS,
             0 if dtype == torch.bfloat16 else 1)
        torch.cuda.synchronize()
        assert same(target.view(-1), want[0].contiguous().view(-1)) and same(q, want[1].view(-1)) and torch.equal(s, want[2])


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
def test_general_kernel_equals_the_tuned_one(cuda_dev, dtype):
    a, b, w = inputs(1300, 2048, dtype, 1)
    tuned = cuda_dev.add_rms_norm_fp8_bf16_dev(a, b, w, 1300, 2048, EPS)
    clef.set_kernel_choice(1)
    try:
        general = cuda_dev.add_rms_norm_fp8_bf16_dev(a, b, w, 1300, 2048, EPS)
    finally:
        clef.set_kernel_choice(0)
    assert all(same(x.view(-1), y.view(-1)) for x, y in zip(tuned, general))


@pytest.mark.parametrize("rows,cols", [(40, 2048), (40, 1000)])
def test_against_64_bits(cuda_dev, rows, cols):
    """The sum rounded once, y within f32 sums of the exact norm, the code within half an E4M3 step of y over the exact scale."""
    a, b, w = inputs(rows, cols, torch.float32, 2)
    total, q, s, copy = cuda_dev.add_rms_norm_fp8_bf16_dev(a, b, w, rows, cols, EPS)
    exact = a.double() + b.double()
    assert ((total.double() - exact).abs() <= exact.abs() * 2.0 ** -24).all()
    x = total.double()
    y = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * (1 + w.double())
    # norm in f32: the sum of `cols` squares, quotient, root, three products: cols / 2 roundings at the very most, halved by the root
    slack = (cols / 4 + 8) * 2.0 ** -24
    assert ((copy.double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * slack)).all()
    step = y.abs().amax(-1, keepdim=True) / 448
    word = (s.int() << 16).view(torch.float32).double()
    assert ((word - step[:, 0]).abs() <= step[:, 0] * (2.0 ** -7 + slack)).all()           # truncated to 16 bits
    code = q.view(torch.float8_e4m3fn).double() * step
    # half a step: 2^-4 of the value; in the subnormal range a full step of 2^-9 scales, its codes are clamped at 7
    assert ((code - y).abs() <= torch.maximum(y.abs() * 2.0 ** -4, step * 2.0 ** -9) + y.abs() * 2 * slack).all()


def test_a_layer_of_the_new_operators(cuda_dev):
    """Two passes of a mixed batch: K/V written to FP8 pages behind RoPE, attention over them, the gated output added to the
    residual stream and normalised for the next projection; every step against the step before in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(11)
    qh, kvh, dim, rotary, page, width = 16, 2, 128, 64, 16, 12
    hidden = qh * dim
    pages = 2 * width
    shape = (pages * page, kvh, dim)
    cache = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(shape[:2], device="cuda") for _ in range(2)]
    angle = torch.arange(256, device="cuda", dtype=torch.float64)[:, None] / 1e7 ** (torch.arange(0, rotary, 2, device="cuda").double() / rotary)
    angle = torch.cat([angle, angle], 1)
    cos, sin = angle.cos().float(), angle.sin().float()
    table = torch.randperm(pages, generator=g, device="cuda").view(2, width).to(torch.int32)
    weight = torch.randn(hidden, generator=g, device="cuda") * 0.1
    k64, v64 = (torch.zeros(2, 256, kvh, dim, dtype=torch.float64, device="cuda") for _ in range(2))
    lens = [0, 0]
    for chunk in ([37, 70], [1, 64], [1, 1]):
        tokens = sum(chunk)
        q, k, v = (torch.randn(tokens, h, dim, generator=g, device="cuda").bfloat16() for h in (qh, kvh, kvh))
        gate, res = (torch.randn(tokens, hidden, generator=g, device="cuda").bfloat16() for _ in range(2))
        seq = torch.tensor([0] * chunk[0] + [1] * chunk[1], device="cuda")
        pos = torch.tensor([lens[0] + i for i in range(chunk[0])] + [lens[1] + i for i in range(chunk[1])], device="cuda")
        rows = (table[seq, pos // page].long() * page + pos % page).to(torch.int32)
        turned = cuda_dev.rope_qkv_write_fp8_dev(q, *cache, *scales, k, v, cos, sin, tokens, qh, kvh, dim, rotary,
                                                 pos_map=pos.to(torch.int32), cache_map=rows)
        lens = [lens[0] + chunk[0], lens[1] + chunk[1]]
        starts = torch.tensor([0, chunk[0], tokens], dtype=torch.int32, device="cuda")
        attn = cuda_dev.paged_attention_dev(turned, *cache, table, starts, torch.tensor(lens, dtype=torch.int32, device="cuda"), qh, kvh, dim,
                                            page, 1 / math.sqrt(dim), k_scales=scales[0], v_scales=scales[1])
        gated = cuda_dev.sigmoid_mul_dev(attn, gate, tokens * hidden).view(tokens, hidden)
        total, codes, words, copy = cuda_dev.add_rms_norm_fp8_bf16_dev(res, gated, weight, tokens, hidden, EPS)
        # what the cache now stands for, read back, is what attention has to have seen
        back_k, back_v = cuda_dev.kv_read_fp8_dev(*cache, *scales, tokens, kvh, dim, row_map=rows, dtype=torch.float32)
        k64[seq, pos], v64[seq, pos] = back_k.double(), back_v.double()
        at = 0
        for s, n in enumerate(chunk):
            length = lens[s]
            mask = torch.arange(length, device="cuda")[None, :] <= (length - n + torch.arange(n, device="cuda"))[:, None]
            kk, vv = (t[s, :length].repeat_interleave(qh // kvh, 1) for t in (k64, v64))
            score = torch.einsum("thd,jhd->htj", turned[at:at + n].double(), kk) / math.sqrt(dim)
            o = torch.einsum("htj,jhd->thd", torch.softmax(score.masked_fill(~mask, -math.inf), -1), vv)
            assert ((attn[at:at + n].double() - o).abs() <= (2.0 ** -7 + 2.0 ** -13) * vv.abs().max()).all()
            at += n
        want = chain(cuda_dev, res, gated, weight, tokens, hidden)
        assert all(same(x.view(-1), y.view(-1)) for x, y in zip((total, codes, words, copy), want))
