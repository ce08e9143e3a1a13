"""clef_paged_attention key by key: every key a row sees counts once, with its own weight, and none beside them; rows past 32-bit
offsets in both kernels and both kinds of cache; q that is not whole rows is refused."""
import math

import pytest
import torch

import aiis_clef_b200 as clef
from test_gpu_attention import Problem

pytestmark = pytest.mark.gpu

# (batch, heads): single tokens, few and many rows; lengths around the multiples of 16, 64 and 128 keys, row tiles that are cut
# over many CTAs and row tiles that are not
COUNTS = {
    "long_token": ([(1, 20011)], (8, 1)),
    "tokens": ([(1, n) for n in (1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 4095, 4097)], (8, 2)),
    "few_rows": ([(3, 130), (2, 2), (4, 2049)], (4, 2)),
    "long_chunk": ([(70, 9001)], (8, 1)),
    "prompts": ([(300, 300), (129, 129), (64, 65)], (4, 2)),
    "chunks": ([(40, 63), (33, 1025), (1, 700), (130, 131)], (16, 2)),
    "one_head_each": ([(257, 1300), (31, 31)], (3, 3)),
}


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16_cache", "fp8_cache"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("batch", list(COUNTS))
def test_every_key_counts_once(cuda_dev, batch, head_dim, fp8):
    """Key t has weight 2^-(t // 7 % 3) and the value 1 at dim t % head_dim alone: an output is the share of the weights that
    fall on the dim. Weights are powers of two, which bf16 and f16 hold: what is left are the f32 exponentials, sums and scores
    (2^-20), and over FP8 the value's scale of 1 / 448 rounded to f16 (2^-11) and its product with 448 (2^-11). The lightest key left
    out or taken twice shows: of 20,011 keys over 64 dims, weights of 0.58 on average, it is 0.25 / 182 = 2^-9.5 of its dim."""
    lens, heads = COUNTS[batch]
    p = Problem(lens, heads, head_dim, 16, fp8, torch.float32, seed=1)
    p.scale = math.log(2.0)
    p.q.zero_()
    p.q[..., 3] = 1.0
    for s, (_, length) in enumerate(lens):
        t, rows = torch.arange(length), p.rows[s]
        k, v = torch.zeros(length, head_dim), torch.zeros(length, head_dim)
        k[:, 3] = -(t // 7 % 3).float()
        v[t, t % head_dim] = 1.0
        for cache, scales, x in ((p.k, p.ks, k), (p.v, p.vs, v)):
            if fp8:      # key scales of 1: their codes are 0, -1 and -2
                scales[rows] = 1.0 if cache is p.k else 1.0 / 448.0
                x = (x if cache is p.k else x * 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
            cache[rows] = x.to(cache.dtype)[:, None]
    out = p.run(cuda_dev).cpu().double()
    bound = 2.0 ** -10 + 2.0 ** -18 if fp8 else 2.0 ** -19
    at = 0
    for n, length in lens:
        t = torch.arange(length)
        share = torch.zeros(length, head_dim, dtype=torch.float64)
        share[t, t % head_dim] = torch.exp2(-(t // 7 % 3).double())
        want = share.cumsum(0)
        want = (want / want.sum(1, keepdim=True))[length - n:]
        err = (out[at:at + n] - want[:, None]).abs()
        assert (err <= bound * want[:, None]).all(), f"{(err / want[:, None].clamp(min=1e-9)).max():.3g} at {(n, length)}"
        at += n


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16_cache", "fp8_cache"])
def test_rows_past_32_bit_offsets_in_chunks(cuda_dev, fp8):
    """2,200,000 rows x 8 x 128 = 2.25e9 values; 1 token, and 40 that go to the kernel for chunks, in the last pages."""
    rows, kvh, d, page = 2_200_000, 8, 128, 16
    dtype = torch.uint8 if fp8 else torch.bfloat16
    k = torch.zeros(rows, kvh, d, dtype=dtype, device="cuda")
    v = torch.zeros_like(k)
    scales = dict(k_scales=torch.zeros(rows, kvh, device="cuda"), v_scales=torch.zeros(rows, kvh, device="cuda")) if fp8 else {}
    first = rows - 3 * page
    k[first:], v[first:] = (0x20, 0x38) if fp8 else (0.125, 3.0)     # 0x20: 2^-3, 0x38: 1
    for name, scale in (("k_scales", 1.0), ("v_scales", 3.0)):
        if fp8:
            scales[name][first:] = scale
    table = torch.tensor([[rows // page - 1, rows // page - 3, rows // page - 2]], dtype=torch.int32, device="cuda")
    for n in (1, 40):
        q = torch.ones(n, kvh, d, dtype=torch.bfloat16, device="cuda")
        out = cuda_dev.paged_attention_dev(q, k, v, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                           torch.tensor([48], dtype=torch.int32, device="cuda"), kvh, kvh, d, page, 0.1, **scales)
        assert (out == 3.0).all()


def test_queries_that_are_not_whole_rows_are_refused(cuda_dev):
    """A remainder would come back as it was in memory."""
    p = Problem([(1, 100)], (6, 2), 128, 16, behind=0)
    at = [t.cuda() for t in (p.q, p.k, p.v, p.table, p.q_start, p.kv_len)]
    with pytest.raises(clef.ClefError, match="whole rows of 4 x 128"):
        cuda_dev.paged_attention_dev(*at, 4, 2, 128, 16, 0.1)
    with pytest.raises(clef.ClefError, match="whole rows of 6 x 256"):
        cuda_dev.paged_attention_dev(*at, 6, 2, 256, 16, 0.1)
    p.check(cuda_dev.paged_attention_dev(*at, 6, 2, 128, 16, p.scale))
