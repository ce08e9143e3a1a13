"""clef_paged_attention over FP8 caches whose scales lie far apart: what a row of the output is must not depend on keys that the
causal mask hides from it, and keys without a value still weigh.

Tolerances, relative to the largest |v| among the keys that the ROW sees (an output is a convex combination of those): the weight
times the value scale is rounded to f16 (2^-11) beside a value rounded to f16 at most twice (2^-11 each), the output to bf16
(2^-8). Below 2^-14 of the row's reference f16 steps by 2^-24, so a weight is off by 2^-25 of it beside that, and the reference
is within 2^5 of what the row's largest weight needs: with 448 / 256 for the distance of a value from the power of two above it,
less than 2^-19 per key, 2^-11 for the 160 keys here at most. f32 sums, exp2 and scores: below 2^-13. In all below 2^-7."""
import pytest
import torch

from test_gpu_attention import Problem

pytestmark = pytest.mark.gpu
BOUND = 2 ** -7


def most_seen(p):
    """Largest |v| of the keys each row sees, per row and head, in 64 bits."""
    most = torch.zeros(p.tokens, p.qh, 1, dtype=torch.float64)
    group, at = p.qh // p.kvh, 0
    for s, (n, length) in enumerate(p.lens):
        top = p.v64[p.rows[s]].abs().amax(-1).cummax(0).values          # [keys, kv heads]
        for i in range(n):
            seen = length - n + i + 1
            if seen > 0:
                most[at + i, :, 0] = top[seen - 1].repeat_interleave(group)
        at += n
    return most


def check(p, out, bound=BOUND):
    want, _ = p.want()
    most = most_seen(p)
    err = (out.cpu().double()[:p.tokens] - want).abs()
    assert torch.isfinite(out).all()
    worst = (err / most.clamp(min=1e-300)).max().item()
    assert (err <= bound * most).all(), f"off by {worst:.3g} of the largest value that the row sees, allowed {bound:.3g}"


# two, four and five tokens go to the kernel for few rows, the others to the one for chunks; the last tokens' 16 keys begin
# inside, at, and before a tile's end
BATCHES = {"two_tokens": [(2, 60)], "four_tokens": [(4, 64), (4, 140)], "five_tokens": [(5, 33)], "chunk": [(40, 100)], "prompt": [(150, 150)],
           "edges": [(33, 129), (20, 64), (17, 17)]}


@pytest.mark.parametrize("power", [6, 12, 16, 20, 24, 40])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_a_late_value_does_not_cost_earlier_rows_precision(cuda_dev, batch, head_dim, power):
    """The last key of each sequence has values 2^power larger: only the last row sees it."""
    p = Problem(BATCHES[batch], (8, 2), head_dim, 16, True, seed=power)
    for rows in p.rows:
        p.vs[rows[-1]] *= 2.0 ** power
        p.v64[rows[-1]] *= 2.0 ** power
    check(p, p.run(cuda_dev))


@pytest.mark.parametrize("power", [6, 16, 24, 40])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_a_late_key_does_not_cost_earlier_rows_precision(cuda_dev, batch, head_dim, power):
    """The last key itself is 2^power larger; the row that sees it has scores to match and is left out."""
    p = Problem(BATCHES[batch], (8, 2), head_dim, 16, True, seed=power)
    last = []
    for s, rows in enumerate(p.rows):
        p.ks[rows[-1]] *= 2.0 ** power
        p.k64[rows[-1]] *= 2.0 ** power
        last.append(sum(n for n, _ in p.lens[:s + 1]) - 1)
    out = p.run(cuda_dev)
    want, _ = p.want()
    out[last] = want[last].to(out.dtype).cuda()
    check(p, out)


@pytest.mark.parametrize("power", [0, 20, 40, 100])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 160)], [(40, 160)]], ids=["token", "chunk"])
def test_keys_without_a_value_beside_large_ones_still_weigh(cuda_dev, lens, head_dim, power):
    """Every other 16 keys have values of zero (scale 0), the others values of 2^power: both count in the sum of the weights."""
    p = Problem(lens, (8, 2), head_dim, 16, True, torch.float32, seed=power)
    for start in range(0, 160, 16):
        rows, factor = p.rows[0][start:start + 16], 0.0 if start % 32 else 2.0 ** power
        p.vs[rows] *= factor
        p.v64[rows] *= factor
    check(p, p.run(cuda_dev))


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 150)], [(3, 150)], [(40, 150)], [(150, 150)]], ids=["token", "tokens", "chunk", "prompt"])
def test_every_key_on_a_scale_of_its_own(cuda_dev, lens, head_dim):
    """Scales of K and V that rise along the sequence from 2^-20 to 2^20, up and down by 2^6 from key to key."""
    p = Problem(lens, (8, 2), head_dim, 16, True, seed=head_dim)
    t = torch.arange(150)
    rise = torch.exp2((t * 40 // 150 - 20 + 6 * (t % 2)).float())
    for scales, values in ((p.ks, p.k64), (p.vs, p.v64)):
        scales[p.rows[0]] *= rise[:, None]
        values[p.rows[0]] *= rise[:, None, None].double()
    p.q = (p.q.float() * 2.0 ** -26).to(p.q.dtype)        # scores stay moderate
    check(p, p.run(cuda_dev))


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("heads", [(16, 2), (4, 4)])
def test_long_chunks_on_scales_far_apart(cuda_dev, heads, head_dim):
    """Chunks cut over many CTAs, every scale a random power of two up to 2^30: 2,500 keys instead of the 160 that the bound at the
    top counts with, 2^-19 each, add 2^-7.7 at the very most."""
    p = Problem([(600, 2500), (1, 900), (300, 300)], heads, head_dim, 16, True, seed=heads[0])
    g = torch.Generator().manual_seed(head_dim)
    for scales, values in ((p.ks, p.k64), (p.vs, p.v64)):
        factor = torch.exp2(torch.randint(0, 31, scales.shape, generator=g).float())
        for rows in p.rows:
            scales[rows] *= factor[rows]
            values[rows] *= factor[rows][..., None].double()
    p.q = (p.q.float() * 2.0 ** -30).to(p.q.dtype)
    check(p, p.run(cuda_dev), BOUND + 2.0 ** -7.7)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("short", [600, 1100, 1700, 3000])
def test_row_tiles_with_and_without_a_second_block_in_turn(cuda_dev, short, head_dim):
    """So many row tiles that a CTA takes several behind each other: of 100 rows (one block of 128, up to 47 steps of 64 keys) and of
    256 (two blocks). The second block has nothing to do in the former and is ahead of the keys when it comes to the latter."""
    p = Problem([(100, short), (256, 700)] * 24, (8, 8), head_dim, 64, True, seed=short)
    g = torch.Generator().manual_seed(short)
    for scales, values in ((p.ks, p.k64), (p.vs, p.v64)):     # every sixteen keys under an exponent of their own
        for rows in p.rows:
            factor = torch.exp2(torch.randint(-6, 1, (len(rows) // 16 + 1,), generator=g).float()).repeat_interleave(16)[:len(rows)]
            scales[rows] *= factor[:, None]
            values[rows] *= factor[:, None, None].double()
    check(p, p.run(cuda_dev), BOUND + 2.0 ** -7.4)
