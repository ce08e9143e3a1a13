"""clef_paged_attention over FP8 caches whose scales lie far apart: keys without a value still weigh beside large ones.

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


def check(p, out):
    want, _ = p.want()
    most = most_seen(p)
    err = (out.cpu().double()[:p.tokens] - want).abs()
    assert torch.isfinite(out).all()
    worst = (err / most.clamp(min=1e-300)).max().item()
    assert (err <= BOUND * most).all(), f"off by {worst:.3g} of the largest value that the row sees, allowed {BOUND:.3g}"


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
