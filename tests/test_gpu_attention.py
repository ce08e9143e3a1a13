"""clef_paged_attention against the definition in 64 bits: lengths from one token to long ones, odd sizes, uneven batches,
bf16 and FP8 caches, masks that leave a row empty, bytes that must not be read or written.

Tolerances, relative to the largest |v| a row sees (an output is a convex combination of values):
  weights rounded to bf16 (half a step, finfo.eps / 2 = 2^-8, of each: 2^-8 of the combination at most), the output's own
  rounding to bf16 (2^-8 again) and f32 sums and exp2 (well below 2^-13 together): 2^-7 + 2^-13 for bf16 outputs,
  2^-8 + 2^-13 for f32. In an FP8 cache the weight times the value scale is what is rounded: the same bound. The inputs q are bf16
  values, so rounding q is exact; f32 q that is not is tested against the rounded q."""
import math

import numpy as np
import pytest
import torch

import aiis_clef_b200 as clef

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cleanup():
    yield
    torch.cuda.empty_cache()


def quantise(x):
    """E4M3 codes (uint8) and f32 scales of the last axis."""
    scale = x.abs().amax(-1, keepdim=True) / 448.0
    codes = torch.where(scale > 0, x / scale, torch.zeros_like(x)).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), scale.squeeze(-1).contiguous()


class Problem:
    """A paged cache in shuffled pages, uneven sequences, and everything a call must not touch filled with NaN."""

    def __init__(self, lens, heads, head_dim, page, fp8=False, dtype=torch.bfloat16, seed=0, behind=3, gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, (self.qh, self.kvh), self.d, self.page, self.fp8 = lens, heads, head_dim, page, fp8
        pages = [-(-l // page) for _, l in lens]
        self.width = max(max(pages), 1) + 1
        self.n_pages = sum(pages) + 2
        order = torch.randperm(self.n_pages, generator=g)
        # entries past the pages in use name pages that are not there
        self.table = torch.randint(-(1 << 30), 1 << 30, (len(lens), self.width), generator=g, dtype=torch.int32)
        self.rows, at = [], 0
        for s, (n, l) in enumerate(lens):
            mine = order[at:at + pages[s]]
            at += pages[s]
            self.table[s, :pages[s]] = mine.to(torch.int32)
            t = torch.arange(l)
            self.rows.append(mine[t // page] * page + t % page if l else t)
        shape = (self.n_pages * page, self.kvh, head_dim)
        k, v = torch.randn(shape, generator=g) * gain, torch.randn(shape, generator=g)
        used = torch.cat(self.rows) if lens else torch.zeros(0, dtype=torch.long)
        hole = torch.ones(shape[0], dtype=torch.bool)
        hole[used] = False
        self.ks = self.vs = None
        if fp8:
            (k, self.ks), (v, self.vs) = quantise(k), quantise(v)
            self.k64 = k.view(torch.float8_e4m3fn).double() * self.ks.double()[..., None]
            self.v64 = v.view(torch.float8_e4m3fn).double() * self.vs.double()[..., None]
            k[hole], v[hole] = 0x7F, 0x7F
            self.ks[hole], self.vs[hole] = math.nan, math.nan
        else:
            k, v = k.bfloat16(), v.bfloat16()
            self.k64, self.v64 = k.double(), v.double()
            k[hole], v[hole] = math.nan, math.nan
        self.k, self.v = k, v
        self.q_start = torch.tensor([0] + list(np.cumsum([n for n, _ in lens])), dtype=torch.int32)
        self.kv_len = torch.tensor([l for _, l in lens], dtype=torch.int32)
        self.tokens = sum(n for n, _ in lens)
        self.q = (torch.randn(self.tokens + behind, self.qh, head_dim, generator=g) * 1.5).bfloat16().to(dtype)
        self.scale = 1.0 / math.sqrt(head_dim)

    def run(self, dev, out=None, **more):
        c = lambda t: None if t is None else t.cuda()  # noqa: E731
        if out is None:
            out = torch.full(self.q.shape, 77.0, dtype=self.q.dtype, device="cuda")
        dev.paged_attention_dev(c(self.q), c(self.k), c(self.v), c(self.table), c(self.q_start), c(self.kv_len), self.qh, self.kvh,
                                self.d, self.page, self.scale, k_scales=c(self.ks), v_scales=c(self.vs), out=out, **more)
        return out

    def want(self):
        """(output, bound on |v|) per row and head in 64 bits."""
        out = torch.zeros(self.tokens, self.qh, self.d, dtype=torch.float64)
        most = torch.zeros(self.tokens, self.qh, 1, dtype=torch.float64)
        group = self.qh // self.kvh
        q64 = self.q.bfloat16().cuda().double()
        for s, (n, l) in enumerate(self.lens):
            first = sum(m for m, _ in self.lens[:s])
            seen = torch.arange(l)[None, :] <= (l - n + torch.arange(n))[:, None]
            some = seen.any(1)
            if not some.any():
                continue
            mask = seen.cuda()
            for h in range(self.qh):
                k, v = self.k64[self.rows[s], h // group].cuda(), self.v64[self.rows[s], h // group].cuda()
                score = (q64[first:first + n, h] @ k.T * self.scale).masked_fill(~mask, -math.inf)
                o = torch.softmax(score[some.cuda()], -1) @ v
                out[first:first + n, h][some] = o.cpu()
                most[first:first + n, h, 0][some] = v.abs().max().item()
        return out, most

    def check(self, out, bound=None):
        bound = bound or ((2 ** -7 if out.dtype == torch.bfloat16 else 2 ** -8) + 2 ** -13)
        want, most = self.want()
        got = out.cpu().double()
        assert (got[self.tokens:] == 77.0).all(), "rows behind the last sequence were written"
        err = (got[:self.tokens] - want).abs()
        assert torch.isfinite(got).all()
        worst = (err / most.clamp(min=1e-30)).max().item() if err.numel() else 0.0
        assert (err <= bound * most).all(), f"off by {worst:.3g} of the largest value, allowed {bound:.3g}"


DTYPES = [torch.bfloat16, torch.float32]
LENS = {
    "one_token": [(1, 1)],
    "one_key_more": [(1, 129)],
    "short_decode": [(1, 777)],
    "uneven_decode": [(1, 5), (1, 128), (1, 1000), (1, 127), (1, 2049), (1, 1)],
    "long_decode": [(1, 20011)],
    "empty_between": [(0, 0), (1, 40), (0, 300), (2, 2), (0, 0)],
    "rows_without_keys": [(5, 3), (4, 0), (1, 0), (3, 3)],
    "short_chunks": [(3, 200), (7, 7), (2, 1500)],
    "chunk": [(130, 300)],
    "prompt": [(333, 333)],
    "mixed": [(1, 900), (65, 400), (1, 1), (200, 200), (17, 1300)],
}


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16_cache", "fp8_cache"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("lens", list(LENS))
def test_lengths(cuda_dev, lens, head_dim, fp8):
    p = Problem(LENS[lens], (8, 2), head_dim, 16, fp8, seed=len(lens) + head_dim)
    p.check(p.run(cuda_dev))


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f32"])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16_cache", "fp8_cache"])
@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (6, 2), (16, 2), (12, 1), (10, 2), (33, 1), (64, 1)])
def test_head_layouts(cuda_dev, heads, fp8, dtype):
    for lens in ([(1, 300), (1, 77)], [(40, 100), (1, 260)]):
        p = Problem(lens, heads, 128, 32, fp8, dtype, seed=heads[0])
        p.check(p.run(cuda_dev))


@pytest.mark.parametrize("page", [1, 3, 8, 48, 100, 128, 1024])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16_cache", "fp8_cache"])
def test_page_sizes(cuda_dev, page, fp8):
    for lens in ([(1, 500), (1, 31)], [(100, 411), (3, 3)]):
        p = Problem(lens, (4, 2), 128, page, fp8, seed=page)
        p.check(p.run(cuda_dev))


@pytest.mark.parametrize("head_dim", [128, 256])
def test_large_scores_and_far_maxima(cuda_dev, head_dim):
    """Scores in the hundreds: the running maximum moves often and weights underflow."""
    for lens in ([(1, 3000)], [(150, 900)]):
        p = Problem(lens, (8, 1), head_dim, 16, seed=5, gain=30.0)
        # score errors: f32 products of exact bf16 operands, sums of 128 terms of ~50 each off by some 2^-24 * 128 * 500;
        # exp2 turns an absolute score error e into a relative one of e: 0.004 at most, next to the roundings above
        p.check(p.run(cuda_dev), bound=2 ** -7 + 2 ** -8)


def test_f32_queries_are_rounded_once(cuda_dev):
    p = Problem([(1, 300), (70, 90)], (4, 2), 128, 16, dtype=torch.float32)
    p.q = p.q + torch.randn(p.q.shape, generator=torch.Generator().manual_seed(1)) * 1e-3
    p.check(p.run(cuda_dev))


def test_pages_that_are_not_there_read_as_zeros(cuda_dev):
    p = Problem([(1, 64), (20, 64)], (4, 2), 128, 16)
    for s in range(2):
        bad = int(p.table[s, 1])
        p.table[s, 1] = (-1, p.n_pages)[s]
        p.k64[bad * 16:bad * 16 + 16] = 0
        p.v64[bad * 16:bad * 16 + 16] = 0
    p.check(p.run(cuda_dev))


def test_lengths_beyond_the_shapes_are_clamped(cuda_dev):
    """kv_len above the table and q_start above total_q: nothing outside the tensors is read or written."""
    p = Problem([(2, 48)], (4, 2), 128, 16, behind=0)
    p.table = p.table[:, :3].contiguous()
    p.kv_len = torch.tensor([1 << 30], dtype=torch.int32)
    p.q_start = torch.tensor([0, 1 << 30], dtype=torch.int32)
    p.check(p.run(cuda_dev))
    p.kv_len, p.lens = torch.tensor([-5], dtype=torch.int32), [(2, 0)]
    p.rows = [p.rows[0][:0]]
    p.check(p.run(cuda_dev))


def test_graph_replay_equals_the_eager_call_and_follows_the_lengths(cuda_dev):
    p = Problem([(1, 900), (1, 300), (1, 700)], (16, 2), 128, 16, fp8=True)
    dev = [t.cuda() for t in (p.q, p.k, p.v, p.table, p.q_start, p.kv_len)]
    ks, vs = p.ks.cuda(), p.vs.cuda()
    out = torch.full(p.q.shape, 77.0, dtype=p.q.dtype, device="cuda")

    def go():
        cuda_dev.paged_attention_dev(*dev, p.qh, p.kvh, p.d, p.page, p.scale, k_scales=ks, v_scales=vs, out=out)

    go()
    torch.cuda.synchronize()
    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    out.fill_(77.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    p.kv_len = torch.tensor([450, 300, 1], dtype=torch.int32)
    p.lens = [(1, 450), (1, 300), (1, 1)]
    p.rows = [r[:l] for r, (_, l) in zip(p.rows, p.lens)]
    dev[5].copy_(p.kv_len)
    graph.replay()
    torch.cuda.synchronize()
    p.check(out)


@pytest.mark.parametrize("lens", [[(1, 5000), (1, 100)], [(300, 700), (1, 900)]])
def test_results_do_not_depend_on_timing_or_stream(cuda_dev, lens):
    p = Problem(lens, (16, 2), 128, 64)
    first = p.run(cuda_dev)
    for _ in range(5):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = p.run(cuda_dev)
        side.synchronize()
        assert torch.equal(first, again)


def test_a_workspace_with_any_contents_serves(cuda_dev):
    p = Problem([(1, 5000), (1, 100)], (16, 2), 128, 64)
    ws = torch.full((clef.paged_attention_workspace(2, p.q.shape[0], 16, 2, 128),), 0xFF, dtype=torch.uint8, device="cuda")
    p.check(p.run(cuda_dev, workspace=ws))
    p.check(p.run(cuda_dev, workspace=ws))


def test_rows_past_32_bit_offsets(cuda_dev):
    """Cache rows whose element offsets pass 2^31: 2,200,000 rows x 8 x 128 = 2.25e9 values."""
    rows, kvh, d, page = 2_200_000, 8, 128, 16
    k = torch.zeros(rows, kvh, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    last = rows // page - 1
    k[last * page:], v[last * page:] = 0.01, 3.0
    table = torch.tensor([[last]], dtype=torch.int32, device="cuda")
    for n in (1, 16):
        q = torch.ones(n, kvh, d, dtype=torch.bfloat16, device="cuda")
        out = cuda_dev.paged_attention_dev(q, k, v, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                           torch.tensor([16], dtype=torch.int32, device="cuda"), kvh, kvh, d, page, 0.1)
        assert (out == 3.0).all()


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16_cache", "fp8_cache"])
def test_more_sequences_than_a_warp_scans_at_once(cuda_dev, fp8):
    g = np.random.default_rng(8)
    decode = [(1, int(n)) for n in g.integers(1, 400, 150)]
    mixed = [(int(n), int(n + m)) for n, m in zip(g.integers(0, 60, 70), g.integers(0, 300, 70))]
    for lens in (decode, mixed):
        p = Problem(lens, (8, 2), 128, 16, fp8, seed=len(lens))
        p.check(p.run(cuda_dev))


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(cuda_dev, seed):
    g = np.random.default_rng(seed)
    lens = []
    for _ in range(int(g.integers(1, 7))):
        n = int(g.choice([1, 1, g.integers(1, 9), g.integers(1, 200)]))
        lens.append((n, int(n + g.choice([0, g.integers(0, 40), g.integers(0, 3000)]))))
    kvh = int(g.choice([1, 2, 3, 8]))
    p = Problem(lens, (kvh * int(g.choice([1, 2, 5, 8, 16])), kvh), int(g.choice([64, 128, 256])), int(g.choice([1, 7, 16, 64, 512])),
                bool(g.integers(2)), DTYPES[int(g.integers(2))], seed=seed)
    p.check(p.run(cuda_dev))


@pytest.mark.parametrize("lens", [[(1, 700)], [(90, 700)]], ids=["token", "chunk"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_fp8_scales_far_apart(cuda_dev, lens, head_dim):
    """Head rows from 2^-40 to 2^12 in one tile, some of them zero. q is scaled down so that scores stay moderate."""
    p = Problem(lens, (8, 2), head_dim, 16, True)
    g = torch.Generator().manual_seed(3)
    for scales, values in ((p.ks, p.k64), (p.vs, p.v64)):
        fine = torch.isfinite(scales)
        factor = torch.exp2(torch.randint(-40, 13, scales.shape, generator=g).float()) * (torch.rand(scales.shape, generator=g) > 0.1)
        scales[fine] = (scales * factor)[fine]
        values *= factor[..., None].double()
    p.q = (p.q.float() * 2.0 ** -10).to(p.q.dtype)
    # as above, and 2^-10 more: a value's scale under the tile's power of two is rounded to f16 (2^-11) and so is the product
    p.check(p.run(cuda_dev), bound=2 ** -7 + 2 ** -10 + 2 ** -13)


@pytest.mark.parametrize("head_dim", [128, 256])
@pytest.mark.parametrize("lens", [[(1, 300)], [(40, 300)]], ids=["token", "chunk"])
def test_fp8_rows_that_held_no_number(cuda_dev, lens, head_dim):
    """A NaN scale, of K or of V, makes NaN of the rows that see the key and leaves those that do not."""
    n = lens[0][0]
    for which in ("ks", "vs"):
        p = Problem(lens, (4, 2), head_dim, 16, True, behind=0)
        key = 300 - (n + 1) // 2 if n > 1 else 250      # the second half of a chunk sees it
        getattr(p, which)[p.rows[0][key], 0] = math.nan
        out = p.run(cuda_dev).cpu().double()
        want, most = p.want()
        sees = torch.arange(n) + 300 - n >= key
        assert torch.isnan(out[sees][:, :2]).all()
        err = (out - want).abs()
        assert (err[~sees] <= 2 ** -6 * most[~sees]).all() and (err[:, 2:] <= 2 ** -6 * most[:, 2:]).all()


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16_cache", "fp8_cache"])
@pytest.mark.parametrize("lens", [[(1, 300), (2, 900)], [(60, 300), (1, 900)]], ids=["tokens", "chunk"])
@pytest.mark.parametrize("scale", [0.0, -0.05])
def test_scales_that_are_not_positive(cuda_dev, lens, fp8, scale):
    p = Problem(lens, (8, 2), 128, 16, fp8)
    p.scale = scale
    p.check(p.run(cuda_dev))


def test_infinite_scores_give_nan_in_their_rows_alone(cuda_dev):
    for lens in ([(1, 300), (1, 300)], [(40, 300), (40, 300)]):
        p = Problem(lens, (4, 2), 128, 16, behind=0)
        p.q[0] = math.inf
        out = p.run(cuda_dev).cpu().double()
        want, most = p.want()
        assert torch.isnan(out[0]).all()
        assert ((out - want).abs()[1:] <= (2 ** -7 + 2 ** -13) * most[1:]).all()


def test_two_calls_at_once(cuda_dev):
    """Two streams, each with a workspace of its own, many times over."""
    a, b = Problem([(1, 6000), (1, 50)], (16, 2), 128, 64), Problem([(200, 2000)], (16, 2), 128, 64, True)
    want = [p.run(cuda_dev) for p in (a, b)]
    torch.cuda.synchronize()
    args = [([t.cuda() for t in (p.q, p.k, p.v, p.table, p.q_start, p.kv_len)], {k: t.cuda() for k, t in (("k_scales", p.ks), ("v_scales", p.vs)) if t is not None}) for p in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.full_like(w, 77.0) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, (x, y), s, o in zip((a, b), args, streams, outs):
            with torch.cuda.stream(s):
                cuda_dev.paged_attention_dev(*x, p.qh, p.kvh, p.d, p.page, p.scale, out=o, **y)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("choice", ["rows", "chunk"])
def test_sequences_longer_than_the_average_rows(cuda_dev, choice):
    """A long chunk among many single tokens stays with the kernel for few rows; a lone token in a batch of chunks with the
    other. Both have to hold whatever the average says."""
    lens = [(1, 40)] * 60 + [(50, 333)] if choice == "rows" else [(150, 150)] * 4 + [(1, 2000), (2, 3)]
    for fp8 in (False, True):
        p = Problem(lens, (16, 2), 128, 16, fp8, seed=9)
        p.check(p.run(cuda_dev))


def test_float8_tensors_and_views_as_caches(cuda_dev):
    p = Problem([(1, 100)], (4, 2), 128, 16, True, behind=0)
    plain = p.run(cuda_dev)
    p.k, p.v = p.k.view(torch.float8_e4m3fn), p.v.view(torch.float8_e4m3fn)
    assert torch.equal(p.run(cuda_dev), plain)


def test_the_binding_refuses_what_does_not_fit(cuda_dev):
    p = Problem([(1, 100)], (4, 2), 128, 16, True)
    good = dict(q=p.q, cache_k=p.k, cache_v=p.v, page_table=p.table, q_start=p.q_start, kv_len=p.kv_len)
    good = {k: t.cuda() for k, t in good.items()}
    rest = dict(q_heads=4, kv_heads=2, head_dim=128, page_size=16, scale=0.1, k_scales=p.ks.cuda(), v_scales=p.vs.cuda())

    def refused(match, **other):
        with pytest.raises(clef.ClefError, match=match):
            cuda_dev.paged_attention_dev(**{**good, **rest, **other})

    refused("kv_len must be .*int32", kv_len=good["kv_len"].long())
    refused("n_seqs", q_start=good["q_start"][:1])
    refused("k_scales", k_scales=None)
    refused("v_scales must be .*float32", v_scales=rest["v_scales"].half())
    refused("cache_v", cache_v=good["cache_v"][:16])
    refused("cache_v must be .*uint8", cache_v=good["cache_v"].view(torch.int8))
    refused("contiguous", cache_k=good["cache_k"].transpose(0, 1))
    refused("CUDA", page_table=p.table)
    refused("out must", out=good["q"].float())
    refused("workspace", workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    for name in ("q_heads", "kv_heads", "head_dim", "page_size"):
        refused("positive", **{name: 0})


def test_calls_without_a_token_or_a_sequence(cuda_dev):
    p = Problem([(1, 100)], (4, 2), 128, 16)
    k, v = p.k.cuda(), p.v.cuda()
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 4, 128, dtype=torch.bfloat16, device="cuda")
    rest = (4, 2, 128, 16, 0.1)
    assert cuda_dev.paged_attention_dev(q, k, v, p.table.cuda()[:0], zero, none, *rest).shape == q.shape
    assert cuda_dev.paged_attention_dev(q, k, v, p.table.cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"), p.kv_len.cuda(), *rest).shape == q.shape
    out = torch.full((3, 4, 128), 5.0, dtype=torch.bfloat16, device="cuda")      # rows, but no sequence to own them
    cuda_dev.paged_attention_dev(out.clone(), k, v, p.table.cuda()[:0], zero, none, *rest, out=out)
    torch.cuda.synchronize()
    assert (out == 5).all()


def test_replayed_with_other_lengths(cuda_dev):
    """A captured call, replayed after its lengths, pages and tokens were changed in place, against a plain call."""
    big = Problem([(5, 900), (60, 700), (1, 1200)], (8, 2), 128, 16, seed=4)
    small = Problem([(30, 901), (2, 697), (34, 1190)], (8, 2), 128, 16, seed=5)
    assert big.table.shape == small.table.shape and big.q.shape == small.q.shape and big.k.shape == small.k.shape
    at = [t.cuda() for t in (big.q, big.k, big.v, big.table, big.q_start, big.kv_len)]
    out = torch.full_like(at[0], 77.0)
    call = lambda: cuda_dev.paged_attention_dev(*at, 8, 2, 128, 16, big.scale, out=out)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for p in (small, big):
        for dst, src in zip(at, (p.q, p.k, p.v, p.table, p.q_start, p.kv_len)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        p.check(out)
