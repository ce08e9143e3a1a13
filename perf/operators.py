"""What the KV-cache, attention and residual-norm operators are measured on: cases, inputs, plain forms and 64-bit forms.

`own = False`: `run` computes an operator from elementary torch operations in 32 bits; `own = True`: through
`aiis_clef_b200.Device`. Serving shapes: 16 query heads over 2 key/value heads of 128 or 256, 64 rotated dims, passes of
up to 8,192 rows, contexts of up to 130,712 tokens.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e7
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HEADS = ((16, 2), (8, 8), (12, 4), (16, 1), (6, 2), (32, 4))


# ---- the cases -------------------------------------------------------------------------------------------------
def listed():
    return [
        # the residual add + norm of one generated token, on the f32 residual stream
        {"name": "add_norm_one_token_f32", "op": "add_norm", "rows": 1, "cols": 4096, "dtype": "f32"},
        # the same step of a full 8,192-row pass on bf16 activations
        {"name": "add_norm_pass_bf16", "op": "add_norm", "rows": 8192, "cols": 2048, "dtype": "bf16"},
        # the cache write of a decode batch: one new token for each of 61 requests, wide heads
        {"name": "kv_write_decode", "op": "kv_write", "tokens": 61, "q_heads": 16, "kv_heads": 2, "head_dim": 256,
         "rotary_dim": 64, "dtype": "bf16"},
        # the cache write of a full pass
        {"name": "kv_write_pass", "op": "kv_write", "tokens": 8192, "q_heads": 16, "kv_heads": 2, "head_dim": 128,
         "rotary_dim": 64, "dtype": "bf16"},
        # a short request's cached rows read back
        {"name": "kv_read_short", "op": "kv_read", "rows": 777, "kv_heads": 2, "head_dim": 256, "dtype": "bf16"},
        # the longest context read back
        {"name": "kv_read_long", "op": "kv_read", "rows": 130712, "kv_heads": 2, "head_dim": 128, "dtype": "bf16"},
        # one request generating a token after a short prompt: latency
        {"name": "decode_one_bf16", "op": "attention", "seqs": 1, "q_len": 1, "kv_len": 777, "q_heads": 16, "kv_heads": 2,
         "head_dim": 128, "page": 16, "cache": "bf16", "shape": 1},
        # a decode batch of 64 requests of uneven lengths on the FP8 cache
        {"name": "decode_batch_fp8", "op": "attention", "seqs": 64, "q_len": 1, "kv_len": 8192, "q_heads": 16,
         "kv_heads": 2, "head_dim": 128, "page": 64, "cache": "fp8", "shape": 2},
        # one request generating a token at the end of the longest context, wide heads
        {"name": "decode_long_bf16", "op": "attention", "seqs": 1, "q_len": 1, "kv_len": 130712, "q_heads": 16,
         "kv_heads": 2, "head_dim": 256, "page": 64, "cache": "bf16", "shape": 3},
        # a whole prompt in one pass
        {"name": "prefill_bf16", "op": "attention", "seqs": 1, "q_len": 8192, "kv_len": 8192, "q_heads": 16,
         "kv_heads": 2, "head_dim": 128, "page": 64, "cache": "bf16", "shape": 4},
        # an odd chunk late in a long prompt, FP8 cache
        {"name": "chunk_fp8", "op": "attention", "seqs": 1, "q_len": 2011, "kv_len": 32768, "q_heads": 16, "kv_heads": 2,
         "head_dim": 128, "page": 64, "cache": "fp8", "shape": 5},
        # a mixed batch: chunks and single tokens of nine requests, wide heads, small pages
        {"name": "mixed_bf16", "op": "attention", "seqs": 9, "q_len": 700, "kv_len": 4096, "q_heads": 16, "kv_heads": 2,
         "head_dim": 256, "page": 16, "cache": "bf16", "shape": 6},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["add_norm", "kv_write", "kv_read", "attention", "attention", "attention"])
    if op == "add_norm":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": 8 * _log(rng, 8, 768), "dtype": rng.choice(["bf16", "f32"])}
    q_heads, kv_heads = rng.choice(HEADS)
    head_dim = rng.choice([64, 128, 256])
    if op == "kv_write":
        return {"op": op, "tokens": _log(rng, 1, 4096), "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "rotary_dim": rng.choice([32, 64, head_dim]), "dtype": rng.choice(["bf16", "f32"])}
    if op == "kv_read":
        return {"op": op, "rows": _log(rng, 1, 32768), "kv_heads": kv_heads, "head_dim": head_dim,
                "dtype": rng.choice(["bf16", "f32"])}
    case = {"op": op, "seqs": _log(rng, 1, 64), "q_len": _log(rng, 1, 4096), "kv_len": _log(rng, 1, 65536),
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([8, 16, 48, 64, 256]),
            "cache": rng.choice(["bf16", "fp8"]), "shape": rng.randrange(1 << 30)}
    case["q_len"] = min(case["q_len"], case["kv_len"])
    # keep the plain form's padded score matrix and gathered cache in bounds
    while case["seqs"] * q_heads * case["q_len"] * case["kv_len"] > 6e8 or case["seqs"] * kv_heads * head_dim * case["kv_len"] > 1.3e8:
        key = max(("seqs", "q_len", "kv_len"), key=lambda k: case[k] if k != "kv_len" else case[k] / 64)
        if case[key] <= 1:
            key = "kv_len"
        case[key] = max(1, case[key] * 2 // 3)
        case["q_len"] = min(case["q_len"], case["kv_len"])
    return case


def _lengths(case):
    """[(new tokens, cached tokens)] of each request: the first has the full lengths, the others uneven ones."""
    rng = random.Random(case["shape"])
    lens = [(case["q_len"], case["kv_len"])]
    for _ in range(case["seqs"] - 1):
        n = rng.choice([1, rng.randint(1, case["q_len"])])
        lens.append((n, rng.randint(max(n, case["kv_len"] // 8), case["kv_len"])))
    return lens


def work(case):
    op = case["op"]
    if op == "add_norm":
        e = 2 if case["dtype"] == "bf16" else 4
        n = case["rows"] * case["cols"]
        return {"bytes": n * (3 * e + 1 + 2) + 2 * case["rows"] + 4 * case["cols"], "flops": 8 * n}
    e = 2 if case.get("dtype", "bf16") == "bf16" else 4
    if op == "kv_write":
        t, q, kv = case["tokens"], case["q_heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        return {"bytes": t * (2 * q * e + 2 * kv * (e + 1) + 8 * case["kv_heads"] + 8 * case["rotary_dim"] + 8),
                "flops": t * (3 * q + 6 * kv)}
    if op == "kv_read":
        n = case["rows"] * case["kv_heads"]
        return {"bytes": n * 2 * (case["head_dim"] * (1 + e) + 4) + 4 * case["rows"], "flops": 2 * n * case["head_dim"]}
    lens = _lengths(case)
    h, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    tokens, cached = sum(n for n, _ in lens), sum(l for _, l in lens)
    pairs = sum(n * l - n * (n - 1) // 2 for n, l in lens)
    row = 2 * d if case["cache"] == "bf16" else d + 4
    return {"bytes": 2 * tokens * h * d * 2 + 2 * cached * kv * row, "flops": 4 * pairs * h * d}


# ---- inputs ----------------------------------------------------------------------------------------------------
def _quantise_rows(x):
    """(e4m3 codes as float8, f32 scale per row) of the last axis."""
    scale = x.abs().amax(-1, keepdim=True) / 448.0
    codes = torch.where(scale > 0, x / scale, torch.zeros_like(x)).clamp(-448.0, 448.0)
    return codes.to(torch.float8_e4m3fn), scale.squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def order(n):
        return torch.randperm(n, generator=g, device="cuda")

    op = case["op"]
    if op == "add_norm":
        rows, cols, t = case["rows"], case["cols"], TYPES[case["dtype"]]
        gain = torch.ones(cols, device="cuda")
        gain[order(cols)[:8]] = 20.0                       # the outlier channels of a residual stream
        return {"case": case, "a": (normal(rows, cols) * gain).to(t), "b": (normal(rows, cols) * 0.5).to(t),
                "weight": normal(cols) * 0.1}
    if op == "attention":
        return _prepare_attention(case, normal, order)
    kv, d = case["kv_heads"], case["head_dim"]
    count = case["tokens"] if op == "kv_write" else case["rows"]
    cache_rows = count + count // 4 + 3
    rows = order(cache_rows)[:count].to(torch.int32)
    k_codes, k_scales = _quantise_rows(normal(cache_rows, kv, d))
    v_codes, v_scales = _quantise_rows(normal(cache_rows, kv, d))
    state = {"case": case, "rows": rows, "cache_k": k_codes.view(torch.uint8), "cache_v": v_codes.view(torch.uint8),
             "k_scales": k_scales, "v_scales": v_scales}
    if op == "kv_write":
        t, r = TYPES[case["dtype"]], case["rotary_dim"]
        angle = torch.arange(case["tokens"] + 64, device="cuda", dtype=torch.float64)[:, None] / THETA ** (
            torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        angle = torch.cat([angle, angle], dim=1)
        state |= {"q": normal(count, case["q_heads"], d).to(t), "k": (normal(count, kv, d) * 2).to(t),
                  "v": normal(count, kv, d).to(t), "cos": angle.cos().float(), "sin": angle.sin().float(),
                  "positions": order(case["tokens"] + 64)[:count].to(torch.int32)}
    return state


def _prepare_attention(case, normal, order):
    lens, page = _lengths(case), case["page"]
    kv, d = case["kv_heads"], case["head_dim"]
    pages = [-(-l // page) for _, l in lens]
    width, total = max(pages), sum(pages) + 2
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    shuffled, at = order(total).to(torch.int32), 0
    for s, n in enumerate(pages):
        table[s, :n] = shuffled[at:at + n]
        at += n
    k, v = normal(total * page, kv, d), normal(total * page, kv, d)
    state = {"case": case, "table": table, "k_scales": None, "v_scales": None,
             "q_start": torch.tensor([0] + list(np.cumsum([n for n, _ in lens])), dtype=torch.int32, device="cuda"),
             "kv_len": torch.tensor([l for _, l in lens], dtype=torch.int32, device="cuda"),
             "q_most": max(n for n, _ in lens), "kv_most": max(l for _, l in lens),
             "q": (normal(sum(n for n, _ in lens), case["q_heads"], d) * 1.5).bfloat16()}
    if case["cache"] == "bf16":
        return state | {"cache_k": k.bfloat16(), "cache_v": v.bfloat16()}
    (k, k_scales), (v, v_scales) = _quantise_rows(k), _quantise_rows(v)
    return state | {"cache_k": k.view(torch.uint8), "cache_v": v.view(torch.uint8), "k_scales": k_scales, "v_scales": v_scales}


# ---- one pass --------------------------------------------------------------------------------------------------
_kept = {}


def _device():
    """The framework's device handle, opened once as a program does."""
    if "device" not in _kept:
        import aiis_clef_b200 as clef

        _kept["device"] = clef.Device(0)
    return _kept["device"]


def _float8(x):
    return x.view(torch.float8_e4m3fn)


def run(state):
    case = state["case"]
    if own:
        return _RUN_OWN[case["op"]](_device(), state, case)
    return _RUN_PLAIN[case["op"]](state, case)


def _own_add_norm(dev, s, case):
    total, codes, scales, copy = dev.add_rms_norm_fp8_bf16_dev(s["a"], s["b"], s["weight"], case["rows"], case["cols"], EPS)
    return {"sum": total, "codes": _float8(codes), "scales": scales.view(torch.bfloat16), "copy": copy}


def _own_kv_write(dev, s, case):
    q = dev.rope_qkv_write_fp8_dev(s["q"], s["cache_k"], s["cache_v"], s["k_scales"], s["v_scales"], s["k"], s["v"], s["cos"],
                                   s["sin"], case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"],
                                   case["rotary_dim"], pos_map=s["positions"], cache_map=s["rows"])
    return {"q": q, "cache_k": _float8(s["cache_k"]), "cache_v": _float8(s["cache_v"]), "k_scales": s["k_scales"],
            "v_scales": s["v_scales"]}


def _own_kv_read(dev, s, case):
    k, v = dev.kv_read_fp8_dev(s["cache_k"], s["cache_v"], s["k_scales"], s["v_scales"], case["rows"], case["kv_heads"],
                               case["head_dim"], row_map=s["rows"], dtype=TYPES[case["dtype"]])
    return {"k": k, "v": v}


def _own_attention(dev, s, case):
    return dev.paged_attention_dev(s["q"], s["cache_k"], s["cache_v"], s["table"], s["q_start"], s["kv_len"], case["q_heads"],
                                   case["kv_heads"], case["head_dim"], case["page"], 1.0 / math.sqrt(case["head_dim"]),
                                   k_scales=s["k_scales"], v_scales=s["v_scales"])


def _plain_add_norm(s, case):
    t = TYPES[case["dtype"]]
    total = (s["a"].float() + s["b"].float()).to(t)
    x = total.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + s["weight"])
    codes, scale = _quantise_rows(y)
    word = (scale.view(torch.int32) >> 16).to(torch.int16)     # the upper 16 bits of the scale
    return {"sum": total, "codes": codes, "scales": word.view(torch.bfloat16), "copy": y.bfloat16()}


def _rotate(x, cos, sin, rotary):
    half = rotary // 2
    lo, hi = x[..., :half], x[..., half:rotary]
    c, s = cos[:, None, :half], sin[:, None, :half]
    return torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., rotary:]], dim=-1)


def _plain_kv_write(s, case):
    at, rows = s["positions"].long(), s["rows"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    q = _rotate(s["q"].float(), cos, sin, case["rotary_dim"]).to(TYPES[case["dtype"]])
    k_codes, k_scale = _quantise_rows(_rotate(s["k"].float(), cos, sin, case["rotary_dim"]))
    v_codes, v_scale = _quantise_rows(s["v"].float())
    s["cache_k"][rows], s["cache_v"][rows] = k_codes.view(torch.uint8), v_codes.view(torch.uint8)
    s["k_scales"][rows], s["v_scales"][rows] = k_scale, v_scale
    return {"q": q, "cache_k": _float8(s["cache_k"]), "cache_v": _float8(s["cache_v"]), "k_scales": s["k_scales"],
            "v_scales": s["v_scales"]}


def _plain_kv_read(s, case):
    rows, t = s["rows"].long(), TYPES[case["dtype"]]
    k = _float8(s["cache_k"][rows]).float() * s["k_scales"][rows][..., None]
    v = _float8(s["cache_v"][rows]).float() * s["v_scales"][rows][..., None]
    return {"k": k.to(t), "v": v.to(t)}


def _plain_attention(s, case):
    h, kv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    group, n, width = h // kv, s["kv_len"].numel(), s["kv_most"]
    j = torch.arange(width, device="cuda")
    there = j[None, :] < s["kv_len"][:, None]                                          # [n, keys]
    rows = torch.where(there, s["table"].long()[:, j // page] * page + j % page, 0)
    k, v = s["cache_k"][rows], s["cache_v"][rows]                                      # [n, keys, kv, d]
    if case["cache"] == "fp8":
        k = _float8(k).float() * s["k_scales"][rows][..., None]
        v = _float8(v).float() * s["v_scales"][rows][..., None]
    k, v = k.float().permute(0, 2, 3, 1), v.float().permute(0, 2, 1, 3)
    i = torch.arange(s["q_most"], device="cuda")
    first, new = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    live = i[None, :] < new[:, None]                                                   # [n, queries]
    token = torch.where(live, first[:, None] + i[None, :], 0)
    q = s["q"][token].float().view(n, -1, kv, group, d).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)
    last = s["kv_len"].long()[:, None] - new[:, None] + i[None, :]                     # the last key a query sees
    seen = (j[None, None, :] <= last[:, :, None]) & there[:, None, :]
    seen = seen[:, None, :, None, :]
    score = torch.matmul(q, k).mul_(1.0 / math.sqrt(d)).view(n, kv, -1, group, width)
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(n, kv, -1, width), v).view(n, kv, -1, group, d) / total.clamp(min=1e-30)
    return out.permute(0, 2, 1, 3, 4).reshape(n, -1, h, d)[live].bfloat16()


_RUN_OWN = {"add_norm": _own_add_norm, "kv_write": _own_kv_write, "kv_read": _own_kv_read, "attention": _own_attention}
_RUN_PLAIN = {"add_norm": _plain_add_norm, "kv_write": _plain_kv_write, "kv_read": _plain_kv_read,
              "attention": _plain_attention}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))


def _exact_add_norm(case, s):
    t = TYPES[case["dtype"]]
    stored = (s["a"].double() + s["b"].double()).to(t).double()            # the sum as it is stored
    norm = stored / (stored.pow(2).sum(-1, keepdim=True) / case["cols"] + EPS).sqrt()
    y = norm + norm * s["weight"].double()
    step = y.abs().max(-1, keepdim=True).values / 448
    word = (step.float().view(torch.int32) & -65536).view(torch.float32).double().squeeze(-1)
    return {"sum": stored, "codes": y / step, "scales": word, "copy": y}


def _turned(x, angle_cos, angle_sin, rotary):
    """Each pair (j, j + rotary / 2) as a complex number times e^(i angle)."""
    half = rotary // 2
    z = torch.complex(x[..., :half].double(), x[..., half:rotary].double())
    z = z * torch.complex(angle_cos[:, :half].double(), angle_sin[:, :half].double())[:, None, :]
    out = x.double().clone()
    out[..., :half], out[..., half:rotary] = z.real, z.imag
    return out


def _exact_kv_write(case, s):
    at, rows = s["positions"].long(), s["rows"].long()
    cos, sin = s["cos"].index_select(0, at), s["sin"].index_select(0, at)
    out = {"q": _turned(s["q"], cos, sin, case["rotary_dim"])}
    for name, x in (("k", _turned(s["k"], cos, sin, case["rotary_dim"])), ("v", s["v"].double())):
        codes, scales = _float8(s["cache_" + name]).double(), s[name + "_scales"].double()
        step = x.abs().max(-1).values / 448
        out["cache_" + name] = codes.index_copy(0, rows, x / step[..., None])
        out[name + "_scales"] = scales.index_copy(0, rows, step)
    return out


def _exact_kv_read(case, s):
    rows = s["rows"].long()
    return {name: _float8(s["cache_" + name].index_select(0, rows)).double()
            * s[name + "_scales"].index_select(0, rows).double().unsqueeze(-1) for name in ("k", "v")}


def _exact_attention(case, s):
    """One request, head and block of queries at a time."""
    h, kv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    out, at = torch.zeros_like(s["q"], dtype=torch.float64), 0
    for r, (n, length) in enumerate(_lengths(case)):
        pages = s["table"][r, : -(-length // page)].long()
        rows = (pages[:, None] * page + torch.arange(page, device="cuda")[None, :]).reshape(-1)[:length]
        for head in range(h):
            g = head * kv // h
            k, v = s["cache_k"][rows, g], s["cache_v"][rows, g]
            if case["cache"] == "fp8":
                k, v = (_float8(x.contiguous()).double() * c[rows, g].double()[:, None]
                        for x, c in ((k, s["k_scales"]), (v, s["v_scales"])))
            k, v = k.double(), v.double()
            for first in range(0, n, 2048):
                last = min(n, first + 2048)
                q = s["q"][at + first:at + last, head].double()
                score = q @ k.T / math.sqrt(d)
                keep = torch.ones_like(score, dtype=torch.bool).tril(length - n + first)
                out[at + first:at + last, head] = torch.softmax(score.masked_fill(~keep, -math.inf), dim=-1) @ v
        at += n
    return out


_EXACT = {"add_norm": _exact_add_norm, "kv_write": _exact_kv_write, "kv_read": _exact_kv_read,
          "attention": _exact_attention}
