"""Performance cases of the operators of a paged KV cache held in 8 bits.

The cache: K and V pools [n_pages, Hkv, page_rows, 128] of float8_e4m3fn, and for each
a pool of scales [n_pages, Hkv, page_rows / 32] of float8_e8m0fnu, a power of two for 32
rows of a head.  A row's values are its codes times its block's scale.  The scale is the
smallest 2^e with every value within 448 2^e (and no smaller than 2^-100); a block that
rows are added to keeps the larger of its scale and what the new rows need, and rows it
already holds are rounded again to a larger one.

`listed()` names the fixed cases and `draw(rng)` gives more of the same ranges.
`prepare(case, seed)` makes on the GPU what a program holds before the call, `run(state)`
makes one pass, `work(case)` says what the pass cannot do without, and
`exact(case, seed)` gives the same outputs in float64, codes before their rounding.

Where `own` is false `run` computes an operator in its plain form, from elementary torch
operations in 32 bits, rounded once at the end.  Where it is true it calls the framework.

Kinds:
  append  the per-head RMS norm and the rotation of new tokens' q and k, and their k and
          v quantised into the pages at every sequence's length
  attn    attention of the S last tokens of every sequence over its rows of the cache
  read    the rows of every sequence as values, side by side
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
BLOCK = 32         # rows of one scale
TOP = 448.0        # largest code
FLOOR = 27         # smallest scale byte: 2^(27 - 127)
EPS = 1e-6
THETA = 1e6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One token of one conversation: the smallest append.
        {"name": "append_token", "kind": "append", "dtype": "bf16", "batch": 1, "hq": 16, "hkv": 8, "page": 256,
         "seq": 1, "len_lo": 77, "len_hi": 77, "order": "norm_then_rope", "pick": 1},
        # A decode step of 32 conversations.
        {"name": "append_step", "kind": "append", "dtype": "bf16", "batch": 32, "hq": 32, "hkv": 8, "page": 256,
         "seq": 1, "len_lo": 512, "len_hi": 4096, "order": "norm_then_rope", "pick": 2},
        # Chunks of three prompts that begin inside a block, in f32, the norm behind the rotation.
        {"name": "append_chunk_f32", "kind": "append", "dtype": "f32", "batch": 3, "hq": 16, "hkv": 8, "page": 512,
         "seq": 77, "len_lo": 1, "len_hi": 300, "order": "rope_then_norm", "pick": 3},
        # Eight prompts of 4096 tokens into an empty cache.
        {"name": "append_prompts", "kind": "append", "dtype": "bf16", "batch": 8, "hq": 28, "hkv": 4, "page": 256,
         "seq": 4096, "len_lo": 0, "len_hi": 0, "order": "rope_only", "pick": 4},
        # A question of 300 tokens being answered: the smallest attention.
        {"name": "decode_one", "kind": "attn", "dtype": "bf16", "batch": 1, "hq": 16, "hkv": 8, "page": 256, "seq": 1,
         "idle": 0, "len_lo": 301, "len_hi": 301, "pick": 5},
        # 32 conversations of 512 to 4096 tokens.
        {"name": "decode_ragged", "kind": "attn", "dtype": "bf16", "batch": 32, "hq": 32, "hkv": 8, "page": 256,
         "seq": 1, "idle": 0, "len_lo": 512, "len_hi": 4096, "pick": 6},
        # Eight long documents, a wide model.
        {"name": "decode_long", "kind": "attn", "dtype": "bf16", "batch": 8, "hq": 64, "hkv": 8, "page": 256, "seq": 1,
         "idle": 0, "len_lo": 32768, "len_hi": 32768, "pick": 7},
        # A model loaded in f32; two of the batch's places are not taken.
        {"name": "decode_f32", "kind": "attn", "dtype": "f32", "batch": 6, "hq": 28, "hkv": 4, "page": 512, "seq": 1,
         "idle": 2, "len_lo": 700, "len_hi": 2900, "pick": 8},
        # Five drafted tokens of each conversation checked in one pass.
        {"name": "chunk_draft", "kind": "attn", "dtype": "bf16", "batch": 16, "hq": 32, "hkv": 8, "page": 256, "seq": 5,
         "idle": 0, "len_lo": 600, "len_hi": 5000, "pick": 9},
        # The last 1024 tokens of four prompts of up to 9000.
        {"name": "chunk_prompts", "kind": "attn", "dtype": "bf16", "batch": 4, "hq": 28, "hkv": 4, "page": 256,
         "seq": 1024, "idle": 0, "len_lo": 5000, "len_hi": 9000, "pick": 10},
        # One short conversation taken out of the cache.
        {"name": "read_one", "kind": "read", "dtype": "f32", "batch": 1, "hkv": 8, "page": 256, "len_lo": 333,
         "len_hi": 333, "pick": 11},
        # 16 conversations taken out of the cache.
        {"name": "read_batch", "kind": "read", "dtype": "bf16", "batch": 16, "hkv": 8, "page": 256, "len_lo": 512,
         "len_hi": 4096, "pick": 12},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    kind = rng.choice(["append", "append", "attn", "attn", "attn", "read"])
    hkv = rng.choice([2, 4, 8])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f32"]), "batch": _log(rng, 1, 64), "hkv": hkv,
            "page": rng.choice([256, 256, 512]), "pick": rng.randrange(1 << 20)}
    if kind == "read":
        case["len_hi"] = _log(rng, 1, 8192)
    else:
        case["hq"] = hkv * rng.choice([1, 2, 4, 5, 7, 8])
        case["seq"] = 1 if rng.random() < 0.5 else _log(rng, 2, 4096 if kind == "append" else 1500)
    if kind == "append":
        case["order"] = rng.choice(["norm_then_rope", "rope_then_norm", "rope_only"])
        case["len_hi"] = _log(rng, 1, 6000) - 1
    elif kind == "attn":
        case["idle"] = rng.choice([0, 0, rng.randint(0, case["batch"] - 1)])
        case["len_hi"] = case["seq"] + _log(rng, 1, 33000) - 1
    case["len_lo"] = rng.randint(case.get("seq", 0) if kind == "attn" else 0, case["len_hi"])
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / (1e15 if case["dtype"] == "bf16" else 2e14))


def draw(rng):
    """A case of the listed ranges: no dearer than the dearest listed one of its kind, its
    rows within 4 GiB as float32."""
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        case = _draw_one(rng)
        wide = case["batch"] * (case["len_hi"] + case.get("seq", 0)) * case["hkv"] * D * 4
        scores = 4 * case["batch"] * case["hq"] * case["seq"] * case["len_hi"] if case["kind"] == "attn" else 0
        if _cost(case) <= most[case["kind"]] and wide <= 4 << 30 and scores <= 8 << 30:
            return case


# --------------------------------------------------------------------- layout

def _lengths(case):
    """Rows of every sequence before the call (append) or with its new rows (attn); the
    first sequence has the most, idle ones have none."""
    rng = random.Random(case["pick"])
    lens = [case["len_hi"]] + [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(case["batch"] - 1)]
    for b in rng.sample(range(1, case["batch"]), case.get("idle", 0)) if case.get("idle") else []:
        lens[b] = 0
    return lens


def _pages_of(case):
    """Pages every sequence holds; an append's are reserved a block ahead of its rows."""
    ahead = case["seq"] + 2 * BLOCK if case["kind"] == "append" else 0
    return [-(-(n + ahead) // case["page"]) for n in _lengths(case)]


# --------------------------------------------------------------------- inputs

def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device=_dev())


def _pow2(byte):
    """2^(byte - 127) of scale bytes (0 for bytes below 1)."""
    return (byte.clamp_min(0).to(torch.int32) << 23).view(torch.float32)


def _scale_byte(amax):
    """The byte of the smallest scale that holds amax: amax = m 2^x, 448 = 0.875 2^9."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, (x - 9 + (m > 0.875) + 127).to(torch.int32), FLOOR).clamp_min(FLOOR)


def _pool(gen, pages, case, spread):
    """A pool of pages that were written before, and its scales."""
    x = torch.randn((pages, case["hkv"], case["page"] // BLOCK, BLOCK, D), generator=gen, device=_dev())
    x *= torch.exp(spread * torch.randn((case["hkv"], 1, 1, D), generator=gen, device=_dev()))
    byte = _scale_byte(x.abs().amax((3, 4)))
    x *= _pow2(254 - byte)[..., None, None]
    return x.to(torch.float8_e4m3fn).view(pages, case["hkv"], case["page"], D), \
        byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _cache(case, seed):
    """Pools (the keys' dims differ in size, as a norm's weights make them) and a block
    table of pages in any order, -1 past a sequence's."""
    gen = torch.Generator(device=_dev()).manual_seed(seed)
    each = _pages_of(case)
    ids = list(range(sum(each) + 1))
    random.Random(seed).shuffle(ids)
    width, table = max(max(each), 1), []
    for n in each:
        table.append(ids[:n] + [-1] * (width - n))
        ids = ids[n:]
    k, k_scale = _pool(gen, sum(each) + 1, case, 0.4)
    v, v_scale = _pool(gen, sum(each) + 1, case, 0.1)
    return gen, {"kind": case["kind"], "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "table": _ints(table),
                 "lens": _ints(_lengths(case)), "max_len": max(_lengths(case)), "dtype": DTYPES[case["dtype"]]}


def prepare(case, seed):
    gen, s = _cache(case, seed)
    B, dtype = case["batch"], DTYPES[case["dtype"]]
    if case["kind"] == "attn":
        shape = (B, case["hq"], D) if case["seq"] == 1 else (B, case["hq"], case["seq"], D)
        s["q"] = (1.5 * torch.randn(shape, generator=gen, device=_dev())).to(dtype)
    if case["kind"] == "append":
        H = case["hq"] + 2 * case["hkv"]
        x = torch.randn((B, case["seq"], H, D), generator=gen, device=_dev())
        x *= torch.exp(0.4 * torch.randn((H, D), generator=gen, device=_dev()))
        freq = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=_dev()) / D)
        angle = torch.arange(s["max_len"] + case["seq"], device=_dev())[:, None] * freq
        s.update(qkv=x.view(B, case["seq"], H * D).to(dtype), cos=angle.cos().to(dtype), sin=angle.sin().to(dtype),
                 hq=case["hq"], order=case["order"], q_w=None, k_w=None)
        if case["order"] != "rope_only":
            s["q_w"], s["k_w"] = ((1 + 0.3 * torch.randn(D, generator=gen, device=_dev())).to(dtype) for _ in "qk")
    return s


# ------------------------------------------------------------------ the passes

def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rope(x, cos, sin):
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _turn(x, w, cos, sin, order):
    if order == "norm_then_rope":
        x = _norm(x, w)
    x = _rope(x, cos, sin)
    return _norm(x, w) if order == "rope_then_norm" else x


def _plain_store(s, pool, scales, x):
    """Rows x [B, S, Hkv, D] into the blocks of 32 they fall in."""
    B, S, hkv, _ = x.shape
    page_rows, codes, bytes_ = pool.shape[2], pool.view(torch.uint8), scales.view(torch.uint8)
    start, dev = s["lens"].long(), x.device
    n = (S + 2 * BLOCK - 2) // BLOCK
    at = torch.arange(n * BLOCK, device=dev) - (start % BLOCK)[:, None]  # a block row's new row; < 0: an older row
    row = start[:, None] + at
    page = s["table"].long().gather(1, row // page_rows)
    old, new = at < 0, (at >= 0) & (at < S)
    x = torch.where(new[..., None, None], x[torch.arange(B, device=dev)[:, None], at.clamp(0, S - 1)], 0.0)
    need = _scale_byte(x.view(B, n, BLOCK, hkv, D).abs().amax((2, 4)))
    block = (page[:, ::BLOCK], slice(None), row[:, ::BLOCK] % page_rows // BLOCK)
    had = bytes_[block].to(torch.int32)
    byte = torch.where(old[:, ::BLOCK, None], torch.maximum(had, need), need)
    mine = byte.repeat_interleave(BLOCK, 1)[..., None]
    was = codes[page, :, row % page_rows]
    held = was.view(torch.float8_e4m3fn).float() * _pow2(127 + had.repeat_interleave(BLOCK, 1)[..., None] - mine)
    code = torch.where(new[..., None, None], x * _pow2(254 - mine), held).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[page, :, row % page_rows] = torch.where((old | new)[..., None, None], code, was)
    touched = new.view(B, n, BLOCK).any(2)[..., None]
    bytes_[block] = torch.where(touched, byte, had).to(torch.uint8)


def _plain_append(s):
    B, S, _ = s["qkv"].shape
    hkv = s["k"].shape[1]
    q, k, v = s["qkv"].float().view(B, S, -1, D).split((s["hq"], hkv, hkv), 2)
    at = s["lens"].long()[:, None] + torch.arange(S, device=q.device)
    cos, sin = s["cos"][at].float()[:, :, None], s["sin"][at].float()[:, :, None]
    q = _turn(q, s["q_w"], cos, sin, s["order"]).transpose(1, 2).to(s["dtype"]).contiguous()
    _plain_store(s, s["k"], s["k_scale"], _turn(k, s["k_w"], cos, sin, s["order"]))
    _plain_store(s, s["v"], s["v_scale"], v)
    return q


def _plain_rows(s, pool, scales):
    """[B, Hkv, longest, D] float32."""
    rows = torch.arange(s["max_len"], device=pool.device)
    page = s["table"].long()[:, rows // pool.shape[2]].clamp_min(0)
    at = rows % pool.shape[2]
    x = pool.view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn).float()
    return (x * _pow2(scales.view(torch.uint8)[page, :, at // BLOCK])[..., None]).transpose(1, 2).contiguous()


def _plain_attn(s):
    q = s["q"] if s["q"].dim() == 4 else s["q"].unsqueeze(2)
    B, hq, S, _ = q.shape
    k, v = _plain_rows(s, s["k"], s["k_scale"]), _plain_rows(s, s["v"], s["v_scale"])
    hkv, n = k.shape[1], k.shape[2]
    scores = torch.matmul(q.float().view(B, hkv, -1, D), k.transpose(2, 3).contiguous()).view(B, hkv, -1, S, n)
    limit = s["lens"][:, None] - S + 1 + torch.arange(S, device=q.device)
    hidden = torch.arange(n, device=q.device) >= limit[..., None]
    scores = scores.mul_(D ** -0.5).masked_fill_(hidden[:, None, None], -math.inf).view(B, hkv, -1, n)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, torch.matmul(p, v) / total, 0.0)
    return out.view(B, hq, S, D).transpose(1, 2).reshape(B, S, hq * D).to(q.dtype)


def _plain_read(s):
    past = torch.arange(s["max_len"], device=s["k"].device) >= s["lens"][:, None]
    return tuple(_plain_rows(s, s[x], s[x + "_scale"]).masked_fill_(past[:, None, :, None], 0.0).to(s["dtype"])
                 for x in "kv")


def run(s):
    pools = s["k"], s["v"], s["k_scale"], s["v_scale"]
    if s["kind"] == "append":
        if own:
            from crane_amd import ops
            q = ops.qk_norm_rope_append_paged_f8(s["qkv"], s["cos"], s["sin"], s["lens"], pools, s["table"], s["lens"],
                                                 s["hq"], s["q_w"], s["k_w"], EPS, s["order"])
        else:
            q = _plain_append(s)
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if s["kind"] == "attn":
        if own:
            from crane_amd import ops
            return ops.attention_paged_f8(s["q"], pools, s["table"], s["lens"], s["max_len"])
        return _plain_attn(s)
    if own:
        from crane_amd import ops
        k, v = ops.read_paged_f8(pools, s["table"], s["lens"], s["max_len"], s["dtype"])
    else:
        k, v = _plain_read(s)
    return {"k": k, "v": v}


# ------------------------------------------------------------- work and answers

def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    lens = _lengths(case)
    row = 2 * case["hkv"] * (D + 1 / BLOCK)  # bytes of a row of the cache
    if case["kind"] == "read":
        return {"bytes": sum(lens) * row + 2 * e * D * case["hkv"] * case["batch"] * max(lens),
                "flops": 2 * D * case["hkv"] * sum(lens)}
    S, hq = case["seq"], case["hq"]
    tokens = case["batch"] * S
    if case["kind"] == "append":
        heads = hq + 2 * case["hkv"]
        return {"bytes": tokens * (e * D * (heads + hq) + row), "flops": 8 * tokens * heads * D}
    seen = sum(max(0, S * n - S * (S - 1) // 2) for n in lens if n)
    return {"bytes": 2 * e * D * hq * tokens + sum(lens) * row, "flops": 4 * D * hq * seen}


def _values(s, b, n, h, pool, scales):
    """Head h's first n rows of sequence b in float64."""
    rows = torch.arange(n, device=_dev())
    page, at = s["table"][b].long()[rows // pool.shape[2]], rows % pool.shape[2]
    exponent = scales.view(torch.uint8)[page, h, at // BLOCK].double() - 127
    return pool.view(torch.uint8)[page, h, at].view(torch.float8_e4m3fn).double() * torch.exp2(exponent)[:, None]


def _exact_append(s):
    B, S, _ = s["qkv"].shape
    hq, hkv, P = s["hq"], s["k"].shape[1], s["k"].shape[2]
    x = s["qkv"].double().view(B, S, -1, D)

    def turn(x, w, c, t):
        def unit(y):
            return y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS) * w.double()
        if s["order"] == "norm_then_rope":
            x = unit(x)
        x = torch.stack((x[..., :64] * c - x[..., 64:] * t, x[..., 64:] * c + x[..., :64] * t), -2).flatten(-2)
        return unit(x) if s["order"] == "rope_then_norm" else x

    q = torch.empty((B, hq, S, D), dtype=torch.float64, device=_dev())
    out = {"q": q, "k": s["k"].double(), "v": s["v"].double(), "k_scale": s["k_scale"].double(),
           "v_scale": s["v_scale"].double()}
    lens = s["lens"].tolist()
    for b in range(B):
        c, t = (s[x][lens[b]:lens[b] + S].double()[:, None] for x in ("cos", "sin"))
        q[b] = turn(x[b, :, :hq], s["q_w"], c, t).transpose(0, 1)
        new = {"k": turn(x[b, :, hq:hq + hkv], s["k_w"], c, t), "v": x[b, :, hq + hkv:]}
        first, end = lens[b] // BLOCK * BLOCK, lens[b] + S
        starts = torch.arange(first, end, BLOCK, device=_dev())
        page, block = s["table"][b].long()[starts // P], starts % P // BLOCK
        held = lens[b] - first
        rows = torch.arange(first, end, device=_dev())
        pages, at = s["table"][b].long()[rows // P], rows % P
        for name in "kv":
            was = out[name][pages[:held], :, at[:held]] * out[name + "_scale"][page[:1], :, block[:1]][..., None]
            fresh = torch.cat((torch.zeros_like(was), new[name], new[name].new_zeros((-end % BLOCK, hkv, D))))
            most = fresh.view(-1, BLOCK, hkv, D).abs().amax((1, 3))
            exponent = torch.ceil(torch.log2((most / TOP).clamp_min(2.0 ** (FLOOR - 127))))
            if held:
                had = torch.log2(out[name + "_scale"][page[0], :, block[0]])
                exponent[0] = torch.maximum(exponent[0], had.round())
            scale = torch.exp2(exponent)
            values = torch.cat((was, new[name])) / scale.repeat_interleave(BLOCK, 0)[:end - first, :, None]
            out[name][pages, :, at] = values
            out[name + "_scale"][page, :, block] = scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    hkv, lens = case["hkv"], s["lens"].tolist()
    if case["kind"] == "read":
        out = {x: torch.zeros((case["batch"], hkv, max(lens), D), dtype=torch.float64, device=_dev()) for x in "kv"}
        for b, n in enumerate(lens):
            for h in range(hkv):
                for x in "kv":
                    out[x][b, h, :n] = _values(s, b, n, h, s[x], s[x + "_scale"])
        return out
    S, hq = case["seq"], case["hq"]
    q = s["q"].double().view(case["batch"], hkv, hq // hkv, S, D)
    out = torch.zeros((case["batch"], hkv, hq // hkv, S, D), dtype=torch.float64, device=_dev())
    for b, n in enumerate(lens):
        seen = torch.arange(n, device=_dev()) <= torch.arange(n - S, n, device=_dev())[:, None]
        for h in range(hkv if n else 0):
            k, v = (_values(s, b, n, h, s[x], s[x + "_scale"]) for x in "kv")
            for g in range(hq // hkv):
                logits = torch.mm(q[b, h, g], k.t()) / math.sqrt(D)
                logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
                weights = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
                out[b, h, g] = torch.mm(weights, v)
    return out.view(case["batch"], hq, S, D).transpose(1, 2).reshape(case["batch"], S, hq * D)
