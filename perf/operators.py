"""Performance cases of the operators for sequences that share pages of a paged KV
cache.

`listed()` names the fixed cases and `draw(rng)` gives more of the same ranges.
`prepare(case, seed)` makes on the GPU what a program holds before the call (pools,
block tables, lengths, the groups of sequences that share rows), `run(state)` makes
one pass, `work(case)` says what the pass cannot do without, and `exact(case, seed)`
gives the same outputs in float64.

Where `own` is false `run` computes an operator in its plain form, from elementary
torch operations in 32 bits, rounded once at the end.  Where it is true it calls the
framework.

Kinds:
  attn  attention of S new tokens of every sequence of a batch over a paged cache, in
        which groups of sequences share their first pages (a system prompt, several
        answers to one prompt)
  copy  rows of pages copied to other pages of the same pools: the partial last page
        of a sequence that is forked, whole pages of a pool that is compacted
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

D = 128
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # Two answers to one short question, a few tokens in: the smallest call.
        {"name": "decode_pair", "kind": "attn", "dtype": "bf16", "batch": 2, "hq": 16, "hkv": 8, "page": 256, "seq": 1,
         "groups": 1, "alone": 0, "shared": 2, "own_lo": 3, "own_hi": 41, "pick": 1},
        # Four answers in f32, as a model loaded without a narrower type runs.
        {"name": "decode_f32", "kind": "attn", "dtype": "f32", "batch": 4, "hq": 16, "hkv": 8, "page": 256, "seq": 1,
         "groups": 1, "alone": 0, "shared": 5, "own_lo": 90, "own_hi": 333, "pick": 2},
        # 32 requests behind one system prompt of 4096 tokens.
        {"name": "decode_system", "kind": "attn", "dtype": "bf16", "batch": 32, "hq": 32, "hkv": 8, "page": 256,
         "seq": 1, "groups": 1, "alone": 0, "shared": 16, "own_lo": 200, "own_hi": 1500, "pick": 3},
        # Five prompts, several answers to each, and requests that share nothing.
        {"name": "decode_groups", "kind": "attn", "dtype": "bf16", "batch": 27, "hq": 28, "hkv": 4, "page": 512,
         "seq": 1, "groups": 5, "alone": 4, "shared": 13, "own_lo": 1, "own_hi": 900, "pick": 4},
        # A long document asked about by 64 requests, a wide model.
        {"name": "decode_document", "kind": "attn", "dtype": "bf16", "batch": 64, "hq": 64, "hkv": 8, "page": 256,
         "seq": 1, "groups": 1, "alone": 0, "shared": 128, "own_lo": 16, "own_hi": 300, "pick": 5},
        # Five drafted tokens of each sequence checked in one pass.
        {"name": "chunk_draft", "kind": "attn", "dtype": "bf16", "batch": 16, "hq": 32, "hkv": 8, "page": 256, "seq": 5,
         "groups": 2, "alone": 1, "shared": 8, "own_lo": 100, "own_hi": 900, "pick": 6},
        # Eight questions of 129 tokens behind one long prompt.
        {"name": "chunk_questions", "kind": "attn", "dtype": "bf16", "batch": 8, "hq": 28, "hkv": 4, "page": 256,
         "seq": 129, "groups": 1, "alone": 0, "shared": 23, "own_lo": 129, "own_hi": 400, "pick": 7},
        # One layer: a sequence forked in three, 77 rows in its last page.
        {"name": "copy_fork", "kind": "copy", "dtype": "bf16", "hkv": 8, "page": 256, "pages": 24, "layers": 1,
         "sources": 1, "pairs": 3, "rows": 77, "pick": 8},
        # Every layer of a 36-layer model: a sequence forked in eight.
        {"name": "copy_fork_layers", "kind": "copy", "dtype": "bf16", "hkv": 8, "page": 256, "pages": 12, "layers": 36,
         "sources": 1, "pairs": 8, "rows": 201, "pick": 9},
        # A fragmented f32 pool compacted.
        {"name": "copy_compact", "kind": "copy", "dtype": "f32", "hkv": 4, "page": 512, "pages": 240, "layers": 1,
         "sources": 97, "pairs": 97, "rows": 512, "pick": 10},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_attn(rng):
    hkv = rng.choice([2, 4, 8])
    seq = 1 if rng.random() < 0.6 else _log(rng, 2, 160)
    page = rng.choice([256, 256, 512])
    batch = _log(rng, 1, 64)
    groups = rng.randint(1, min(6, batch))
    alone = rng.choice([0, 0, rng.randint(0, batch - groups)])
    own_hi = seq + _log(rng, 1, 1600)
    return {"kind": "attn", "dtype": rng.choice(["bf16", "bf16", "bf16", "f32"]), "batch": batch,
            "hq": hkv * rng.choice([1, 2, 4, 7, 8]), "hkv": hkv, "page": page, "seq": seq, "groups": groups,
            "alone": alone, "shared": max(1, _log(rng, 256, 32768) // page),
            "own_lo": rng.randint(seq, own_hi), "own_hi": own_hi, "pick": rng.randrange(1 << 20)}


def _draw_copy(rng):
    pages = _log(rng, 8, 240)
    fork = rng.random() < 0.6
    pairs = _log(rng, 1, min(64, pages // 2)) if fork else _log(rng, 1, pages // 2)
    page = rng.choice([256, 512])
    return {"kind": "copy", "dtype": rng.choice(["bf16", "bf16", "f32"]), "hkv": rng.choice([2, 4, 8]), "page": page,
            "pages": pages, "layers": rng.choice([1, _log(rng, 1, 36)]),
            "sources": rng.randint(1, min(4, pairs)) if fork else pairs, "pairs": pairs,
            "rows": rng.randint(1, page) if fork else page, "pick": rng.randrange(1 << 20)}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / (1e15 if case["dtype"] == "bf16" else 1e14))


def draw(rng):
    """A case of the listed ranges: no dearer than the largest listed one, its pools
    within 2 GiB."""
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw_attn(rng) if rng.random() < 0.7 else _draw_copy(rng)
        e = 2 if case["dtype"] == "bf16" else 4
        pages = case["layers"] * case["pages"] if case["kind"] == "copy" else _attn_layout(case)["pages"]
        if _cost(case) <= most and 2 * pages * case["hkv"] * case["page"] * D * e <= 2 << 30:
            return case


# --------------------------------------------------------------------- layout

def _attn_layout(case):
    """Which sequences share how many pages, and every sequence's length: groups of
    uneven size in a shuffled batch, the first with case["shared"] pages, then
    `alone` sequences that share none."""
    rng = random.Random(case["pick"])
    B, page = case["batch"], case["page"]
    ids = list(range(B))
    rng.shuffle(ids)
    together = ids[:B - case["alone"]]
    n = case["groups"]
    cuts = [0] + sorted(rng.sample(range(1, len(together)), n - 1)) + [len(together)]
    groups = [together[cuts[g]:cuts[g + 1]] for g in range(n)]
    shared = [case["shared"]] + [rng.randint(1, case["shared"]) for _ in range(n - 1)]
    own_rows = [rng.randint(case["own_lo"], case["own_hi"]) for _ in range(B)]
    own_rows[ids[0]] = case["own_hi"]
    rows = [0] * B
    for members, pages in zip(groups, shared):
        for b in members:
            rows[b] = pages * page
    pages = sum(shared) + sum(-(-r // page) for r in own_rows)
    return {"groups": groups, "group_rows": [p * page for p in shared], "rows": rows,
            "lens": [r + o for r, o in zip(rows, own_rows)], "pages": pages}


def _copy_pairs(case):
    """Source pages, `pairs` copies of them spread over other pages, and the rows of
    each copy."""
    rng = random.Random(case["pick"])
    ids = list(range(case["pages"]))
    rng.shuffle(ids)
    src = ids[:case["sources"]]
    dst = ids[case["sources"]:case["sources"] + case["pairs"]]
    rows = [case["rows"] if i == 0 or case["rows"] == case["page"] else rng.randint(1, case["rows"])
            for i in range(case["sources"])]
    return [src[i % len(src)] for i in range(case["pairs"])], dst, [rows[i % len(src)] for i in range(case["pairs"])]


# --------------------------------------------------------------------- inputs

def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _ints(a):
    return torch.as_tensor(np.asarray(a, np.int32), device=_dev())


def _attn_inputs(case, seed):
    """Normed queries and keys (unit variance, the queries' peaks raised), values, and
    pools whose rows past a sequence's end hold what an earlier owner left."""
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    lay = _attn_layout(case)
    B, page = case["batch"], case["page"]
    order = np.random.default_rng(seed).permutation(lay["pages"] + 2).astype(np.int32)
    width = max(-(-n // page) for n in lay["lens"]) + 1
    table = np.full((B, width), -1, np.int32)
    at = 0
    for members, rows in zip(lay["groups"], lay["group_rows"]):
        n = rows // page
        table[members, :n] = order[at:at + n]
        at += n
    for b in range(B):
        first, last = lay["rows"][b] // page, -(-lay["lens"][b] // page)
        table[b, first:last] = order[at:at + last - first]
        at += last - first
    shape = (lay["pages"] + 2, case["hkv"], page, D)
    k = torch.randn(shape, generator=gen, dtype=dtype, device=_dev())
    v = torch.randn(shape, generator=gen, dtype=dtype, device=_dev())
    q = torch.randn((B, case["hq"], case["seq"], D), generator=gen, dtype=dtype, device=_dev()).mul_(1.5)
    return {"q": q, "k": k, "v": v, "table": table, "lens": lay["lens"], "groups": lay["groups"],
            "group_rows": lay["group_rows"]}


def _copy_inputs(case, seed):
    """The K and V pools of every layer, in one allocation."""
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    shape = (case["pages"], case["hkv"], case["page"], D)
    cache = torch.randn((2 * case["layers"],) + shape, generator=gen, dtype=dtype, device=_dev())
    src, dst, rows = _copy_pairs(case)
    return {"cache": cache, "src": src, "dst": dst, "rows": rows}


def prepare(case, seed):
    if case["kind"] == "copy":
        s = _copy_inputs(case, seed)
        return {"kind": "copy", "pools": list(s["cache"].unbind(0)), **s}
    s = _attn_inputs(case, seed)
    if case["seq"] == 1:
        s["q"] = s["q"].view(case["batch"], case["hq"], D)
    s.update(kind="attn", table=_ints(s["table"]), kv_len=_ints(s["lens"]), max_kv=max(s["lens"]))
    if own:
        from crane_amd import ops
        s["shared"] = ops.prefix_groups(s["groups"], s["group_rows"], case["batch"])
    return s


# ------------------------------------------------------------------ the passes

def _plain_attn(s):
    """Every sequence by itself: its pages gathered, the scores of all its queries, a
    softmax over the rows each may see, and the product with the values."""
    q = s["q"] if s["q"].dim() == 4 else s["q"].unsqueeze(2)
    B, hq, S, _ = q.shape
    hkv, page = s["k"].shape[1], s["k"].shape[2]
    group = hq // hkv
    out = torch.empty((B, S, hq * D), dtype=q.dtype, device=q.device)
    for b, n in enumerate(s["lens"]):
        pages = s["table"][b, :-(-n // page)].long()
        k = s["k"][pages].transpose(0, 1).reshape(hkv, -1, D)[:, :n].float()
        v = s["v"][pages].transpose(0, 1).reshape(hkv, -1, D)[:, :n].float()
        scores = torch.matmul(q[b].float().view(hkv, group * S, D), k.transpose(1, 2).contiguous()) * D ** -0.5
        limit = torch.arange(n - S + 1, n + 1, device=q.device).repeat(group)
        hidden = torch.arange(n, device=q.device)[None, :] >= limit[:, None]
        scores.masked_fill_(hidden, -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[b] = o.view(hq, S, D).transpose(0, 1).reshape(S, hq * D).to(q.dtype)
    return out


def _plain_copy(s):
    for i, j, n in zip(s["src"], s["dst"], s["rows"]):
        for pool in s["pools"]:
            pool[j, :, :n] = pool[i, :, :n]
    return s["cache"]


def run(s):
    if not own:
        return _plain_attn(s) if s["kind"] == "attn" else _plain_copy(s)
    from crane_amd import ops
    if s["kind"] == "attn":
        return ops.attention_shared_paged(s["q"], s["k"], s["v"], s["table"], s["kv_len"], s["max_kv"], s["shared"])
    ops.copy_pages(s["pools"], s["src"], s["dst"], s["rows"])
    return s["cache"]


# ------------------------------------------------------------- work and answers

def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "copy":
        src, _, rows = _copy_pairs(case)
        moved = sum(dict(zip(src, rows)).values()) + sum(rows)
        return {"bytes": 2 * case["layers"] * case["hkv"] * D * e * moved, "flops": 0}
    lay = _attn_layout(case)
    S = case["seq"]
    cached = sum(lay["group_rows"]) + sum(n - r for n, r in zip(lay["lens"], lay["rows"]))
    seen = sum(S * n - S * (S - 1) // 2 for n in lay["lens"])
    return {"bytes": e * D * (2 * case["batch"] * case["hq"] * S + 2 * case["hkv"] * cached),
            "flops": 4 * D * case["hq"] * seen}


def exact(case, seed):
    if case["kind"] == "copy":
        c = _copy_inputs(case, seed)
        dst, src, rows = _ints(c["dst"]).long(), _ints(c["src"]).long(), _ints(c["rows"])
        taken = (torch.arange(case["page"], device=_dev())[None, :] < rows[:, None])[None, :, None, :, None]
        wide = c["cache"].double()
        wide.index_copy_(1, dst, torch.where(taken, wide[:, src], wide[:, dst]))
        return wide
    s = _attn_inputs(case, seed)
    S, hq, hkv, page = case["seq"], case["hq"], case["hkv"], case["page"]
    answers = []
    for b, n in enumerate(s["lens"]):
        rows = torch.arange(n, device=_dev())
        at = _ints(s["table"][b]).long()[rows // page]
        heads = []
        for h in range(hkv):
            k, v = s["k"][at, h, rows % page].double(), s["v"][at, h, rows % page].double()
            x = s["q"][b, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            logits = torch.mm(x.reshape(-1, D), k.t()).view(-1, S, n) / math.sqrt(D)
            seen = rows[None, :] <= torch.arange(n - S, n, device=_dev())[:, None]
            logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
            weights = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
            heads.append(torch.mm(weights.view(-1, n), v).view(-1, S, D))
        answers.append(torch.cat(heads).permute(1, 0, 2).reshape(S, hq * D))
    return torch.stack(answers)
