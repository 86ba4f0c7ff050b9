"""Attention over shared pages (include/crane_shared.h) at random sizes against the
definition in 64 bits, with the element-wise bounds of test_shared: batches of groups whose
members end anywhere, page sizes, wide page tables, loose and tight host bounds, causal
and not, a workspace full of NaN, an output that has to be written whole, pool rows that no
query may see NaN.  Page copies captured into a graph."""
import math

import numpy as np
import pytest

import cases
import test_shared as ts

D = 128


def draw(seed):
    """Sizes of a call: about 2^21 (query row, key) pairs at most per kv head and group."""
    r = cases.rng(4000 + seed)
    log = lambda lo, hi: int(round(math.exp(r.uniform(math.log(lo), math.log(hi)))))
    Hkv = int(r.choice([1, 2, 3, 8]))
    G = int(r.choice([1, 2, 3, 5, 7, 8, 12]))
    S = 1 if r.random() < 0.5 else log(2, 600)
    P = int(r.choice([256, 512, 768]))
    B = min(log(1, 48), max(1, 24000 // (S * G)))
    n_groups = int(r.integers(0, min(3, B) + 1))
    pages = [max(1, log(256, 9000) // P) for _ in range(n_groups)]
    free = [int(x) for x in r.permutation(B)]
    groups = []
    for g in range(n_groups):                      # one or more of what is left, some in no group
        n = int(r.integers(1, max(2, len(free) - (n_groups - g - 1) + 1)))
        groups.append(free[:n])
        free = free[n:]
    rows = [p * P for p in pages]
    lens = [0] * B
    for b in range(B):
        shared = next((rows[g] for g in range(n_groups) if b in groups[g]), 0)
        lens[b] = shared + int(r.integers(0, log(1, 1500) + 1))
        if r.random() < 0.08:
            lens[b] = int(r.integers(0, lens[b] + 1))  # ends inside the shared rows, or has none
    return dict(lens=lens, groups=groups, rows=rows, P=P, Hq=Hkv * G, Hkv=Hkv, S=S, causal=bool(r.random() < 0.8),
                loose=int(r.choice([0, 0, 1, 5000])), tight=bool(r.random() < 0.5), wide=int(r.choice([0, 0, 70])))


def definition(q, k, v, table, lens, P, causal, gpu):
    """(out, sum of w |v|, largest sum |q k| scale) in float64 on the GPU, from host arrays."""
    import torch
    B, Hq, S, _ = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    scale = D ** -0.5
    out = torch.zeros((B, S, Hkv, G, D), dtype=torch.float64, device=gpu)
    mag = torch.zeros_like(out)
    most = 0.0
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(gpu).double()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        kb, vb = (t(ts.rows_of(x, table, b, n, P)) for x in (k, v))
        qb = t(q[b]).view(Hkv, G, S, D)
        limit = torch.arange(n - S + 1, n + 1, device=gpu) if causal else torch.full((S,), n, device=gpu)
        seen = torch.arange(n, device=gpu)[None, :] < limit[:, None]
        some = (limit > 0)[:, None]
        for h in range(Hkv):
            kt = kb[h].t().contiguous()
            for g in range(G):
                sc = torch.mm(qb[h, g], kt) * scale
                most = max(most, float(torch.mm(qb[h, g].abs(), kt.abs()).max()) * scale)
                sc = torch.where(seen, sc, torch.full_like(sc, -math.inf))
                w = torch.where(some, torch.softmax(torch.where(some, sc, torch.zeros_like(sc)), -1),
                                torch.zeros_like(sc))
                out[b, :, h, g] = torch.mm(w, vb[h])
                mag[b, :, h, g] = torch.mm(w, vb[h].abs())
    flat = lambda x: x.view(B, S, -1).cpu().numpy()
    return flat(out), flat(mag), most


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("seed", range(30))
def test_random_calls(gpu, seed, dtype):
    import torch
    from crane_amd import _lib, ops
    c = draw(seed)
    lens, groups, rows, P, Hq, Hkv, S = (c[x] for x in ("lens", "groups", "rows", "P", "Hq", "Hkv", "S"))
    B = len(lens)
    print(f"random {seed} {dtype} B={B} S={S} {Hq}/{Hkv} P={P} lens={lens[:8]} groups={groups[:2]} rows={rows} {c}",
          flush=True)
    full = list(lens)                              # members name every shared page, also past their own end
    for members, n in zip(groups, rows):
        for b in members:
            full[b] = max(full[b], n)
    table, total = ts.layout(4100 + seed, full, groups, rows, P)
    k, v = (cases.cast(x, dtype) for x in ts.pools(4200 + seed, total, Hkv, P, table, full, False))
    table = np.concatenate([table, np.full((B, c["wide"]), -1, np.int32)], 1)
    q = cases.cast(cases.normal(cases.rng(4300 + seed), (B, Hq, S, D)) * np.float32(1.5), dtype)
    shared = [0] * B
    for members, n in zip(groups, rows):
        for b in members:
            shared[b] = n
    max_kv = min(max(full + [1]) + c["loose"], table.shape[1] * P)
    own = max(max(n - s for n, s in zip(lens, shared)), 0) if c["tight"] else max(max_kv - min(shared), 0)
    mean = sum(max(n - s, 0) for n, s in zip(lens, shared)) // B if c["tight"] else 6 * (max_kv - max(shared)) // 10
    g = ops.prefix_groups(groups, rows, B, gpu)
    t = [ts.tens(q, dtype, gpu), ts.tens(k, dtype, gpu), ts.tens(v, dtype, gpu), ts.ints(table, gpu),
         ts.ints(lens, gpu)]
    L, dt = _lib.lib(), int(dtype == "bf16")
    need = L.crane_hip_attn_shared_workspace(g.groups_host, g.n_groups, max_kv, own, mean, B, S, Hq, Hkv, D, dt)
    ws = torch.full((max(need // 4, 4),), math.nan, dtype=torch.float32, device=gpu)
    got = torch.full((B, S, Hq * D), math.nan, dtype=t[0].dtype, device=gpu)
    rc = L.crane_hip_attn_shared_paged(
        t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), total, P, t[3].data_ptr(), table.shape[1], t[4].data_ptr(),
        max_kv, g.shared_rows.data_ptr(), g.groups.data_ptr(), g.members.data_ptr(), g.groups_host, g.n_groups, own,
        mean, B, S, Hq, Hkv, D, D ** -0.5, int(c["causal"]), ws.data_ptr(), need, got.data_ptr(), dt,
        torch.cuda.current_stream(gpu).cuda_stream)
    assert rc == _lib.OK
    out, mag, most = definition(q, k, v, table, lens, P, c["causal"], gpu)
    err = np.abs(got.float().cpu().numpy() - out) / ts.bounds(out, mag, most, max(lens + [1]), dtype)
    assert (err <= 1).all(), float(np.nanmax(err))
    if S > 1 or not c["tight"]:                    # and the entry point in Python, with its guesses
        a = ops.attention_shared_paged(t[0] if S > 1 else t[0].view(B, Hq, D), *t[1:], max_kv, g, causal=c["causal"])
        err = np.abs(a.float().cpu().numpy() - out) / ts.bounds(out, mag, most, max(lens + [1]), dtype)
        assert (err <= 1).all(), float(np.nanmax(err))


@pytest.mark.gpu
def test_captured_page_copies(gpu):
    """A captured copy runs on what the pages hold at every replay, with the lists that were
    given when it was captured."""
    import torch
    from crane_amd import ops
    pools = [torch.zeros((9, 3, 256, D), dtype=torch.bfloat16, device=gpu) for _ in range(4)]
    src, dst, rows = [2, 2, 5], [0, 7, 8], [256, 77, 1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages(pools, src, dst, rows)
    src[0], rows[1] = 1, 0
    for step in range(4):
        for p in pools:
            p.copy_(torch.randn(p.shape, device=gpu))
        want = [p.clone() for p in pools]
        for p in want:
            for i, j, n in ((2, 0, 256), (2, 7, 77), (5, 8, 1)):
                p[j, :, :n] = p[i, :, :n]
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(pools, want)), step
