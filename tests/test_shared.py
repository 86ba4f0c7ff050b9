"""Attention over pages that sequences share and page copies (include/crane_shared.h).

Crane has no counterpart of either, so the reference is the definition in 64 bits:
every sequence by itself over its own rows.  Two kinds of inputs:

  exact  q = 0 and V of -1 and 1: every weight is 1, all sums are whole numbers below
         2^24, and the result is T(f32(sum) / f32(count)) to the last bit.  A key
         lost, taken twice or taken past a row's limit changes it (by at least
         1 / count, against values of about count^-1/2 whose rounding is 2^-8 of
         that).
  close  normal q, K, V with element-wise bounds (bounds() derives them).

Pool rows that no query may see hold NaN."""
import ctypes
import math

import numpy as np
import pytest

import cases

D = 128
U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of f32 and bf16, relative


# ------------------------------------------------------------------ inputs

def layout(seed, lens, groups, rows, P, spare=2):
    """Tables on shuffled pages: a group's members name the same pages for its first
    rows[g] rows (up to the page that rows[g] ends in, when they have rows past it in
    other pages only; else the caller passes whole pages or identical sequences)."""
    r = cases.rng(seed)
    B = len(lens)
    width = max(1, max(math.ceil(n / P) for n in lens)) + 1
    total = sum(math.ceil(n / P) for n in lens) + sum(math.ceil(x / P) for x in rows) + spare
    perm = r.permutation(total).astype(np.int32)
    table = np.full((B, width), -1, np.int32)
    at = 0
    for members, n in zip(groups, rows):
        pages = math.ceil(n / P)
        for b in members:
            table[b, :pages] = perm[at:at + pages]
        at += pages
    for b, n in enumerate(lens):
        for i in range(math.ceil(n / P)):
            if table[b, i] < 0:
                table[b, i] = perm[at]
                at += 1
    for b, n in enumerate(lens):  # entries past a sequence's rows are of no page
        table[b, math.ceil(n / P):] = -7
    return table, total


def pools(seed, total, Hkv, P, table, lens, exact):
    """K and V pools: NaN but for the rows some sequence holds."""
    r = cases.rng(seed)
    k = np.full((total, Hkv, P, D), np.nan, np.float32)
    v = np.full_like(k, np.nan)
    for b, n in enumerate(lens):
        for i in range(math.ceil(n / P)):
            m = min(P, n - i * P)
            page = table[b, i]
            fresh = np.isnan(k[page, 0, :m, 0])
            if exact:
                kk, vv = cases.normal(r, (Hkv, m, D)), r.integers(0, 2, (Hkv, m, D)).astype(np.float32) * 2 - 1
            else:
                kk, vv = cases.normal(r, (Hkv, m, D)), cases.normal(r, (Hkv, m, D))
            k[page][:, :m][:, fresh] = kk[:, fresh]
            v[page][:, :m][:, fresh] = vv[:, fresh]
    return k, v


def rows_of(pool, table, b, n, P):
    return np.concatenate([pool[table[b, i], :, :min(P, n - i * P)] for i in range(math.ceil(n / P))], 1) \
        if n else pool[0, :, :0]


def reference(q, k, v, table, lens, P, scale, causal):
    """(out [B, S, Hq D], sum of w |v| of the same shape, largest sum |q k| scale) in
    float64."""
    B, Hq, S, _ = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    out = np.zeros((B, S, Hq, D))
    mag = np.zeros_like(out)
    most = 0.0
    for b, n in enumerate(lens):
        kb, vb = (rows_of(x, table, b, n, P).astype(np.float64) for x in (k, v))
        for h in range(Hq):
            for s in range(S):
                L = n - S + 1 + s if causal else n
                if L <= 0:
                    continue
                x, kk, vv = q[b, h, s].astype(np.float64), kb[h // G, :L], vb[h // G, :L]
                sc = kk @ x * scale
                w = np.exp(sc - sc.max())
                w /= w.sum()
                out[b, s, h] = w @ vv
                mag[b, s, h] = w @ np.abs(vv)
                most = max(most, float((np.abs(kk) @ np.abs(x)).max()) * scale)
    return out.reshape(B, S, -1), mag.reshape(B, S, -1), most


def bounds(out, mag, most, n, dtype):
    """|kernel - exact| per element.  With weights w (1 + d), |d| <= e, over their own
    sum: |o' - o| <= e / (1 - e) (sum w |v| + |o|).  e: bf16 rounds every weight once,
    2^-8.  f32 arithmetic, for both types: a 128-term product errs by at most 128 half
    steps of sum |q k| scale, its scaling and the reference's subtraction by 4 more
    (the exponent's size is at most twice that sum, log2 e < 2), and an exponent's
    error is the weight's relative one; exp2 2 steps; the sums' order n half steps
    each, the joins' scalings 16.  The result is rounded once."""
    e = U32 * (2 * 132 * most + 4 + 2 * n + 16) + (U16 if dtype == "bf16" else 0)
    last = U16 if dtype == "bf16" else U32
    return e / (1 - e) * (mag + np.abs(out)) * (1 + last) + last * np.abs(out) + 1e-30


def tens(x, dtype, dev):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t.to(torch.bfloat16) if dtype == "bf16" else t).to(dev)


def ints(x, dev):
    import torch
    return torch.as_tensor(np.asarray(x, np.int32), device=dev)


def call(gpu, q, k, v, table, lens, groups, rows, dtype, **kw):
    from crane_amd import ops
    B = len(lens)
    g = ops.prefix_groups(groups, rows, B, gpu)
    qq = tens(q, dtype, gpu)
    if kw.pop("flat", q.shape[2] == 1):
        qq = qq.view(B, q.shape[1], D)
    return ops.attention_shared_paged(qq, tens(k, dtype, gpu), tens(v, dtype, gpu), ints(table, gpu), ints(lens, gpu),
                                      max(max(lens), 1), g, **kw)


def check_exact(gpu, seed, lens, groups, rows, P, Hq, Hkv, S, dtype, causal=True, **kw):
    import torch
    print(f"exact {seed} lens={lens[:6]} groups={len(groups)} rows={rows} P={P} {Hq}/{Hkv} S={S} {dtype} {causal}",
          flush=True)
    table, total = layout(seed, lens, groups, rows, P)
    k, v = pools(seed + 1, total, Hkv, P, table, lens, True)
    q = np.zeros((len(lens), Hq, S, D), np.float32)
    got = call(gpu, q, cases.cast(k, dtype), v, table, lens, groups, rows, dtype, causal=causal, **kw)
    want = np.zeros((len(lens), S, Hkv, Hq // Hkv, D), np.float32)
    for b, n in enumerate(lens):
        total_v = np.cumsum(rows_of(v, table, b, n, P).astype(np.float64), 1)
        for s in range(S):
            L = n - S + 1 + s if causal else n
            if L > 0:
                want[b, s] = (total_v[:, L - 1].astype(np.float32) / np.float32(L))[:, None, :]
    want = torch.from_numpy(want.reshape(len(lens), S, -1)).to(got.dtype)
    assert got.shape == want.shape
    wrong = int((got.cpu() != want).sum())
    assert wrong == 0, wrong


def check_close(gpu, seed, lens, groups, rows, P, Hq, Hkv, S, dtype, causal=True, q_scale=1.5, **kw):
    print(f"close {seed} lens={lens[:6]} groups={len(groups)} rows={rows} P={P} {Hq}/{Hkv} S={S} {dtype} {causal}",
          flush=True)
    table, total = layout(seed, lens, groups, rows, P)
    k, v = pools(seed + 1, total, Hkv, P, table, lens, False)
    q = cases.normal(cases.rng(seed + 2), (len(lens), Hq, S, D)) * np.float32(q_scale)
    q, k, v = (cases.cast(x, dtype) for x in (q, k, v))
    got = call(gpu, q, k, v, table, lens, groups, rows, dtype, causal=causal, **kw).float().cpu().numpy()
    out, mag, most = reference(q, k, v, table, lens, P, D ** -0.5, causal)
    tol = bounds(out, mag, most, max(lens), dtype)
    assert np.isfinite(got).all()
    worst = float((np.abs(got - out) / tol).max())
    assert worst <= 1, worst
    return got


# ------------------------------------------------------------------ refusals (CPU)

BASE = dict(q=16, k=16, v=16, n_pages=64, P=256, table=16, stride=8, kv_len=16, max_kv=1024, shared=16, groups=16, members=16,
            groups_host=[0, 4, 0, 512], n_groups=1, max_own=512, mean_own=100, B=4, S=1, Hq=32, Hkv=8, D=128, scale=0.088, flags=1,
            ws=16, ws_bytes=1 << 40, out=16, dtype=1, stream=None)


def host(groups):
    return None if groups is None else (ctypes.c_int32 * max(len(groups), 1))(*groups)


def shared_call(**kw):
    from crane_amd import _lib
    a = {**BASE, **kw}
    a["groups_host"] = host(a["groups_host"])
    return _lib.lib().crane_hip_attn_shared_paged(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), "E_DTYPE"), (dict(D=64), "E_HEAD_DIM"), (dict(Hq=30), "E_GQA"), (dict(Hkv=0), "E_INVALID"),
    (dict(P=100), "E_INVALID"), (dict(n_pages=0), "E_INVALID"), (dict(table=None), "E_INVALID"),
    (dict(stride=0), "E_INVALID"), (dict(max_kv=8 * 256 + 1), "E_CAPACITY"), (dict(max_kv=0), "E_INVALID"),
    (dict(groups_host=[0, 4, 0, 1025]), "E_CAPACITY"), (dict(max_own=1025), "E_CAPACITY"),
    (dict(max_own=-1), "E_INVALID"), (dict(n_groups=5, groups_host=[0, 0, 0, 0] * 5), "E_INVALID"),
    (dict(n_groups=-1), "E_INVALID"), (dict(groups_host=None), "E_INVALID"),
    (dict(groups_host=[0, 5, 0, 512]), "E_INVALID"), (dict(groups_host=[-1, 2, 0, 512]), "E_INVALID"),
    (dict(groups_host=[0, -1, 0, 512]), "E_INVALID"), (dict(groups_host=[0, 4, 4, 512]), "E_INVALID"),
    (dict(groups_host=[0, 4, -1, 512]), "E_INVALID"), (dict(groups_host=[0, 4, 0, -1]), "E_INVALID"),
    (dict(groups_host=[3, 0x7fffffff, 0, 512]), "E_INVALID"), (dict(groups_host=[0, 4, 0, 0x7fffffff]), "E_INVALID"),
    (dict(flags=2), "E_INVALID"), (dict(flags=3), "E_INVALID"), (dict(scale=0.0), "E_INVALID"),
    (dict(scale=float("nan")), "E_INVALID"), (dict(scale=float("inf")), "E_INVALID"), (dict(q=None), "E_INVALID"),
    (dict(out=None), "E_INVALID"), (dict(kv_len=None), "E_INVALID"), (dict(shared=None), "E_INVALID"),
    (dict(groups=None), "E_INVALID"), (dict(members=None), "E_INVALID"), (dict(groups=8), "E_ALIGN"), (dict(q=8), "E_ALIGN"), (dict(k=24), "E_ALIGN"),
    (dict(v=8), "E_ALIGN"), (dict(out=8), "E_ALIGN"), (dict(ws=None), "E_WORKSPACE"), (dict(ws=8), "E_WORKSPACE"),
    (dict(ws_bytes=100), "E_WORKSPACE"), (dict(B=-1), "E_INVALID"), (dict(S=-1), "E_INVALID"),
    (dict(B=65536), "E_INVALID"), (dict(B=0, n_groups=0), "OK"), (dict(S=0), "OK"),
    (dict(S=1 << 30), "E_INVALID"), (dict(S=1 << 19), "E_INVALID"),    # 2^26 query rows or more
    (dict(P=1 << 28, stride=7, n_pages=1, max_kv=7 << 28, max_own=7 << 28,
          groups_host=[0, 4, 0, 7 << 28]), "E_INVALID"),
])
def test_attention_refusals(kw, code):
    from crane_amd import _lib
    assert shared_call(**kw) == getattr(_lib, code)


def test_workspace_query():
    from crane_amd import _lib
    L = _lib.lib()
    def ws(**kw):
        a = {**BASE, **kw}
        a["groups_host"] = host(a["groups_host"])
        return L.crane_hip_attn_shared_workspace(*[a[x] for x in ("groups_host", "n_groups", "max_kv", "max_own", "mean_own", "B", "S",
                                                                  "Hq", "Hkv", "D", "dtype")])

    need = ws()
    assert need > 0 and shared_call(ws_bytes=need - 1) == _lib.E_WORKSPACE
    assert ws(n_groups=0, max_own=60, mean_own=60) == 0                          # one chunk: written directly
    assert ws(D=64) == 0 and ws(dtype=9) == 0 and ws(B=0, n_groups=0) == 0 and ws(S=0) == 0 and ws(max_own=-1) == 0
    assert ws(groups_host=[0, 9, 0, 512]) == 0


def copy_call(pools=(16, 32), n_pages=8, P=256, Hkv=4, D=128, src=(0,), dst=(1,), rows=None, dtype=1, n=None):
    from crane_amd import _lib
    arr = lambda x: None if x is None else (ctypes.c_int32 * max(len(x), 1))(*x)
    ptr = (ctypes.c_void_p * max(len(pools), 1))(*pools)
    return _lib.lib().crane_hip_copy_pages(ptr, len(pools), n_pages, P, Hkv, D, arr(src), arr(dst), arr(rows),
                                           len(src) if n is None else n, dtype, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), "E_DTYPE"), (dict(D=96), "E_HEAD_DIM"), (dict(Hkv=0), "E_INVALID"), (dict(P=100), "E_INVALID"),
    (dict(n_pages=0), "E_INVALID"), (dict(n=-1), "E_INVALID"), (dict(pools=(16, None)), "E_INVALID"),
    (dict(pools=(16, 24)), "E_ALIGN"), (dict(src=(8,)), "E_INVALID"), (dict(src=(-1,)), "E_INVALID"),
    (dict(dst=(8,)), "E_INVALID"), (dict(dst=(-1,)), "E_INVALID"), (dict(rows=(257,)), "E_INVALID"),
    (dict(rows=(-1,)), "E_INVALID"), (dict(src=(1,), dst=(1,)), "E_INVALID"),
    (dict(src=(0, 2), dst=(3, 3)), "E_INVALID"),                      # one destination twice
    (dict(src=(0, 1), dst=(1, 2)), "E_INVALID"),                      # a destination that is a source
    (dict(src=(1, 0), dst=(2, 1)), "E_INVALID"),
    (dict(src=(), dst=()), "OK"),
    (dict(pools=()), "OK"), (dict(src=(0, 0), dst=(1, 2), rows=(0, 0)), "OK"),
])
def test_copy_refusals(kw, code):
    from crane_amd import _lib
    assert copy_call(**kw) == getattr(_lib, code)


def test_prefix_groups_checks():
    from crane_amd import ops
    from crane_amd._lib import CraneHipError
    g = ops.prefix_groups([[3, 0], [1]], [512, 100], 5, "cpu")
    assert g.shared_rows.tolist() == [512, 100, 0, 512, 0]
    assert g.groups.tolist() == [[0, 2, 3, 512], [2, 1, 1, 100]] and g.members.tolist() == [3, 0, 1]
    assert (g.n_groups, g.min_shared, list(g.groups_host)) == (2, 0, g.groups.flatten().tolist())
    g = ops.prefix_groups([], [], 3, "cpu")
    assert (g.n_groups, g.min_shared) == (0, 0)
    for groups, rows in (([[0, 1], [1]], [1, 2]), ([[5]], [1]), ([[-1]], [1]), ([[0, 0]], [4]), ([[]], [1]),
                         ([[0]], [-1]), ([[0]], [1, 2]), ([[0]], [1 << 31])):
        with pytest.raises(CraneHipError):
            ops.prefix_groups(groups, rows, 5, "cpu")


def test_host_tensors_are_refused():
    import torch
    from crane_amd import ops
    from crane_amd._lib import CraneHipError
    pool = torch.zeros(4, 2, 256, D)
    with pytest.raises(CraneHipError, match="GPU only"):
        ops.copy_pages([pool, pool], [0], [1])
    with pytest.raises(CraneHipError, match="GPU only"):
        ops.attention_shared_paged(torch.zeros(1, 4, D), pool, pool, torch.zeros(1, 2, dtype=torch.int32),
                                   torch.zeros(1, dtype=torch.int32), 4, ops.prefix_groups([], [], 1, "cpu"))


# ------------------------------------------------------------------ GPU: attention

SHAPES = [  # lens, groups, rows, P, Hq, Hkv, S
    ([257], [], [], 256, 8, 8, 1),
    ([1], [], [], 256, 4, 1, 1),
    ([31, 32, 33, 0, 1], [], [], 256, 4, 2, 1),
    ([513, 530], [[0, 1]], [512], 256, 16, 8, 1),
    ([256, 256, 256], [[0, 1, 2]], [256], 256, 8, 2, 1),               # nothing of their own
    ([700, 530, 1025, 512, 90, 2300], [[3, 0, 1], [5, 2]], [512, 1024], 512, 14, 2, 1),
    ([640] * 9 + [700] * 8, [list(range(0, 17, 2)), list(range(1, 17, 2))], [512, 256], 256, 8, 8, 1),
    ([2049 + 7 * i for i in range(21)], [list(range(21))], [2048], 256, 28, 4, 1),
    ([300, 310, 280], [[0, 1, 2]], [256], 256, 8, 2, 5),               # queries inside and past the shared rows
    ([260, 257, 256], [[0, 1, 2]], [256], 256, 7, 1, 17),
    ([40, 5, 70, 0], [], [], 256, 4, 2, 40),                           # fewer rows than queries
    ([1500, 1400], [[0, 1]], [1280], 256, 4, 4, 129),
    ([900, 3000, 1200], [[1, 2]], [512], 512, 16, 2, 64),
    ([4100], [[0]], [4096], 256, 8, 1, 3),                             # a group of one
    ([9000, 9100], [[0, 1]], [8704], 512, 2, 2, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_every_key_once(gpu, case, dtype):
    lens, groups, rows, P, Hq, Hkv, S = SHAPES[case]
    check_exact(gpu, 100 + case, lens, groups, rows, P, Hq, Hkv, S, dtype)
    check_exact(gpu, 200 + case, lens, groups, rows, P, Hq, Hkv, S, dtype, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", [i for i in range(len(SHAPES)) if i not in (11, 12)])
def test_attention_close(gpu, case, dtype):
    lens, groups, rows, P, Hq, Hkv, S = SHAPES[case]
    check_close(gpu, 300 + case, lens, groups, rows, P, Hq, Hkv, S, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 100, 255, 300])
@pytest.mark.parametrize("S", [1, 4])
def test_shared_rows_of_any_number(gpu, rows, S):
    """Rows shared up to the middle of a page or a tile: the sequences are one and the
    same, described as sharing only their first rows."""
    import torch
    from crane_amd import ops
    for dtype in ("bf16", "f32"):
        lens, P, Hq, Hkv = [333, 333], 256, 8, 2
        table, total = layout(50 + rows, lens, [[0, 1]], [333], P)
        k, v = pools(51 + rows, total, Hkv, P, table, lens, True)
        q = np.zeros((2, Hq, S, D), np.float32)
        got = call(gpu, q, cases.cast(k, dtype), v, table, lens, [[1, 0]], [rows], dtype)
        want = call(gpu, q, cases.cast(k, dtype), v, table, lens, [], [], dtype)
        assert torch.equal(got, want) and torch.equal(got[0], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores(gpu, dtype):
    """Scores of many hundreds: the running maximum moves often and most weights
    vanish."""
    check_close(gpu, 400, [800, 1100, 777], [[0, 2], [1]], [512, 768], 256, 8, 2, 1, dtype, q_scale=60.0)
    check_close(gpu, 403, [333, 290], [[0, 1]], [256], 256, 8, 2, 6, dtype, q_scale=60.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_rows_have_no_influence(gpu, dtype, bad):
    """A key that a causal query does not see, NaN or infinite in K and in V, has no
    influence on it; the queries that see it are as the definition says."""
    lens, groups, rows, P, Hq, Hkv, S = [300, 290], [[0, 1]], [256], 256, 8, 2, 9
    table, total = layout(61, lens, groups, rows, P)
    k, v = pools(62, total, Hkv, P, table, lens, False)
    q = cases.normal(cases.rng(63), (2, Hq, S, D))
    q, k, v = (cases.cast(x, dtype) for x in (q, k, v))
    out, mag, most = reference(q, k, v, table, lens, P, D ** -0.5, True)
    tol = bounds(out, mag, most, 300, dtype)
    untouched = np.ones(out.shape, bool)
    for which in ("k", "v"):
        k2, v2 = k.copy(), v.copy()
        j = 300 - 4                                # seen by sequence 0's last 4 queries only
        (k2 if which == "k" else v2)[table[0, j // P], :, j % P, ::3] = bad
        got = call(gpu, q, k2, v2, table, lens, groups, rows, dtype).float().cpu().numpy()
        untouched[0, S - 4:] = False
        if which == "v":                           # the other dims of those queries, too
            seen = untouched[0, S - 4:].reshape(4, Hq, D)
            seen[..., np.arange(D) % 3 != 0] = True
            hit = got[0, S - 4:].reshape(4, Hq, D)[..., ::3]
            assert np.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
        assert (np.abs(got - out)[untouched] <= tol[untouched]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 5])
def test_members_shorter_than_the_shared_rows(gpu, S):
    """A member whose length ends inside the group's shared rows sees its own rows
    only (a page id of its table past its end is not used)."""
    lens, P = [700, 512, 300, 2, 0], 256
    for dtype in ("bf16", "f32"):
        table, total = layout(70, [700, 512, 512, 512, 512], [list(range(5))], [512], P)
        k, v = pools(71, total, 2, P, table, [700, 512, 512, 512, 512], False)
        q = cases.cast(cases.normal(cases.rng(72), (5, 8, S, D)), dtype)
        k, v = cases.cast(k, dtype), cases.cast(v, dtype)
        got = call(gpu, q, k, v, table, lens, [[0, 1, 2, 3, 4]], [512], dtype).float().cpu().numpy()
        out, mag, most = reference(q, k, v, table, lens, P, D ** -0.5, True)
        assert (np.abs(got - out) <= bounds(out, mag, most, 700, dtype)).all()
        assert (got[4] == 0).all()


@pytest.mark.gpu
def test_pages_outside_the_pool_read_as_zero(gpu):
    import torch
    lens, groups, rows, P = [900, 820], [[0, 1]], [512], 256
    for dtype in ("bf16", "f32"):
        table, total = layout(80, lens, groups, rows, P)
        k, v = pools(81, total, 2, P, table, lens, False)
        q, k, v = (cases.cast(x, dtype) for x in (cases.normal(cases.rng(82), (2, 8, 1, D)), k, v))
        kz, vz, bad = k.copy(), v.copy(), table.copy()
        for b, i, x in ((0, 1, 10 ** 6), (1, 1, 10 ** 6), (1, 3, -5)):
            kz[table[b, i]] = 0
            vz[table[b, i]] = 0
            bad[b, i] = x
        got = call(gpu, q, k, v, bad, lens, groups, rows, dtype)
        assert torch.equal(got, call(gpu, q, kz, vz, table, lens, groups, rows, dtype))


@pytest.mark.gpu
def test_inconsistent_descriptions_stay_in_bounds(gpu):
    """Members and starts outside the batch, and lengths past the host's bounds, are
    not followed; sequences the description gets right keep their results."""
    import torch
    from crane_amd import ops
    lens, P = [600, 700, 300], 256
    table, total = layout(90, lens, [[0, 1]], [512], P)
    k, v = pools(91, total, 2, P, table, lens, False)
    q, k, v = (cases.cast(x, "bf16") for x in (cases.normal(cases.rng(92), (3, 8, 1, D)), k, v))
    want = call(gpu, q, k, v, table, lens, [[0, 1]], [512], "bf16")
    g = ops.prefix_groups([[0, 1]], [512], 3, gpu)
    args = lambda: (tens(q, "bf16", gpu).view(3, 8, D), tens(k, "bf16", gpu), tens(v, "bf16", gpu), ints(table, gpu),
                    ints(lens, gpu), 700, g)
    for groups, members in (([[0, 2, 0, 512]], [0, 99]), ([[0, 2, 0, 512]], [-3, 1]),
                            ([[-50, 1 << 30, 0, 512]], [0, 1, 2]), ([[0, 2, 99, 512]], [0, 1]),
                            ([[0, 2, -1, 512]], [0, 1]), ([[0, -4, 0, 512]], [0, 1]),
                            ([[0, 2, 0, 1 << 30]], [0, 1]), ([[0, 2, 0, -9]], [0, 1]), ([[1 << 30, 2, 0, 512]], [0, 1])):
        print(groups, members, flush=True)
        g.groups, g.members = ints(groups, gpu), ints(members + [0] * 3, gpu)
        got = ops.attention_shared_paged(*args())
        assert torch.equal(got[2], want[2])


@pytest.mark.gpu
def test_replays_and_streams(gpu):
    """A captured call replayed with other lengths and other eager calls between
    equals the eager call; another stream and a repeated call give the same bits."""
    import torch
    from crane_amd import ops
    lens, groups, rows, P, Hq, Hkv = [1100, 1300, 1030, 600], [[0, 1, 2]], [1024], 256, 16, 2
    table, total = layout(95, lens, groups, rows, P)
    k, v = pools(96, total, Hkv, P, table, lens, False)
    q = cases.cast(cases.normal(cases.rng(97), (4, Hq, 1, D)), "bf16")
    t = dict(q=tens(q, "bf16", gpu).view(4, Hq, D), k=tens(k, "bf16", gpu), v=tens(v, "bf16", gpu),
             table=ints(table, gpu), n=ints(lens, gpu))
    g = ops.prefix_groups(groups, rows, 4, gpu)
    run = lambda n: ops.attention_shared_paged(t["q"], t["k"], t["v"], t["table"], n, 1300, g)
    want = run(t["n"])
    assert torch.equal(run(t["n"]), want)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        other = run(t["n"])
    torch.cuda.current_stream(gpu).wait_stream(side)
    assert torch.equal(other, want)
    graphs = []
    for _ in range(2):  # two graphs of one call, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(t["n"])
        graphs.append((graph, out))
    for step in range(4):
        t["n"].copy_(ints([x - 5 * step for x in lens], gpu))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize(gpu)
        want = run(t["n"])
        for _, out in graphs:
            assert torch.equal(out, want), step


# ------------------------------------------------------------------ GPU: sizes at which sharing pays

SHARED_SHAPES = [  # members, shared rows, own rows from, other sequences, P, Hq, Hkv, S
    (16, 2048, 40, (100, 0), 256, 2, 2, 1),        # 16 rows a kv head in all
    (33, 1536, 200, (700,), 256, 4, 2, 1),         # 66
    (96, 512, 50, (), 512, 8, 4, 1),               # 192
    (4, 4096, 20, (), 256, 8, 8, 20),              # 80, 20 a sequence
    (16, 2560, 20, (30, 2), 512, 4, 2, 20),        # 640, 40
    (16, 4096, 65, (), 256, 2, 1, 65),             # 2080, 130
    (40, 1024, 0, (), 256, 8, 2, 1),               # little or nothing of their own
    (24, 1024, 0, (), 256, 8, 4, 5),               # queries inside and past the shared rows
    (6, 16896, 40, (), 256, 2, 2, 1),              # block table rows of 67 pages
]


def shared_shape(i):
    n, shared, own, others, P, Hq, Hkv, S = SHARED_SHAPES[i]
    lens = [shared + own + x % 7 for x in range(n)] + list(others)
    order = cases.rng(i).permutation(len(lens))    # the members in any order in the batch
    members = [int(np.where(order == x)[0][0]) for x in range(n)]
    return [lens[x] for x in order], [members], [shared], P, Hq, Hkv, S


def only_first_names(table, members, pages):
    """The table with the shared pages named by the group's first member only."""
    t = table.copy()
    for b in members[1:]:
        t[b, :pages] = -7
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(SHARED_SHAPES)))
def test_shared_rows_are_read_once(gpu, case, dtype):
    """Exact as above; and the members' own entries for shared pages are not read, which
    says that these calls share."""
    import torch
    lens, groups, rows, P, Hq, Hkv, S = shared_shape(case)
    for causal in (True, False):
        check_exact(gpu, 500 + case, lens, groups, rows, P, Hq, Hkv, S, dtype, causal)
    table, total = layout(520 + case, lens, groups, rows, P)
    k, v = pools(521 + case, total, Hkv, P, table, lens, False)
    q = cases.cast(cases.normal(cases.rng(522 + case), (len(lens), Hq, S, D)), dtype)
    args = (q, cases.cast(k, dtype), cases.cast(v, dtype))
    want = call(gpu, *args, table, lens, groups, rows, dtype)
    got = call(gpu, *args, only_first_names(table, groups[0], rows[0] // P), lens, groups, rows, dtype)
    if (case, dtype) != (4, "bf16"):               # (whole row blocks hold 3 sequences: no gain)
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", [0, 1, 2, 3, 6, 7])
@pytest.mark.parametrize("q_scale", [1.5, 60.0])
def test_shared_attention_close(gpu, case, dtype, q_scale):
    lens, groups, rows, P, Hq, Hkv, S = shared_shape(case)
    check_close(gpu, 540 + case, lens, groups, rows, P, Hq, Hkv, S, dtype, q_scale=q_scale)


def one_sequence_for_all(seed, n, Hkv, P):
    """A table row, K and V of one sequence of n rows."""
    pages = math.ceil(n / P)
    table, total = layout(seed, [n], [], [], P)
    k, v = pools(seed + 1, total, Hkv, P, table, [n], False)
    return table[:, :pages + 1], k, v


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,Hq,Hkv,S,n,shared", [
    (300, 2, 2, 1, 1400, 0), (150, 4, 2, 10, 1400, 0), (60, 4, 1, 33, 1400, 0), (64, 8, 8, 1, 4200, 4096),
    (256, 8, 8, 1, 2100, 2048), (16, 2, 1, 65, 4200, 4096)])
def test_rising_scores(gpu, B, Hq, Hkv, S, n, shared, dtype):
    """Scores that rise by 0.8 (natural units) from key to key: past any fixed maximum of a
    chunk's first keys by hundreds of powers of two."""
    P = 256
    table, k, v = one_sequence_for_all(560, n, Hkv, P)
    r = cases.rng(562)
    u = np.sign(cases.normal(r, (D,)))
    ramp = np.arange(n) * (0.8 * math.sqrt(D) / D)
    for i in range(math.ceil(n / P)):
        m = min(P, n - i * P)
        k[table[0, i], :, :m] = 0.05 * k[table[0, i], :, :m] + ramp[i * P:i * P + m, None] * u
    q = u + 0.05 * cases.normal(r, (B, Hq, S, D))
    lens = [n - b % 50 for b in range(B)]
    q, k, v = (cases.cast(x.astype(np.float32), dtype) for x in (q, k, v))
    table = np.repeat(table, B, 0)
    groups, rows = ([list(range(B))], [shared]) if shared else ([], [])
    got = call(gpu, q, k, v, table, lens, groups, rows, dtype).float().cpu().numpy()
    some = sorted({0, 1, 49, B - 1} & set(range(B)))   # sequences checked (all differ in q)
    out, mag, most = reference(q[some], k, v, table[some], [lens[b] for b in some], P, D ** -0.5, True)
    assert np.isfinite(got).all()
    assert (np.abs(got[some] - out) <= bounds(out, mag, most, n, dtype)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("B,Hq,Hkv,S,n,shared", [(2, 8, 2, 33, 400, 0), (24, 8, 4, 5, 1024, 1024), (16, 2, 1, 65, 4100, 4096)])
def test_hidden_rows_in_blocks(gpu, B, Hq, Hkv, S, n, shared, bad, dtype):
    """As test_hidden_rows_have_no_influence, in blocks of 128 rows and in shared rows: key
    n - 4 is NaN or infinite in K or in V, and the last 4 queries of the sequences that are
    n long see it."""
    P = 256
    table, k, v = one_sequence_for_all(570, n, Hkv, P)
    table = np.repeat(table, B, 0)
    lens = [n - b % 2 * 3 for b in range(B)]
    q = cases.normal(cases.rng(572), (B, Hq, S, D))
    q, k, v = (cases.cast(x, dtype) for x in (q, k, v))
    groups, rows = ([list(range(B))], [shared // P * P]) if shared else ([], [])
    j = n - 4
    some = [0, 1, B - 1]
    out, mag, most = reference(q[some], k, v, table[some], [lens[b] for b in some], P, D ** -0.5, True)
    tol = bounds(out, mag, most, n, dtype).reshape(3, S, Hq, D)
    out = out.reshape(3, S, Hq, D)
    for which in ("k", "v"):
        k2, v2 = k.copy(), v.copy()
        (k2 if which == "k" else v2)[table[0, j // P], :, j % P, ::3] = bad
        got = call(gpu, q, k2, v2, table, lens, groups, rows, dtype).float().cpu().numpy()
        got = got.reshape(B, S, Hq, D)[some]
        for x, b in enumerate(some):
            unseen = np.array([lens[b] - S + 1 + i <= j for i in range(S)])
            assert (np.abs(got[x] - out[x])[unseen] <= tol[x][unseen]).all()
            if which == "v":
                hit = got[x][~unseen][..., ::3]
                assert np.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
                clean = np.arange(D) % 3 != 0
                assert (np.abs(got[x] - out[x])[~unseen][..., clean] <= tol[x][~unseen][..., clean]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_short_members_and_bad_pages(gpu, dtype):
    """Members that end inside the shared rows, a page outside the pool among the shared
    ones, and one among a member's own."""
    import torch
    P, B, Hq, Hkv, S = 256, 40, 8, 2, 1
    full = [1024 + 3 * b for b in range(B)]
    lens = list(full)
    lens[3], lens[7], lens[20], lens[39] = 1024, 300, 2, 0
    table, total = layout(580, full, [list(range(B))], [1024], P)
    k, v = pools(581, total, Hkv, P, table, full, False)
    q = cases.cast(cases.normal(cases.rng(582), (B, Hq, S, D)), dtype)
    k, v = cases.cast(k, dtype), cases.cast(v, dtype)
    groups, rows = [list(range(B))], [1024]
    got = call(gpu, q, k, v, table, lens, groups, rows, dtype)
    out, mag, most = reference(q, k, v, table, lens, P, D ** -0.5, True)
    assert (np.abs(got.float().cpu().numpy() - out) <= bounds(out, mag, most, max(lens), dtype)).all()
    assert (got[39] == 0).all()
    kz, vz, bad = k.copy(), v.copy(), table.copy()
    for b, i, x in ((0, 2, 10 ** 6), (5, 4, -5)):
        kz[table[b, i]] = 0
        vz[table[b, i]] = 0
        bad[b, i] = x
    got = call(gpu, q, k, v, only_first_names(bad, groups[0], 4), lens, groups, rows, dtype)
    assert torch.equal(got, call(gpu, q, kz, vz, table, lens, groups, rows, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 5])
def test_shared_inconsistent_descriptions(gpu, S):
    """As test_inconsistent_descriptions_stay_in_bounds, where the call shares."""
    import torch
    from crane_amd import ops
    P, B = 256, 41
    lens = [1024 + b for b in range(B - 1)] + [300]
    table, total = layout(590, lens, [list(range(B - 1))], [1024], P)
    k, v = pools(591, total, 2, P, table, lens, False)
    q, k, v = (cases.cast(x, "bf16") for x in (cases.normal(cases.rng(592), (B, 8, S, D)), k, v))
    t = [tens(q, "bf16", gpu), tens(k, "bf16", gpu), tens(v, "bf16", gpu), ints(table, gpu), ints(lens, gpu)]
    g = ops.prefix_groups([list(range(B - 1))], [1024], B, gpu)
    want = ops.attention_shared_paged(*t, 1024 + B, g)
    members = list(range(B - 1))
    for groups, of in (([[0, 40, 0, 1024]], [99] * 40), ([[0, 40, 0, 1024]], [-3] + members[1:]),
                       ([[-50, 1 << 30, 0, 1024]], members), ([[0, 40, 99, 1024]], members),
                       ([[0, 40, -1, 1024]], members), ([[0, -4, 0, 1024]], members),
                       ([[0, 40, 0, 1 << 30]], members), ([[0, 40, 0, -9]], members),
                       ([[1 << 30, 40, 0, 1024]], members), ([[0, 40, 0, 1024]], [7] * 20 + [8] * 20)):
        print(groups, of[:3], flush=True)
        g.groups, g.members = ints(groups, gpu), ints(of, gpu)
        got = ops.attention_shared_paged(*t, 1024 + B, g)
        assert torch.equal(got[B - 1], want[B - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 8])
def test_shared_replays_streams_and_threads(gpu, S):
    """Two captured calls that share, replayed with other lengths and eager calls between;
    calls of two threads at once on streams of their own."""
    import threading

    import torch
    from crane_amd import ops
    lens, P, B, Hq, Hkv = [1100 + 5 * b for b in range(40)], 256, 40, 8, 2
    table, total = layout(600, lens, [list(range(B))], [1024], P)
    k, v = pools(601, total, Hkv, P, table, lens, False)
    q = cases.cast(cases.normal(cases.rng(602), (B, Hq, S, D)), "bf16")
    q, k, v, table, n = tens(q, "bf16", gpu), tens(k, "bf16", gpu), tens(v, "bf16", gpu), ints(table, gpu), ints(lens, gpu)
    g = ops.prefix_groups([list(range(B))], [1024], B, gpu)
    run = lambda n: ops.attention_shared_paged(q, k, v, table, n, max(lens), g)
    want = run(n)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(n)
        graphs.append((graph, out))
    for step in range(3):
        n.copy_(ints([x - 5 * step for x in lens], gpu))
        for graph, _ in graphs:
            graph.replay()
        want = run(n)
        torch.cuda.synchronize(gpu)
        for _, out in graphs:
            assert torch.equal(out, want), step
    results = [None, None]
    def work(i):
        stream = torch.cuda.Stream(gpu)
        with torch.cuda.stream(stream):
            results[i] = [run(n) for _ in range(20)]
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(x, want) for r in results for x in r)


@pytest.mark.gpu
def test_pools_past_31_bits(gpu):
    """Pages past the first 2^31 elements of a pool: attention over them, and copies."""
    import torch
    from crane_amd import ops
    P, Hq, Hkv, B = 256, 8, 8, 24
    far = 2 ** 31 // (Hkv * P * D)
    lens = [1024 + 9 * b for b in range(B)]
    table, total = layout(610, lens, [list(range(B))], [1024], P)
    k, v = pools(611, total, Hkv, P, table, lens, True)
    q = torch.zeros(B, Hq, D, dtype=torch.bfloat16, device=gpu)
    near = [tens(cases.cast(x, "bf16"), "bf16", gpu) for x in (k, v)]
    big = [torch.empty(far + total, Hkv, P, D, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    for x, y in zip(big, near):
        x[far:] = y
    for groups, rows in (([list(range(B))], [1024]), ([], [])):
        g = ops.prefix_groups(groups, rows, B, gpu)
        want = ops.attention_shared_paged(q, *near, ints(table, gpu), ints(lens, gpu), max(lens), g)
        got = ops.attention_shared_paged(q, *big, ints(np.where(table < 0, table, table + far), gpu), ints(lens, gpu),
                                         max(lens), g)
        assert torch.equal(got, want)
    ops.copy_pages(big, [far, far + 1, far + 2], [0, 1, far + 5], [P, 77, P])
    for x, y in zip(big, near):
        assert torch.equal(x[0].view(torch.int16), y[0].view(torch.int16))
        assert torch.equal(x[1, :, :77].view(torch.int16), y[1, :, :77].view(torch.int16))
        assert torch.equal(x[far + 5].view(torch.int16), y[2].view(torch.int16))


# ------------------------------------------------------------------ GPU: copies

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,P,Hkv,n_pools", [("bf16", 256, 8, 2), ("f32", 512, 3, 2), ("bf16", 256, 1, 74),
                                                 ("bf16", 256, 2, 131)])
def test_copy_pages(gpu, dtype, P, Hkv, n_pools):
    import torch
    from crane_amd import ops
    r = cases.rng(500 + n_pools)
    n_pages = 300 if n_pools == 2 else 12
    for pairs in ([1, 3, 140] if n_pools == 2 else [5]):  # 140: more than one launch's pairs
        ids = r.permutation(n_pages)
        src = [int(ids[i % max(1, min(7, pairs // 2))]) for i in range(pairs)]
        dst = [int(x) for x in ids[-pairs:]]
        for rows in (None, [int(x) for x in r.integers(0, P + 1, pairs)]):
            print(f"copy {dtype} P={P} Hkv={Hkv} pools={n_pools} pairs={pairs} rows={rows and rows[:4]}", flush=True)
            pools_ = [torch.randn((n_pages, Hkv, P, D), device=gpu).to(torch.bfloat16 if dtype == "bf16" else
                                                                      torch.float32) for _ in range(n_pools)]
            want = [p.clone() for p in pools_]
            ops.copy_pages(pools_, src, dst, rows)
            for p in want:
                for i, (a, b) in enumerate(zip(src, dst)):
                    n = P if rows is None else rows[i]
                    p[b, :, :n] = p[a, :, :n]
            assert all(torch.equal(a, b) for a, b in zip(pools_, want))


@pytest.mark.gpu
def test_copy_pages_python_refusals(gpu):
    import torch
    from crane_amd import ops
    from crane_amd._lib import CraneHipError
    a = torch.zeros((4, 2, 256, D), device=gpu)
    for args in (([a, a[:3]], [0], [1]), ([a, a.bfloat16()], [0], [1]), ([a], [0, 1], [2]), ([a], [0], [4]),
                 ([a], [1 << 32], [1]), ([a], [0], [1], [257]), ([a], [0], [1], [1, 2]), ([a], [0, 0], [1, 1]),
                 ([a.transpose(1, 2)], [0], [1]), ([a[..., :64].contiguous()], [0], [1]),
                 ([a], bytes(4), bytes([1, 0, 0, 0]))):
        with pytest.raises(CraneHipError):
            ops.copy_pages(*args)
    ops.copy_pages([], [0], [1])
    ops.copy_pages([a], [], [])


# ------------------------------------------------------------------ grouping (CPU)

def partitions(items):
    if not items:
        yield []
        return
    first, rest = items[0], items[1:]
    for p in partitions(rest):
        yield [[first]] + p
        for i in range(len(p)):
            yield p[:i] + [[first] + p[i]] + p[i + 1:]


def common(tables, members):
    n = 0
    while all(len(tables[b]) > n and tables[b][n] == tables[members[0]][n] >= 0 for b in members):
        n += 1
    return n


@pytest.mark.parametrize("seed", range(40))
def test_group_prefixes_saves_most(seed):
    """Against every partition of up to six page lists that branch from one another."""
    from crane_amd import ops
    r = cases.rng(seed)
    tables, nxt = [[]], 1
    for _ in range(int(r.integers(1, 6))):
        src = tables[int(r.integers(len(tables)))]
        t = src[:int(r.integers(0, len(src) + 1))] if seed % 4 else list(src)
        n = int(r.integers(0, 5))
        t = t + list(range(nxt, nxt + n))
        nxt += n
        tables.append(t)
    if seed % 5 == 0:
        tables[0] = [-1, 7]
        tables[-1] = [-1, 7]
    groups, pages = ops.group_prefixes(tables)
    assert len(groups) == len(pages)
    flat = [b for g in groups for b in g]
    assert len(flat) == len(set(flat))
    for g, n in zip(groups, pages):
        assert len(g) > 1 and n == common(tables, g) > 0
    saved = sum((len(g) - 1) * n for g, n in zip(groups, pages))
    best = max(sum((len(g) - 1) * common(tables, g) for g in p) for p in partitions(list(range(len(tables)))))
    assert saved == best


def test_group_prefixes_edges():
    from crane_amd import _lib, ops
    from crane_amd._lib import CraneHipError
    assert ops.group_prefixes([]) == ([], [])
    assert ops.group_prefixes([[], []]) == ([], [])
    assert ops.group_prefixes([[5, 6], [1], [5, 6]]) == ([[0, 2]], [2])
    with pytest.raises(CraneHipError):
        ops.group_prefixes([[0], [1 << 32]])
    L, n = _lib.lib(), ctypes.c_int()
    buf = (ctypes.c_int32 * 8)()
    assert L.crane_hip_group_prefixes(buf, 2, (ctypes.c_int32 * 1)(3), 1, buf, buf, buf, ctypes.byref(n)) == \
        _lib.E_INVALID                                                  # more pages than the table's stride
    assert L.crane_hip_group_prefixes(None, 2, (ctypes.c_int32 * 1)(1), 1, buf, buf, buf, ctypes.byref(n)) == \
        _lib.E_INVALID
    assert L.crane_hip_group_prefixes(buf, 2, buf, 1, buf, None, buf, ctypes.byref(n)) == _lib.E_INVALID
    assert L.crane_hip_group_prefixes(buf, 2, buf, -1, buf, buf, buf, ctypes.byref(n)) == _lib.E_INVALID


def test_group_prefixes_nested_deep():
    """Lists that each extend the last: the nesting stays within a bound, the groups valid."""
    from crane_amd import ops
    tables = [list(range(n)) for n in range(1, 2501)]
    groups, pages = ops.group_prefixes(tables)
    flat = [b for g in groups for b in g]
    assert len(flat) == len(set(flat)) and len(groups) == len(pages) >= 1
    for g, n in zip(groups, pages):
        assert len(g) > 1 and 0 < n <= min(len(tables[b]) for b in g)
    assert sum((len(g) - 1) * n for g, n in zip(groups, pages)) >= 1900 * 500   # one group of the longest does that


def test_manager_refusals_without_a_cache():
    from crane_amd import _lib
    L = _lib.lib()
    ids, null = (ctypes.c_int * 4)(), (ctypes.c_void_p * 2)(None, None)
    assert L.crane_pkv_fork(null, 2, 0, -1, 1, ids, None) == _lib.E_INVALID
    assert L.crane_pkv_fork(None, 1, 0, -1, 1, ids, None) == _lib.E_INVALID
    assert L.crane_pkv_fork(null, -1, 0, -1, 1, ids, None) == _lib.E_INVALID
    assert L.crane_pkv_truncate(null, 1, 0, 0, None) == _lib.E_INVALID
    assert L.crane_pkv_compact(null, 1, None, None) == _lib.E_INVALID
    assert L.crane_pkv_shared_workspace(None, 8, 1) == 0
    assert L.crane_pkv_attention_shared(None, 16, 8, 1, 0.1, 1, None, 0, 16, None) == _lib.E_INVALID


# ------------------------------------------------------------------ GPU: the manager

class Model:
    """What the caches should hold: every sequence's rows per layer, and which
    sequences hold which pages (a page is named by the object that filled it)."""

    def __init__(self, layers, P):
        self.rows, self.pages, self.P, self.layers, self.made = {}, {}, P, layers, 0

    def new(self):
        self.made += 1
        return self.made

    def grow(self, sid):
        n = self.rows[sid][0][0].shape[1]
        while len(self.pages[sid]) * self.P < n:
            self.pages[sid].append(self.new())

    def cut(self, sid, n):
        need = math.ceil(n / self.P)
        held = [p for s, ps in self.pages.items() if s != sid for p in ps]
        self.pages[sid] = self.pages[sid][:need]
        if n % self.P and self.pages[sid][-1] in held:
            self.pages[sid][-1] = self.new()

    def used(self):
        return len({p for ps in self.pages.values() for p in ps})


@pytest.mark.gpu
@pytest.mark.parametrize("seed,dtype", [(1, "bf16"), (2, "f32"), (3, "bf16")])
def test_forks_appends_cuts_and_compactions(gpu, seed, dtype):
    """A random run over two layers' caches: sequences written, forked, appended to in
    batches, cut, freed and compacted, against rows kept apart; every step's attention
    against the definition, and the pages in use counted."""
    import torch
    from crane_amd import kv
    from crane_amd._lib import CraneHipError
    r = cases.rng(900 + seed)
    Hkv, Hq, P, n_pages = 2, 8, 256, 24
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    caches = [kv.PagedKvCache(Hkv, n_pages, td, P, max_seqs=8, max_pages_per_seq=8, device=gpu) for _ in range(2)]
    m = Model(2, P)
    rand = lambda *shape: tens(cases.normal(r, shape), dtype, gpu)
    batch = []

    def check(sids):
        for sid in sids:
            for c, layer in zip(caches, m.rows[sid]):
                k, v = c.read_sequence(sid)
                assert torch.equal(k, layer[0]) and torch.equal(v, layer[1]), sid
        assert all(c.free_pages == n_pages - m.used() for c in caches)

    for step in range(60):
        what = ["write", "fork", "append", "append", "cut", "free", "compact", "append"][int(r.integers(8))]
        live = sorted(m.rows)
        idle = [s for s in live if s not in batch]
        print(f"step {step}: {what} live={live} used={m.used()}", flush=True)
        try:
            if what == "write":
                n = int(r.integers(0, 3 * P))
                new = not idle or r.integers(2)
                sids = [c.add_sequence() for c in caches] if new else [idle[0]] * 2
                assert sids[0] == sids[1]
                rows = [[rand(Hkv, n, D), rand(Hkv, n, D)] for _ in caches]
                if new:
                    m.rows[sids[0]], m.pages[sids[0]] = [[x[:, :0] for x in l] for l in rows], []
                for c, (k, v) in zip(caches, rows):
                    c.write_sequence(sids[0], k, v)
                held = [p for s, ps in m.pages.items() if s != sids[0] for p in ps]
                m.pages[sids[0]] = [p for p in m.pages[sids[0]] if p not in held][:math.ceil(n / P)]
                m.rows[sids[0]] = rows
                m.grow(sids[0])
            elif what == "fork" and live:
                sid, count = live[int(r.integers(len(live)))], int(r.integers(1, 4))
                full = m.rows[sid][0][0].shape[1]
                n = None if r.integers(2) else int(r.integers(0, full + 1))
                ids = kv.fork_sequence(caches, sid, count, n)
                n = full if n is None else n
                assert len(set(ids)) == count and not set(ids) & set(live)
                for i in ids:
                    m.rows[i] = [[x[:, :n].clone() for x in l] for l in m.rows[sid]]
                    m.pages[i] = m.pages[sid][:n // P] + ([m.new()] if n % P else [])
            elif what == "append" and live:
                batch = [s for s in live if r.integers(4)] or live[:1]
                for c in caches:
                    c.set_batch(batch)
                S = int(r.integers(1, 6)) if r.integers(3) else int(r.integers(100, 300))
                new = [[rand(len(batch), Hkv, S, D), rand(len(batch), Hkv, S, D)] for _ in caches]
                for c, (k, v) in zip(caches, new):
                    c.update_kv_cache(k, v)
                for i, sid in enumerate(batch):
                    m.rows[sid] = [[torch.cat([x, y[i]], 1) for x, y in zip(l, nl)] for l, nl in zip(m.rows[sid], new)]
                    m.grow(sid)
                Sq = min(S, 3)
                q = cases.cast(cases.normal(r, (len(batch), Hq, Sq, D)), dtype)
                for c, layer in zip(caches, range(2)):
                    got = c.attention_shared(tens(q, dtype, gpu) if Sq > 1 else tens(q, dtype, gpu)[:, :, 0])
                    for i, sid in enumerate(batch):
                        k, v = (x.float().cpu().numpy() for x in m.rows[sid][layer])
                        n = k.shape[1]
                        t = np.zeros((1, 1), np.int32)
                        out, mag, most = reference(q[i:i + 1], k[None], v[None], t, [n], n, D ** -0.5, True)
                        err = np.abs(got[i:i + 1].float().cpu().numpy() - out)
                        assert (err <= bounds(out, mag, most, n, dtype)).all(), (sid, n)
            elif what == "cut" and idle:
                sid = idle[int(r.integers(len(idle)))]
                n = int(r.integers(0, m.rows[sid][0][0].shape[1] + 1))
                kv.truncate_sequence(caches, sid, n)
                m.rows[sid] = [[x[:, :n].clone() for x in l] for l in m.rows[sid]]
                m.cut(sid, n)
            elif what == "free" and idle:
                for c in caches:
                    c.free_sequence(idle[-1])
                del m.rows[idle[-1]], m.pages[idle[-1]]
            elif what == "compact":
                kv.compact(caches)
                assert kv.compact(caches) == 0
                for c in caches:
                    assert c.block_table().max() < m.used() if batch else True
        except CraneHipError as e:              # (both layers refuse alike, the first before the second)
            assert "capacity" in str(e), e      # out of pages or ids: nothing has changed
        check(m.rows)
    for c in caches:
        c.close()


@pytest.mark.gpu
def test_answers_to_one_prompt(gpu):
    """A prompt prefilled once, forked into answers that decode together, beside copies
    of it that share nothing: the same appends give the same rows, the attention is
    the definition's for both, and freeing the answers leaves the prompt."""
    import torch
    from crane_amd import kv, ops
    Hq, Hkv, P, S0, n = 16, 2, 256, 700, 5
    g = torch.Generator(device=gpu).manual_seed(5)
    r16 = lambda *s: torch.randn(s, generator=g, device=gpu).to(torch.bfloat16)
    cos, sin = ops.rope_tables(D, 1e6, 2048, device=gpu, dtype=torch.bfloat16)
    c = kv.PagedKvCache(Hkv, 40, torch.bfloat16, P, max_seqs=16, max_pages_per_seq=6, device=gpu)
    first = c.add_sequence()
    c.set_batch([first])
    qkv, at = r16(1, S0, (Hq + 2 * Hkv) * D), torch.zeros(1, dtype=torch.int32, device=gpu)
    q = c.append_qkv(qkv, cos, sin, at, Hq)
    got = c.attention_shared(q).float().cpu().numpy()   # the prompt itself: one sequence, no groups
    k, v = c.read_sequence(first)
    kk, vv = k.float().cpu().numpy(), v.float().cpu().numpy()
    out, mag, most = reference(q.float().cpu().numpy(), kk[None], vv[None], np.zeros((1, 1), np.int32), [S0], S0,
                               D ** -0.5, True)
    assert (np.abs(got - out) <= bounds(out, mag, most, S0, "bf16")).all()
    used = 40 - c.free_pages
    answers = c.fork_sequence(first, n)
    assert 40 - c.free_pages == used + n                # the 188 rows past two whole pages, copied
    copies = []
    for _ in range(n):
        copies.append(c.add_sequence())
        c.write_sequence(copies[-1], k, v)
    for step in range(3):
        tok = r16(n, 1, (Hq + 2 * Hkv) * D)
        at = torch.full((n,), S0 + step, dtype=torch.int32, device=gpu)
        outs, rows = [], []
        for ids in (answers, copies):
            c.set_batch(ids)
            q = c.append_qkv(tok, cos, sin, at, Hq)
            outs.append(c.attention_shared(q.view(n, Hq, D)).float().cpu().numpy())
            rows.append([c.read_sequence(i) for i in ids])
        for (ka, va), (kb, vb) in zip(*rows):
            assert torch.equal(ka, kb) and torch.equal(va, vb)
        qn = q.float().cpu().numpy()
        for i, (ka, va) in enumerate(rows[0]):
            kk, vv = ka.float().cpu().numpy(), va.float().cpu().numpy()
            out, mag, most = reference(qn[i:i + 1], kk[None], vv[None], np.zeros((1, 1), np.int32), [kk.shape[1]],
                                       kk.shape[1], D ** -0.5, True)
            tol = bounds(out, mag, most, kk.shape[1], "bf16")
            assert (np.abs(outs[0][i] - out[0]) <= tol[0]).all() and (np.abs(outs[1][i] - out[0]) <= tol[0]).all()
        if step == 1:
            c.set_batch([])
            c.free_sequence(copies.pop())
            copies.append(c.fork_sequence(answers[-1])[0])  # and a fork of a fork in a copy's place
            moved = c.compact()
            assert moved >= 0 and c.compact() == 0
    c.set_batch([])
    for i in answers + copies:
        c.free_sequence(i)
    assert 40 - c.free_pages == used
    k2, v2 = c.read_sequence(first)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    c.close()


@pytest.mark.gpu
def test_manager_refusals(gpu):
    import torch
    from crane_amd import _lib, kv
    from crane_amd._lib import CraneHipError
    c = kv.PagedKvCache(2, 8, torch.bfloat16, 256, max_seqs=4, max_pages_per_seq=4, device=gpu)
    a = c.add_sequence()
    z = torch.zeros((2, 300, D), dtype=torch.bfloat16, device=gpu)
    c.write_sequence(a, z, z)
    c.set_batch([a])

    def refused(code, f, *args):
        with pytest.raises(CraneHipError) as e:
            f(*args)
        assert e.value.code == code, e.value

    refused(_lib.E_INVALID, c.fork_sequence, 3)                # not live
    refused(_lib.E_INVALID, c.fork_sequence, a, 1, 301)        # more rows than it has
    refused(_lib.E_INVALID, c.fork_sequence, a, 1, -1)
    refused(_lib.E_INVALID, c.fork_sequence, a, -1)
    refused(_lib.E_CAPACITY, c.fork_sequence, a, 4)            # 3 ids left
    refused(_lib.E_INVALID, c.truncate_sequence, a, 10)        # in the batch
    refused(_lib.E_INVALID, kv.fork_sequence, [c, c], a)       # one cache twice
    refused(_lib.E_INVALID, kv.compact, [])
    assert c.fork_sequence(a, 0) == []
    b, = c.fork_sequence(a, 1, 256)                            # a whole page: nothing copied
    assert c.seq_len(b) == 256 and c.free_pages == 6
    refused(_lib.E_INVALID, c.truncate_sequence, b, 257)
    refused(_lib.E_INVALID, c.truncate_sequence, b, -1)
    q = torch.zeros((1, 4, D), dtype=torch.bfloat16, device=gpu)
    refused(_lib.E_INVALID, c.attention_shared, q.expand(2, 4, D))
    refused(_lib.E_DTYPE, c.attention_shared, q.float())
    refused(_lib.E_INVALID, c.attention_shared, q.view(1, 4, 1, D).expand(1, 4, 301, D))
    refused(_lib.E_INVALID, c.attention_shared, q, -1.0)
    other = kv.PagedKvCache(2, 3, torch.bfloat16, 256, max_seqs=4, max_pages_per_seq=4, device=gpu)
    other.write_sequence(other.add_sequence(), z[:, :200], z[:, :200])
    refused(_lib.E_INVALID, kv.fork_sequence, [c, other], a, 1, 256)   # `other` has 200 rows
    assert c.free_pages == 6 and other.free_pages == 2
    other.set_batch([])
    d, = other.fork_sequence(0)
    e, = other.fork_sequence(0)
    assert other.free_pages == 0
    refused(_lib.E_CAPACITY, other.fork_sequence, 0)           # no page for the copied rows
    assert [other.seq_len(i) for i in (0, d, e, 3)] == [200, 200, 200, -1]
    c.close()
    other.close()
