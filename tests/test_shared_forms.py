"""Every kernel form of the attention over shared pages, shared row counts off every
bound, and descriptions that contradict the host's, at sizes whose plan shares
(include/crane_shared.h).  A test on the host pins the form that each case takes; that a
call shares is shown by page tables that name the shared pages in the first member's row
only.  The inputs and the derived bounds are those of test_shared."""
import numpy as np
import pytest

import cases
import test_shared as ts
from test_shared_plan import host, plan  # noqa: F401  (host: a fixture)

D = 128

FORMS = [  # members, shared rows, own rows from, other sequences, P, Hq, Hkv, S, {type: (shared role's rows, own's, one block)}
    (16, 2048, 40, (), 256, 2, 2, 1, {"bf16": (16, 16, True), "f32": (16, 16, True)}),
    (11, 2048, 30, (5,), 256, 8, 4, 1, {"bf16": (32, 16, True), "f32": (32, 16, True)}),
    (33, 1536, 200, (700,), 256, 4, 2, 1, {"bf16": (32, 16, False), "f32": (32, 16, False)}),
    (8, 2816, 30, (), 256, 8, 8, 5, {"bf16": (32, 16, False), "f32": (32, 16, False)}),
    (4, 4096, 20, (), 256, 8, 8, 20, {"bf16": (32, 32, False), "f32": (32, 32, False)}),
    (40, 1024, 60, (), 256, 8, 2, 1, {"bf16": (128, 16, False), "f32": (32, 16, False)}),
    (32, 4096, 30, (), 256, 8, 2, 5, {"bf16": (128, 32, False), "f32": (32, 32, False)}),
    (12, 8192, 20, (), 512, 8, 8, 20, {"bf16": (128, 32, False), "f32": (32, 32, False)}),
    (16, 4096, 70, (), 256, 2, 1, 65, {"bf16": (128, 128, False), "f32": (32, 32, False)}),
]
ODD = [  # members, shared rows, own rows from, P, Hq, Hkv, S: one sequence, cut at several lengths
    (16, 2600, 40, 256, 2, 2, 1),
    (11, 2079, 30, 256, 8, 4, 1),
    (40, 1057, 60, 256, 8, 2, 1),
    (40, 2040, 60, 512, 8, 2, 5),
    (33, 1841, 30, 256, 8, 2, 4),
    (32, 4097, 30, 256, 8, 2, 5),
    (8, 3001, 30, 256, 4, 2, 20),
    (16, 4159, 70, 256, 2, 1, 65),
]


def shuffled(i, n, lens):
    """The sequences of `lens`, the members first, in any order in the batch."""
    order = cases.rng(i).permutation(len(lens))
    return [lens[x] for x in order], [int(np.where(order == x)[0][0]) for x in range(n)]


def form_case(i):
    n, shared, own, others, P, Hq, Hkv, S, forms = FORMS[i]
    lens, members = shuffled(800 + i, n, [shared + own + x % 7 for x in range(n)] + list(others))
    return lens, members, shared, P, Hq, Hkv, S, forms


def odd_case(i):
    n, shared, own, P, Hq, Hkv, S = ODD[i]
    lens, members = shuffled(840 + i, n, [shared + own + x % 7 for x in range(n)])
    return lens, members, shared, P, Hq, Hkv, S


def ops_plan(host, lens, members, shared, Hq, Hkv, S, dtype, max_own=None):
    """The plan of a call through ops, whose bounds are guessed from the longest sequence."""
    rows = [shared if b in members else 0 for b in range(len(lens))]
    own = max(lens) - min(rows) if max_own is None else max_own
    return plan(host, [(len(members), shared)], max(lens), own, 6 * (max(lens) - max(rows)) // 10, len(lens), S, Hq,
                Hkv, dtype == "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cases_take_every_form(host, dtype):  # noqa: F811
    seen = set()
    for i in range(len(FORMS)):
        lens, members, shared, P, Hq, Hkv, S, forms = form_case(i)
        p = ops_plan(host, lens, members, shared, Hq, Hkv, S, dtype)
        once = p["shared_tiles"] == 1 if p["own_rows"] == 16 else False
        assert p["share"] and (p["shared_rows"], p["own_rows"], once) == forms[dtype], (i, p)
        seen.add(forms[dtype])
    assert seen == {(16, 16, True), (32, 16, True), (32, 16, False), (32, 32, False)} | (
        {(128, 16, False), (128, 32, False), (128, 128, False)} if dtype == "bf16" else set())
    for i in range(len(ODD)):
        lens, members, shared, P, Hq, Hkv, S = odd_case(i)
        assert ops_plan(host, lens, members, shared, Hq, Hkv, S, dtype)["share"] and shared % 64, i


def check(got, want, bound):
    got = got.float().cpu().numpy()
    worst = float((np.abs(got - want) / bound).max())
    assert worst <= 1, worst


def some_of(lens, members):
    """A few sequences: the first, second and last member, one outside the group."""
    rest = [b for b in range(len(lens)) if b not in members]
    return [members[0], members[1], members[-1]] + rest[:1]


def exact_want(v, table, lens, S, Hq, Hkv, P, causal):
    """q = 0: T(f32(sum of V) / f32(count)), as in test_shared."""
    want = np.zeros((len(lens), S, Hkv, Hq // Hkv, D), np.float32)
    for b, n in enumerate(lens):
        sums = np.cumsum(ts.rows_of(v, table, b, n, P).astype(np.float64), 1)
        for s in range(S):
            L = n - S + 1 + s if causal else n
            if L > 0:
                want[b, s] = (sums[:, L - 1].astype(np.float32) / np.float32(L))[:, None, :]
    return want.reshape(len(lens), S, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(FORMS)))
def test_forms(gpu, case, dtype):
    """Every key once, and the definition in 64 bits, in every form; the members' own
    entries for the shared pages are not read."""
    lens, members, shared, P, Hq, Hkv, S, _ = form_case(case)
    print(f"form {case} {dtype}", flush=True)
    table, total = ts.layout(860 + case, lens, [members], [shared], P)
    first_only = ts.only_first_names(table, members, shared // P)
    zero = np.zeros((len(lens), Hq, S, D), np.float32)
    k, v = ts.pools(861 + case, total, Hkv, P, table, lens, True)
    for causal in (True, False):
        got = ts.call(gpu, zero, cases.cast(k, dtype), v, first_only, lens, [members], [shared], dtype, causal=causal)
        want = cases.cast(exact_want(v, table, lens, S, Hq, Hkv, P, causal), dtype)
        wrong = int((got.float().cpu().numpy() != want).sum())
        assert wrong == 0, wrong
    k, v = (cases.cast(x, dtype) for x in ts.pools(862 + case, total, Hkv, P, table, lens, False))
    q = cases.cast(cases.normal(cases.rng(863 + case), (len(lens), Hq, S, D)) * np.float32(1.5), dtype)
    got = ts.call(gpu, q, k, v, first_only, lens, [members], [shared], dtype)
    some = some_of(lens, members)
    out, mag, most = ts.reference(q[some], k, v, table[some], [lens[b] for b in some], P, D ** -0.5, True)
    check(got[some], out, ts.bounds(out, mag, most, max(lens), dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(ODD)))
def test_shared_rows_off_every_bound(gpu, case, dtype):
    """Shared rows that end inside a page, a tile and a step: the members are one sequence
    at several lengths, so that the page they end in may be named by all; the whole
    shared pages are named by the first member only."""
    lens, members, shared, P, Hq, Hkv, S = odd_case(case)
    print(f"odd {case} {dtype}", flush=True)
    B = len(lens)
    row, k, v = ts.one_sequence_for_all(880 + case, max(lens), Hkv, P)
    table = np.repeat(row, B, 0)
    first_only = ts.only_first_names(table, members, shared // P)
    # every key once
    exact = np.where(np.isnan(v), v, np.sign(v))
    zero = np.zeros((B, Hq, S, D), np.float32)
    for causal in (True, False):
        got = ts.call(gpu, zero, cases.cast(k, dtype), exact, first_only, lens, [members], [shared], dtype,
                      causal=causal)
        want = cases.cast(exact_want(exact, table, lens, S, Hq, Hkv, P, causal), dtype)
        wrong = int((got.float().cpu().numpy() != want).sum())
        assert wrong == 0, wrong
    # the definition
    k, v = cases.cast(k, dtype), cases.cast(v, dtype)
    q = cases.cast(cases.normal(cases.rng(882 + case), (B, Hq, S, D)) * np.float32(1.5), dtype)
    got = ts.call(gpu, q, k, v, first_only, lens, [members], [shared], dtype)
    some = some_of(lens, members)
    out, mag, most = ts.reference(q[some], k, v, table[some], [lens[b] for b in some], P, D ** -0.5, True)
    check(got[some], out, ts.bounds(out, mag, most, max(lens), dtype))


CONTRADICTIONS = [  # the device's group, its members
    ([0, 40, 0, 4096], [99] * 40), ([0, 40, 0, 4096], [-3] + list(range(1, 40))), ([-50, 1 << 30, 0, 4096], None),
    ([0, 40, 99, 4096], None), ([0, 40, -1, 4096], None), ([0, -4, 0, 4096], None), ([0, 40, 0, 1 << 30], None),
    ([0, 40, 0, -9], None), ([1 << 30, 40, 0, 4096], None), ([39, 40, 0, 4096], None), ([40, 1, 0, 4096], None),
    ([0, 40, 0, 4096], [7] * 20 + [8] * 20), ([0, 7, 0, 100], None)]


def contradiction_case():
    B, shared = 41, 4096
    return [shared + 1 + b for b in range(B - 1)] + [300], list(range(B - 1)), shared, 256, 8, 2


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 5])
def test_contradictions_are_of_a_plan_that_shares(host, S, dtype):  # noqa: F811
    lens, members, shared, P, Hq, Hkv = contradiction_case()
    assert ops_plan(host, lens, members, shared, Hq, Hkv, S, dtype, max_own=300)["share"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 5])
def test_contradictions_stay_in_bounds(gpu, S, dtype):
    """Device groups and members outside the batch and the members array (which has the
    group's 40 entries and no more), with a sequence outside the group whose result they
    leave alone; the description that is right gives the definition."""
    import torch
    from crane_amd import ops
    lens, members, shared, P, Hq, Hkv = contradiction_case()
    B = len(lens)
    table, total = ts.layout(900, lens, [members], [shared], P)
    k, v = (cases.cast(x, dtype) for x in ts.pools(901, total, Hkv, P, table, lens, False))
    q = cases.cast(cases.normal(cases.rng(902), (B, Hq, S, D)) * np.float32(1.5), dtype)
    qq = ts.tens(q, dtype, gpu)
    t = [qq.view(B, Hq, D) if S == 1 else qq, ts.tens(k, dtype, gpu), ts.tens(v, dtype, gpu),
         ts.ints(ts.only_first_names(table, members, shared // P), gpu), ts.ints(lens, gpu)]
    g = ops.prefix_groups([members], [shared], B, gpu)
    call = lambda: ops.attention_shared_paged(*t, max(lens), g, max_own=300)
    want = call()
    some = [0, 20, 39, 40]
    out, mag, most = ts.reference(q[some], k, v, table[some], [lens[b] for b in some], P, D ** -0.5, True)
    check(want[some], out, ts.bounds(out, mag, most, max(lens), dtype))
    right = g.groups, g.members
    for group, of in CONTRADICTIONS:
        print(group, of and of[:3], flush=True)
        g.groups, g.members = ts.ints([group], gpu), ts.ints(members if of is None else of, gpu)
        assert torch.equal(call()[B - 1], want[B - 1])
    g.groups, g.members = right
    assert torch.equal(call(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_replayed_call_shares(host, dtype):  # noqa: F811
    lens = [4200 + 5 * b for b in range(32)]
    assert ops_plan(host, lens, list(range(32)), 4096, 8, 2, 8, dtype)["share"] == (dtype == "bf16")
    assert ops_plan(host, lens, list(range(32)), 4096, 8, 2, 5, dtype)["share"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,S", [("bf16", 8), ("f32", 5)])
def test_replays_of_several_tokens_that_share(gpu, dtype, S):
    """Two captured calls of several tokens, replayed with other lengths and eager calls
    between them, and the same call on another stream."""
    import torch
    from crane_amd import ops
    lens, P, B, Hq, Hkv = [4200 + 5 * b for b in range(32)], 256, 32, 8, 2
    table, total = ts.layout(910, lens, [list(range(B))], [4096], P)
    k, v = ts.pools(911, total, Hkv, P, table, lens, False)
    q = cases.normal(cases.rng(912), (B, Hq, S, D))
    q, k, v, table, n = (ts.tens(q, dtype, gpu), ts.tens(k, dtype, gpu), ts.tens(v, dtype, gpu), ts.ints(table, gpu),
                         ts.ints(lens, gpu))
    g = ops.prefix_groups([list(range(B))], [4096], B, gpu)
    run = lambda: ops.attention_shared_paged(q, k, v, table, n, max(lens), g)
    want = run()
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream(gpu).wait_stream(side)
    assert torch.equal(other, want)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for step in range(4):
        n.copy_(ts.ints([x - 5 * step for x in lens], gpu))
        for graph, _ in graphs:
            graph.replay()
        want = run()
        torch.cuda.synchronize(gpu)
        for _, out in graphs:
            assert torch.equal(out, want), step


# ------------------------------------------------------------------ the manager

def manager_lens(step):
    """Lengths of the batch of test_manager_batches_that_share: 24 forks of a prompt of
    3000 rows (11 pages shared), 9 of another of 2304 (9 pages), one alone, in this order."""
    return [3000 + step + b % 3 for b in range(24)] + [2304 + step + b % 2 for b in range(9)] + [70 + step]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_manager_batches_share(host, dtype):  # noqa: F811
    for step, S in ((1, 1), (4, 3)):
        lens = manager_lens(step)
        own = [n - (11 * 256 if b < 24 else 9 * 256 if b < 33 else 0) for b, n in enumerate(lens)]
        p = plan(host, [(24, 11 * 256), (9, 9 * 256)], max(lens), max(own), sum(own) // len(own), len(lens), S, 8, 2,
                 dtype == "bf16")
        assert p["share"], (step, S, p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_manager_batches_that_share(gpu, dtype):
    """Two forked prompts and a sequence of its own in one batch, in a shuffled order:
    the cache's own groups steer calls that share, of one and of three tokens, before and
    after a compaction that moves the shared pages."""
    import torch
    from crane_amd import kv
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    r = cases.rng(930)
    Hkv, Hq, P = 2, 8, 256
    c = kv.PagedKvCache(Hkv, 140, td, P, max_seqs=40, max_pages_per_seq=16, device=gpu)
    rand = lambda *shape: ts.tens(cases.normal(r, shape), dtype, gpu)
    filler = c.add_sequence()
    c.write_sequence(filler, rand(Hkv, 2000, D), rand(Hkv, 2000, D))
    ids = []
    for n, count in ((3000, 24), (2304, 9)):
        sid = c.add_sequence()
        c.write_sequence(sid, rand(Hkv, n, D), rand(Hkv, n, D))
        ids += [sid] + c.fork_sequence(sid, count - 1)
    ids.append(c.add_sequence())
    c.write_sequence(ids[-1], rand(Hkv, 70, D), rand(Hkv, 70, D))
    start = manager_lens(0)
    for b, sid in enumerate(ids):                                # lengths apart by up to 2 rows
        extra = start[b] - c.seq_len(sid)
        if extra:
            c.set_batch([sid])
            c.update_kv_cache(rand(1, Hkv, extra, D), rand(1, Hkv, extra, D))
    order = [int(x) for x in r.permutation(len(ids))]
    batch = [ids[x] for x in order]
    c.set_batch(batch)
    step = 0
    for S, compacted in ((1, False), (3, False), (1, True), (3, True)):
        if compacted and S == 1:
            c.free_sequence(filler)
            assert c.compact() > 0                               # the batch and its table follow
        c.update_kv_cache(rand(len(ids), Hkv, S, D), rand(len(ids), Hkv, S, D))
        step += S
        assert c.lengths == [manager_lens(step)[x] for x in order]
        q = cases.cast(cases.normal(r, (len(ids), Hq, S, D)), dtype)
        qq = ts.tens(q, dtype, gpu)
        got = c.attention_shared(qq if S > 1 else qq.view(len(ids), Hq, D))
        for x in (0, 7, 23, 24, 32, 33):
            b = order.index(x)
            kk, vv = (y.float().cpu().numpy() for y in c.read_sequence(batch[b]))
            n = kk.shape[1]
            out, mag, most = ts.reference(q[b:b + 1], kk[None], vv[None], np.zeros((1, 1), np.int32), [n], n,
                                          D ** -0.5, True)
            check(got[b:b + 1], out, ts.bounds(out, mag, most, n, dtype))
    c.close()
