"""The paged cache manager with rows in 8 bits (include/crane_pkv.h): what it holds is
checked against the format's definition in 64 bits, its append and attention against the
launchers they stand for, to the last bit."""
import ctypes

import pytest
import torch

D, BLOCK, FLOOR = 128, 32, 27
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
gpu_test = pytest.mark.gpu


def held(k, start=0, before=None):
    """What a cache gives back for rows k [Hkv, n, D] appended in one call behind the `start`
    rows of `before` [(rows as held, float64), (scale exponents [Hkv, blocks])]: the same pair."""
    Hkv, n, _ = k.shape
    rows = torch.zeros((Hkv, start + n, D), dtype=torch.float64)
    exps = torch.full((Hkv, -(-(start + n) // BLOCK)), FLOOR - 127, dtype=torch.int64)
    if start:
        rows[:, :start] = before[0][:, :start]
        exps[:, :-(-start // BLOCK)] = before[1][:, :-(-start // BLOCK)]
    rows[:, start:] = k.double().cpu()
    for j in range(start // BLOCK * BLOCK, start + n, BLOCK):
        new = rows[:, max(j, start):min(j + BLOCK, start + n)].abs().amax((1, 2))
        e = torch.ceil(torch.log2(new.clamp_min(2.0 ** -300) / 448)).long()
        exps[:, j // BLOCK] = torch.maximum(exps[:, j // BLOCK], e)
        s = torch.exp2(exps[:, j // BLOCK].double())[:, None, None]
        x = rows[:, j:min(j + BLOCK, start + n)] / s  # a held row's code anew, or a new row's
        rows[:, j:min(j + BLOCK, start + n)] = x.float().to(E4M3).double() * s
    return rows, exps


def rows_of(g, n, Hkv, dtype, spread=1.0):
    return [(torch.randn((Hkv, n, D), generator=g) * spread).to(dtype) for _ in "kv"]


def cache_of(gpu, Hkv, dtype, n_pages=12, P=256, max_seqs=6, pps=4):
    from crane_amd.kv import PagedKvCache
    return PagedKvCache(Hkv, n_pages, dtype, P, max_seqs, pps, gpu, kv_dtype=E4M3)


def qkv_of(g, B, S, H, dtype, gpu):
    return torch.randn((B, S, H * D), generator=g).to(dtype).to(gpu)


def tables(n, dtype, gpu):
    freq = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    angle = torch.arange(n)[:, None] * freq
    return angle.cos().to(dtype).to(gpu), angle.sin().to(dtype).to(gpu)


@gpu_test
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hkv,P", [(1, 256), (2, 512), (3, 256)])
def test_write_update_read(gpu, dtype, Hkv, P):
    """Rows that come in are held by the definition, wherever in a block they begin."""
    g = torch.Generator().manual_seed(Hkv)
    c = cache_of(gpu, Hkv, dtype, P=P)
    lens = [0, 1, 31, 32, 300]
    ids = [c.add_sequence() for _ in lens]
    want = {}
    for sid, n in zip(ids, lens):
        k, v = rows_of(g, n, Hkv, dtype)
        c.write_sequence(sid, k.to(gpu), v.to(gpu))
        want[sid] = [held(x) if n else (torch.zeros((Hkv, 0, D), dtype=torch.float64), None) for x in (k, v)]
    c.set_batch(ids)
    for S, spread in ((1, 1.0), (40, 5.0), (3, 2.0 ** -6), (1, 300.0)):
        new = [rows_of(g, S, Hkv, dtype, spread) for _ in ids]
        c.update_kv_cache(*(torch.stack([x[i] for x in new]).to(gpu) for i in (0, 1)))
        for i, sid in enumerate(ids):
            want[sid] = [held(new[i][w], lens[i], want[sid][w]) for w in (0, 1)]
        lens = [n + S for n in lens]
    assert c.lengths == lens
    for sid, n in zip(ids, lens):
        for got, ref in zip(c.read_sequence(sid), want[sid]):
            assert got.shape == (Hkv, n, D) and got.dtype == dtype
            assert torch.equal(got.cpu().double(), ref[0])


@gpu_test
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompts_then_tokens(gpu, dtype):
    """append_qkv, prefill and decode are the launchers' over the manager's pools; pages open
    as the sequences grow."""
    from crane_amd import ops
    Hq, Hkv, P = 4, 2, 256
    g = torch.Generator().manual_seed(5)
    c = cache_of(gpu, Hkv, dtype, P=P)
    cos, sin = tables(800, dtype, gpu)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(gpu) for _ in "qk"]
    ids = [c.add_sequence() for _ in range(3)]
    start = [0, 250, 33]
    for sid, n in zip(ids, start):
        c.write_sequence(sid, *(x.to(gpu) for x in rows_of(g, n, Hkv, dtype)))
    c.set_batch(ids)
    for S in (60, 1, 1, 5):
        lens = torch.tensor(start, dtype=torch.int32, device=gpu)
        qkv = qkv_of(g, 3, S, Hq + 2 * Hkv, dtype, gpu)
        before = [x.clone() for x in c.pools()]
        q = c.append_qkv(qkv, cos, sin, lens, Hq, *w)
        q2 = ops.qk_norm_rope_append_paged_f8(qkv, cos, sin, lens, before, c.block_table(), lens, Hq, *w)
        start = [n + S for n in start]
        assert torch.equal(q, q2) and c.lengths == start and c.device_lengths().tolist() == start
        for sid, n, row in zip(ids, start, c.block_table().cpu()):
            ks, vs = ops.read_paged_f8(before, row[None].to(gpu), torch.tensor([n], dtype=torch.int32, device=gpu), n,
                                       dtype)
            k, v = c.read_sequence(sid)
            assert torch.equal(k, ks[0]) and torch.equal(v, vs[0])
        now = torch.tensor(start, dtype=torch.int32, device=gpu)
        for causal in (True, False):
            ref = ops.attention_paged_f8(q, c.pools(), c.block_table(), now, max(start), causal=causal)
            assert torch.equal(c.prefill(q, causal=causal), ref)
        if S == 1:
            assert torch.equal(c.decode(q[:, :, 0]), ops.attention_paged_f8(q, c.pools(), c.block_table(), now,
                                                                            max(start)))


@gpu_test
def test_workspace(gpu):
    """A batch long enough for its sequences to be cut: with the workspace that the call
    takes, with one that is given, and one too small."""
    from crane_amd import CraneHipError, _lib, ops
    g = torch.Generator().manual_seed(6)
    c = cache_of(gpu, 1, torch.bfloat16, n_pages=20, pps=16)
    sid = c.add_sequence()
    c.write_sequence(sid, *(x.to(gpu) for x in rows_of(g, 4000, 1, torch.bfloat16)))
    c.set_batch([sid])
    q = torch.randn((1, 4, D), generator=g).bfloat16().to(gpu)
    need = _lib.lib().crane_pkv_attention_f8_workspace(c._h, 4, 1)
    assert need == _lib.lib().crane_hip_attn_paged_f8_workspace(4000, 1, 1, 4, 1, D, _lib.BF16) > 0
    ref = ops.attention_paged_f8(q, c.pools(), c.block_table(), c.device_lengths(), 4000)
    assert torch.equal(c.decode(q), ref)
    assert torch.equal(c.decode(q, workspace=torch.full((need,), 0xff, dtype=torch.uint8, device=gpu)), ref)
    with pytest.raises(CraneHipError) as e:
        c.decode(q, workspace=torch.empty(need - 16, dtype=torch.uint8, device=gpu))
    assert e.value.code == _lib.E_WORKSPACE


@gpu_test
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hkv", [1, 2])
def test_fork_truncate_compact(gpu, dtype, Hkv):
    """Rows keep their values through copies of pages; what a child appends is its own."""
    from crane_amd import kv
    g = torch.Generator().manual_seed(7 + Hkv)
    layers = [cache_of(gpu, Hkv, dtype, n_pages=16) for _ in range(2)]
    plain = kv.PagedKvCache(Hkv, 16, dtype, 256, 6, 4, gpu)  # a layer in the model's type, driven along
    caches = layers + [plain]
    first, sid = ([c.add_sequence() for c in caches][0] for _ in "ab")
    for c in caches:
        c.write_sequence(first, *(x.to(gpu) for x in rows_of(g, 300, Hkv, dtype)))
    rows = [rows_of(g, 700, Hkv, dtype) for _ in caches]
    for c, (k, v) in zip(caches, rows):
        c.write_sequence(sid, k.to(gpu), v.to(gpu))
    was = [c.read_sequence(sid) for c in caches]
    kids = kv.fork_sequence(caches, sid, 2, 590)  # two full pages shared, 78 rows of the third copied
    new = [rows_of(g, 20, Hkv, dtype, 40.0) for _ in caches]
    for c, (k, v) in zip(caches, new):
        assert c.free_pages == 16 - 2 - 3 - 2
        c.set_batch(kids[:1])
        c.update_kv_cache(k[None].to(gpu), v[None].to(gpu))
        c.set_batch([])
    for c, w in zip(caches, was):
        for got, ref in zip(c.read_sequence(sid), w):
            assert torch.equal(got, ref)  # the parent's rows are as they were
        for got, ref in zip(c.read_sequence(kids[1]), w):
            assert torch.equal(got, ref[:, :590])
        for got, ref in zip(c.read_sequence(kids[0]), w):
            assert got.shape[1] == 610 and torch.equal(got[:, :576], ref[:, :576])
    for c, (k, v) in zip(layers, new):
        # rows 576 .. 589 were held with rows up to 607 of the parent, whose scale stays the least
        for which, x in ((0, k), (1, v)):
            src = rows[caches.index(c)][which]
            exps = held(src)[1][:, :19]
            want = held(x, 590, (was[caches.index(c)][which].cpu().double(), exps))[0]
            assert torch.equal(c.read_sequence(kids[0])[which].cpu().double(), want)
    kv.truncate_sequence(caches, kids[1], 300)  # a shared page becomes partial
    for c in caches:
        c.free_sequence(first)
    assert kv.compact(caches) > 0
    for c, w in zip(caches, was):
        for got, ref in zip(c.read_sequence(kids[1]), w):
            assert torch.equal(got, ref[:, :300])
        for got, ref in zip(c.read_sequence(sid), w):
            assert torch.equal(got, ref)
        used = 16 - c.free_pages
        c.set_batch([sid, kids[0], kids[1]])
        table = c.block_table()
        assert int(table[table >= 0].max()) == used - 1
    for c in layers:  # attention follows the moved pages
        from crane_amd import ops
        q = torch.randn((3, 2 * Hkv, D), generator=g).to(dtype).to(gpu)
        k, v = c.pools()[:2]
        assert k.shape == (16, Hkv, 256, D)
        out = c.decode(q)
        assert torch.equal(out, ops.attention_paged_f8(q, c.pools(), c.block_table(), c.device_lengths(), 700))


@gpu_test
def test_block_begun_anew_forgets_its_scale(gpu):
    """Truncated to a multiple of 32 rows, the next block's old scale has no part; cut inside a
    block, its scale stays.  (Codes from 256 on are 32 apart: 400, halfway from 384 to 416, is
    held as the even one, 1.5 2^8.)"""
    c = cache_of(gpu, 1, torch.bfloat16)
    big = torch.full((1, 64, D), 400.0, dtype=torch.bfloat16, device=gpu)
    small = torch.full((1, 1, 8, D), 2.0 ** -12, dtype=torch.bfloat16, device=gpu)
    for rows, expect in ((32, 2.0 ** -12), (40, 0.0)):
        sid = c.add_sequence()
        c.write_sequence(sid, big, big)
        c.truncate_sequence(sid, rows)
        c.set_batch([sid])
        c.update_kv_cache(small, small)
        c.set_batch([])
        for x in c.read_sequence(sid):
            assert (x[:, :rows] == 384).all() and (x[:, rows:] == expect).all()


@gpu_test
def test_sizes_and_refusals(gpu):
    from crane_amd import CraneHipError, _lib, kv, ops
    c = cache_of(gpu, 2, torch.bfloat16)
    pools = c.pools()
    assert [x.dtype for x in pools] == [E4M3, E4M3, E8M0, E8M0]
    assert [x.shape for x in pools] == [x.shape for x in ops.f8_pools(12, 2, 256, gpu)]
    assert c.bytes == sum(x.numel() for x in pools) and c.kv_dtype == E4M3 and c.dtype == torch.bfloat16
    plain = kv.PagedKvCache(2, 12, torch.bfloat16, device=gpu)
    assert plain.kv_dtype == torch.bfloat16
    sid = c.add_sequence()
    z = torch.zeros((2, 5, D), dtype=torch.bfloat16, device=gpu)
    c.write_sequence(sid, z, z)
    c.set_batch([sid])
    q = torch.zeros((1, 2, D), dtype=torch.bfloat16, device=gpu)

    def refused(code, f):
        with pytest.raises(CraneHipError) as e:
            f()
        assert e.value.code == code

    refused(_lib.E_DTYPE, lambda: kv.PagedKvCache(2, 12, torch.bfloat16, device=gpu, kv_dtype=torch.float32))
    refused(_lib.E_DTYPE, lambda: kv.PagedKvCache(2, 12, torch.bfloat16, device=gpu, kv_dtype=torch.float8_e5m2))
    refused(_lib.E_INVALID, lambda: c.decode(q, score_mode="candle"))
    refused(_lib.E_INVALID, lambda: c.prefill(q[:, :, None], long_rows_one_rounding=True))
    refused(_lib.E_DTYPE, lambda: c.attention_shared(q))
    refused(_lib.E_DTYPE, lambda: c.decode(q.float()))
    refused(_lib.E_INVALID, lambda: c.prefill(torch.zeros((1, 2, 6, D), dtype=torch.bfloat16, device=gpu)))
    L, p, st = _lib.lib(), q.data_ptr(), torch.cuda.current_stream().cuda_stream
    assert L.crane_pkv_decode(c._h, p, 2, 0.1, 0, None, 0, p, st) == _lib.E_DTYPE
    assert L.crane_pkv_prefill(c._h, p, 2, 1, 0.1, 1, p, st) == _lib.E_DTYPE
    assert L.crane_pkv_attention_f8(plain._h, p, 2, 1, 0.1, 1, None, 0, p, st) == _lib.E_DTYPE
    assert L.crane_pkv_attention_f8_workspace(plain._h, 2, 1) == 0
    a, b = ctypes.c_void_p(), ctypes.c_void_p()
    assert L.crane_pkv_scales_f8(plain._h, ctypes.byref(a), ctypes.byref(b)) == _lib.E_DTYPE
    # rows on the host, of another width, and a workspace that is not what its size says
    one = z[None, :, :1]
    refused(_lib.E_INVALID, lambda: c.update_kv_cache(one.cpu(), one.cpu()))
    refused(_lib.E_INVALID, lambda: c.update_kv_cache(one, one.cpu()))
    refused(_lib.E_INVALID, lambda: c.update_kv_cache(one[..., :64], one[..., :64]))
    other = c.add_sequence()
    refused(_lib.E_INVALID, lambda: c.write_sequence(other, z.cpu(), z.cpu()))
    refused(_lib.E_INVALID, lambda: c.decode(q, workspace=torch.empty(1, device=gpu).expand(1 << 20)))
    c.free_sequence(other)
    # a batch without rows, and a full cache: nothing changes
    empty = c.add_sequence()
    c.set_batch([empty])
    refused(_lib.E_INVALID, lambda: c.decode(q))
    many = torch.zeros((1, 2, 4 * 256 + 1, D), dtype=torch.bfloat16, device=gpu)
    refused(_lib.E_CAPACITY, lambda: c.update_kv_cache(many, many))
    cos, sin = tables(2000, torch.bfloat16, gpu)
    at = torch.zeros(1, dtype=torch.int32, device=gpu)
    refused(_lib.E_CAPACITY, lambda: c.append_qkv(torch.zeros((1, 1025, 6 * D), dtype=torch.bfloat16, device=gpu), cos,
                                                  sin, at, 2))
    assert c.lengths == [0] and c.free_pages == 11


def test_create_refuses():
    from crane_amd import _lib
    L, h = _lib.lib(), ctypes.c_void_p()
    make = lambda *a: L.crane_pkv_create_f8(*a, ctypes.byref(h))  # noqa: E731
    assert make(8, 128, 1, 100, 16, 4, 4) == _lib.E_INVALID  # page_rows
    assert make(8, 64, 1, 256, 16, 4, 4) == _lib.E_HEAD_DIM
    assert make(8, 128, 3, 256, 16, 4, 4) == _lib.E_DTYPE
    assert make(0, 128, 1, 256, 16, 4, 4) == _lib.E_INVALID
    assert make(8, 128, 1, 256, 0, 4, 4) == _lib.E_INVALID
    assert make(65535, 128, 1, 33024, 16, 4, 4) == _lib.E_INVALID  # a page's scales pass 2^31
    assert L.crane_pkv_create_f8(8, 128, 1, 256, 16, 4, 4, None) == _lib.E_INVALID
    assert L.crane_pkv_attention_f8(None, None, 1, 1, 0.1, 1, None, 0, None, None) == _lib.E_INVALID
    assert L.crane_pkv_attention_f8_workspace(None, 1, 1) == 0
    assert L.crane_pkv_scales_f8(None, None, None) == _lib.E_INVALID
