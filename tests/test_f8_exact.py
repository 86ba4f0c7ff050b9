"""The paged KV cache in 8 bits (include/crane_f8.h) where a result is known to the bit, or to
a bound on its norm: what the elementwise bounds of test_f8.py leave room for."""
import math

import pytest
import torch

import test_f8 as f8
from test_f8 import BLOCK, D, DTYPES, gpu_test, ints

# Every form: 16 query rows a wave, whole and cut, its chunks joined by 1, 4 and 16 waves; 32
# rows (bf16), whole and cut; blocks of 128.  [lengths], S, Hq, Hkv
FORMS = [([700], 1, 2, 1), ([5000] * 100, 1, 4, 1), ([3000], 1, 8, 4), ([9000], 1, 4, 1), ([700] * 20, 48, 8, 8),
         ([3000] * 11 + [1700], 5, 32, 8), ([700], 700, 300, 1)]


def set_rows(c, which, b, x, byte=127):
    """Rows of sequence b: x [n, D] of every head, under one scale."""
    code = f8.encode(x.double(), torch.tensor(byte))
    for j in range(0, x.shape[0], c.P):
        page, m = int(c.table[b, j // c.P]), min(c.P, x.shape[0] - j)
        c.codes[which, page, :, :m] = code[j:j + m]
        c.scales[which, page, :, :-(-m // BLOCK)] = byte


# ------------------------------------------------------------------ the append

@gpu_test
@pytest.mark.parametrize("stale", [0xff, 254, 200, 0])
@pytest.mark.parametrize("skipped", [1, 2, 5, 40])
@pytest.mark.parametrize("S", [1, 3])
def test_block_that_begins_with_rows_that_are_not_written(gpu, S, skipped, stale):
    """New rows whose positions are outside the tables begin blocks, over scales that earlier
    owners left; the rows that come after them are as in blocks of the smallest scale."""
    from crane_amd import ops
    lens = [64, 0, 32]
    cos, sin = (x.to(gpu) for x in f8.tables(200, torch.bfloat16))
    g = torch.Generator().manual_seed(skipped)
    first, then = (torch.randn((3, n, 8 * D), generator=g).to(gpu, torch.bfloat16) for n in (skipped, S))
    outs = []
    for byte in (stale, f8.FLOOR):
        c = f8.Cache(2, lens, 2, ahead=skipped + S)
        for b, n in enumerate(lens):
            page, block = c.block(b, torch.arange(n, n + skipped + S, BLOCK))
            c.scales[0, page, :, block] = byte
        pools, table = c.to(gpu)
        at = ints(lens, gpu)
        ops.qk_norm_rope_append_paged_f8(first, cos, sin, ints([300, -skipped, 1000], gpu), pools, table, at, 4)
        at = at + skipped
        ops.qk_norm_rope_append_paged_f8(then, cos, sin, at, pools, table, at, 4)
        outs.append(pools)
    for b, n in enumerate(lens):
        page, row = c.at(b, torch.arange(n + skipped, n + skipped + S))
        for which in (0, 1):
            codes, want = (p[which].view(torch.uint8).cpu()[page, :, row] for p in outs)
            assert torch.equal(codes, want) and ((codes & 0x7f) != 0x7f).all() and (codes & 0x7f).any()
            scales, want = (p[2 + which].view(torch.uint8).cpu()[page, :, row // BLOCK] for p in outs)
            assert torch.equal(scales, want)


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 3])
@pytest.mark.parametrize("held", [0, 5])
def test_finite_values_stay_finite(gpu, dtype, S, held):
    """The largest values of the types: their codes times their scales are finite too, and read
    so; an infinity is a NaN."""
    from crane_amd import ops
    t = DTYPES[dtype]
    top = 2.0 ** 127
    x = torch.tensor([torch.finfo(t).max, -torch.finfo(t).max, 1.9375 * top, 1.921875 * top, 1.875 * top, -1.8125 * top,
                      1.78125 * top, 3e38, 1e38, -1e36, math.inf, math.nan], dtype=torch.float64).to(t)
    want = torch.tensor([1.875, -1.875, 1.875, 1.875, 1.875, -1.75, 1.75, 1.75, 0.5625, -0.00585937500, math.nan, math.nan],
                        dtype=torch.float64) * top
    c = f8.Cache(2, [held], 1, ahead=S)
    pools, table = c.to(gpu)
    cos, sin = (y.to(gpu) for y in f8.tables(64, t))
    qkv = torch.zeros((1, S, 3 * D), dtype=t)
    qkv[0, S - 1, 2 * D:2 * D + len(x)] = x
    at = ints([held], gpu)
    ops.qk_norm_rope_append_paged_f8(qkv.to(gpu), cos, sin, at, pools, table, at, 1, order="rope_only")
    v = ops.read_paged_f8(pools, table, at + S, held + S, torch.float32)[1][0, 0, held + S - 1, :len(x)]
    assert torch.equal(torch.nan_to_num(v.cpu().double(), nan=7.0), torch.nan_to_num(want, nan=7.0))


@gpu_test
@pytest.mark.parametrize("byte", [1, 26, 247, 253, 254])
@pytest.mark.parametrize("S", [1, 3])
def test_append_to_scales_that_no_append_writes(gpu, S, byte):
    """Rows that join a block whose scale is any of the format's: the smallest, below the append's
    own, and the largest."""
    from crane_amd import ops
    c = f8.Cache(2, [5], 1, ahead=S)
    page, block = (int(x) for x in c.block(0, 0))
    c.scales[1, page, :, block] = byte
    pools, table = c.to(gpu)
    qkv = torch.zeros((1, S, 3 * D))
    x = torch.tensor([1.5, 1.0, -1.25, 0.75]) * 2.0 ** min(byte - 127, 127)
    qkv[0, S - 1, 2 * D:2 * D + 4] = x
    cos, sin = (y.to(gpu) for y in f8.tables(64, torch.float32))
    at = ints([5], gpu)
    ops.qk_norm_rope_append_paged_f8(qkv.to(gpu), cos, sin, at, pools, table, at, 1, order="rope_only")
    have = int(pools[3].view(torch.uint8)[page, 0, block])
    assert have == max(byte, f8.FLOOR)
    want = f8.encode(x.double(), torch.tensor(have))
    assert torch.equal(pools[1].view(torch.uint8)[page, 0, 5 + S - 1, :4].cpu(), want)


# ------------------------------------------------------------------ attention

@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,G", [(6, 3), (140, 3), (500, 400)])
def test_hidden_largest_values_reach_nobody(gpu, dtype, S, G):
    """A chunk whose last token's v is the largest there is: earlier queries get what they get
    with zeros in its place."""
    from crane_amd import ops
    t, n = DTYPES[dtype], S + 90
    c = f8.Cache(8, [90], 1, ahead=S)
    pools, table = c.to(gpu)
    cos, sin = (x.to(gpu) for x in f8.tables(n, t))
    qkv = torch.randn((1, S, (G + 2) * D), generator=torch.Generator().manual_seed(1)).to(t)
    qkv[0, S - 1, (G + 1) * D:] = torch.finfo(t).max
    at = ints([90], gpu)
    q = ops.qk_norm_rope_append_paged_f8(qkv.to(gpu), cos, sin, at, pools, table, at, G)
    got = ops.attention_paged_f8(q, pools, table, at + S, n)
    page, row = (int(x) for x in c.at(0, n - 1))
    pools[1].view(torch.uint8)[page, :, row] = 0
    want = ops.attention_paged_f8(q, pools, table, at + S, n)
    assert torch.isfinite(got[:, :-1]).all() and torch.equal(got[:, :-1], want[:, :-1])


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,S,Hq,Hkv", FORMS)
def test_rows_of_one_value(gpu, dtype, lens, S, Hq, Hkv):
    """Where all rows of V are the same, so is the result, whatever the weights: 1 for the first
    64 keys and 1 + 0.99 2^-8 for the others, which bf16 rounds to 1, in the product as in the
    sum.  The result is v to the sums' n + 64 half steps of f32, and to the bit after bf16's
    rounding."""
    from crane_amd import ops
    c = f8.Cache(1, lens, Hkv)
    v = torch.where(torch.arange(D) % 2 == 0, 1.0, -1.0) * (1 + torch.arange(D) % 8 / 8)
    for b, n in enumerate(lens):
        k = torch.zeros((n, D))
        k[64:, 0] = 1.0
        set_rows(c, 0, b, k)
        set_rows(c, 1, b, v.expand(n, D))
    q = torch.zeros((len(lens), Hq, S, D), dtype=DTYPES[dtype])
    q[..., 0] = 1.0
    pools, table = c.to(gpu)
    got = ops.attention_paged_f8(q.to(gpu), pools, table, ints(lens, gpu), max(lens), math.log1p(0.99 * 2.0 ** -8))
    want = v.double().repeat(Hq).expand(got.shape)
    if dtype == "bf16":
        assert torch.equal(got.cpu().double(), want)
    else:
        assert ((got.cpu().double() - want).abs() <= (max(lens) + 64) * 2.0 ** -24 * want.abs()).all()


def large_scores(c, lens, S, Hq, seed, rising):
    """Keys whose scores are 2^20 + d, d whole numbers up to 11 in any order or up to 48 and
    rising, all exact in f32, for queries of (2^20, 1, 0 ..); (q, [d] per sequence)."""
    g = torch.Generator().manual_seed(seed)
    steps = torch.tensor([*range(17), *range(18, 33, 2), *range(36, 49, 4)])
    ds = []
    for b, n in enumerate(lens):
        d = steps[torch.arange(n) * len(steps) // max(n, 1)] if rising else torch.randint(0, 12, (n,), generator=g)
        k = torch.zeros((n, D))
        k[:, 0], k[:, 1] = 1.0, d.float()
        set_rows(c, 0, b, k)
        ds.append(d.double())
    q = torch.zeros((len(lens), Hq, S, D))
    q[..., 0], q[..., 1] = 2.0 ** 20, 1.0
    return q, ds


@gpu_test
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,S,Hq,Hkv", FORMS)
def test_weights_of_large_scores(gpu, dtype, lens, S, Hq, Hkv, rising):
    """Scores near 2^20, where half a step of f32 is 2^-5 and a weight that far off 2%: the maxima
    that tiles, waves and chunks count from differ, and their partial results have to join
    as if there was no rounding.  A weight's exponent, 24 at most where the weight counts, is off
    by 4 of its half steps (scale, log2 e, their product, the result's)."""
    from crane_amd import ops
    c = f8.Cache(5, lens, Hkv)
    q, ds = large_scores(c, lens, S, Hq, 6, rising)
    scale = float(torch.tensor(0.7))
    pools, table = c.to(gpu)
    got = ops.attention_paged_f8(q.to(gpu, DTYPES[dtype]), pools, table, ints(lens, gpu), max(lens), scale).cpu().double()
    for b, n in enumerate(lens):
        v = c.rows(1, b, n)
        w = torch.exp(scale * (ds[b] - ds[b].max()))[None, :, None]
        at = torch.arange(n - S, n)
        den = w.cumsum(1)[:, at]
        ref, mag = ((w * x).cumsum(1)[:, at] / den for x in (v, v.abs()))
        tol = f8.HALF[dtype] * (ref.abs() + mag) + mag * (2 * 24 * 4 + n + 64) * 2.0 ** -24
        have = got[b].view(S, Hkv, Hq // Hkv, D)
        for i in range(Hq // Hkv):
            bad = ~((have[:, :, i].transpose(0, 1) - ref).abs() <= tol)
            assert not bad.any(), (b, i, float(((have[:, :, i].transpose(0, 1) - ref).abs() / tol).max()))


@gpu_test
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S,Hq,bound", [(1, 4, 300), (5, 4, 300), (40, 2, 1100), (200, 400, 256)])
def test_a_longer_sequence_counts_as_the_bound(gpu, S, Hq, bound, causal):
    """Chunks of a sequence past max_kv: its queries sit at the last rows of max_kv."""
    from crane_amd import ops
    c = f8.Cache(2, [1400, 90], 1)
    pools, table = c.to(gpu)
    q = torch.randn((2, Hq, S, D), generator=torch.Generator().manual_seed(3)).to(gpu, torch.bfloat16)
    a, b = (ops.attention_paged_f8(q, pools, table, ints([n, 90], gpu), bound, causal=causal) for n in (1400, bound))
    assert torch.equal(a, b)


# Of f32 attention in the norm, random rows.  A weight's exponent is up to 16 in size and rounded
# once, uniformly within 2^-20 (a root mean square of 3.8e-7 of the weight), its score is a sum
# of 12 such steps of sums a quarter as large (3.3e-7), exp2, the weights' product and the sums
# are off by a few half steps of 1 (2e-7); half as much again for the inputs at hand.
NORM = 8e-7 * 1.5


def parts(x, n):
    """The first n bf16 parts of f32 values, each the rounding of what the ones before leave."""
    out = torch.zeros_like(x)
    for _ in range(n):
        out = out + (x - out).bfloat16().float()
    return out


@pytest.mark.parametrize("n", [33, 700, 5000])
@pytest.mark.parametrize("q_parts,w_parts", [(3, 3), (2, 3), (3, 2)])
def test_the_norm_tells_parts_apart(n, q_parts, w_parts):
    """With two bf16 parts of q or of the weights the result is past the bound, with three it is
    a tenth of it (everything else exact)."""
    c = f8.Cache(1, [n], 1)
    q = 1.5 * torch.randn((1, 4, 1, D), generator=torch.Generator().manual_seed(2))
    ref, _, _ = f8.reference(c, q, [n], D ** -0.5, True)
    s = parts(q[0, :, 0], q_parts).double() @ c.rows(0, 0, n)[0].T * D ** -0.5
    w = torch.exp(s - s.amax(1, keepdim=True))
    out = parts(w.float(), w_parts).double() @ c.rows(1, 0, n)[0] / w.sum(1, keepdim=True)
    off = (out.view(-1) - ref.view(-1)).norm() / ref.norm()
    assert off < NORM / 10 if q_parts == w_parts == 3 else off > NORM


@gpu_test
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,S,Hq,Hkv", FORMS)
def test_f32_keeps_its_bits(gpu, lens, S, Hq, Hkv, causal):
    """f32 calls carry q and the weights in three parts: within a bound that two exceed."""
    from crane_amd import ops
    c = f8.Cache(7, lens, Hkv)
    q = 1.5 * torch.randn((len(lens), Hq, S, D), generator=torch.Generator().manual_seed(8))
    pools, table = c.to(gpu)
    got = ops.attention_paged_f8(q.to(gpu), pools, table, ints(lens, gpu), max(lens), causal=causal).cpu().double()
    ref, _, _ = f8.reference(c, q, lens, D ** -0.5, causal)
    assert (got - ref).norm() <= NORM * ref.norm(), float((got - ref).norm() / ref.norm())


@pytest.mark.parametrize("scale,code", [(3.4e38, 1), (2.4e38, 1), (2.3e38, 0), (1e-45, 0)])
def test_scales_whose_product_overflows_are_refused(scale, code):
    """In base 2 the exponents' factor is scale log2 e: past 2^128 every weight would be NaN."""
    assert f8._attn(scale=scale) == code
