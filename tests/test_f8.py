"""The paged KV cache in 8 bits (include/crane_f8.h): the append that quantises, attention
over the codes, and the read.

Crane has no counterpart, so the reference is the definition in 64 bits, on the CPU.
Codes are checked two ways: v, which the append only quantises, to the last code, and k,
whose norm and rotation are f32 sums, to half a step of its code and the error of those
sums.  Attention is checked element by element against the bound that reference() gives.
Rows that no query may see hold NaN codes, under scale bytes of blocks without rows that
are NaN, too."""
import ctypes
import math

import pytest
import torch

D, BLOCK, FLOOR = 128, 32, 27
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # half a step, relative
gpu_test = pytest.mark.gpu


# ------------------------------------------------------------------ the format

def pow2(byte):
    return torch.exp2(byte.double() - 127)


def values(codes, scales):
    """Codes [..., rows, D] and scale bytes [..., rows / 32] (uint8, CPU) as float64."""
    return codes.view(E4M3).double() * pow2(scales).repeat_interleave(BLOCK, -1)[..., None]


def scale_byte(amax):
    """Of the smallest scale with amax <= 448 2^e, float64."""
    e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -300) / 448))
    return (e + 127).clamp_min(FLOOR).to(torch.int64)


def encode(x, byte):
    """Codes of float64 values for scale bytes of the same shape, nearest even (the values are
    f32's and times a power of two, so the cast to f32 is exact)."""
    y = (x * pow2(254 - byte)).float()
    code = y.to(E4M3).view(torch.uint8)
    return torch.where(torch.isfinite(y), code, 0x7f)


def same_codes(a, b):
    """Equal, any NaN counting as another."""
    return torch.equal(torch.where((a & 0x7f) == 0x7f, 0x7f, a), torch.where((b & 0x7f) == 0x7f, 0x7f, b))


class Cache:
    """Pools on the CPU with pages in shuffled order; entries of the table past a
    sequence's rows are of no page."""

    def __init__(self, seed, lens, Hkv, P=256, ahead=0, spread=1.0, spare=2, least=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.Hkv, self.P, self.B = list(lens), Hkv, P, len(lens)
        each = [-(-(n + ahead) // P) for n in lens]
        total = sum(each) + spare + least
        ids = (torch.randperm(total - least, generator=g) + least).tolist()
        width = max(each + [1]) + 1
        self.table = torch.full((self.B, width), -7, dtype=torch.int32)
        for b, n in enumerate(each):
            self.table[b, :n] = torch.tensor(ids[:n], dtype=torch.int32)
            ids = ids[n:]
        self.codes = torch.full((2, total, Hkv, P, D), 0x7f, dtype=torch.uint8)
        self.scales = torch.full((2, total, Hkv, P // BLOCK), 0xff, dtype=torch.uint8)
        for b, n in enumerate(lens):
            for j in range(0, n, BLOCK):
                m = min(BLOCK, n - j)
                page, row = int(self.table[b, j // P]), j % P
                x = torch.randn((2, Hkv, m, D), generator=g, dtype=torch.float64) * spread
                x = x.float().double()
                byte = scale_byte(x.abs().amax((2, 3)))
                self.codes[:, page, :, row:row + m] = encode(x, byte[..., None, None])
                self.scales[:, page, :, row // BLOCK] = byte.to(torch.uint8)

    def at(self, b, rows):
        """(pages, rows of them) of a sequence's rows."""
        rows = torch.as_tensor(rows)
        return self.table[b].long()[rows // self.P], rows % self.P

    def block(self, b, rows):
        """(pages, blocks of them) that a sequence's rows are in."""
        page, at = self.at(b, rows)
        return page, at // BLOCK

    def rows(self, which, b, n):
        """[Hkv, n, D] float64; zeros where the page is none of the pool's."""
        out = torch.zeros((self.Hkv, n, D), dtype=torch.float64)
        for j in range(0, n, self.P):
            page, m = int(self.table[b, j // self.P]), min(self.P, n - j)
            if 0 <= page < self.codes.shape[1]:
                out[:, j:j + m] = values(self.codes[which, page], self.scales[which, page])[:, :m]
        return out

    def to(self, dev):
        pools = (self.codes[0].to(dev).view(E4M3), self.codes[1].to(dev).view(E4M3),
                 self.scales[0].to(dev).view(E8M0), self.scales[1].to(dev).view(E8M0))
        return pools, self.table.to(dev)


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------ the append

def tables(n, dtype):
    freq = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    angle = torch.arange(n)[:, None] * freq
    return angle.cos().to(dtype), angle.sin().to(dtype)


def turn(x, w, cos, sin, order, eps):
    """x [S, H, D] float64 normed and rotated."""
    def unit(y):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        return y if w is None else y * w.double()
    if order == "norm_then_rope":
        x = unit(x)
    a, b = x[..., :64], x[..., 64:]
    x = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return unit(x) if order == "rope_then_norm" else x


def check_append(gpu, dtype, lens, S, Hq, Hkv, order, P=256, seed=0, shift=0, eps=1e-6, weights=True, edit=None,
                 spread=1.0, table_rows=None, drop_page=None):
    """The append at those lengths against the definition; edit(qkv [B, S, H, D]) changes the rows."""
    from crane_amd import ops
    t = DTYPES[dtype]
    c = Cache(seed, lens, Hkv, P, ahead=S, spread=spread)
    g = torch.Generator().manual_seed(seed + 1)
    B, H = len(lens), Hq + 2 * Hkv
    qkv = torch.randn((B, S, H, D), generator=g).to(t)
    if edit is not None:
        edit(qkv)
    q_w, k_w = ((1 + 0.3 * torch.randn(D, generator=g)).to(t) for _ in "qk") if weights else (None, None)
    n_table = table_rows or max(lens) + S + shift + 1
    cos, sin = tables(n_table, t)
    positions = [n + shift for n in lens]
    if drop_page is not None:
        c.table[drop_page] = c.codes.shape[1] + 3
    pools, table = c.to(gpu)
    up = lambda x: None if x is None else x.to(gpu)  # noqa: E731
    q = ops.qk_norm_rope_append_paged_f8(qkv.view(B, S, H * D).to(gpu), cos.to(gpu), sin.to(gpu), ints(positions, gpu),
                                         pools, table, ints(lens, gpu), Hq, up(q_w), up(k_w), eps, order)
    torch.cuda.synchronize()
    got = torch.stack([x.view(torch.uint8).cpu() for x in pools[:2]])
    got_scales = torch.stack([x.view(torch.uint8).cpu() for x in pools[2:]])
    want, want_scales = c.codes.clone(), c.scales.clone()
    q = q.cpu().double()
    for b in range(B):
        p = torch.arange(S) + positions[b]
        inside = (p >= 0) & (p < n_table)
        cs, sn = (x.double()[p.clamp(0, n_table - 1)][:, None] for x in (cos, sin))
        x = qkv[b].double()
        ref = turn(x[:, :Hq], q_w, cs, sn, order, eps).transpose(0, 1)[:, inside]
        # one rounding, and the f32 sums before it: 160 steps at most on a row's largest
        tol = HALF[dtype] * ref.abs() + 2.0 ** -16 * ref.abs().amax(-1, keepdim=True)
        assert ((q[b][:, inside] - ref).abs() <= tol).all(), (b, (q[b][:, inside] - ref).abs().max())
        if drop_page is not None and drop_page[0] == b:
            assert drop_page[1] * P <= lens[b] and lens[b] + S <= (drop_page[1] + 1) * P
            continue  # every row lands on the missing page
        rows = torch.arange(lens[b], lens[b] + S)
        for which in (0, 1):
            new = turn(x[:, Hq:Hq + Hkv], k_w, cs, sn, order, eps) if which == 0 else x[:, Hq + Hkv:]
            new = new.transpose(0, 1)                                                       # [Hkv, S, D]
            keep = inside if which == 0 else torch.ones(S, dtype=torch.bool)
            for j in range(lens[b] // BLOCK * BLOCK, lens[b] + S, BLOCK):
                mine = (rows >= j) & (rows < j + BLOCK) & keep
                if not mine.any():
                    continue
                page, block = (int(y) for y in c.block(b, j))
                y = new[:, mine]
                most = torch.where(torch.isfinite(y), y.abs(), 0.0).amax((1, 2))
                byte, had = scale_byte(most), want_scales[which, page, :, block].long()
                held = max(0, lens[b] - j)
                byte = torch.maximum(byte, had) if held else byte
                have = got_scales[which, page, :, block].long()
                if which == 0:  # the largest is an f32 sum: at a border either scale may be taken
                    near = (most / 448 / pow2(scale_byte(most)) - 1).abs() < 2.0 ** -16
                    near |= (most / 448 / pow2(scale_byte(most) - 1) - 1).abs() < 2.0 ** -16
                    byte = torch.where(near & ((have - byte).abs() == 1), have, byte)
                assert torch.equal(have, byte), (b, which, j, have, byte)
                want_scales[which, page, :, block] = byte.to(torch.uint8)
                old = want[which, page, :, j % P:j % P + held]
                want[which, page, :, j % P:j % P + held] = torch.where(
                    (byte > had)[:, None, None], encode(old.view(E4M3).double(), (127 + byte - had)[:, None, None]), old)
                r = rows[mine] % P
                if which == 1:
                    want[which, page, :, r] = encode(y, byte[:, None, None])
                else:
                    have = got[0, page][:, r]
                    val = have.view(E4M3).double() * pow2(byte)[:, None, None]
                    finite = torch.isfinite(y).all(-1, keepdim=True).expand_as(y)
                    size = y.abs().amax(-1, keepdim=True)
                    tol = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * pow2(byte)[:, None, None]) + 2.0 ** -16 * size
                    assert ((val - y).abs() <= tol)[finite].all(), (b, j)
                    want[0, page, :, r] = have
    assert torch.equal(got_scales, want_scales)
    for which in (0, 1):
        assert same_codes(got[which], want[which]), which
    return got, got_scales


@gpu_test
@pytest.mark.parametrize("order", ["norm_then_rope", "rope_then_norm", "rope_only"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,S,Hq,Hkv,P", [
    ([0], 1, 1, 1, 256), ([5, 31, 32, 255, 256, 0], 1, 4, 2, 256), ([100] * 9, 1, 14, 2, 512),
    ([0, 1, 31, 32], 2, 2, 2, 256), ([30, 255, 250, 7], 33, 4, 4, 256), ([0, 511, 77], 64, 5, 1, 512),
    ([3, 224], 300, 7, 1, 256)])
def test_append(gpu, dtype, order, lens, S, Hq, Hkv, P):
    check_append(gpu, dtype, lens, S, Hq, Hkv, order, P, seed=len(lens) + S)


@gpu_test
@pytest.mark.parametrize("S", [1, 3, 40])
@pytest.mark.parametrize("spread", [2.0 ** -20, 2.0 ** -3, 1.0, 300.0])
def test_append_grows_or_keeps_a_scale(gpu, S, spread):
    """Blocks that hold rows much smaller than the new ones (their codes are rounded again, most
    to subnormal ones or 0), somewhat smaller, of a size, and larger (the scale stays)."""
    check_append(gpu, "bf16", [31, 1, 20, 64, 0], S, 2, 2, "rope_only", spread=spread, seed=S)


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 6])
def test_append_extreme_values(gpu, dtype, S):
    """Zeros, values at and next to a scale's border, tiny and huge ones, infinities and NaN."""
    def edit(x):
        Hkv, s = 2, S - 1
        v = x[:, :, 4:]
        v[0] = 0                                    # nothing but zeros: the smallest scale
        v[1, s, 0, 0] = 448.0
        v[1, s, 1, 0] = 450.0                       # past it: the next scale
        v[2] *= 2.0 ** -110                         # below the smallest scale's steps
        v[3, s, 0] = 3e38
        v[4, s, 0, 7], v[4, s, 1, 9] = math.inf, -math.inf
        v[5, s, 0, 3] = math.nan
        v[6, s] = math.nan                          # a whole row
        x[7, s, 2:4, 5] = math.nan                  # k: the norm carries it through the row
        assert v.shape[2] == Hkv
    check_append(gpu, dtype, [5, 32, 9, 40, 0, 17, 64, 3], S, 2, 2, "rope_only", edit=edit, seed=3)


@gpu_test
@pytest.mark.parametrize("S", [1, 5])
def test_append_skips_what_has_no_place(gpu, S):
    """Positions outside the tables (q and k are not written, v is), a page outside the pool."""
    check_append(gpu, "bf16", [40, 7], S, 2, 1, "rope_only", shift=10, table_rows=20, seed=5)
    check_append(gpu, "bf16", [40, 9], S, 2, 1, "rope_only", shift=-42, table_rows=64, seed=6)
    check_append(gpu, "bf16", [40, 300, 9], S, 2, 1, "norm_then_rope", drop_page=(1, 1), seed=7, weights=False)


@gpu_test
def test_append_rows_of_wider_tensors(gpu):
    """qkv and the tables as views with a row stride of their own."""
    from crane_amd import ops
    c = Cache(1, [33, 2], 1, ahead=3)
    wide = torch.randn((2, 3, 5 * D), generator=torch.Generator().manual_seed(2)).to(gpu, torch.bfloat16)
    cos, sin = (x.to(gpu) for x in tables(64, torch.bfloat16))
    lens = ints([33, 2], gpu)
    outs = []
    for rows in (wide[:, :, D:4 * D], wide[:, :, D:4 * D].contiguous()):
        pools, table = c.to(gpu)
        q = ops.qk_norm_rope_append_paged_f8(rows, cos, sin, lens, pools, table, lens, 1)
        outs.append([q.view(torch.uint8)] + [p.view(torch.uint8) for p in pools])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@gpu_test
@pytest.mark.parametrize("S", [1, 5])
def test_append_before_the_first_row(gpu, S):
    """Rows before row 0 are not written; those from it on are, as in an empty sequence."""
    from crane_amd import ops
    cos, sin = (x.to(gpu) for x in tables(64, torch.bfloat16))
    qkv = torch.randn((1, S, 3 * D), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(gpu)
    got, want = ([x.clone() for x in Cache(1, [0], 1, ahead=S).to(gpu)[0]] for _ in "ab")
    table = Cache(1, [0], 1, ahead=S).to(gpu)[1]
    ops.qk_norm_rope_append_paged_f8(qkv, cos, sin, ints([7], gpu), got, table, ints([-3], gpu), 1)
    if S > 3:
        ops.qk_norm_rope_append_paged_f8(qkv[:, 3:].contiguous(), cos, sin, ints([10], gpu), want, table,
                                         ints([0], gpu), 1)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))


# ------------------------------------------------------------------ attention

def reference(c, q, lens, scale, causal):
    """(out [B, S, Hq D], bound on |result - out|) in float64; q [B, Hq, S, D]."""
    B, Hq, S, _ = q.shape
    G = Hq // c.Hkv
    out, mag = torch.zeros((B, S, Hq, D), dtype=torch.float64), torch.zeros((B, S, Hq, D), dtype=torch.float64)
    slack = torch.zeros((B, S, Hq, 1), dtype=torch.float64)
    for b, n in enumerate(lens):
        k, v = c.rows(0, b, n), c.rows(1, b, n)
        limit = torch.arange(n - S + 1, n + 1) if causal else torch.full((S,), n)
        hidden = torch.arange(n)[None, :] >= limit[:, None]
        for h in range(Hq if n else 0):
            x, kk, vv = q[b, h].double(), k[h // G], v[h // G]
            logits = (scale * (x @ kk.T)).masked_fill(hidden, -math.inf)
            w = torch.nan_to_num(torch.softmax(logits, 1))  # a row of nothing: zeros
            out[b, :, h], mag[b, :, h] = w @ vv, w @ vv.abs()
            # a score's sum of 128 products, its difference to the largest and its product with
            # log2 e are off by 132 half steps of f32 of the size of their terms at most, and so
            # is the largest; the sums over n keys by n
            most = scale * (x.abs() @ kk.abs().T).masked_fill(hidden, 0.0).amax(1)
            slack[b, :, h, 0] = 2 * 132 * 2.0 ** -24 * most + (n + 64) * 2.0 ** -24
    return out.view(B, S, Hq * D), mag.view(B, S, Hq * D), slack.expand(B, S, Hq, D).reshape(B, S, Hq * D)


def check_attention(gpu, dtype, lens, S, Hq, Hkv, P=256, causal=True, seed=0, scale=None, c=None, q=None, q3=True,
                    max_kv=None):
    from crane_amd import ops
    c = c or Cache(seed, lens, Hkv, P)
    if q is None:
        g = torch.Generator().manual_seed(seed + 1)
        q = (1.5 * torch.randn((len(lens), Hq, S, D), generator=g)).to(DTYPES[dtype])
    pools, table = c.to(gpu)
    qq = q[:, :, 0] if S == 1 and q3 else q
    got = ops.attention_paged_f8(qq.contiguous().to(gpu), pools, table, ints(lens, gpu), max_kv or max(max(lens), 1), scale,
                                 causal).cpu().double()
    ref, mag, slack = reference(c, q, lens, scale or D ** -0.5, causal)
    # the result's rounding, the probabilities' (bf16: half a step each; f32: three parts, 2^-24), the sums'
    tol = HALF[dtype] * (ref.abs() + mag) + mag * slack
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[:5], float(((got - ref).abs() / tol.clamp_min(1e-300)).max()))
    return got


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 2), (7, 1), (8, 1), (10, 2), (16, 1), (33, 1)])
def test_decode(gpu, dtype, Hq, Hkv):
    check_attention(gpu, dtype, [0, 1, 2, 31, 32, 33, 63, 64, 65, 129], 1, Hq, Hkv, seed=Hq)


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,P", [([255, 256, 257], 256), ([1000, 3, 0, 513], 512), ([2100, 1024], 256), ([5000], 256)])
def test_decode_lengths(gpu, dtype, lens, P):
    check_attention(gpu, dtype, lens, 1, 6, 2, P, seed=sum(lens))
    check_attention(gpu, dtype, lens, 1, 6, 2, P, seed=sum(lens), max_kv=P * (-(-max(lens) // P) + 1))


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,S,Hq,Hkv", [
    ([2, 5, 64, 300], 2, 4, 2), ([5, 0, 70, 260], 5, 4, 1), ([17, 100], 17, 7, 1), ([33, 129, 40], 33, 2, 2),
    ([130, 700], 130, 2, 1), ([3, 1, 0], 4, 3, 1)])
def test_chunk(gpu, dtype, causal, lens, S, Hq, Hkv):
    """S tokens; a sequence may have fewer rows than that (its first queries see none)."""
    check_attention(gpu, dtype, lens, S, Hq, Hkv, causal=causal, seed=S)


def spread_lengths(B, longest, seed):
    """Lengths from 0 to `longest`, most of them short."""
    g = torch.Generator().manual_seed(seed)
    lens = (longest ** torch.rand(B, generator=g)).long().tolist()
    return [0, longest] + [0 if b % 7 == 3 else n for b, n in enumerate(lens)][2:]


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,S,Hq,Hkv,max_kv", [
    (spread_lengths(70, 2500, 1), 1, 4, 1, None), (spread_lengths(200, 1500, 2), 1, 6, 2, None),
    (spread_lengths(256, 1300, 3), 1, 1, 1, None), (spread_lengths(257, 1300, 4), 1, 1, 1, None),
    ([9000] + [10] * 40, 1, 8, 4, None), ([5000, 0, 17, 4999], 5, 8, 2, None), ([3000, 39, 1500], 40, 4, 1, None),
    ([1100] * 16, 1, 16, 8, None), ([300, 20], 1, 4, 2, 60000), ([70, 1300], 3, 20, 2, 30000), ([0, 0], 1, 4, 2, 2000)])
def test_sequences_cut_into_chunks(gpu, dtype, lens, S, Hq, Hkv, max_kv):
    """Batches whose sequences are cut, by their lengths, into as many chunks as fill the device:
    very different lengths, more sequences than a wave's lanes, bounds far above the lengths."""
    c = Cache(len(lens), lens, Hkv, 512)
    if max_kv:
        c.table = torch.cat((c.table, torch.full((c.B, max_kv // 512 + 1), -7, dtype=torch.int32)), 1)
    check_attention(gpu, dtype, lens, S, Hq, Hkv, 512, c=c, max_kv=max_kv, seed=len(lens))


@gpu_test
@pytest.mark.parametrize("dtype,lens,S,Hq,Hkv", [
    ("bf16", [3000, 70, 2100, 0, 3000, 12, 1500, 900, 3000, 41, 2999, 3000], 5, 32, 8),  # 32 rows a wave, cut
    ("bf16", [3000], 66, 64, 8), ("bf16", [4000] * 3 + [300], 20, 32, 8),                # the same, R > 32; whole
    ("bf16", [2500, 1300, 20], 12, 16, 4), ("bf16", [1500] * 8, 9, 32, 8),               # 16 rows a wave, cut; whole
    ("bf16", [2000, 1999], 5, 28, 4),
    ("f32", [3000, 17, 2100], 12, 16, 4), ("f32", [1500] * 6, 24, 32, 8), ("f32", [2000], 150, 16, 2)])
def test_rows_of_a_wave(gpu, dtype, lens, S, Hq, Hkv):
    """16 and 32 query rows a wave, over sequences that are cut and that are not."""
    check_attention(gpu, dtype, lens, S, Hq, Hkv, seed=S)
    check_attention(gpu, dtype, lens, S, Hq, Hkv, seed=S, causal=False)


@gpu_test
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,B,S,Hq,Hkv,P", [("bf16", 13, 260, 56, 8, 256), ("bf16", 50, 129, 32, 8, 512),
                                                 ("f32", 9, 260, 56, 8, 256), ("f32", 70, 40, 32, 8, 256)])
def test_chunk_of_many(gpu, dtype, B, S, Hq, Hkv, P, causal):
    """As many query rows as run in blocks of 128 that share their keys."""
    lens = [0, S // 2, S, S + 1] + [S + 37 * b % 300 for b in range(4, B)]
    check_attention(gpu, dtype, lens, S, Hq, Hkv, P, causal=causal, seed=B)


@gpu_test
@pytest.mark.parametrize("seed", range(40))
def test_drawn_calls(gpu, seed):
    """Sizes drawn over what the rules for rows, cuts and blocks tell apart."""
    g = torch.Generator().manual_seed(100 + seed)
    pick = lambda lo, hi: int(lo * (hi / lo) ** float(torch.rand((), generator=g)))  # noqa: E731
    Hkv, G, S = pick(1, 9), pick(1, 17), 1 if seed % 3 == 0 else pick(2, 300)
    longest = pick(300, 5000)
    B = min(pick(1, 60), max(1, int(2e8 / (Hkv * G * S * longest))))
    lens = [0 if float(torch.rand((), generator=g)) < 0.1 else pick(1, longest + 1) for _ in range(B)]
    lens[0] = longest
    check_attention(gpu, "f32" if seed % 4 == 1 else "bf16", lens, S, Hkv * G, Hkv, 256 * pick(1, 3), seed % 5 != 2,
                    seed=seed, max_kv=longest if seed % 2 else None)


@gpu_test
@pytest.mark.parametrize("lens,S,Hq", [([17000] + [3] * 256, 1, 2), ([17000, 16385, 70], 3, 2), ([17000, 30], 128, 256)])
def test_more_pages_than_lanes(gpu, lens, S, Hq):
    """Sequences of 67 pages: whole, cut, and in blocks of 128 rows."""
    check_attention(gpu, "bf16", lens, S, Hq, 1, seed=S)


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,Hq", [(1, 1), (12, 1), (150, 1), (700, 300)])
def test_scores_far_apart(gpu, dtype, S, Hq):
    """Keys sorted by score, both ways: the running maximum moves at every tile, or never; scores
    from -3000 to 3000, and one scale of 2^-30 the softmax is flat at."""
    lens = [700]
    for way in (1, -1):
        c = Cache(3, lens, 1)
        q = torch.zeros((1, Hq, S, D))
        q[..., 0] = 256.0
        k = way * torch.linspace(-240, 240, 700, dtype=torch.float64)
        for j in range(0, 700, BLOCK):
            page, block = (int(y) for y in c.block(0, j))
            m = min(BLOCK, 700 - j)
            c.scales[0, page, :, block] = 127
            c.codes[0, page, :, j % 256:j % 256 + m, 0] = encode(k[j:j + m].float().to(E4M3).double(),
                                                                 torch.tensor(127))
        check_attention(gpu, dtype, lens, S, Hq, 1, c=c, q=q.to(DTYPES[dtype]), scale=0.05)
        check_attention(gpu, dtype, lens, S, Hq, 1, c=c, q=q.to(DTYPES[dtype]), scale=2.0 ** -30)


@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,G", [(6, 3), (140, 3), (500, 400)])
def test_hidden_nan_reaches_nobody(gpu, dtype, S, G):
    """A token whose k and v are NaN: earlier queries of the chunk are what they are without
    it, it and the later ones get NaN (v's only in the dims that hold one)."""
    from crane_amd import ops
    n, bad = S + 90, S + 90 - 3
    for which in (0, 1):
        c = Cache(8, [n], 1)
        page, row = (int(y) for y in c.at(0, bad))
        q = torch.randn((1, G, S, D), generator=torch.Generator().manual_seed(1)).to(DTYPES[dtype])
        args = (ints([n], gpu), n)
        pools, table = c.to(gpu)
        clean = ops.attention_paged_f8(q.to(gpu), pools, table, *args)
        c.codes[which, page, :, row, 5:9] = 0xff
        pools, table = c.to(gpu)
        got = ops.attention_paged_f8(q.to(gpu), pools, table, *args)
        last = S - 3  # the query at the row `bad`
        assert torch.equal(got[:, :last], clean[:, :last])
        nan = torch.isnan(got[:, last:].view(1, -1, G, D))
        if which == 0:
            assert nan.all()
        else:
            assert nan[..., 5:9].all() and not nan[..., :5].any() and not nan[..., 9:].any()
            a, b = (x[:, last:].view(1, -1, G, D) for x in (got, clean))  # the other dims: the same bits
            assert torch.equal(a[..., :5], b[..., :5]) and torch.equal(a[..., 9:], b[..., 9:])


@gpu_test
def test_values_a_scale_holds(gpu):
    """Blocks of scales 2^-100 to 2^100 side by side; and visible NaN and queries of infinities
    give NaN."""
    from crane_amd import ops
    c = Cache(4, [256], 1)
    page = int(c.table[0, 0])
    for block, byte in enumerate([27, 60, 100, 127, 140, 170, 200, 227]):
        c.scales[1, page, :, block] = byte
    check_attention(gpu, "bf16", [256], 1, 2, 1, c=c)
    check_attention(gpu, "f32", [256], 1, 2, 1, c=c)
    c = Cache(4, [100], 1)
    page = int(c.table[0, 0])
    pools, table = c.to(gpu)
    q = torch.randn((1, 2, D), device=gpu)
    q[0, 1, 3] = math.inf
    for t in (torch.bfloat16, torch.float32):
        out = ops.attention_paged_f8(q.to(t), pools, table, ints([100], gpu), 100).view(2, D)
        assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()
    c.codes[1, page, :, 50, 7] = 0x7f
    pools, table = c.to(gpu)
    out = ops.attention_paged_f8(q, pools, table, ints([100], gpu), 100).view(2, D)
    assert torch.isnan(out[0, 7]) and torch.isfinite(out[0, :7]).all()


@gpu_test
@pytest.mark.parametrize("S,Hq", [(1, 2), (9, 2), (150, 2), (250, 400)])
def test_pages_outside_the_pool_count_as_zeros(gpu, S, Hq):
    for bad in (-1, 1 << 30, 2 ** 31 - 1):
        c = Cache(2, [600, 300], 1)
        c.table[0, 1] = bad
        check_attention(gpu, "bf16", [600, 300], S, Hq, 1, c=c, causal=False)


@gpu_test
def test_length_past_the_bound(gpu):
    """Rows past max_kv are not attended: as if kv_len were max_kv."""
    from crane_amd import ops
    c = Cache(2, [700], 1)
    pools, table = c.to(gpu)
    q = torch.randn((1, 2, D), device=gpu, dtype=torch.bfloat16)
    a = ops.attention_paged_f8(q, pools, table, ints([700], gpu), 300)
    assert torch.equal(a, ops.attention_paged_f8(q, pools, table, ints([300], gpu), 300))


@gpu_test
def test_pools_past_4_gib(gpu):
    """Pages whose bytes lie past 2^32 in the pools, for all three operators."""
    from crane_amd import ops
    Hkv, P, B, S = 4, 512, 2, 3
    n_pages = (1 << 32) // (Hkv * P * D) + 8
    lens = [700, 40]
    small = Cache(6, lens, Hkv, P, ahead=S)
    pools, _ = small.to(gpu)
    high = n_pages - small.codes.shape[1]
    big = ops.f8_pools(n_pages, Hkv, P, gpu)
    for x, y in zip(big, pools):
        x.view(torch.uint8)[high:] = y.view(torch.uint8)
    far = torch.where(small.table >= 0, small.table + high, small.table).to(gpu)
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn((B, S, 3 * Hkv * D), generator=g).to(gpu, torch.bfloat16)
    cos, sin = (x.to(gpu) for x in tables(710, torch.bfloat16))
    outs = []
    for ps, table in ((pools, small.table.to(gpu)), (big, far)):
        q = ops.qk_norm_rope_append_paged_f8(qkv, cos, sin, ints(lens, gpu), ps, table, ints(lens, gpu), Hkv)
        after = ints([n + S for n in lens], gpu)
        outs.append([q, ops.attention_paged_f8(q, ps, table, after, 703)] + list(ops.read_paged_f8(ps, table, after, 703)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    for x, y in zip(big, pools):
        assert torch.equal(x.view(torch.uint8)[high:], y.view(torch.uint8))


# ------------------------------------------------------------------ the read

@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,P", [([1], 256), ([0, 31, 32, 300], 256), ([700, 511, 512], 512)])
def test_read(gpu, dtype, lens, P):
    from crane_amd import ops
    c = Cache(sum(lens), lens, 2, P)
    if len(lens) > 3:
        c.table[3, 0] = -1
    pools, table = c.to(gpu)
    top = max(lens) + 7
    k, v = ops.read_paged_f8(pools, table, ints(lens, gpu), top, DTYPES[dtype])
    for which, x in enumerate((k, v)):
        want = torch.zeros((len(lens), 2, top, D), dtype=torch.float64)
        for b, n in enumerate(lens):
            want[b, :, :n] = c.rows(which, b, n)
        assert torch.equal(x.cpu().double(), want)


# ------------------------------------------------------------------ together

@gpu_test
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_then_tokens(gpu, dtype):
    """A prompt in two chunks, then tokens one by one, for two sequences: attention after every
    step against the definition over the rows that read_paged_f8 gives, and those against the
    rows that went in (two roundings to 4 bits at most)."""
    from crane_amd import ops
    t, Hq, Hkv, lens = DTYPES[dtype], 6, 2, [0, 0]
    g = torch.Generator().manual_seed(3)
    c = Cache(0, [400, 400], Hkv)
    pools = ops.f8_pools(c.codes.shape[1], Hkv, 256, gpu)
    table = c.table.to(gpu)
    cos, sin = (x.to(gpu) for x in tables(400, t))
    put = []
    for S in (150, 101, 1, 1, 1, 1, 1, 7, 1):
        qkv = torch.randn((2, S, (Hq + 2 * Hkv) * D), generator=g).to(t)
        qkv *= 2.0 ** len(put)  # later rows are larger: scales grow
        put.append(qkv.view(2, S, -1, D)[:, :, Hq + Hkv:].double())
        at = ints(lens, gpu)
        q = ops.qk_norm_rope_append_paged_f8(qkv.to(gpu), cos, sin, at, pools, table, at, Hq, order="norm_then_rope")
        lens = [n + S for n in lens]
        out = ops.attention_paged_f8(q, pools, table, ints(lens, gpu), lens[0])
        k, v = ops.read_paged_f8(pools, table, ints(lens, gpu), lens[0], torch.float32)
        rows = torch.cat(put, 1).transpose(1, 2)
        big = rows.abs().amax((2, 3), keepdim=True)
        assert ((v.cpu().double() - rows).abs() <= 2.0 ** -3 * rows.abs() + 2.0 ** -16 * big).all()
        c.codes, c.scales = (torch.stack([p.view(torch.uint8).cpu() for p in pair]) for pair in (pools[:2], pools[2:]))
        assert torch.equal(c.rows(1, 1, lens[1]), v[1].cpu().double())
        ref, mag, slack = reference(c, q.cpu(), lens, D ** -0.5, True)
        assert ((out.cpu().double() - ref).abs() <= HALF[dtype] * (ref.abs() + mag) + mag * slack).all()


@gpu_test
@pytest.mark.parametrize("B,Hq,Hkv,S", [(2, 4, 2, 1), (3, 4, 2, 5), (1, 4, 1, 200)])
def test_captured_step(gpu, B, Hq, Hkv, S):
    """A step (append, attention, read) captured in a graph and replayed on changing inputs, beside
    another graph of the same calls and eager calls of the program's own."""
    from crane_amd import ops
    lens = [300 + 50 * b for b in range(B)]
    c = Cache(1, lens, Hkv, ahead=S)
    base, table = c.to(gpu)
    cos, sin = (x.to(gpu) for x in tables(800, torch.bfloat16))
    qkv = torch.zeros((B, S, (Hq + 2 * Hkv) * D), dtype=torch.bfloat16, device=gpu)
    at, after, top = ints(lens, gpu), ints([n + S for n in lens], gpu), max(lens) + S

    def step(pools):
        q = ops.qk_norm_rope_append_paged_f8(qkv, cos, sin, at, pools, table, at, Hq)
        return (q, ops.attention_paged_f8(q, pools, table, after, top)) + ops.read_paged_f8(pools, table, after, top)

    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        pools = tuple(p.clone() for p in base)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(pools)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(pools)
        graphs.append((graph, pools, out))
    g = torch.Generator().manual_seed(4)
    for turn_ in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(torch.bfloat16))
        for graph, pools, out in graphs:
            for p, x in zip(pools, base):
                p.view(torch.uint8).copy_(x.view(torch.uint8))
        mine = tuple(p.clone() for p in base)
        want = step(mine)
        for graph, pools, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, pools, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn_
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pools, mine))


@gpu_test
@pytest.mark.parametrize("S", [1, 30])
def test_captured_attention_follows_the_lengths(gpu, S):
    """One captured call, its bound the longest there may be, replayed as the lengths change, in
    a workspace that others write to between the replays."""
    from crane_amd import _lib, ops
    top = 6000
    c = Cache(3, [top, 5000, 40], 2)
    pools, table = c.to(gpu)
    n = ints([top, 5000, 40], gpu)
    q = torch.randn((3, 4, S, D), device=gpu).bfloat16()
    need = _lib.lib().crane_hip_attn_paged_f8_workspace(top, 3, S, 4, 2, D, _lib.BF16)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_paged_f8(q, pools, table, n, top, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_paged_f8(q, pools, table, n, top, workspace=ws)
    for lens in ([top, 5000, 40], [1, 0, 7], [300, 4097, 0], [0, 0, 0], [64, 4999, 33], [top, 5000, 40]):
        n.copy_(ints(lens, gpu))
        ws.fill_(0xff)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attention_paged_f8(q, pools, table, n, top)), lens
        ref, mag, slack = reference(c, q.cpu(), lens, D ** -0.5, True)
        tol = HALF["bf16"] * (ref.abs() + mag) + mag * slack
        assert ((out.cpu().double() - ref).abs() <= tol).all(), lens


@gpu_test
def test_streams_and_repeats(gpu):
    """Calls on two streams at once give what each gives alone, every time."""
    from crane_amd import ops
    lens = [900, 1500, 40]
    c = Cache(9, lens, 2)
    pools, table = c.to(gpu)
    q = torch.randn((3, 8, D), device=gpu, dtype=torch.bfloat16)
    n = ints(lens, gpu)
    want = ops.attention_paged_f8(q, pools, table, n, 1500)
    rows = ops.read_paged_f8(pools, table, n, 1500)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append((ops.attention_paged_f8(q, pools, table, n, 1500), ops.read_paged_f8(pools, table, n, 1500)))
    torch.cuda.synchronize()
    for a, r in outs:
        assert torch.equal(a, want) and torch.equal(r[0], rows[0]) and torch.equal(r[1], rows[1])


@gpu_test
def test_given_workspace(gpu):
    """A workspace of any contents and at least the size asked for; a smaller one is refused."""
    from crane_amd import _lib, ops
    lens = [5000]
    c = Cache(9, lens, 1)
    pools, table = c.to(gpu)
    q = torch.randn((1, 2, D), device=gpu, dtype=torch.bfloat16)
    need = _lib.lib().crane_hip_attn_paged_f8_workspace(5000, 1, 1, 2, 1, D, _lib.BF16)
    assert need > 0
    want = ops.attention_paged_f8(q, pools, table, ints(lens, gpu), 5000)
    for fill in (0, 0xff):
        ws = torch.full((need,), fill, dtype=torch.uint8, device=gpu)
        assert torch.equal(ops.attention_paged_f8(q, pools, table, ints(lens, gpu), 5000, workspace=ws), want)
    with pytest.raises(_lib.CraneHipError) as e:
        ops.attention_paged_f8(q, pools, table, ints(lens, gpu), 5000, workspace=ws[:need - 16])
    assert e.value.code == _lib.E_WORKSPACE
    for bad in (ws[:1].expand(need), torch.empty(2 * need, dtype=torch.uint8, device=gpu)[::2]):
        with pytest.raises(_lib.CraneHipError) as e:
            ops.attention_paged_f8(q, pools, table, ints(lens, gpu), 5000, workspace=bad)
        assert e.value.code == _lib.E_INVALID


# ------------------------------------------------------------------ refusals

def _append(**kw):
    from crane_amd import _lib
    a = dict(qkv=16, stride=768, qw=None, kw=None, eps=1e-6, order=0, cos=16, sin=16, cs=64, rows=100, pos=16, q=16,
             k=16, v=16, ks=16, vs=16, n_pages=4, P=256, table=16, width=2, len=16, B=0, S=1, Hq=4, Hkv=1, D=128, dtype=1)
    a.update(kw)
    return _lib.lib().crane_hip_qknorm_rope_append_paged_f8(*a.values(), None)


def _attn(**kw):
    from crane_amd import _lib
    a = dict(q=16, k=16, v=16, ks=16, vs=16, n_pages=4, P=256, table=16, width=2, len=16, max_kv=512, B=0, S=1, Hq=4,
             Hkv=1, D=128, scale=0.1, flags=1, ws=None, bytes=0, out=16, dtype=1)
    a.update(kw)
    return _lib.lib().crane_hip_attn_paged_f8(*a.values(), None)


def _read(**kw):
    from crane_amd import _lib
    a = dict(k=16, v=16, ks=16, vs=16, n_pages=4, P=256, table=16, width=2, len=16, max_kv=512, B=0, Hkv=1, D=128, ko=16,
             vo=16, dtype=1)
    a.update(kw)
    return _lib.lib().crane_hip_read_paged_f8(*a.values(), None)


SHARED = [(dict(dtype=2), 2), (dict(dtype=-1), 2), (dict(D=64), 3), (dict(B=-1), 1), (dict(Hkv=0), 1),
          (dict(n_pages=0), 1), (dict(P=128), 1), (dict(P=0), 1), (dict(table=None), 1), (dict(width=0), 1),
          (dict(B=1, k=None), 1), (dict(B=1, v=None), 1), (dict(B=1, ks=None), 1), (dict(B=1, vs=None), 1),
          (dict(B=1, len=None), 1), (dict(B=1, k=8), 8), (dict(B=1, v=8), 8), (dict(B=1, ks=8), 8), (dict(B=1, vs=4), 8)]


@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(S=-1), 1), (dict(Hq=0), 1), (dict(Hq=3, Hkv=2), 4), (dict(order=3), 1), (dict(order=-1), 1), (dict(eps=-1.0), 1),
    (dict(eps=math.nan), 1), (dict(S=513), 5), (dict(B=1, qkv=None), 1), (dict(B=1, cos=None), 1), (dict(B=1, sin=None), 1),
    (dict(B=1, pos=None), 1), (dict(B=1, q=None), 1), (dict(B=1, cs=32), 1), (dict(B=1, rows=0), 1),
    (dict(B=1, stride=760), 1), (dict(B=1, stride=772), 8), (dict(B=1, cs=68), 8), (dict(B=1, qkv=8), 8),
    (dict(B=1, cos=8), 8), (dict(B=1, q=8), 8), (dict(B=1, qw=8), 8), (dict(B=1, kw=8), 8),
    (dict(B=1 << 30, S=500), 1), (dict(), 0), (dict(B=1, S=0), 0)])
def test_append_refuses(kw, code):
    assert _append(**kw) == code


@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(S=-1), 1), (dict(Hq=0), 1), (dict(Hq=3, Hkv=2), 4), (dict(flags=2), 1), (dict(scale=0.0), 1),
    (dict(scale=-1.0), 1), (dict(scale=math.inf), 1), (dict(scale=math.nan), 1), (dict(max_kv=0), 1), (dict(max_kv=-5), 1),
    (dict(max_kv=513), 5), (dict(max_kv=2 ** 31), 1), (dict(B=70000), 1), (dict(B=1, q=None), 1), (dict(B=1, out=None), 1),
    (dict(B=1, q=8), 8), (dict(B=1, out=8), 8), (dict(B=60000, Hq=40000, Hkv=1), 1), (dict(B=2, S=2 ** 30), 1),
    (dict(), 0), (dict(B=1, S=0), 0)])
def test_attention_refuses(kw, code):
    assert _attn(**kw) == code


def test_attention_wants_its_workspace():
    from crane_amd import _lib
    args = (4096, 1, 1, 4, 1, 128, 1)
    need = _lib.lib().crane_hip_attn_paged_f8_workspace(*args)
    assert need > 0
    call = dict(B=1, max_kv=4096, width=16)
    assert _attn(**call) == _lib.E_WORKSPACE
    assert _attn(**call, ws=16, bytes=need - 1) == _lib.E_WORKSPACE
    assert _attn(**call, ws=24, bytes=need) == _lib.E_WORKSPACE
    for bad in ((4096, 0, 1, 4, 1, 128, 1), (4096, 1, 0, 4, 1, 128, 1), (0, 1, 1, 4, 1, 128, 1), (4096, 1, 1, 4, 1, 64, 1),
                (4096, 1, 1, 4, 3, 128, 1), (4096, 1, 1, 4, 1, 128, 5), (2 ** 31, 1, 1, 4, 1, 128, 1)):
        assert _lib.lib().crane_hip_attn_paged_f8_workspace(*bad) == 0


@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(max_kv=-1), 1), (dict(max_kv=513), 5), (dict(B=1, ko=None), 1), (dict(B=1, vo=None), 1), (dict(B=1, ko=8), 8),
    (dict(B=1, vo=8), 8), (dict(B=2 ** 30, Hkv=8), 1), (dict(B=2 ** 22, max_kv=512), 1), (dict(), 0), (dict(B=1, max_kv=0), 0)])
def test_read_refuses(kw, code):
    assert _read(**kw) == code


def test_host_tensors_are_refused():
    from crane_amd import ops
    from crane_amd._lib import CraneHipError
    pools, table = Cache(0, [5], 1).to("cpu")
    n = ints([5], "cpu")
    with pytest.raises(CraneHipError):
        ops.attention_paged_f8(torch.zeros((1, 2, D)), pools, table, n, 5)
    with pytest.raises(CraneHipError):
        ops.read_paged_f8(pools, table, n, 5)
    with pytest.raises(CraneHipError):
        ops.qk_norm_rope_append_paged_f8(torch.zeros((1, 1, 3 * D)), *tables(8, torch.float32), n, pools, table, n, 1)


@gpu_test
def test_python_refusals(gpu):
    """Every argument the kernels rely on is checked before anything runs."""
    from crane_amd import _lib, ops
    from crane_amd._lib import CraneHipError
    pools, table = Cache(0, [5, 9], 2).to(gpu)
    n, q = ints([5, 9], gpu), torch.zeros((2, 4, D), device=gpu, dtype=torch.bfloat16)
    qkv = torch.zeros((2, 1, 8 * D), device=gpu, dtype=torch.bfloat16)
    cos, sin = (x.to(gpu) for x in tables(16, torch.bfloat16))

    def swap(i, t):
        return pools[:i] + (t,) + pools[i + 1:]

    def refused(code, f, *args, **kw):
        with pytest.raises(CraneHipError) as e:
            f(*args, **kw)
        assert e.value.code == code, e.value

    def all_three(code, ps=pools, tb=table):
        refused(code, ops.attention_paged_f8, q, ps, tb, n, 9)
        refused(code, ops.read_paged_f8, ps, tb, n, 9)
        refused(code, ops.qk_norm_rope_append_paged_f8, qkv, cos, sin, n, ps, tb, n, 4)

    all_three(_lib.E_INVALID, pools[:3])
    all_three(_lib.E_DTYPE, swap(0, pools[0].view(torch.uint8)))
    all_three(_lib.E_DTYPE, swap(3, pools[3].view(torch.uint8)))
    all_three(_lib.E_INVALID, swap(1, pools[1][:, :, :128].contiguous()))
    all_three(_lib.E_INVALID, swap(2, pools[2][:, :1].contiguous()))
    all_three(_lib.E_INVALID, swap(0, pools[0].transpose(1, 2).contiguous().transpose(1, 2)))
    all_three(_lib.E_INVALID, swap(2, pools[2].cpu()))
    all_three(_lib.E_INVALID, tb=table.long())
    all_three(_lib.E_INVALID, tb=table.t().contiguous().t())
    refused(_lib.E_INVALID, ops.attention_paged_f8, q[:, :3].contiguous(), pools, table[:1], n, 9)
    refused(_lib.E_GQA, ops.attention_paged_f8, q[:, :3].contiguous(), pools, table, n, 9)
    refused(_lib.E_INVALID, ops.attention_paged_f8, q.transpose(0, 1).contiguous().transpose(0, 1), pools, table, n, 9)
    refused(_lib.E_DTYPE, ops.attention_paged_f8, q.half(), pools, table, n, 9)
    refused(_lib.E_HEAD_DIM, ops.attention_paged_f8, q[..., :64].contiguous(), pools, table, n, 9)
    refused(_lib.E_INVALID, ops.attention_paged_f8, q, pools, table, n.long(), 9)
    refused(_lib.E_INVALID, ops.attention_paged_f8, q, pools, table, n[:1], 9)
    refused(_lib.E_INVALID, ops.attention_paged_f8, q, pools, table, n.cpu(), 9)
    refused(_lib.E_CAPACITY, ops.attention_paged_f8, q, pools, table, n, table.shape[1] * 256 + 1)
    refused(_lib.E_INVALID, ops.attention_paged_f8, q, pools, table, n, 0)
    refused(_lib.E_DTYPE, ops.read_paged_f8, pools, table, n, 9, torch.float16)
    refused(_lib.E_INVALID, ops.read_paged_f8, pools, table, n, -1)
    refused(_lib.E_INVALID, ops.qk_norm_rope_append_paged_f8, qkv, cos, sin, n, pools, table, n, 5)
    refused(_lib.E_INVALID, ops.qk_norm_rope_append_paged_f8, qkv, cos, sin, n, pools, table, n.long(), 4)
    refused(_lib.E_DTYPE, ops.qk_norm_rope_append_paged_f8, qkv, cos.float(), sin.float(), n, pools, table, n, 4)
    refused(_lib.E_INVALID, ops.qk_norm_rope_append_paged_f8, qkv, cos, sin, n, pools, table, n, 4, order="rope")


@gpu_test
def test_nothing_to_do(gpu):
    from crane_amd import ops
    pools, table = Cache(0, [5, 9], 2).to(gpu)
    n = ints([5, 9], gpu)
    none = table[:0].contiguous()
    cos, sin = (x.to(gpu) for x in tables(16, torch.bfloat16))
    e = torch.zeros((0,), dtype=torch.int32, device=gpu)
    before = [p.view(torch.uint8).clone() for p in pools]
    assert ops.attention_paged_f8(torch.zeros((0, 4, D), device=gpu), pools, none, e, 5).shape == (0, 1, 4 * D)
    assert ops.attention_paged_f8(torch.zeros((2, 4, 0, D), device=gpu), pools, table, n, 9).shape == (2, 0, 4 * D)
    assert ops.read_paged_f8(pools, none, e, 5)[0].shape == (0, 2, 5, D)
    assert ops.read_paged_f8(pools, table, n, 0)[1].shape == (2, 2, 0, D)
    x = torch.zeros((0, 3, 8 * D), device=gpu, dtype=torch.bfloat16)
    assert ops.qk_norm_rope_append_paged_f8(x, cos, sin, e, pools, none, e, 4).shape == (0, 4, 3, D)
    assert all(torch.equal(a, p.view(torch.uint8)) for a, p in zip(before, pools))
