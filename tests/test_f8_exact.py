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


# ------------------------------------------------------------------ attention

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
