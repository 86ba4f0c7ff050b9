"""Attention over shared pages (include/crane_shared.h) with scores of any size f32 holds.

Keys are a_j u and queries b u with u of -1 and 1, a_j small whole numbers and b a power
of two, so every score is exact and the scores' differences are hundreds or more: the
weights are equal for the keys of the largest score and 0 for the others, and the result
is the mean of those keys' V (of -1 and 1).

Where every maximum m = scale log2 e max s is past 2^26, the walk takes differences of
scores: the weights are 1, all sums are whole numbers, and the result is T(f32(sum) /
f32(count)) to the last bit.  Below that the weights are exp2(d), d the rounding of m, of
which bf16 calls round the product's operand but not the sum: test_shared.bounds() with no
error of a score."""
import numpy as np
import pytest

import cases
import test_shared as ts

D = 128

SHAPES = [  # lens, groups, rows, P, Hq, Hkv, S
    ([1], [], [], 256, 4, 1, 1),
    ([700, 530, 1025, 512, 90, 2300, 0], [[3, 0, 1], [5, 2]], [512, 1024], 512, 14, 2, 1),
    ([300, 310, 280], [[0, 1, 2]], [256], 256, 8, 2, 5),
    ([1500, 1400], [[0, 1]], [1280], 256, 4, 4, 129),
    ([40, 5, 70, 0], [], [], 256, 4, 2, 40),
] + [ts.shared_shape(i) for i in (0, 1, 2, 3, 5, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("b", [2.0 ** 12, 2.0 ** 20, -2.0 ** 20, 2.0 ** 33, -2.0 ** 70, 2.0 ** 100])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_scores_of_any_size(gpu, case, b, dtype):
    lens, groups, rows, P, Hq, Hkv, S = SHAPES[case]
    print(f"scores case {case} b={b} {dtype}", flush=True)
    table, total = ts.layout(700 + case, lens, groups, rows, P)
    k, v = ts.pools(701 + case, total, Hkv, P, table, lens, True)
    r = cases.rng(702 + case)
    u = np.sign(cases.normal(r, (D,))).astype(np.float32)
    a = r.integers(1, 200, k.shape[:3]).astype(np.float32)          # [page, kv head, row]
    k = np.where(np.isnan(k), k, a[..., None] * u)
    q = np.broadcast_to(np.float32(b) * u, (len(lens), Hq, S, D))
    got = ts.call(gpu, q, k, v, table, lens, groups, rows, dtype)
    want = np.zeros((len(lens), S, Hkv, Hq // Hkv, D), np.float32)
    for x, n in enumerate(lens):
        if n == 0:
            continue
        vv, aa = ts.rows_of(v, table, x, n, P), ts.rows_of(a[..., None], table, x, n, P)[..., 0]
        for s in range(S):
            L = n - S + 1 + s
            if L <= 0:
                continue
            sc = aa[:, :L] * np.sign(b)
            top = sc == sc.max(-1, keepdims=True)
            want[x, s] = (np.where(top[..., None], vv[:, :L], 0).sum(1, dtype=np.float64).astype(np.float32)
                          / top.sum(-1).astype(np.float32)[:, None])[:, None, :]
    want = want.reshape(len(lens), S, -1)
    got = got.float().cpu().numpy()
    if abs(b) >= 2.0 ** 33:                                         # m >= 2^33 128 D^-1/2 log2 e > 2^37
        assert (got == cases.cast(want, dtype)).all(), (int((got != want).sum()), int(np.isnan(got).sum()))
    else:
        err = np.abs(got - want) / ts.bounds(want, np.float32(1), 0.0, max(lens), dtype)
        assert (err <= 1).all(), float(err.max())
