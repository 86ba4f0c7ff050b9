"""How the attention over shared pages is cut (crane_amd/csrc/shared_plan.h, compiled for
the host alone): the order of a role's workgroups."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crane_amd", "csrc")
SOURCE = """
#include "shared_plan.h"
using namespace crane;
extern "C" void plan(const int32_t* groups, int n_groups, int64_t max_kv, int64_t max_own, int64_t mean_own, int B,
                     int S, int Hq, int Hkv, int bf16, int64_t* out) {
    const Plan p = plan_for(Sizes{groups, n_groups, max_kv, max_own, mean_own, B, S, Hq, Hkv, bf16 != 0});
    const int64_t r[] = {p.share, p.shared_rows, p.own_rows, p.shared_tiles, p.own_tiles, p.chunk,
                         p.shared_splits, p.own_splits, p.shared_items, p.own_items, p.fits};
    std::copy(r, r + 11, out);
}
// A device group's {first place, members} as the kernel takes them, and the entries of
// the host's groups.
extern "C" void members(const int32_t* groups, int n_groups, int B, int first, int count, int32_t* out) {
    const Plan p = plan_for(Sizes{groups, n_groups, 1024, 512, 100, B, 1, 8, 2, true});
    const Members m(first, count, p.members);
    const int32_t r[] = {m.first, m.n, p.members};
    std::copy(r, r + 3, out);
}
// Every item of a role: {block, kv head, segment, chunk}, or -1 for none.
extern "C" void items(int n, int blocks, int Hkv, int segs, int chunks, int32_t* out) {
    for (int x = 0; x < n; ++x) {
        const Item i(x, blocks, Hkv, segs, chunks);
        const int32_t r[] = {i.block, i.kvh, i.seg, i.chunk};
        for (int e = 0; e < 4; ++e) out[4 * x + e] = i.ok ? r[e] : -1;
    }
}
"""
FIELDS = ("share", "shared_rows", "own_rows", "shared_tiles", "own_tiles", "chunk", "shared_splits", "own_splits",
          "shared_items", "own_items", "fits")
_i, _i64 = ctypes.c_int, ctypes.c_int64


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The header behind two C functions."""
    at = tmp_path_factory.mktemp("shared_plan")
    src, lib = at / "plan.cpp", at / "plan.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover=undefined", "-shared", "-fPIC", "-D__host__=", "-D__device__=",
                    "-D__forceinline__=inline", "-I", CSRC, str(src), "-o", str(lib)], check=True)
    L = ctypes.CDLL(str(lib))
    L.plan.argtypes = [ctypes.POINTER(ctypes.c_int32), _i, _i64, _i64, _i64, _i, _i, _i, _i, _i, ctypes.POINTER(_i64)]
    L.items.argtypes = [_i] * 5 + [ctypes.c_void_p]
    L.members.argtypes = [ctypes.POINTER(ctypes.c_int32), _i, _i, _i, _i, ctypes.POINTER(ctypes.c_int32)]
    L.plan.restype = L.items.restype = L.members.restype = None
    return L


def plan(host, groups, max_kv, max_own, mean_own, B, S, Hq, Hkv, bf16):
    """The plan of groups [(members, rows)]."""
    desc, at = [], 0
    for n, rows in groups:
        desc += [at, n, at, rows]
        at += n
    out = (_i64 * len(FIELDS))()
    host.plan((ctypes.c_int32 * max(len(desc), 1))(*desc), len(groups), max_kv, max_own, mean_own, B, S, Hq, Hkv, bf16,
              out)
    return dict(zip(FIELDS, out))


def items(host, blocks, Hkv, segs, chunks):
    n = 8 * blocks * -(-segs * Hkv * chunks // 8)
    out = np.zeros((n, 4), np.int32)
    host.items(n, blocks, Hkv, segs, chunks, out.ctypes.data)
    return out


@pytest.mark.parametrize("blocks", [1, 2, 7])
@pytest.mark.parametrize("Hkv", [1, 2, 3, 4, 8, 16])
def test_items_are_each_unit_once(host, Hkv, blocks):
    """Every (block, kv head, segment, chunk) is one workgroup's, and a unit's blocks are
    on one XCD (workgroups go to the 8 XCDs in turn)."""
    for segs in (1, 2, 3, 4, 5, 8, 12, 31):
        for chunks in (1, 2, 5, 16):
            got = items(host, blocks, Hkv, segs, chunks)
            some = got[:, 0] >= 0
            place = np.ravel_multi_index(got[some].T, (blocks, Hkv, segs, chunks))
            assert sorted(place) == list(range(blocks * Hkv * segs * chunks))
            unit, xcd = place % (Hkv * segs * chunks), np.flatnonzero(some) % 8
            order = np.argsort(unit, kind="stable")
            assert (xcd[order].reshape(-1, blocks) == xcd[order][::blocks, None]).all()


@pytest.mark.parametrize("host_groups,entries", [([(0, 2)], 2), ([(0, 2), (2, 5)], 7), ([(38, 3)], 41), ([(4, 0)], 4)])
def test_device_groups_stay_in_the_members_array(host, host_groups, entries):
    """Whatever a device group says, only entries that the host's groups account for are
    read: those of a batch of 41 with fewer members, too."""
    desc = (ctypes.c_int32 * (4 * len(host_groups)))(*[x for s, n in host_groups for x in (s, n, 0, 256)])
    out = (ctypes.c_int32 * 3)()
    edges = (-2 ** 31, -50, -1, 0, 1, 2, 3, 6, 7, 8, 38, 40, 41, 42, 1 << 30, 2 ** 31 - 1)
    for first in edges:
        for count in edges:
            host.members(desc, len(host_groups), 41, first, count, out)
            at, n, total = out
            assert total == entries
            assert 0 <= at and 0 <= n and at + n <= entries
            if 0 <= first and 0 <= count and first + count <= entries:
                assert (at, n) == (first, count)      # what is consistent is taken as it is


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("S", [1, 40, 300])
@pytest.mark.parametrize("groups", [[], [(2, 0)], [(3, 0), (1, 0)]])
def test_no_keys_are_one_chunk(host, groups, S, bf16):
    """Where the bounds leave no key, the own role's workgroups still write the zeros."""
    p = plan(host, groups, 256, 0, 0, 4, S, 8, 2, bf16)
    assert (p["shared_splits"], p["own_splits"], p["shared_items"]) == (0, 1, 0)
    assert p["own_items"] == 8 * p["own_tiles"]


@pytest.mark.parametrize("groups,max_own,B,Hq,Hkv,bf16,share", [
    ([(1, 446_000_000)] + [(1, 61_000_000)] * 75 + [(73, 61_000_000)], 29_000, 149, 16, 2, 1, 0),
                                                                # sharing is cheaper, not sharing fits
    ([(60, 100_000)] + [(1, 30_000)] * 7, 3_500_000, 67, 16, 4, 1, 1),         # what is chosen fits
    ([], 45_000, 65535, 64, 64, 1, None),                                     # nothing does
    ([(268, 2_000_000)], 300_000_000, 268, 8, 2, 0, None),
])
def test_a_cut_that_fits_the_grid_is_taken(host, groups, max_own, B, Hq, Hkv, bf16, share):
    """A grid has fewer than 2^32 threads: cuts into more workgroups are passed over."""
    p = plan(host, groups, max_own + max((r for _, r in groups), default=0), max_own, max_own, B, 1, Hq, Hkv, bf16)
    assert bool(p["fits"]) == (share is not None)
    if share is not None:
        assert p["share"] == share and p["shared_items"] + p["own_items"] <= (2 ** 32 - 1) // 256


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("groups,rows", [([], []), ([[0, 2]], [0])])
@pytest.mark.parametrize("S", [1, 40, 300])
def test_sequences_without_rows_get_zeros(gpu, S, groups, rows, dtype):
    """kv_len 0 everywhere with the tight bound max_own = 0."""
    import torch
    from crane_amd import _lib, ops
    B, Hq, Hkv, P = 4, 8, 2, 256
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    k = torch.full((3, Hkv, P, 128), float("nan"), dtype=td, device=gpu)
    q = torch.ones((B, Hq, S, 128), dtype=td, device=gpu)
    table = torch.zeros((B, 2), dtype=torch.int32, device=gpu)
    n = torch.zeros(B, dtype=torch.int32, device=gpu)
    g = ops.prefix_groups(groups, rows, B, gpu)
    for causal in (True, False):
        got = ops.attention_shared_paged(q, k, k, table, n, P, g, causal=causal, max_own=0)
        assert got.shape == (B, S, Hq * 128) and (got == 0).all()
        out = torch.full((B, S, Hq * 128), float("nan"), dtype=td, device=gpu)   # and every element is written
        rc = _lib.lib().crane_hip_attn_shared_paged(
            q.data_ptr(), k.data_ptr(), k.data_ptr(), 3, P, table.data_ptr(), 2, n.data_ptr(), P,
            g.shared_rows.data_ptr(), g.groups.data_ptr(), g.members.data_ptr(), g.groups_host, g.n_groups, 0, 0,
            B, S, Hq, Hkv, 128, 0.1, int(causal), None, 0, out.data_ptr(), int(dtype == "bf16"),
            torch.cuda.current_stream(gpu).cuda_stream)
        assert rc == _lib.OK and (out == 0).all()
