"""Pools that share memory: the moves of two workgroups would race, so such calls are refused."""

import ctypes
import itertools
import os
import random
import shutil
import subprocess

import pytest
import torch

from tests.conftest import ROOT

NULL, FAKE = None, 0x1000


def test_c_entry_refuses_shared_memory(pkg):
    from vllm_rlt_amd import _lib

    def commit(key=FAKE, value=FAKE, blocks=10, layers=2, bs=16, strides=(4096, 2048, 128), n=2):
        return _lib.library().rlt_kv_commit_path(
            FAKE, n, 1, 4, bs, FAKE, FAKE, 5, 5, FAKE, layers, blocks, key, value, *strides, 256, 2, NULL)

    assert commit() == 1 and commit(n=0) == 0
    for strides in ((0, 2048, 128), (4096, 0, 128), (4096, 2048, 0)):
        assert commit(value=FAKE + 1024, strides=strides) == 1


def test_c_entry_refuses_views_that_meet(pkg):
    """Two views of one allocation that are a layer, a block or a part of a row apart."""
    from vllm_rlt_amd import _lib

    def commit(apart, strides=(4096, 2048, 128), layers=2):
        return _lib.library().rlt_kv_commit_path(
            FAKE, 2, 1, 4, 16, FAKE, FAKE, 5, 5, FAKE, layers, 10, FAKE, FAKE + apart, *strides, 256, 2, NULL)

    for apart in (256, 2 * 2048, 2 * 4096, 2 * (3 * 4096 + 128), 2 * (9 * 4096 + 2048 + 15 * 128)):
        assert commit(apart) == 1
    # keys and values side by side in a token's 512 bytes, one byte too near
    assert commit(255, strides=(8192, 4096, 256)) == 1
    assert commit(257, strides=(8192, 4096, 256)) == 1


def test_overlap_of_layouts(tmp_path):
    """The host check against all pairs of rows: right for nested axes in any order, with gaps;
    elsewhere it names no layout that does not overlap."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    src = tmp_path / "overlap.cpp"
    src.write_text("""#include "pool_overlap.h"
extern "C" int overlap(int64_t d, const int64_t* s, const int64_t* n, int64_t row) {
  return pools::overlap(d, {{s[0], n[0]}, {s[1], n[1]}, {s[2], n[2]}}, row);
}
""")
    out = tmp_path / "overlap.so"
    subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "vllm-rlt_amd", "csrc"), str(src), "-o", str(out)], check=True)
    check = ctypes.CDLL(str(out)).overlap
    i64 = ctypes.c_int64

    def truth(delta, strides, counts, row):
        rows = [sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, counts))]
        own = sorted(rows)
        if any(b - a < row for a, b in zip(own, own[1:])):
            return True
        return any(abs(a - b - delta) < row for a in rows for b in rows)

    r = random.Random(3)
    seen = [0, 0]
    for nested in (True, False):
        for _ in range(1500):
            row, counts = r.randint(1, 6), [r.randint(1, 4) for _ in range(3)]
            strides, inside = [0, 0, 0], row
            for axis in r.sample(range(3), 3):
                strides[axis] = inside + r.choice((0, 0, row, r.randint(0, 9))) if nested else r.randint(0, 40)
                inside += (counts[axis] - 1) * strides[axis]
            delta = r.randint(-inside - 9, inside + 9)
            got = check(i64(delta), (i64 * 3)(*strides), (i64 * 3)(*counts), i64(row))
            want = truth(delta, strides, counts, row)
            seen[want] += nested
            assert got == want if nested else got <= want, (delta, strides, counts, row)
    assert min(seen) > 200


@pytest.mark.gpu
def test_operator_refuses_shared_memory(pkg, dev):
    """Refused before a launch; views side by side in one allocation are taken."""
    tables = torch.arange(4, device=dev).view(1, 4).int()
    starts, accepted = torch.tensor([3], device=dev), torch.tensor([2], device=dev)
    path = torch.tensor([[0, 2, 4]], device=dev)
    rest = (tables, starts, path, accepted, 4)
    both = torch.randn(9, 2, 4, 2, 16, device=dev)
    old = both.clone()
    shared = both[:1].expand(8, 2, 4, 2, 16)
    layer = both[:8, :1].expand(8, 2, 4, 2, 16)
    token = both[:8, :, :1].expand(8, 2, 4, 2, 16)
    other = torch.randn(9, 2, 4, 2, 16, device=dev)[:8]
    wide = torch.randn(9, 3, 4, 1, 32, device=dev)
    for k, v in ((both, both), (both[:8], both[:8]), (both[:8], both[1:]), (both[1:], both[:8]),
                 (shared, other[:1].expand(8, 2, 4, 2, 16)), (layer, other[:, :1].expand_as(layer)),
                 (token, other[:, :, :1].expand_as(token)),
                 # a layer, or half a row, apart
                 (wide[:8, :2], wide[:8, 1:]), (wide[:8, :2, :, :, :16], wide[:8, :2, :, :, 8:24])):
        with pytest.raises(ValueError, match="overlap"):
            pkg.commit_tree_kv(k, v, *rest)
    torch.cuda.synchronize()
    assert torch.equal(both, old)
    # keys and values of one allocation: interleaved by layer, and one behind the other
    for k, v in ((both[:, :1], both[:, 1:]), (both[:4], both[4:8]), (wide[..., :16], wide[..., 16:]),
                 (wide[:, :1, :2], wide[:, 1:2, :2])):
        if k.shape[2] != 4:  # (blocks of two tokens)
            rest = (tables, starts, path, accepted, 2)
        a, b = k.clone(), v.clone()
        pkg.commit_tree_kv(k, v, *rest)
        pkg.commit_tree_kv(a, b, *rest)
        assert torch.equal(k, a) and torch.equal(v, b)
    assert not torch.equal(both, old)
