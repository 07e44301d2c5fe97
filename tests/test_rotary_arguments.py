"""Rotary plans and the refusals of the rotation, the append and the load, without a GPU."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import rotary as orot


def test_plain_frequencies(pkg):
    r = pkg.Rotary(8, 100.0, device="cpu")
    want = torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64) / (2 * math.pi)
    torch.testing.assert_close(r.turns, want, rtol=1e-15, atol=0)
    assert r.amplitude == 1.0 and r.rotary_dim == 8 and not r.interleaved


def test_scaled_frequencies(pkg):
    base = pkg.Rotary(64, device="cpu").turns
    linear = pkg.Rotary(64, scaling="linear", factor=8.0, device="cpu").turns
    torch.testing.assert_close(linear, base / 8, rtol=1e-15, atol=0)
    ntk = pkg.Rotary(64, scaling="ntk", factor=8.0, device="cpu").turns
    torch.testing.assert_close(ntk[0], base[0], rtol=1e-15, atol=0)
    torch.testing.assert_close(ntk[-1], base[-1] / 8, rtol=1e-12, atol=0)
    bands = pkg.Rotary(64, scaling="bands", factor=8.0, original_length=4096, device="cpu").turns
    n = 4096 * base
    assert torch.equal(bands[n >= 4], base[n >= 4])
    torch.testing.assert_close(bands[n <= 1], base[n <= 1] / 8, rtol=1e-15, atol=0)
    mid = (n > 1) & (n < 4)
    assert mid.any() and (bands[mid] < base[mid]).all() and (bands[mid] > base[mid] / 8).all()
    yarn = pkg.Rotary(64, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    assert yarn.amplitude == pytest.approx(0.1 * math.log(8) + 1)
    low = math.floor(64 * math.log(4096 / (64 * math.pi)) / (2 * math.log(10000)))
    high = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000)))
    assert torch.equal(yarn.turns[:low + 1], base[:low + 1])
    torch.testing.assert_close(yarn.turns[high:], base[high:] / 8, rtol=1e-15, atol=0)
    assert (yarn.turns.diff() < 0).all()
    divided = pkg.Rotary(64, divisors=[2.0] * 32, amplitude=1.5, device="cpu")
    torch.testing.assert_close(divided.turns, base / 2, rtol=1e-15, atol=0)
    assert divided.amplitude == 1.5


@pytest.mark.parametrize("args,kwargs", [
    ((7,), {}), ((0,), {}), ((258,), {}), ((64, -1.0), {}), ((64, float("nan")), {}),
    ((64,), {"scaling": "other"}), ((64,), {"scaling": "linear", "factor": 0.0}),
    ((64,), {"scaling": "yarn", "factor": 2.0}), ((2,), {"scaling": "ntk", "factor": 2.0}),
    ((64,), {"scaling": "bands", "factor": 2.0, "original_length": 10, "fast": 1.0}),
    ((64,), {"divisors": [1.0]}), ((4,), {"divisors": [1.0, 0.0]}),
    ((4,), {"divisors": [1.0, math.inf]}), ((64,), {"amplitude": math.nan}),
    ((64,), {"scaling": "yarn", "factor": 2.0, "original_length": math.inf}),
    ((64,), {"scaling": "bands", "factor": 2.0, "original_length": 10, "fast": math.inf}),
])
def test_plans_refuse(pkg, args, kwargs):
    with pytest.raises(ValueError):
        pkg.Rotary(*args, device="cpu", **kwargs)


def test_host_tensors_are_refused(pkg):
    x = torch.zeros(2, 4, 64)
    plan = pkg.Rotary(64, device="cpu")
    with pytest.raises(ValueError, match="ROCm"):
        pkg.apply_rotary(x, None, torch.zeros(2, dtype=torch.long), plan)
    pool = torch.zeros(4, 16, 4, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm"):
        pkg.append_kv(pool, pool, x, x, i[:, None], i, i, 1)
    with pytest.raises(ValueError, match="ROCm"):
        pkg.load_kv(pool, pool, i[:, None], i, i, 1, 2)


def test_fake_shapes(pkg):
    with FakeTensorMode():
        pool = torch.empty(8, 16, 4, 64, dtype=torch.int8)
        scale = torch.empty(8, 4)
        tables, lengths = torch.empty(2, 3, dtype=torch.int32), torch.empty(2, dtype=torch.int32)
        cu = torch.empty(3, dtype=torch.int32)
        k, v = torch.ops.rlt_mi355x.load_kv(pool, pool, tables, lengths, cu, 9, 11, scale, scale,
                                            torch.float16)
        assert k.shape == v.shape == (11, 4, 64) and k.dtype == torch.float16
        x = torch.empty(11, 4, 64)
        q = torch.ops.rlt_mi355x.append_kv(pool, pool, x, x, tables, lengths, cu, 9, scale, scale, q=x)
        assert q.shape == x.shape


def test_c_entries_refuse(pkg):
    """The C entries answer bad sizes, types and modes before they touch a device."""
    from vllm_rlt_amd import _lib

    lib = _lib.library()
    n, p = 0, 16  # null and a pointer that is never followed

    def rotary(rows=1, turns=p, rot=64, hq=1, hkv=1, d=64, dtype=2, pos=p, q=p):
        return lib.rlt_rotary(q, 64, 64, p, 64, 64, pos, rows, turns, rot, 1.0, 0, 0, hq, hkv, d,
                              dtype, p, 64, 64, p, 64, 64, n)

    assert rotary(rows=0) == 0
    for bad in (dict(rows=-1), dict(rot=3), dict(rot=66), dict(turns=n), dict(d=257, rot=0), dict(d=0, rot=0),
                dict(dtype=3), dict(dtype=4), dict(pos=n), dict(q=n), dict(hq=-1)):
        assert rotary(**bad) == 1, bad

    def append(rows=1, dtype=2, kv=4, mode=3, scale=p, blocks=4, bs=16, hkv=2, d=64, seqs=1, maxq=1,
               rot=0, k=p):
        return lib.rlt_kv_append(k, 128, 64, p, 128, 64, dtype, p, p, 2048, 128, 64, 2048, 128, 64,
                                 blocks, bs, kv, scale, scale, mode, 2, 0, 1, p, 1, 1, p, p, seqs,
                                 maxq, rows, hkv, d, n, n, rot, 1.0, 0, n, 0, 0, 0, n, 0, 0, n)

    assert append(rows=0) == append(seqs=0) == append(maxq=0) == 0
    for bad in (dict(rows=-1), dict(dtype=3), dict(mode=0), dict(mode=1), dict(mode=2), dict(kv=2, mode=3),
                dict(kv=1, mode=0), dict(scale=n), dict(blocks=0), dict(bs=0), dict(d=257), dict(hkv=0),
                dict(rot=2), dict(k=n), dict(maxq=-1)):
        assert append(**bad) == 1, bad
    assert append(hkv=257) == 2

    def load(kv=4, mode=3, scale=p, out=2, rows=1, bs=16):
        return lib.rlt_kv_load(p, p, 2048, 128, 64, 2048, 128, 64, 4, bs, kv, scale, scale, mode, 2, 0,
                               1, p, 1, 1, p, p, 1, 1, rows, 2, 64, out, p, p, n)

    assert load(rows=0) == 0
    for bad in (dict(mode=0), dict(mode=1), dict(mode=2), dict(scale=n), dict(kv=2), dict(kv=3, mode=0),
                dict(kv=5), dict(bs=0), dict(rows=-1), dict(mode=4)):
        assert load(**bad) == 1, bad


def test_oracle_rotation_is_a_rotation():
    """Norms times the amplitude, the inverse, and a closed form at a quarter turn."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 2, 12, generator=g, dtype=torch.float64)
    turns, pos = torch.rand(4, generator=g, dtype=torch.float64), torch.tensor([0, 1, -3, 70000, 5])
    for inter in (False, True):
        y = orot.rotate(x, pos, turns, 1.5, inter)
        torch.testing.assert_close(y[..., :8].norm(dim=-1), 1.5 * x[..., :8].norm(dim=-1))
        assert torch.equal(y[..., 8:], x[..., 8:])
        back = orot.rotate(y, pos, turns, 1 / 1.5, inter, inverse=True)
        torch.testing.assert_close(back, x)
    y = orot.rotate(torch.tensor([[[1.0, 2.0]]]), torch.tensor([1]), torch.tensor([0.25]))
    torch.testing.assert_close(y, torch.tensor([[[-2.0, 1.0]]], dtype=torch.float64))


def test_oracle_append_rescales():
    """A larger value raises the scale of its block and head alone, and the earlier codes follow."""
    cache = torch.zeros(2, 4, 1, 2, dtype=torch.int8)
    scale = torch.zeros(2, 1)
    tables = torch.tensor([[1]], dtype=torch.int32)
    orot.append(cache, scale, torch.tensor([[[127.0, -3.0]]]), tables, [1], [1])
    assert scale[1, 0] == 1 and cache[1, 0, 0].tolist() == [127, -3]
    orot.append(cache, scale, torch.tensor([[[254.0, 1.0]]]), tables, [2], [1])
    assert scale[1, 0] == 2 and cache[1, :2, 0].tolist() == [[64, -2], [127, 0]]
    orot.append(cache, scale, torch.tensor([[[2.0, 8.0]]]), tables, [3], [1])
    assert scale[1, 0] == 2 and cache[1, :3, 0].tolist() == [[64, -2], [127, 0], [1, 4]]
    orot.append(cache, scale, torch.tensor([[[1.0, 0.0]]]), tables, [1], [1])
    assert scale[1, 0] == torch.tensor(1 / 127) and cache[1, 0, 0].tolist() == [127, 0]
    assert not cache[0].any() and scale[0, 0] == 0
