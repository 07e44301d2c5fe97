"""Rotary positions on the GPU against the rotation in float64 (``oracle/rotary.py``)."""

import pytest
import torch

from oracle import rotary as orot

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _say(*args):
    print("[case]", *args, flush=True)


def _check(got, x, positions, plan, inverse=False):
    turns = plan.turns.cpu()
    want = orot.rotate(x, positions, turns, plan.amplitude, plan.interleaved, inverse)
    near = orot.rotate_error(x, turns, plan.amplitude, plan.interleaved)
    # rounded once to the type: half a step (or of the smallest subnormal)
    info = torch.finfo(got.dtype)
    near = near + (want.abs() + near) * (info.eps / 2) + info.smallest_normal * info.eps / 2
    assert ((got.double() - want).abs() <= near).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (96, 96), (96, 32), (256, 256),
                                     (256, 64), (80, 80), (20, 12), (7, 6), (7, 2), (1, 0), (33, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation(pkg, dev, dtype, dim, rot, interleaved):
    _say("rotary", dtype, dim, rot, interleaved)
    g = torch.Generator().manual_seed(dim + rot)
    if rot == 0:
        with pytest.raises(ValueError):
            pkg.Rotary(rot, device=dev)
        return
    plan = pkg.Rotary(rot, interleaved=interleaved, amplitude=1.25, device=dev)
    for rows, hq, hkv in ((1, 16, 16), (3, 5, 1), (17, 4, 2), (100, 2, 1)):
        q, k = (torch.randn(rows, h, dim, generator=g).to(dtype) for h in (hq, hkv))
        pos = torch.randint(-5, 1 << 20, (rows,), generator=g)
        a, b = pkg.apply_rotary(q.to(dev), k.to(dev), pos.to(dev), plan)
        _check(a.cpu(), q, pos, plan)
        _check(b.cpu(), k, pos, plan)
        a, none = pkg.apply_rotary(q.to(dev), None, pos.to(dev), plan, inverse=True)
        assert none is None
        _check(a.cpu(), q, pos, plan, inverse=True)


def test_far_positions(pkg, dev):
    """Positions up to 2^31: the product position * turns is off by 2^-53 of itself, 2^31 / 2 pi
    turns at most, so an angle by 2.4e-7 beyond the sines' own error."""
    plan = pkg.Rotary(128, device=dev)
    pos = torch.tensor([0, 1, 4095, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31)])
    g = torch.Generator().manual_seed(1)
    q = torch.randn(len(pos), 4, 128, generator=g)
    got = pkg.apply_rotary(q.to(dev), None, pos.to(dev), plan)[0].cpu().double()
    turns = plan.turns.cpu()
    want = orot.rotate(q, pos, turns)
    a, b = q.double()[..., :64].abs(), q.double()[..., 64:].abs()
    near = orot.rotate_error(q, turns) + torch.cat([a + b] * 2, -1) * 2.4e-7 + want.abs() * 2.0 ** -24
    assert ((got - want).abs() <= near).all()


def test_strided_in_place_and_broadcast(pkg, dev):
    """Heads of a fused projection turned in place leave the rest alone; rows that share memory
    can be read but not turned in place; odd offsets take the elementwise form."""
    g = torch.Generator().manual_seed(2)
    plan = pkg.Rotary(64, device=dev)
    pos = torch.randint(0, 9999, (37,), generator=g)
    fused = torch.randn(37, 12, 64, generator=g).to(torch.bfloat16)
    x = fused.to(dev)
    pkg.apply_rotary(x[:, :8], x[:, 8:10], pos.to(dev), plan, inplace=True)
    _check(x[:, :8].cpu(), fused[:, :8], pos, plan)
    _check(x[:, 8:10].cpu(), fused[:, 8:10], pos, plan)
    assert torch.equal(x[:, 10:].cpu(), fused[:, 10:])
    one = torch.randn(37, 1, 64, generator=g)
    wide = one.to(dev).expand(37, 4, 64)
    _check(pkg.apply_rotary(wide, None, pos.to(dev), plan)[0].cpu(), one.expand(37, 4, 64), pos, plan)
    with pytest.raises(ValueError, match="in place"):
        pkg.apply_rotary(wide, None, pos.to(dev), plan, inplace=True)
    flat = torch.randn(37 * 3 * 65 + 1, generator=g).to(torch.float16)
    odd = flat[1:].view(37, 3, 65)[..., 1:]  # rows 65 apart, no 16-byte address
    y = flat.to(dev)[1:].view(37, 3, 65)[..., 1:]
    _check(pkg.apply_rotary(y, None, pos.to(dev), plan)[0].cpu(), odd, pos, plan)
    across = torch.randn(37, 64, 3, generator=g)
    y = across.to(dev).transpose(1, 2)  # dims apart: copied first
    _check(pkg.apply_rotary(y, None, pos.to(dev), plan)[0].cpu(), across.transpose(1, 2), pos, plan)


def test_special_values_and_empty_calls(pkg, dev):
    """A NaN or an infinity stays within its pair; no rows and no heads are calls too."""
    plan = pkg.Rotary(32, device=dev)
    q = torch.ones(2, 1, 64)
    q[0, 0, 3], q[1, 0, 50] = float("nan"), float("inf")
    y = pkg.apply_rotary(q.to(dev), None, torch.tensor([3, 4], device=dev), plan)[0].cpu()
    assert y[0, 0].isnan().nonzero().flatten().tolist() == [3, 19]
    assert y[1, 0, 50] == float("inf") and y[1, 0].isfinite().sum() == 63
    e = pkg.apply_rotary(q[:0].to(dev), q[:0, :0].to(dev), torch.zeros(0, dtype=torch.long, device=dev), plan)
    assert e[0].shape == (0, 1, 64) and e[1].shape == (0, 0, 64)
    e = pkg.apply_rotary(q[:, :0].to(dev), q.to(dev), torch.tensor([0, 0], device=dev), plan)
    assert torch.equal(e[1].cpu()[..., 32:], q[..., 32:])


def test_gradient_is_the_inverse(pkg, dev):
    """<apply(x), y> = <x, inverse(y)>, and against differences of the rotation."""
    g = torch.Generator().manual_seed(4)
    plan = pkg.Rotary(48, interleaved=True, amplitude=0.7, device=dev)
    pos = torch.randint(0, 99999, (9,), generator=g).to(dev)
    x, y, d = (torch.randn(9, 3, 64, generator=g).to(dev) for _ in range(3))
    fx = pkg.apply_rotary(x, None, pos, plan)[0].double()
    gy = pkg.apply_rotary(y, None, pos, plan, inverse=True)[0].double()
    # 1728 products of N(0, 1) values, each side within 2^-20 of itself per product
    assert abs((fx * y.double()).sum() - (x.double() * gy).sum()) <= 1728 * 2.0 ** -17
    step = pkg.apply_rotary(x + d, None, pos, plan)[0].double() - fx
    assert abs((step * y.double()).sum() - (d.double() * gy).sum()) <= 1728 * 2.0 ** -16


def test_refusals(pkg, dev):
    plan = pkg.Rotary(64, device=dev)
    q, pos = torch.zeros(4, 2, 64, device=dev), torch.zeros(4, dtype=torch.long, device=dev)
    for bad in (lambda: pkg.apply_rotary(q, None, pos[:3], plan),
                lambda: pkg.apply_rotary(q[0], None, pos, plan),
                lambda: pkg.apply_rotary(q.double(), None, pos, plan),
                lambda: pkg.apply_rotary(q, q.half(), pos, plan),
                lambda: pkg.apply_rotary(q, q[:3], pos, plan),
                lambda: pkg.apply_rotary(q[..., :32], None, pos, plan),
                lambda: pkg.apply_rotary(torch.zeros(4, 2, 260, device=dev), None, pos, plan),
                lambda: pkg.apply_rotary(q, None, pos.cpu(), plan),
                lambda: pkg.apply_rotary(q, None, pos, pkg.Rotary(64, device="cpu"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="share"):
        pkg.apply_rotary(q, q, pos, plan, inplace=True)
    fused = torch.zeros(4, 12, 64, device=dev)
    for a, b in ((fused[:, :8], fused[:, 7:9]), (fused[:, 2:10], fused[:, 1:3]), (fused[:, :3], fused[..., :2, :]),
                 (fused[:2], fused[1:3]), (fused[::2], fused[:2])):
        with pytest.raises(ValueError, match="share"):
            pkg.apply_rotary(a, b, pos[:len(a)], plan, inplace=True)
    for a, b in ((fused[:, :8], fused[:, 8:10]), (fused[:, 2:10], fused[:, :2]), (fused[:, 4:], fused[:, :4]),
                 (fused[:2], fused[2:])):
        pkg.apply_rotary(a, b, pos[:len(a)], plan, inplace=True)
    with pytest.raises(ValueError, match="stride"):
        pkg.apply_rotary(torch.zeros(4, 64, 2, device=dev).transpose(1, 2), None, pos, plan, inplace=True)
