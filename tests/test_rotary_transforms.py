"""Derivatives of rotary positions in every direction, and torch.func's transforms of them.

On the CPU the launch is replaced by the formula in 64 bits, so that torch's own checks against differences say whether the
derivatives are wired right; on the GPU every one of them is a rotation, and equal to the rotation made by itself."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.func import grad, jacfwd, jacrev, jvp, vjp, vmap

import _hip
import rotary as R

GPU = pytest.mark.gpu


@pytest.fixture
def on_cpu(monkeypatch):
    """Rotations on the CPU: the launch's arguments are not made, its values are the formula's."""
    launches = []

    def rotate(self, xs, positions, back):
        launches.append(len(xs))
        angle = positions.expand(xs[0].shape[:-2]).double()[..., None, None] * self.turns * 2 * torch.pi
        c, s = self.amplitude * torch.cos(angle), (-1 if back else 1) * self.amplitude * torch.sin(angle)
        out, half = [], self.rotated // 2
        for x in xs:
            a, b = x[..., :half], x[..., half:self.rotated]
            out.append(torch.cat([a * c - b * s, b * c + a * s, x[..., self.rotated:]], -1))
        return tuple(out)

    monkeypatch.setattr(_hip, "require_device", lambda t: None)
    monkeypatch.setattr(R, "_TYPES", {torch.float64: 0})
    monkeypatch.setattr(R.Rotary, "_rotate", rotate)
    return launches


def small(device, dtype):
    g = torch.Generator().manual_seed(3)
    rot = R.Rotary(6, rotated=4, scaling=R.Yarn(8., 4096), device=device)
    q, k, dq, dk = (torch.randn(5, h, 6, generator=g).to(device, dtype) for h in (3, 1, 3, 1))
    return rot, q, k, dq, dk, torch.tensor([0, 7, 300, -2, 11], device=device)


def test_derivatives_against_differences(on_cpu):
    rot, q, k, _, _, positions = small("cpu", torch.float64)
    q.requires_grad_(), k.requires_grad_()

    def both(q, k):
        return rot(q, k, positions=positions)

    assert torch.autograd.gradcheck(both, (q, k), check_forward_ad=True, check_batched_grad=True, check_batched_forward_grad=True,
                                    check_undefined_grad=True)
    assert torch.autograd.gradgradcheck(lambda q, k: [y * y for y in both(q, k)], (q, k), check_fwd_over_rev=True, check_rev_over_rev=True)
    assert torch.autograd.gradcheck(lambda q: rot(q, k.detach(), positions=positions), (q,), check_forward_ad=True)


def test_a_call_that_nothing_follows_makes_no_node(on_cpu, monkeypatch):
    rot, q, k, _, _, positions = small("cpu", torch.float64)
    monkeypatch.setattr(R, "_Rotation", None)
    with fwAD.dual_level():
        rot(q, k, positions=positions)
    with torch.no_grad():
        rot(q.requires_grad_(), k, positions=positions)
    assert on_cpu == [2, 2]


def check_all(rot, q, k, dq, dk, positions):
    """Every way to a derivative gives the rotation of the direction, in the same bits."""
    def turned(*xs):
        return rot(*xs, positions=positions)

    with torch.no_grad():
        y, dy = turned(q, k), turned(dq, dk)
        back = rot._rotate((dq, dk), positions, True)
    with fwAD.dual_level():
        out = turned(fwAD.make_dual(q, dq), fwAD.make_dual(k, dk))
        assert all(torch.equal(fwAD.unpack_dual(o).primal, a) and torch.equal(fwAD.unpack_dual(o).tangent, b) for o, a, b in zip(out, y, dy))
        out = turned(q, fwAD.make_dual(k, dk))  # one of two
        assert fwAD.unpack_dual(out[0]).tangent is None or not fwAD.unpack_dual(out[0]).tangent.any()
        assert torch.equal(fwAD.unpack_dual(out[1]).tangent, dy[1])
        out = turned(fwAD.make_dual(q.detach().requires_grad_(), dq))  # forward, of what backward is wanted of too
        assert torch.equal(fwAD.unpack_dual(out).tangent, dy[0])
        leaf = q.detach().requires_grad_()  # a gradient with a direction of its own
        (g,) = torch.autograd.grad(turned(leaf), (leaf,), fwAD.make_dual(dq, q))
        assert torch.equal(fwAD.unpack_dual(g).tangent, rot._rotate((q,), positions, True)[0])
    values, tangents = jvp(turned, (q, k), (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip((*values, *tangents), (*y, *dy)))
    assert all(torch.equal(a, b) for a, b in zip(vjp(turned, q, k)[1]((dq, dk)), back))
    assert torch.equal(grad(lambda q: (turned(q, k)[0] * dq).sum())(q), back[0])
    assert torch.equal(jacfwd(turned)(q), jacrev(turned)(q))
    # mapped over new axes, wherever they stand, with positions mapped or not, within a map
    qs, ks = torch.stack([q, dq, 2 * q], 1), torch.stack([k, dk, 2 * k], 0)
    ps = torch.stack([positions, positions + 1, positions * 2])
    got = vmap(lambda q, k, p: rot(q, k, positions=p), (1, 0, 0))(qs, ks, ps)
    for i in range(3):
        assert all(torch.equal(a[i], b) for a, b in zip(got, rot(qs[:, i], ks[i], positions=ps[i])))
    got = vmap(turned, (1, None))(qs, k)
    for i in range(3):
        assert all(torch.equal(a[i], b) for a, b in zip(got, turned(qs[:, i], k)))
    got = vmap(lambda p: rot(q, positions=p))(ps[:, :1])
    assert all(torch.equal(a, rot(q, positions=p)) for a, p in zip(got, ps[:, :1]))
    batch = torch.stack([q, dq])  # two axes before the heads, and the mapped one makes three; twice over, four
    got = vmap(vmap(lambda x: rot(x, positions=positions)))(torch.stack([torch.stack([batch, -batch]), torch.stack([2 * batch, batch])]))
    assert torch.equal(got[1, 0], rot(2 * batch, positions=positions)) and torch.equal(got[0, 1], rot(-batch, positions=positions))
    got = vmap(grad(lambda x, w: (turned(x) * w).sum()), (1, None))(qs, dq)  # of each of many
    assert all(torch.equal(g, back[0]) for g in got)


def test_every_way_to_a_derivative(on_cpu):
    check_all(*small("cpu", torch.float64))


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_way_to_a_derivative_on_the_gpu(dtype):
    check_all(*small("cuda", dtype))
