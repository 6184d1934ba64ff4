"""GPU tests of rotary positions (rotary.py over csrc/rotary.hip) against the formula in 64 bits on the CPU.

Tolerance, from the kernel's roundings: the result's own, half a step (2^-8 of it for bf16, 2^-11 fp16, 2^-24 fp32; a step of
the subnormal numbers for fp16); cosine and sine, amplitude in them, are off by at most 2^-22 a (the angle's rounding to fp32 2^-24, the series'
evaluation 2^-23 at most, the product with a 2^-24), the product that the fused sum takes rounded by 2^-24: together 2^-21.5 a (|x1| +
|x2|); and angles of far positions, whose turns carry two roundings in 64 bits and the reference's own one: 2^-51 |t|."""

import copy
import math

import pytest
import torch

import _hip
import rotary as R

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def pairs(x, rotated, interleaved):
    if interleaved:
        return x[..., 0:rotated:2], x[..., 1:rotated:2]
    return x[..., :rotated // 2], x[..., rotated // 2:rotated]


def formula(x, positions, f, a, rotated, interleaved, back=False):
    """(result, what cosine and sine multiply, |t|) in 64 bits; x [..., heads, dim], positions its leading axes."""
    x = x.detach().cpu().double()
    t = positions.cpu().double()[..., None, None] * torch.tensor(f, dtype=torch.float64)
    c, s = a * torch.cos(t), a * torch.sin(t) * (-1 if back else 1)
    y, size, angle = x.clone(), torch.zeros_like(x), torch.zeros_like(x)
    x1, x2 = pairs(x, rotated, interleaved)
    for out, value in ((y, (x1 * c - x2 * s, x2 * c + x1 * s)), (size, (a * (x1.abs() + x2.abs()),) * 2),
                       (angle, (t.abs().expand_as(x1),) * 2)):
        for to, v in zip(pairs(out, rotated, interleaved), value):
            to.copy_(v)
    return y, size, angle


def check(got, want, dtype):
    y, size, angle = want
    eps = torch.finfo(dtype).eps
    allowed = eps / 2 * y.abs() * 1.01 + size * (2. ** -21.5 + 2. ** -51 * angle) * (1 + eps) + torch.finfo(dtype).smallest_normal * eps
    off = (got.detach().cpu().double() - y).abs()
    assert got.dtype is dtype and bool((off <= allowed).all()), f"off by {float((off / allowed).max()):.3g} of what is allowed"


SHAPES = [(128, 128, False), (128, 128, True), (80, 44, True), (80, 44, False), (64, 2, False), (2, 2, True), (3, 2, False),
          (250, 250, False), (256, 192, True), (37, 36, False), (37, 20, True), (1024, 1024, False), (1024, 6, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,rotated,interleaved", SHAPES)
def test_rotation(dtype, dim, rotated, interleaved):
    print(f"rotary {dtype} dim {dim} rotated {rotated} interleaved {interleaved}", flush=True)
    g = torch.Generator().manual_seed(dim)
    rot = R.Rotary(dim, rotated=rotated, interleaved=interleaved)
    f, a = R.rotary_frequencies(rotated)
    for tokens, hq, hkv in ((1, 1, 1), (7, 5, 1), (300, 12, 3), (0, 4, 4), (33, 64, 8), (1500, 1, 1)):
        x = torch.randn(tokens, hq + 2 * hkv, dim, generator=g).to(DEV, TYPES[dtype])
        q, k = x[:, :hq], x[:, hq:hq + hkv]  # strided parts of one projection's result
        positions = torch.randint(0, 200000, (tokens,), generator=g).to(DEV, torch.int32)
        yq, yk = rot(q, k, positions=positions)
        check(yq, formula(q, positions, f, a, rotated, interleaved), TYPES[dtype])
        check(yk, formula(k, positions, f, a, rotated, interleaved), TYPES[dtype])
        assert torch.equal(rot(k, positions=positions), yk)
        assert torch.equal(yk[..., rotated:], k[..., rotated:])


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [None, R.Linear(8.), R.Ntk(4.), R.Bands(8., 8192), R.Yarn(16., 4096), R.Yarn(4., 4096, amplitude=1.5)])
def test_scalings_and_far_positions(scaling):
    rot = R.Rotary(96, rotated=64, base=500000., scaling=scaling)
    f, a = R.rotary_frequencies(64, 500000., scaling)
    x = torch.randn(6, 3, 96, generator=torch.Generator().manual_seed(2)).to(DEV)
    for kind in (torch.int32, torch.int64):
        positions = torch.tensor([0, 1, -5, 131071, 10 ** 6 + 1, 2 ** 31 - 1], dtype=kind, device=DEV)
        check(rot(x, positions=positions), formula(x, positions, f, a, 64, False), torch.float32)


@pytest.mark.gpu
def test_batches_strides_and_broadcast_positions():
    """[batch, tokens, heads, dim] as views of [batch, heads, tokens, dim], expanded, of a last axis that is no row; and
    positions of one row for all, of a row each, of one for everything."""
    g = torch.Generator().manual_seed(5)
    rot = R.Rotary(40, interleaved=True)
    f, a = R.rotary_frequencies(40)
    x = torch.randn(3, 4, 50, 40, generator=g).to(DEV, torch.bfloat16)
    shapes = {"heads before tokens": x.transpose(1, 2), "rows": x, "every second": x[:, :, ::2], "expanded": x[:1].expand(3, 4, 50, 40),
              "transposed": torch.randn(3, 4, 40, 50, generator=g).to(DEV, torch.bfloat16).transpose(2, 3)}
    for name, v in shapes.items():
        b, t = v.shape[:2]
        for p in (torch.randint(0, 9999, (t,), generator=g), torch.randint(0, 9999, (b, t), generator=g),
                  torch.randint(0, 9999, (b, 1), generator=g), torch.randint(0, 9999, (), generator=g)):
            for kind in (torch.int32, torch.int64):
                p = p.to(DEV, kind)
                y = rot(v, positions=p)
                assert y.shape == v.shape, name
                check(y, formula(v, p.expand(b, t), f, a, 40, True), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,rotated,interleaved", [(128, 128, False), (80, 44, True), (37, 20, False)])
def test_gradients(dtype, dim, rotated, interleaved):
    g = torch.Generator().manual_seed(7)
    rot = R.Rotary(dim, rotated=rotated, interleaved=interleaved, scaling=R.Yarn(8., 4096))
    f, a = R.rotary_frequencies(rotated, scaling=R.Yarn(8., 4096))
    q, k, gq, gk = (torch.randn(19, h, dim, generator=g).to(DEV, TYPES[dtype]) for h in (6, 2, 6, 2))
    q.requires_grad_(), k.requires_grad_()
    positions = torch.randint(0, 100000, (19,), generator=g).to(DEV)
    yq, yk = rot(q, k, positions=positions)
    check(yq, formula(q, positions, f, a, rotated, interleaved), TYPES[dtype])
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    check(dq, formula(gq, positions, f, a, rotated, interleaved, back=True), TYPES[dtype])
    check(dk, formula(gk, positions, f, a, rotated, interleaved, back=True), TYPES[dtype])
    # one of two, a gradient that is one number for all, and of a part
    yq, yk = rot(q, k.detach(), positions=positions)
    (dq,) = torch.autograd.grad(yq[:, 1:].sum(), (q,))
    ones = torch.ones_like(gq)
    ones[:, 0] = 0
    check(dq, formula(ones, positions, f, a, rotated, interleaved, back=True), TYPES[dtype])


@pytest.mark.gpu
def test_gradient_against_differences():
    """The rotation is linear: a difference over any step is the derivative, off by the results' roundings only (of two sums
    of 3 x 2 x 10 products of numbers below 5: 2 x 60 x 25 x 2^-23, over the step of 8)."""
    g = torch.Generator().manual_seed(8)
    rot = R.Rotary(10, rotated=6)
    x, w = (torch.randn(3, 2, 10, generator=g).clamp(-5, 5).to(DEV) for _ in range(2))
    positions = torch.tensor([3, 1000, 77], device=DEV)
    x.requires_grad_()
    (grad,) = torch.autograd.grad((rot(x, positions=positions) * w).sum(), (x,))
    with torch.no_grad():
        at = lambda v: float((rot(v, positions=positions) * w).double().sum())
        base = at(x)
        for i in range(x.numel()):
            step = torch.zeros_like(x)
            step.view(-1)[i] = 8.
            assert abs((at(x + step) - base) / 8 - float(grad.view(-1)[i])) <= 2 * 60 * 25 * 2. ** -23 / 8


@pytest.mark.gpu
def test_second_gradient():
    rot = R.Rotary(16)
    x = torch.randn(5, 2, 16, device=DEV, requires_grad=True)
    v = torch.randn(5, 2, 16, device=DEV, requires_grad=True)
    p = torch.arange(5, device=DEV)
    y = rot(x, positions=p)
    (gx,) = torch.autograd.grad(y, (x,), v, create_graph=True)  # a rotation back of v
    (gv,) = torch.autograd.grad(gx, (v,), x.detach())
    assert torch.equal(gv, y)


@pytest.mark.gpu
def test_values_that_are_no_numbers_stay_in_their_pair():
    rot = R.Rotary(32, rotated=16)
    x = torch.zeros(2, 3, 32, device=DEV)
    x[0, 1, 3], x[1, 2, 20], x[1, 0, 9] = float("nan"), float("inf"), float("inf")
    bad = ~rot(x, positions=torch.tensor([5, 9], device=DEV)).isfinite()
    want = torch.zeros_like(bad)
    want[0, 1, [3, 11]] = want[1, 2, 20] = want[1, 0, [1, 9]] = True
    assert torch.equal(bad, want)


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(9)
    rot = R.Rotary(64)
    f, a = R.rotary_frequencies(64)
    q, k = (torch.randn(20, h, 64, generator=g).to(DEV, torch.bfloat16) for h in (8, 2))
    positions = torch.randint(0, 5000, (20,), generator=g).to(DEV, torch.int32)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        rot(q, k, positions=positions)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, yk = rot(q, k, positions=positions)
    for turn in range(3):
        q.copy_(torch.randn(20, 8, 64, generator=g))
        positions.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        check(yq, formula(q, positions, f, a, 64, False), torch.bfloat16)
        check(yk, formula(k, positions, f, a, 64, False), torch.bfloat16)


@pytest.mark.gpu
def test_captured_training_step():
    """Forward and backward in one graph, replayed with other inputs."""
    g = torch.Generator().manual_seed(10)
    rot = R.Rotary(32, interleaved=True)
    f, a = R.rotary_frequencies(32)
    q, k, gq, gk = (torch.randn(9, h, 32, generator=g).to(DEV) for h in (4, 2, 4, 2))
    q.requires_grad_(), k.requires_grad_()
    positions = torch.randint(0, 5000, (9,), generator=g).to(DEV)

    def step():
        return torch.autograd.grad(rot(q, k, positions=positions), (q, k), (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dq, dk = step()
    for _ in range(3):
        gq.copy_(torch.randn(9, 4, 32, generator=g))
        positions.add_(7)
        graph.replay()
        torch.cuda.synchronize()
        check(dq, formula(gq, positions, f, a, 32, True, back=True), torch.float32)
        check(dk, formula(gk, positions, f, a, 32, True, back=True), torch.float32)


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(4, 2, 8, device=DEV)
    p = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        R.Rotary(1026)
    for kw in (dict(rotated=3), dict(rotated=0), dict(rotated=10), dict(base=1.), dict(scaling=R.Linear(0.)), dict(frequencies=[1.]),
               dict(scaling=R.Bands(2., 100, 4., 4.)), dict(scaling=R.Yarn(2., 0)), dict(scaling=R.Linear(2.), frequencies=[1.] * 4)):
        with pytest.raises(ValueError):
            R.Rotary(8, **kw)
    rot = R.Rotary(8)
    bad = [((), p), ((x, x, x), p), ((x[..., :6],), p), ((x[0],), p), ((x.double(),), p), ((x, x.half()), p), ((x, x[:3]), p),
           ((x,), p.float()), ((x,), p[:3]), ((x,), p[:, None, None]), ((x.cpu(),), p), ((x,), p.cpu())]
    for xs, positions in bad:
        with pytest.raises(ValueError):
            rot(*xs, positions=positions)
    with pytest.raises(_hip.GPTQ2DError):
        R.Rotary(8, device="cpu")


def test_frequencies():
    """What the scalings keep and divide, and where they meet."""
    plain, a = R.rotary_frequencies(64, 10000.)
    assert a == 1 and plain[0] == 1 and len(plain) == 32 and math.isclose(plain[16], 0.01)
    assert R.rotary_frequencies(64, 10000., R.Linear(4.))[0] == [f / 4 for f in plain]
    ntk = R.rotary_frequencies(64, 10000., R.Ntk(4.))[0]
    assert ntk[0] == 1 and math.isclose(ntk[-1], plain[-1] / 4)
    bands = R.rotary_frequencies(64, 10000., R.Bands(4., 8192))[0]
    yarn, amplitude = R.rotary_frequencies(64, 10000., R.Yarn(4., 8192))
    assert math.isclose(amplitude, 0.1 * math.log(4) + 1) and R.rotary_frequencies(64, 10000., R.Yarn(4., 8192, amplitude=2.))[1] == 2
    for f, b, y in zip(plain, bands, yarn):
        turns = 8192 * f / (2 * math.pi)
        assert f / 4 <= b <= f and f / 4 * (1 - 1e-12) <= y <= f * (1 + 1e-12)
        if turns >= 4:
            assert b == f
        if turns <= 1:
            assert math.isclose(b, f / 4)
        if turns > 64:
            assert y == f
        if turns < 0.5:
            assert math.isclose(y, f / 4)
    assert R.rotary_frequencies(2, 10000., R.Ntk(4.))[0] == [1.]


@pytest.mark.gpu
def test_copies_have_frequencies_of_their_own():
    rotary = R.Rotary(64)
    x, positions = torch.randn(5, 2, 64, device=DEV), torch.arange(5, device=DEV)
    want, twin = rotary(x, positions=positions), copy.deepcopy(rotary)
    rotary.turns.zero_()
    assert torch.equal(rotary(x, positions=positions), x)
    assert torch.equal(twin(x, positions=positions), want)
