"""Group normalisation with an activation (``groupnorm_forward`` / ``_backward``, the autograd wrapper and module) against the
formulas in 64 bits, on the CPU reference and - marked gpu - on the HIP kernels.

Tolerances are bounds, element by element (u = 2^-24, h = half a step of the tensors' type): the mean is kept to 4 u of the
largest deviation, 1 / standard deviation to 8 u, so xhat is off by 16 u (1 + |xhat|); u = gamma xhat + beta by |gamma| times that
and 4 u of its terms; the activations and their slopes have first and second derivatives of at most 1.1, and are off by
(8 + 4 |u|) u themselves; relu's slope jumps, so elements with |u| inside the bound are left out by construction (dy is
zero there); sums over n terms by n u of the absolute sum, which is generous for sums in pieces; outputs by h."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import autograd as A
from distributed_tensorflow_amd.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "relu", "sigmoid", "tanh", "silu"]
U = 2.0 ** -24


def _inputs(shape, groups, dtype, device, act, seed=0, offset=0.0):
    C = shape[-1]
    g = torch.Generator().manual_seed(seed + sum(shape) + 31 * groups)
    x = (torch.randn(shape, generator=g) * (0.5 + torch.rand(C, generator=g)) + torch.randn(C, generator=g) + offset).to(dtype)
    gamma, beta = torch.rand(C, generator=g) + 0.5, torch.randn(C, generator=g) * 0.3
    dy = (torch.randn(shape, generator=g) + 0.5).to(dtype)
    if act == "relu":
        # no gradient where u is next to zero: the slope of either side is right there
        v = x.double().reshape(shape[0], -1, groups, C // groups)
        mean, var = v.mean((1, 3), keepdim=True), v.var((1, 3), unbiased=False, keepdim=True)
        u = ((v - mean) / torch.sqrt(var + 1e-3)).reshape(shape) * gamma + beta
        dy = torch.where(u.abs() < (1e-3 if dtype == torch.float32 else 2e-2), torch.zeros_like(dy), dy)
    return [t.to(device) for t in (x, gamma, beta, dy)]


def _act(u, act):
    return {None: lambda: u, "relu": lambda: torch.relu(u), "sigmoid": lambda: torch.sigmoid(u), "tanh": lambda: torch.tanh(u),
            "silu": lambda: u * torch.sigmoid(u)}[act]()


def _check(shape, groups, dtype, device, act, offset=0.0, affine=True, eps=1e-3):
    x, gamma, beta, dy = _inputs(shape, groups, dtype, device, act, offset=offset)
    if not affine:
        gamma = beta = None
        if act == "relu":
            act = None
    half = torch.finfo(dtype).eps / 2
    leaves = [t.clone().requires_grad_() for t in (x, gamma, beta) if t is not None]
    y = A.group_norm(leaves[0], *(leaves[1:] if affine else (None, None)), groups, eps=eps, activation=act)
    assert y.dtype == dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, leaves, dy)
    # 64 bits
    B, C = shape[0], shape[-1]
    r = [t.detach().double().requires_grad_() for t in leaves]
    v = r[0].reshape(B, -1, groups, C // groups)
    mean, var = v.mean((1, 3), keepdim=True), v.var((1, 3), unbiased=False, keepdim=True)
    xhat = ((v - mean) / torch.sqrt(var + eps)).reshape(shape)
    ga, be = (r[1], r[2]) if affine else (torch.ones((), device=device), torch.zeros((), device=device))
    u = xhat * ga + be
    want = _act(u, act)
    rg = torch.autograd.grad(want, r, dy.double(), retain_graph=True)
    with torch.no_grad():
        big = (v - mean).abs().amax((1, 3), keepdim=True).expand_as(v).reshape(shape) / torch.sqrt(var + eps).expand_as(v).reshape(shape)
        exhat = 16 * U * (1 + xhat.abs() + big)
        eu = exhat * ga.abs() + 4 * U * ((xhat * ga).abs() + be.abs())
        eact = 1.1 * eu + (8 + 4 * u.abs()) * U
        yb = eact + half * (want.abs() + eact) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert bool(((y.double() - want).abs() <= yb).all()), float(((y.double() - want).abs() - yb).max())
        # backward: du, d = gamma du and the two means
        slope = torch.ones_like(u) if act is None else (u > 0).double() if act == "relu" else _slope(u, act)
        du = dy.double() * slope
        edu = dy.double().abs() * ((0.0 if act in (None, "relu") else 1.1) * eu + (8 + 4 * u.abs()) * U)
        lead = tuple(range(len(shape) - 1))
        n = x.numel() // C
        if affine:
            terms = du.abs() * exhat + edu * xhat.abs() + edu * exhat
            bounds = (terms + n * U * (du * xhat).abs()).sum(lead), (edu + n * U * du.abs()).sum(lead)
            for got, w, b, name in zip(grads[1:], rg[1:], bounds, ("dgamma", "dbeta")):
                assert bool(((got.double() - w).abs() <= b + U * w.abs()).all()), name
        d, ed = du * ga, edu * ga.abs()
        m = v[0].numel() // groups
        gv = lambda t: t.reshape(B, -1, groups, C // groups)
        mean_of = lambda t: gv(t).mean((1, 3), keepdim=True).expand_as(v).reshape(shape)
        ed1 = mean_of(ed) + m * U * mean_of(d.abs())
        m2 = mean_of(d * xhat).abs()
        ed2 = mean_of(ed * xhat.abs() + d.abs() * exhat) + m * U * mean_of((d * xhat).abs())
        inv = (1 / torch.sqrt(var + eps)).expand_as(v).reshape(shape)
        e = inv * (ed + ed1 + xhat.abs() * ed2 + exhat * m2 + 16 * U * (d.abs() + mean_of(d).abs() + xhat.abs() * m2))
        b = e + half * (rg[0].abs() + e) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert bool(((grads[0].double() - rg[0]).abs() <= b).all()), float(((grads[0].double() - rg[0]).abs() - b).max())


def _slope(u, act):
    s = torch.sigmoid(u)
    return {"sigmoid": lambda: s * (1 - s), "tanh": lambda: 1 - torch.tanh(u) ** 2, "silu": lambda: s * (1 + u * (1 - s))}[act]()


SMALL = [((1, 1), 1), ((2, 3), 1), ((3, 8), 4), ((1, 7, 7, 64), 32), ((2, 5, 3, 15), 5), ((4, 9, 10), 5), ((2, 33, 1, 20), 20),
         ((3, 4, 6, 36), 9)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", SMALL)
def test_values_and_gradients(device, dtype, shape, groups):
    _check(shape, groups, dtype, device, ACTS[(sum(shape) + groups) % 5])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ACTS)
def test_activations_and_no_affine(device, act):
    _check((2, 6, 5, 24), 3, torch.float32, device, act)
    _check((2, 6, 5, 24), 6, torch.float32, device, act, affine=False)


@pytest.mark.parametrize("device", DEVICES)
def test_a_mean_far_above_the_deviation(device):
    _check((3, 40, 16), 4, torch.float32, device, "silu", offset=300.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups,act", [
    ((5, 24, 24, 32), 8, "relu"), ((1, 200, 201, 32), 8, "silu"), ((2, 65, 67, 225), 25, "silu"), ((700, 3, 3, 64), 1, "tanh"),
    ((2, 3, 5, 1031), 1, "sigmoid"), ((3, 17, 2048), 32, None), ((2, 40, 8200), 8, "relu"), ((2, 9, 9001), 1, "silu"),
    ((1, 50000, 3), 3, "silu"), ((1, 30011, 1), 1, None), ((3000, 2, 40), 20, "relu"), ((70000, 4), 2, "silu")])
def test_values_and_gradients_of_larger_sizes(gpu_device, dtype, shape, groups, act):
    _check(shape, groups, dtype, "cuda", act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [((47, 90, 34, 6), 3), ((9, 2500, 3), 1), ((5, 8100, 1), 1), ((6, 1021, 5), 5), ((3, 400, 2), 2)])
def test_few_channels_of_many_positions(gpu_device, dtype, shape, groups):
    # the channels' own means differ by more than their deviations: long sums of like numbers
    _check(shape, groups, dtype, "cuda", "tanh")
    x = _inputs(shape, groups, dtype, "cuda", None)[0]
    stats = F.groupnorm_forward(x, None, None, groups)[1].double()
    v = x.double().reshape(shape[0], -1, groups, shape[-1] // groups)
    mean, var = v.mean((1, 3)), v.var((1, 3), unbiased=False)
    assert bool(((stats[0] + stats[1] - mean).abs() <= 4 * U * (v - mean[:, None, :, None]).abs().amax((1, 3))).all())
    assert bool(((stats[2] * torch.sqrt(var + 1e-3) - 1).abs() <= 8 * U).all())


@pytest.mark.parametrize("device", DEVICES)
def test_one_gradient_at_a_time(device):
    x, gamma, beta, dy = _inputs((3, 5, 7, 12), 4, torch.float32, device, "silu")
    full = [t.clone().requires_grad_() for t in (x, gamma, beta)]
    want = torch.autograd.grad(A.group_norm(*full, 4, activation="silu"), full, dy)
    for k in range(3):
        one = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, gamma, beta))]
        assert torch.equal(torch.autograd.grad(A.group_norm(*one, 4, activation="silu"), one[k], dy)[0], want[k])


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_against_differences(device):
    # central differences, h = 2^-7: u changes by less than 8 h a step, silu's third derivative is below 1, the second
    # derivatives of xhat below 8; what rounding leaves is n (8 u) / h
    x, gamma, beta, dy = _inputs((2, 4, 12), 3, torch.float32, device, "silu")
    g = torch.Generator().manual_seed(5)
    d = [torch.randn(t.shape, generator=g).to(device) * 0.25 for t in (x, gamma, beta)]
    leaves = [t.clone().requires_grad_() for t in (x, gamma, beta)]
    grads = torch.autograd.grad(A.group_norm(*leaves, 3, activation="silu"), leaves, dy)
    slope = float(sum((a * b).double().sum() for a, b in zip(grads, d)))
    h = 2.0 ** -7
    at = lambda s: (A.group_norm(*[t + s * e for t, e in zip((x, gamma, beta), d)], 3, activation="silu").double() * dy.double()).sum()
    n = x.numel()
    assert abs(float((at(h) - at(-h)) / (2 * h)) - slope) <= float(dy.abs().sum()) * (8 * h) ** 2 / 6 + n * 40 * U / h


@pytest.mark.parametrize("device", DEVICES)
def test_layouts_empty_batches_and_other_float_types(device):
    x, gamma, beta, dy = _inputs((4, 6, 8), 2, torch.float32, device, None)
    want = A.group_norm(x, gamma, beta, 2)
    assert torch.equal(A.group_norm(x.transpose(0, 1).contiguous().transpose(0, 1), gamma, beta, 2), want)
    assert A.group_norm(x[:0], gamma, beta, 2).shape == (0, 6, 8)
    leaves = [t.clone().requires_grad_() for t in (x[:0], gamma, beta)]
    grads = torch.autograd.grad(A.group_norm(*leaves, 2), leaves, dy[:0])
    assert grads[0].shape == (0, 6, 8) and not grads[1].any() and not grads[2].any()
    # one sample that starts at an odd element of a larger buffer
    buf = torch.zeros(4 * 48 + 1, device=device)
    view = buf[1:].view(4, 6, 8)
    view.copy_(x)
    assert torch.equal(A.group_norm(view, gamma, beta, 2), want)
    g16 = gamma.to(torch.bfloat16).requires_grad_()
    (dg,) = torch.autograd.grad(A.group_norm(x, g16, beta, 2), g16, dy)
    assert dg.dtype == torch.bfloat16


def test_refusals():
    x, gamma, beta, _ = _inputs((2, 3, 8), 2, torch.float32, "cpu", None)
    with pytest.raises(ValueError, match="do not divide"):
        A.group_norm(x, gamma, beta, 3)
    with pytest.raises(ValueError, match="do not divide"):
        A.group_norm(x, gamma, beta, 0)
    with pytest.raises(ValueError, match="16384 groups"):
        A.group_norm(torch.zeros(1, 2, 20000), None, None, 20000)
    with pytest.raises(ValueError, match="unsupported activation"):
        A.group_norm(x, gamma, beta, 2, activation="gelu")
    with pytest.raises(ValueError, match="gamma must"):
        A.group_norm(x, gamma[:7], beta, 2)
    with pytest.raises(ValueError, match="batch"):
        A.group_norm(x[0, 0], gamma, beta, 2)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        F.groupnorm_forward(x.double(), gamma, beta, 2)
    with pytest.raises(ValueError, match="contiguous"):
        F.groupnorm_forward(x, gamma, beta, 2, out=torch.empty(2, 8, 3).transpose(1, 2))
    y, stats = F.groupnorm_forward(x, gamma, beta, 2)
    with pytest.raises(ValueError, match="stats"):
        F.groupnorm_backward(x, y, gamma, beta, 2, stats[:2])
    with pytest.raises(ValueError, match="dgamma"):
        F.groupnorm_backward(x, y, gamma, beta, 2, stats, dgamma=torch.empty(7))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((5, 24, 24, 32), 8), ((2, 65, 67, 225), 25)])
def test_captured_and_replayed(gpu_device, shape, groups):
    x, gamma, beta, dy = _inputs(shape, groups, torch.float32, "cuda", "silu")

    def step():
        y, stats = F.groupnorm_forward(x, gamma, beta, groups, act=F.groupnorm_activation("silu"))
        dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
        F.groupnorm_backward(x, dy, gamma, beta, groups, stats, F.groupnorm_activation("silu"), dg, db, dx)
        return y, dx, dg, db

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        for t, n in zip((x, gamma, beta, dy), _inputs(shape, groups, torch.float32, "cuda", "silu", seed=50 + k)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step())), k
