"""Softmax cross-entropy of a linear head over a large vocabulary (``linear_xent_forward`` / ``_backward`` and the autograd
wrapper) against the formulas in 64 bits, on the CPU reference and - marked gpu - on the HIP kernels.

Tolerances are bounds, element by element, propagated through the formulas (u = 2^-24; h = half a step of the type, 2^-8 for
bfloat16): a logit is off by at most dz_ = 2 (K + 4) u (|x| |w| + |b|) - K products summed in any order, operands exact or split
into limbs that lose less than u; the row's logsumexp by the p-weighted mean of that plus 2 V u (sums of V exponentials, each
off by (4 + |z|) u); a probability relatively by the sum of both; dz besides by two roundings to bfloat16 where the products
take bfloat16; sums over rows or classes by their length times u of the absolute sum; an output by h of itself."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import autograd as A
from distributed_tensorflow_amd.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def _inputs(M, K, V, dtype, device, seed=0, bias=True, ignored=0.2, scale=2.0):
    g = torch.Generator().manual_seed(seed + 7 * M + 3 * K + V)
    x = torch.randn(M, K, generator=g).to(dtype)
    w = (torch.randn(K, V, generator=g) * (scale / math.sqrt(K))).to(dtype)
    b = torch.randn(V, generator=g).to(dtype) if bias else None
    labels = torch.randint(0, V, (M,), generator=g)
    labels[torch.rand(M, generator=g) < ignored] = -1
    to = lambda t: None if t is None else t.to(device)
    return to(x), to(w), to(b), to(labels)


def _reference(x, w, b, labels, g, bf16=False, ignore=-1):
    """(loss, dx, dw, db) in 64 bits on the operands' device with a bound of the error of each; g: weight of every row."""
    half = torch.finfo(x.dtype).eps / 2 if x.dtype == torch.bfloat16 else U
    counted = labels != ignore
    r = (lambda t: t.float().bfloat16().double()) if bf16 else (lambda t: t.double())
    x64 = torch.where(counted[:, None], r(x), torch.zeros((), dtype=torch.float64, device=x.device))
    w64 = r(w)
    b64 = torch.zeros(w.shape[1], dtype=torch.float64, device=x.device) if b is None else b.double()
    M, K = x.shape
    V = w.shape[1]
    z = x64 @ w64 + b64
    ez = 2 * (K + 4) * U * (x64.abs() @ w64.abs() + b64.abs().clamp(max=1e30)) + 4 * U
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    zf = z.abs().masked_fill(p == 0, 0.0)
    rel = ez + (p * ez).sum(1, keepdim=True) + (2 * V + 16) * U + (zf + lse.abs()[:, None]) * 4 * U
    at = labels.clamp(min=0)[:, None]
    zl = z.gather(1, at)[:, 0]
    loss = torch.where(counted, lse - zl, torch.zeros_like(lse))
    eloss = rel.gather(1, at)[:, 0] + (p * rel).sum(1) + U * (lse.abs() + zl.abs()) * 2
    g = torch.where(counted, g.double(), torch.zeros_like(lse))
    dz = p * g[:, None]
    edz = dz.abs() * rel
    dz = dz.scatter_add(1, at, -g[:, None])
    own = p.gather(1, at) * rel.gather(1, at) * g.abs()[:, None] + 4 * U * dz.gather(1, at).abs()
    edz = edz.scatter(1, at, own) + 4 * U * dz.abs()
    db, edb = dz.sum(0), edz.sum(0) + 2 * M * U * dz.abs().sum(0)
    if bf16 or x.dtype == torch.bfloat16:
        edz = edz + 2.02 * 2.0 ** -8 * dz.abs()
        edb = edb + 2.02 * 2.0 ** -8 * dz.abs().sum(0)
    out = lambda v, e: (v, e + half * (v.abs() + e) + 1e-37)
    dx, edx = dz @ w64.t(), edz @ w64.abs().t() + 2 * (V + 4) * U * (dz.abs() @ w64.abs().t())
    dw, edw = x64.t() @ dz, x64.abs().t() @ edz + 2 * (M + 4) * U * (x64.abs().t() @ dz.abs())
    return (loss, eloss + U), out(dx, edx), out(dw, edw), out(db, edb)


def _within(got, want_bound, name):
    want, bound = want_bound
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), name
    assert bool((off <= bound).all()), "%s: off by %.3g where %.3g is allowed" % (
        name, float(off.max()), float(bound.reshape(-1)[(off - bound).argmax()]))


def _check(x, w, b, labels, bf16=False, reduction="mean"):
    M = x.shape[0]
    leaves = [t.detach().clone().requires_grad_() for t in (x, w) + (() if b is None else (b,))]
    bl = leaves[2] if b is not None else None
    loss = A.linear_softmax_cross_entropy(leaves[0], leaves[1], labels, bl, reduction=reduction, bf16=bf16)
    n = max(int((labels != -1).sum()), 1)
    up = torch.linspace(0.5, 1.5, M, device=x.device) if reduction == "none" else torch.tensor(0.75, device=x.device)
    g = {"none": up, "sum": up.expand(M), "mean": up.expand(M) / n}[reduction]
    rl, rdx, rdw, rdb = _reference(x, w, b, labels, g.float(), bf16)
    grads = torch.autograd.grad(loss, leaves, up)
    if reduction == "none":
        _within(loss.detach(), rl, "loss")
    else:
        d = n if reduction == "mean" else 1
        _within(loss.detach(), (rl[0].sum() / d, rl[1].sum() / d + 4 * U * rl[0].abs().sum() / d), "loss")
    for got, want, name in zip(grads, (rdx, rdw, rdb), ("dx", "dw", "db")):
        # the row weights themselves are float32 products and quotients
        _within(got, (want[0], want[1] + 4 * U * want[0].abs()), name)
    return loss


SMALL = [(1, 1, 1), (1, 64, 257), (3, 7, 2), (5, 33, 1000), (64, 64, 64), (65, 129, 255), (130, 96, 513)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", SMALL)
def test_loss_and_gradients(device, dtype, size):
    _check(*_inputs(*size, dtype, device, bias=size[0] != 5), reduction=["mean", "sum", "none"][size[1] % 3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(1, 512, 32001), (17, 1000, 4096), (257, 72, 12345), (300, 520, 2049), (1024, 256, 8192),
                                  (2047, 128, 33000), (9000, 64, 4097), (33, 2056, 8200),
                                  (1500, 1100, 12000), (700, 260, 40000), (2100, 520, 8000)])
def test_loss_and_gradients_of_larger_sizes(gpu_device, dtype, size):
    _check(*_inputs(*size, dtype, "cuda", bias=size[1] != 72), reduction=["mean", "none"][size[2] % 2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tiles", [0, 1, 3])
@pytest.mark.parametrize("size", [(100, 72, 1500), (300, 130, 1290)])
def test_exponentials_that_were_not_kept_are_computed_again(gpu_device, monkeypatch, dtype, tiles, size):
    x, w, b, labels = _inputs(*size, dtype, "cuda")
    monkeypatch.setattr(F, "LINEAR_XENT_KEEP_BYTES", tiles * 256 * size[0] * torch.finfo(dtype).bits // 8)
    state = F.linear_xent_forward(x, w, b, labels, keep=True)[1]
    assert (state.kept is None) if tiles == 0 else tuple(state.kept.shape) == (size[0], 256 * tiles)
    _check(x, w, b, labels)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_vocabulary_in_several_pieces(gpu_device, dtype):
    # dz of more than 512 MB; in float32 the exponentials exceed the budget besides
    _check(*_inputs(9000, 40, 33001, dtype, "cuda"))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("size", [(65, 129, 255), (5, 64, 1000)])
def test_rounded_operands(device, size):
    _check(*_inputs(*size, torch.float32, device), bf16=True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_confident_row_keeps_its_small_gradient(device, dtype):
    # the label's probability is 1 - 1e-4: p - 1 must not come from a rounded p
    x, w, b, labels = _inputs(4, 64, 300, dtype, device, ignored=0.0, bias=True)
    b[:] = 0.0
    b[7] = 22.0
    labels[:] = 7
    _check(x, w, b, labels)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ignored_rows_may_hold_anything(device, dtype):
    x, w, b, labels = _inputs(70, 64, 300, dtype, device, ignored=0.0)
    labels[3], labels[64] = -1, -1
    ref = [t.clone() for t in (x, w, b)]
    x[3], x[64] = float("nan"), float("inf")
    got, want = [], []
    for xx, out in ((x, got), (ref[0], want)):
        leaves = [t.detach().clone().requires_grad_() for t in (xx, w, b)]
        loss = A.linear_softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2])
        out += [loss.detach(), *torch.autograd.grad(loss, leaves)]
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert not got[1][3].any() and not got[1][64].any()


@pytest.mark.parametrize("device", DEVICES)
def test_no_counted_row(device):
    x, w, b, labels = _inputs(9, 16, 40, torch.float32, device)
    labels[:] = -5
    leaves = [t.requires_grad_() for t in (x, w, b)]
    loss = A.linear_softmax_cross_entropy(x, w, labels, b, ignore_index=-5)
    assert float(loss.detach()) == 0.0
    assert all(not g.any() for g in torch.autograd.grad(loss, leaves))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", ["inf", "lowest"])
def test_masked_classes_have_no_probability(device, dtype, mask):
    x, w, b, labels = _inputs(66, 40, 900, dtype, device, ignored=0.0)
    b[128:700] = -math.inf if mask == "inf" else torch.finfo(dtype).min
    labels = labels % 128
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    loss = A.linear_softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2], reduction="none")
    dx, dw, db = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    assert not dw[:, 128:700].any() and not db[128:700].any()
    keep = torch.cat([torch.arange(128), torch.arange(700, 900)]).to(device)
    want = _reference(x, w[:, keep], b[keep], labels, torch.ones(66, device=device))
    _within(loss.detach(), want[0], "loss")
    _within(dx, (want[1][0], want[1][1] * 900 / 328), "dx")
    _within(dw[:, keep], want[2], "dw")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_ignored_class_of_the_vocabulary(device, dtype):
    # rows labelled 7 count for nothing, and class 7 keeps its share of the others' probability
    x, w, b, labels = _inputs(70, 64, 300, dtype, device, ignored=0.0)
    labels[::3] = 7
    got, want = [], []
    for lab, ignore, out in ((labels, 7, got), (torch.where(labels == 7, -1, labels), -1, want)):
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
        loss = A.linear_softmax_cross_entropy(leaves[0], leaves[1], lab, leaves[2], ignore_index=ignore)
        out += [loss.detach(), *torch.autograd.grad(loss, leaves)]
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
def test_other_orders_in_memory(device):
    # a head that shares the table of an embedding, w = table.t(); features and labels as views with steps
    x, w, b, labels = _inputs(40, 64, 300, torch.float32, device)
    table = w.t().contiguous().requires_grad_()
    wide = torch.stack([x, x], dim=1).transpose(0, 1).requires_grad_()
    loss = A.linear_softmax_cross_entropy(wide[0], table.t(), torch.stack([labels, labels], dim=1)[:, 0], b)
    dx, dt = torch.autograd.grad(loss, (wide, table))
    x, w = x.requires_grad_(), w.requires_grad_()
    plain = A.linear_softmax_cross_entropy(x, w, labels, b)
    ex, ew = torch.autograd.grad(plain, (x, w))
    assert torch.equal(loss, plain) and torch.equal(dx[0], ex) and not dx[1].any() and torch.equal(dt, ew.t())


@pytest.mark.parametrize("device", DEVICES)
def test_a_label_outside_the_vocabulary_is_seen(device):
    x, w, b, labels = _inputs(8, 16, 40, torch.float32, device, ignored=0.0)
    labels[2], labels[5] = 40, -3
    leaf = x.clone().requires_grad_()
    loss = A.linear_softmax_cross_entropy(leaf, w, labels, b, reduction="none")
    (dx,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    bad = torch.zeros(8, dtype=torch.bool, device=device)
    bad[2] = bad[5] = True
    assert torch.equal(torch.isnan(loss), bad) and torch.equal(torch.isnan(dx).any(1), bad)


@pytest.mark.parametrize("device", DEVICES)
def test_shapes_reductions_and_empty_batches(device):
    x, w, b, labels = _inputs(12, 16, 40, torch.float32, device)
    rows = A.linear_softmax_cross_entropy(x, w, labels, b, reduction="none")
    cube = A.linear_softmax_cross_entropy(x.view(3, 4, 16), w, labels.view(3, 4), b, reduction="none")
    assert cube.shape == (3, 4) and torch.equal(cube.reshape(-1), rows)
    strided = A.linear_softmax_cross_entropy(x.t().contiguous().t(), w.t().contiguous().t(), labels, b, reduction="none")
    assert torch.equal(strided, rows)
    n = int((labels != -1).sum())
    total = A.linear_softmax_cross_entropy(x, w, labels, b, reduction="sum")
    torch.testing.assert_close(total, A.linear_softmax_cross_entropy(x, w, labels, b) * n, rtol=1e-6, atol=0)
    leaves = [t[:0].detach().clone().requires_grad_() if t is x else t.detach().clone().requires_grad_() for t in (x, w, b)]
    none = A.linear_softmax_cross_entropy(leaves[0], leaves[1], labels[:0], leaves[2])
    grads = torch.autograd.grad(none, leaves)
    assert float(none.detach()) == 0.0 and grads[0].shape == (0, 16) and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_gradient_at_a_time_and_twice(device, dtype):
    x, w, b, labels = _inputs(66, 72, 700, dtype, device)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    loss = A.linear_softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2])
    both = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, c) for a, c in zip(both, again))
    for k in range(3):
        args = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        one = A.linear_softmax_cross_entropy(args[0], args[1], labels, args[2])
        assert torch.equal(torch.autograd.grad(one, args[k])[0], both[k])


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_against_differences(device):
    # central differences along one direction, h = 2^-5: the third derivative of a row's loss along a direction that changes the
    # logits by at most s is below s^3, so h^2 s^3 / 6 a row; the losses are off by their bound / h
    x, w, b, labels = _inputs(6, 24, 50, torch.float32, device, ignored=0.0)
    g = torch.Generator().manual_seed(1)
    d = [torch.randn(t.shape, generator=g).to(device) * 0.1 for t in (x, w, b)]
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    loss = A.linear_softmax_cross_entropy(leaves[0], leaves[1], labels, leaves[2], reduction="sum")
    slope = sum((gr * dd).sum() for gr, dd in zip(torch.autograd.grad(loss, leaves), d))
    h = 2.0 ** -5
    at = lambda s: A.linear_softmax_cross_entropy(x + s * d[0], w + s * d[1], labels, b + s * d[2], reduction="sum")
    change = (d[0] @ w + x @ d[1] + d[2]).abs().max() * 2 + 2 * h * (d[0] @ d[1]).abs().max()
    tol = 6 * float(change) ** 3 * h * h / 6 * 4 + 6 * float((d[0] @ d[1]).abs().max()) * h * h * float(change) * 6 + 6e-5 / h
    assert abs(float((at(h) - at(-h)) / (2 * h) - slope)) <= tol


def test_refusals():
    x, w, b, labels = _inputs(4, 8, 20, torch.float32, "cpu")
    bad = [((x.half(), w.half(), None, labels), "float32 or all bfloat16"), ((x, w.bfloat16(), b, labels), "float32 or all bfloat16"),
           ((x, w, b.bfloat16(), labels), "float32 or all bfloat16"), ((x[:, :7].contiguous(), w, b, labels), "do not fit"),
           ((x, w, b[:19].contiguous(), labels), "20 elements"), ((x, w, b, labels.int()), "int64"),
           ((x, w, b, labels[:3]), "int64"), ((x, w.t().contiguous().t(), b, labels), "contiguous"),
           ((x, w[:, :0], None, labels), "do not fit")]
    for args, text in bad:
        with pytest.raises(ValueError, match=text):
            F.linear_xent_forward(*args)
    _, state = F.linear_xent_forward(x, w, b, labels)
    for dloss in (torch.ones(3), torch.ones(4, dtype=torch.float64), torch.ones(1), torch.ones(2, 2)):
        with pytest.raises(ValueError, match="dloss"):
            F.linear_xent_backward(x, w, b, labels, state, dloss)
    with pytest.raises(ValueError, match="db must"):
        F.linear_xent_backward(x, w, None, labels, state, torch.ones(()), db=torch.empty(20))
    with pytest.raises(ValueError, match="reduction"):
        A.linear_softmax_cross_entropy(x, w, labels, b, reduction="average")
    with pytest.raises(ValueError, match="integers"):
        A.linear_softmax_cross_entropy(x, w, labels.float(), b)
    with pytest.raises(ValueError, match="do not fit"):
        A.linear_softmax_cross_entropy(x, w, labels[:3], b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(gpu_device, dtype):
    x, w, b, labels = _inputs(70, 128, 1500, dtype, "cuda")
    dl = torch.ones((), device="cuda")

    def step():
        loss, state = F.linear_xent_forward(x, w, b, labels)
        out = [torch.empty_like(t) for t in (x, w, b)]
        F.linear_xent_backward(x, w, b, labels, state, dl, True, dx=out[0], dw=out[1], db=out[2])
        return [loss, F.linear_xent_totals(state, 70)] + out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        new = _inputs(70, 128, 1500, dtype, "cuda", seed=100 + k)
        for t, n in zip((x, w, b, labels), new):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, c) for a, c in zip(captured, eager)), k


@pytest.mark.gpu
def test_two_streams_at_once(gpu_device):
    sets = [_inputs(260, 256, 9000, torch.bfloat16, "cuda", seed=s) for s in range(2)]
    want = []
    for x, w, b, labels in sets:
        loss, state = F.linear_xent_forward(x, w, b, labels)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        F.linear_xent_backward(x, w, b, labels, state, torch.ones((), device="cuda"), True, dx=dx, dw=dw)
        want.append((loss, dx, dw))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    one = torch.ones((), device="cuda")
    torch.cuda.synchronize()
    for (x, w, b, labels), s in zip(sets, streams):
        with torch.cuda.stream(s):
            loss, state = F.linear_xent_forward(x, w, b, labels)
            dx, dw = torch.empty_like(x), torch.empty_like(w)
            F.linear_xent_backward(x, w, b, labels, state, one, True, dx=dx, dw=dw)
            got.append((loss, dx, dw, state))
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for g, v in zip(got, want) for a, c in zip(g, v))
