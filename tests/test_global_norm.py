"""``global_norm`` / ``clip_by_global_norm`` over lists of tensors against 64 bits.  The norm is one rounding to float32 away
from the exact one (2^-23 with the fp64 sum's own error), a clipped element two more and the rounding to its type."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import autograd as A
from distributed_tensorflow_amd.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _list(sizes, device, seed=0, types=TYPES, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * (1 + i % 5)).to(types[i % len(types)]).to(device) for i, n in enumerate(sizes)]


def _norm(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors if t is not None))


def _check(tensors, clip, out=None):
    want = _norm(tensors)
    before = [None if t is None else t.clone() for t in tensors]
    got, norm = F.clip_by_global_norm(tensors, clip, out=out)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= 2 * U * want
    assert float(F.global_norm(before)) == float(norm)
    f = min(1.0, clip / want) if want else 1.0
    for t, o in zip(before, got):
        if t is None:
            assert o is None
            continue
        assert o.dtype == t.dtype and o.shape == t.shape
        exact = t.double() * f
        bound = (torch.finfo(t.dtype).eps / 2 + 4 * U) * exact.abs() + torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps
        assert bool(((o.double() - exact).abs() <= bound).all())
        if out is None:
            assert torch.equal(t, tensors[[id(x) for x in got].index(id(o))])  # the inputs stay
    return got, norm


SIZES = [[1], [0, 5, 0], [7, 8191, 8192, 8193, 1], [64] * 5, [100000, 3, 77777]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("clip", [0.25, 1e6, math.inf])
def test_lists(device, sizes, clip):
    _check(_list(sizes, device), clip)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1 + (37 * i) % 900 for i in range(97)], [5] * 1000, [1 << 24, 3], [(1 << 20) + i for i in range(9)]])
def test_longer_lists(gpu_device, sizes):
    _check(_list(sizes, "cuda", scale=0.1), 1.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", TYPES)
def test_views_at_any_element(device, offset, dtype):
    buf = _list([40000], device, types=[dtype])[0]
    dst = torch.zeros(40000, dtype=dtype, device=device)
    tensors = [buf[offset:offset + 9001], buf[20000 - offset:30003], buf[35001:35002]]
    out = [dst[2 * offset + 1:2 * offset + 1 + 9001], dst[15000:15000 + tensors[1].numel()], dst[39999:]]
    _check(tensors, 0.5, out=out)
    covered = torch.zeros(40000, dtype=torch.bool, device=device)
    for o in out:
        start = (o.data_ptr() - dst.data_ptr()) // o.element_size()
        covered[start:start + o.numel()] = True
    assert not dst[~covered].any()


@pytest.mark.parametrize("device", DEVICES)
def test_in_place_none_and_empty(device):
    tensors = _list([300, 1000], device)
    tensors.insert(1, None)
    kept = [None if t is None else t.clone() for t in tensors]
    got, _ = F.clip_by_global_norm(tensors, 1e9, out=tensors)
    assert all(a is b for a, b in zip(got, tensors))
    assert all(t is None or torch.equal(t, k) for t, k in zip(tensors, kept))
    _check(tensors, 0.5, out=tensors)
    assert F.clip_by_global_norm([], 1.0)[0] == [] and float(F.global_norm([None])) == 0.0
    none, norm = F.clip_by_global_norm([torch.zeros(0, device=device), torch.zeros(10, device=device)], 1.0)
    assert float(norm) == 0.0 and none[0].numel() == 0 and not none[1].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_norm_that_is_not_finite(device, bad):
    tensors = _list([300, 100], device, types=[torch.float32])
    tensors[1][7] = bad
    got, norm = F.clip_by_global_norm(tensors, 1.0)
    assert not math.isfinite(float(norm)) and all(torch.isnan(t).all() for t in got)


@pytest.mark.parametrize("device", DEVICES)
def test_values_whose_squares_leave_float32(device):
    big = [torch.full((1000,), 1e30, device=device), torch.full((10,), 1e-3, device=device)]
    got, norm = F.clip_by_global_norm(big, 1.0)
    assert abs(float(norm) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    assert abs(float(got[0][0]) * math.sqrt(1000) - 1) < 1e-6
    assert abs(float(F.global_norm([torch.full((4,), 1e-30, device=device)])) / 2e-30 - 1) < 1e-6


@pytest.mark.parametrize("device", DEVICES)
def test_clip_grad_norm(device):
    p = [torch.nn.Parameter(torch.ones(5, 3, device=device)), torch.nn.Parameter(torch.ones(4, device=device)),
         torch.nn.Parameter(torch.ones(2, device=device))]
    (p[0].sum() * 2 + p[1].sum()).backward()
    assert abs(float(A.clip_grad_norm(p, 1.0)) - 8.0) < 1e-5          # sqrt(15 * 4 + 4)
    assert p[2].grad is None and abs(_norm([q.grad for q in p]) - 1.0) < 1e-6


def test_refusals():
    t = [torch.ones(4), torch.ones(3)]
    for clip in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="clip_norm"):
            F.clip_by_global_norm(t, clip)
    with pytest.raises(ValueError, match="float32, bfloat16 and float16"):
        F.global_norm([torch.ones(3, dtype=torch.float64)])
    with pytest.raises(ValueError, match="contiguous"):
        F.global_norm([torch.ones(4, 4).t()[:2]])
    with pytest.raises(ValueError, match="every tensor of the list"):
        F.clip_by_global_norm(t, 1.0, out=[t[0]])
    with pytest.raises(ValueError, match="like its tensor"):
        F.clip_by_global_norm(t, 1.0, out=[torch.ones(4), torch.ones(4)])
    buf = torch.zeros(8)
    with pytest.raises(ValueError, match="share memory"):
        F.clip_by_global_norm(t, 1.0, out=[buf[:4], buf[3:6]])
    with pytest.raises(ValueError, match="share memory"):
        F.clip_by_global_norm([t[0], t[0]], 1.0, out=[t[0], t[0]])


@pytest.mark.gpu
def test_captured_and_replayed(gpu_device):
    tensors = _list([1000, 30000, 5], "cuda")
    F.clip_by_global_norm(tensors, 1.0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got, norm = F.clip_by_global_norm(tensors, 1.0)
    for k in range(4):
        for t, n in zip(tensors, _list([1000, 30000, 5], "cuda", seed=9 + k, scale=0.01 if k == 2 else 1.0)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want, wnorm = F.clip_by_global_norm(tensors, 1.0)
        assert float(norm) == float(wnorm) and all(torch.equal(a, b) for a, b in zip(got, want)), k
