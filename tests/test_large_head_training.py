"""Group normalisation, a softmax head over a large vocabulary and clipping by the global norm together in models: gradients
and one update against the same network written out in 64 bits, on the CPU and - marked gpu - on the HIP kernels; the layer's
configuration and checkpoints, graph-captured steps, ranks, and what is refused.

Tolerances: every float32 layer of these small networks is off by a few hundred roundings of its largest terms at most (sums of
up to 1300 products, 2^-24 each); values are compared to 2e-5 of the largest value of their tensor, some 300 roundings, through
four layers to 1e-4."""
import math
import socket
import sys

import pytest
import torch
import torch.multiprocessing as mp

from distributed_tensorflow_amd import optimizers
from distributed_tensorflow_amd.layers import (Conv2D, Dense, Dropout, Flatten, GroupNormalization, MaxPooling2D,
                                               layer_from_config)
from distributed_tensorflow_amd.models import Sequential
from distributed_tensorflow_amd.models.sequential import load_model
from distributed_tensorflow_amd.ops import autograd as A
from distributed_tensorflow_amd.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _close(a, b, tol=1e-4):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert float((a - b).abs().max()) <= tol * float(b.abs().max().clamp(min=1e-30)), float((a - b).abs().max())


def _model(device, classes, optimizer="sgd", **kw):
    m = Sequential([Conv2D(16, (3, 3), padding="same", input_shape=(8, 8, 4)), GroupNormalization(groups=4, activation="silu"),
                    MaxPooling2D((2, 2)), Flatten(), Dense(32, activation="relu"), Dense(classes, activation="softmax")])
    m.compile(loss="sparse_categorical_crossentropy", optimizer=optimizer, metrics=["accuracy"], device=device, seed=4, **kw)
    with torch.no_grad():
        g = torch.Generator().manual_seed(9)
        for v in m.store.trainable:
            if v.name.endswith("gamma"):
                v.tensor.copy_(torch.rand(v.shape, generator=g) + 0.5)
            elif v.name.endswith(("beta", "bias")):
                v.tensor.copy_(torch.randn(v.shape, generator=g) * 0.1)
    return m


def _batch(n, classes, device):
    g = torch.Generator().manual_seed(n + classes)
    return torch.randn(n, 8, 8, 4, generator=g).to(device), torch.randint(0, classes, (n,), generator=g).to(device)


def _torch(m, x, y):
    """Loss, logits and gradients of the model in 64 bits."""
    w = {v.name: v.tensor.detach().cpu().double().requires_grad_() for v in m.store.trainable}
    h = torch.nn.functional.conv2d(x.cpu().double().permute(0, 3, 1, 2), w["conv2d_1/kernel"].permute(3, 2, 0, 1), w["conv2d_1/bias"],
                                   padding=1)
    h = torch.nn.functional.silu(torch.nn.functional.group_norm(h, 4, w["group_normalization_1/gamma"],
                                                                w["group_normalization_1/beta"], 1e-3))
    h = torch.nn.functional.max_pool2d(h, 2).permute(0, 2, 3, 1).reshape(x.shape[0], -1)
    h = torch.relu(h @ w["dense_1/kernel"] + w["dense_1/bias"])
    z = h @ w["dense_2/kernel"] + w["dense_2/bias"]
    loss = torch.nn.functional.cross_entropy(z, y.cpu())
    loss.backward()
    return float(loss.detach()), z.detach(), {n: t.grad for n, t in w.items()}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("classes", [10, 1301])
def test_gradients_loss_and_accuracy(device, classes):
    m = _model(device, classes)
    x, y = _batch(48, classes, device)
    loss, z, grads = _torch(m, x, y)
    y[:5] = z.argmax(1)[:5].to(device)          # some rows are right
    loss, z, grads = _torch(m, x, y)
    m.compute_gradients(x, y)
    logs = m.read_stats()
    assert abs(logs["loss"] - loss) <= 1e-5 * loss
    assert logs["acc"] == pytest.approx(float((z.argmax(1) == y.cpu()).double().mean()))
    for v in m.store.trainable:
        _close(v.grad, grads[v.name])
    again = m.test_on_batch(x, y)
    assert again["loss"] == pytest.approx(logs["loss"], rel=1e-6) and again["acc"] == logs["acc"]
    assert m.evaluate(x, y, batch_size=20)[0] == pytest.approx(loss, rel=1e-5)
    p = m.predict(x[:7])
    _close(p, torch.softmax(z[:7], 1))


@pytest.mark.gpu
def test_wide_head_is_taken_by_class_count(gpu_device):
    for classes, wide in ((F.SOFTMAX_XENT_MAX_CLASSES, False), (F.SOFTMAX_XENT_MAX_CLASSES + 1, True)):
        m = _model("cuda", classes)
        x, y = _batch(9, classes, "cuda")
        assert (m.wide_head(y) is not None) == wide
        m.compute_gradients(x, y)
        _, _, grads = _torch(m, x, y)
        for v in m.store.trainable:
            _close(v.grad, grads[v.name])


@pytest.mark.gpu
def test_wide_head_with_rounded_operands(gpu_device):
    m = _model("cuda", 600, matmul_dtype="bf16")
    x, y = _batch(40, 600, "cuda")
    _, _, grads = _torch(m, x, y)
    m.compute_gradients(x, y)
    # the head's two roundings of its operands and two of dz, 2^-8 each, on sums of terms of either sign
    for name in ("dense_2/kernel", "dense_2/bias", "dense_1/kernel"):
        v = m.store.variables[name]
        assert float((v.grad.cpu().double() - grads[name]).norm() / grads[name].norm()) <= 4 * 2.0 ** -8


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("clip", [0.05, 1e3])
def test_one_clipped_update(device, clip):
    m = _model(device, 400, optimizers.SGD(lr=0.5, global_clipnorm=clip))
    x, y = _batch(32, 400, device)
    _, _, grads = _torch(m, x, y)
    before = {v.name: v.tensor.clone() for v in m.store.trainable}
    m.train_step(x, y)
    norm = math.sqrt(sum(float(g.square().sum()) for g in grads.values()))
    assert norm > 0.05
    f = min(1.0, clip / norm)
    for v in m.store.trainable:
        _close(before[v.name].cpu().double() - v.tensor.cpu().double(), 0.5 * f * grads[v.name], 2e-4)
    assert m.global_step == 1


@pytest.mark.gpu
def test_captured_steps_match_eager_ones(gpu_device):
    x, y = _batch(64, 700, "cuda")
    out = []
    for graph in (0, 2):
        m = _model("cuda", 700, optimizers.Adam(global_clipnorm=0.5))
        m.fit(x, y, batch_size=16, epochs=3, shuffle=False, verbose=0, steps_per_graph=graph)
        out.append((m.store.flat.clone(), m.global_step))
    assert out[0][1] == out[1][1] == 12
    _close(out[1][0], out[0][0], 1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_fused_small_network_still_clips(device):
    # the reference network's whole-step kernel updates as it goes: with clipping the layer-wise step has to run
    def net(opt):
        m = Sequential([Dense(128, input_dim=64, activation="relu"), Dropout(0.3), Dense(128, activation="relu"), Dropout(0.3),
                        Dense(32, activation="sigmoid")])
        m.compile(loss="mean_squared_error", optimizer=opt, device=device, seed=1)
        return m
    m = net(optimizers.SGD(lr=1.0, global_clipnorm=1e-3))
    assert m.fused_step_plan(50) is None
    g = torch.Generator().manual_seed(0)
    x, y = torch.rand(50, 64, generator=g).to(device), (torch.rand(50, 32, generator=g) > 0.5).float().to(device)
    before = m.store.flat.clone()
    m.train_step(x, y)
    assert float((m.store.flat - before).double().norm()) == pytest.approx(1e-3, rel=1e-4)


@pytest.mark.parametrize("device", DEVICES)
def test_together_under_autograd(device):
    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = A.GroupNormalization(24, groups=6, activation="relu")
            self.head = A.SoftmaxCrossEntropyHead(24, 500)

        def forward(self, x, labels):
            return self.head(self.norm(x), labels)

    torch.manual_seed(3)
    net = Net().to(device)
    x = torch.randn(5, 9, 24, device=device)
    labels = torch.randint(0, 500, (5, 9), device=device)
    labels[0, 4:] = -1
    net(x, labels).backward()
    grads = [p.grad.clone() for p in net.parameters()]
    w = [p.detach().cpu().double().requires_grad_() for p in net.parameters()]
    gamma, beta, kernel, bias = w
    h = torch.relu(torch.nn.functional.group_norm(x.cpu().double().transpose(1, 2), 6, gamma, beta, 1e-3)).transpose(1, 2)
    torch.nn.functional.cross_entropy((h @ kernel + bias).reshape(-1, 500), labels.cpu().reshape(-1), ignore_index=-1).backward()
    for a, b in zip(grads, w):
        _close(a, b.grad)
    norm = A.clip_grad_norm(net.parameters(), 1e-2)
    want = math.sqrt(sum(float(b.grad.square().sum()) for b in w))
    assert float(norm) == pytest.approx(want, rel=1e-4)
    for p, b in zip(net.parameters(), w):
        _close(p.grad, b.grad * (1e-2 / want))


def test_layer_configuration_and_checkpoint(tmp_path):
    layer = GroupNormalization(groups=4, epsilon=1e-5, center=False, activation="tanh", name="gn")
    assert layer_from_config(layer.get_config()).get_config() == layer.get_config()
    m = _model("cpu", 20)
    m.save(str(tmp_path / "m"))
    again = load_model(str(tmp_path / "m"), dict(loss="sparse_categorical_crossentropy", optimizer="sgd", device="cpu"))
    x, _ = _batch(3, 20, "cpu")
    assert torch.equal(again.predict(x), m.predict(x))
    assert "group_normalization_1/gamma" in m.store.variables


def test_layer_without_variables_and_first_in_the_model():
    m = Sequential([GroupNormalization(groups=2, center=False, scale=False, input_shape=(6, 6, 4)), Flatten(),
                    Dense(3, activation="sigmoid")])
    m.compile(loss="mean_squared_error", optimizer="sgd", device="cpu", seed=0)
    x = torch.randn(5, 6, 6, 4)
    m.train_step(x, torch.rand(5, 3))
    want = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 2, eps=1e-3).permute(0, 2, 3, 1)
    _close(m.layers[0].forward(x, False), want, 1e-5)


def test_graph_model_and_keras_namespace():
    import distributed_tensorflow_amd.compat as tf
    assert tf.keras.layers.GroupNormalization is not None
    layer = GroupNormalization(groups=2, activation="relu")
    from distributed_tensorflow_amd.variables import VariableStore
    store = VariableStore()
    layer.build((3, 3, 4), store)
    store.finalize("cpu", seed=0)
    x = torch.randn(2, 3, 3, 4)
    _close(layer.forward(x, True), A.group_norm(x, layer.gamma.tensor, layer.beta.tensor, 2, 1e-3, "relu"), 1e-6)


def test_refusals():
    with pytest.raises(ValueError, match="do not divide"):
        _bad = Sequential([GroupNormalization(groups=3, input_shape=(4, 4, 8))])
        _bad.build()
    with pytest.raises(ValueError, match="unsupported activation"):
        GroupNormalization(activation="softmax")
    with pytest.raises(ValueError, match="last axis"):
        GroupNormalization(axis=2)
    with pytest.raises(ValueError, match="global_clipnorm must be positive"):
        optimizers.Adam(global_clipnorm=0.0)

    class Sharded:
        def prepare(self, model):
            pass

    m = Sequential([Dense(3, input_dim=4)])
    with pytest.raises(ValueError, match="global_clipnorm needs the whole gradient"):
        m.compile(loss="mse", optimizer=optimizers.SGD(global_clipnorm=1.0), strategy=Sharded(), device="cpu", seed=0)


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _rank(rank, world, port, below, out_q):
    torch.set_num_threads(1)
    from distributed_tensorflow_amd.parallel import Communicator, SyncReplicasStrategy, init_process_group
    init_process_group("gloo", rank=rank, world_size=world, master_addr="127.0.0.1", master_port=port)
    strat = SyncReplicasStrategy(Communicator(), allreduce_below_bytes=below)
    try:
        m = _model("cpu", 40, optimizers.SGD(lr=0.5, global_clipnorm=0.05), strategy=strat)
    except ValueError as e:
        out_q.put((rank, str(e), None))
    else:
        x, y = _batch(16 * world, 40, "cpu")
        m.train_step(x[rank * 16:(rank + 1) * 16], y[rank * 16:(rank + 1) * 16])
        out_q.put((rank, None, {v.name: v.tensor.numpy().copy() for v in m.store.trainable}))
    import torch.distributed as dist
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("below", [8 << 20, 0], ids=["replicated", "sharded"])
def test_two_ranks_clip_the_averaged_gradient(below):
    port, ctx = _free_port(), mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, below, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted([q.get(timeout=120) for _ in range(2)], key=lambda t: t[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    if not below:
        assert all("whole gradient" in r[1] for r in res)
        return
    m = _model("cpu", 40, optimizers.SGD(lr=0.5, global_clipnorm=0.05))
    before = {v.name: v.tensor.clone() for v in m.store.trainable}
    x, y = _batch(32, 40, "cpu")
    m.train_step(x, y)
    for v in m.store.trainable:
        for r in res:
            _close(torch.from_numpy(r[2][v.name]).double() - before[v.name].double(), v.tensor.double() - before[v.name].double(), 1e-3)
