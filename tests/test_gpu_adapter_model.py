"""GPU: adapters and clipping where a user meets them - DeviceModel.predict / detect with an AdapterBank, AdapterTrainer, and
Trainer / the facade with global_clipnorm - against the oracle and against the operators run by hand."""
import numpy as np
import pytest
import torch

from oracle import loss_ref
from test_gpu_api import _labels
from yolo_amd import ops, params as P
from yolo_amd.adapters import AdapterBank
from yolo_amd.engine import AdapterTrainer, DeviceModel, Trainer
from yolo_amd.keras_facade import Adam

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
N = 6


def _setup(dtype='f32', dense_init='spread'):
    prm = P.make_random_params(seed=5, dense_init=dense_init, bn='random')
    model = DeviceModel(prm, device=DEV, dtype=dtype)
    x = torch.rand((N, 448, 448, 3), generator=torch.Generator().manual_seed(3)).to(DEV)
    bank = AdapterBank(model, 3, 8, scale=0.75)
    g = torch.Generator().manual_seed(4)
    bank.b.copy_(torch.randn(bank.b.shape, generator=g) * 0.1)
    bank.changed()
    return prm, model, x, bank, [1, -1, 0, 2, 1, None]


def _activated(z):
    n = z.shape[0]
    return torch.cat([torch.softmax(z[:, :980].reshape(n, 7, 7, 20), -1), torch.sigmoid(z[:, 980:1078].reshape(n, 7, 7, 2)),
                      torch.sigmoid(z[:, 1078:].reshape(n, 7, 7, 8))], -1)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_a_batch_of_mixed_adapters(dtype):
    prm, model, x, bank, which = _setup(dtype)
    index = bank.index(which)
    feats = model.backbone(x).double().cpu()
    plain = model.predict(x).clone()
    y = model.predict(x, bank, index).clone()
    a, b = (t.double().cpu() for t in bank.weights(torch.float32 if dtype == 'f32' else torch.bfloat16))
    w = (model.dense_wt if dtype == 'f32' else model.dense_wt_bf16)[:model.units].double().cpu()
    z = feats @ w.T + model.dense_b.double().cpu()
    for n, i in enumerate(which):
        if i is not None and i >= 0:
            z[n] += 0.75 * ((feats[n] @ a[i].T) @ b[i])
    # the head's own tolerance (an error of the logits of some 1e-5 of their size, through softmax and sigmoid)
    np.testing.assert_allclose(y.cpu().numpy(), _activated(z).numpy(), rtol=1e-3, atol=1e-4)
    for n in (1, 5):                                  # no adapter: the shared model's bits
        assert torch.equal(y[n], plain[n])
    assert all(not torch.allclose(y[n], plain[n], rtol=1e-3, atol=1e-4) for n in (0, 2, 3, 4))
    # detect: the same logits through the fused tail
    det = [t.clone() for t in model.detect(x, adapters=bank, index=index)]
    want = ops.decode_nms(y)
    assert all(torch.equal(p, q) for p, q in zip(det, want))
    # a bank that was written to is read anew, also in bf16
    bank.b.zero_()
    bank.changed()
    assert torch.equal(model.predict(x, bank, index), plain)


def test_a_captured_detection_follows_the_bank():
    """detect() with adapters as one graph: same bits, and new weights and another index take effect at the next replay."""
    for dtype in ('f32', 'bf16'):
        _, model, x, bank, which = _setup(dtype)
        index = bank.index(which)
        other = bank.index([2, 2, -1, 0, 1, 0])
        want = [[t.clone() for t in model.detect(x, adapters=bank, index=i)] for i in (index, other)]
        live = index.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model.detect(x, adapters=bank, index=live)
        for rep in range(4):
            live.copy_((index, other)[rep % 2])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want[rep % 2])), (dtype, rep)
        bank.b.zero_()
        bank.changed()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, model.detect(x)))


def test_one_image_and_refusals():
    _, model, x, bank, _ = _setup()
    one = model.predict(x[:1], bank, bank.index([2])).clone()
    batch = model.predict(x, bank, bank.index([2] * N))[:1]
    np.testing.assert_allclose(one.cpu().numpy(), batch.cpu().numpy(), rtol=1e-3, atol=1e-4)
    with pytest.raises(ValueError, match='index'):
        model.predict(x, bank)
    with pytest.raises(ValueError, match='without adapters'):
        model.detect(x, index=bank.index([0] * N))
    with pytest.raises(ValueError, match='shape'):
        model.predict(x, bank, bank.index([0] * (N - 1)))
    bank.units = 539
    with pytest.raises(ValueError, match='do not fit'):
        model.predict(x, bank, bank.index([0] * N))


def _adam64(p, g, m, v, t, lr):
    m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
    return p - lr * np.sqrt(1 - 0.999 ** t) / (1 - 0.9 ** t) * m / (v.sqrt() + 1e-7), m, v


@pytest.mark.parametrize('clip', [None, 0.5])
def test_adapter_training_against_autograd(clip):
    """The whole run as it is used: adapted forward, loss, adapter gradients, the global norm over all adapters, the clipped Adam
    step; gradients against autograd through the oracle's loss in float64, the update against the formula on those gradients."""
    _, model, x, bank, which = _setup(dense_init='glorot')
    index = bank.index(which)
    yt = _labels(N, 20, 9)
    yd = torch.from_numpy(yt).to(DEV)
    tr = AdapterTrainer(model, bank, lr=1e-3, global_clipnorm=clip)
    feats = model.backbone(x).clone()
    assert torch.equal(tr.gradients_from_features(feats, yd, index), tr.loss)
    a, b = (t.double().cpu().requires_grad_(True) for t in (bank.a, bank.b))
    f = feats.double().cpu()
    z = f @ model.dense_wt[:model.units].double().cpu().T + model.dense_b.double().cpu()
    rows = []
    for n, i in enumerate(which):
        rows.append(z[n] if i in (None, -1) else z[n] + 0.75 * ((f[n] @ a[i].T) @ b[i]))
    loss = loss_ref.yolo_loss_ref(torch.from_numpy(yt).double(), _activated(torch.stack(rows)))
    loss.backward()
    assert abs(float(tr.loss) - float(loss.detach())) <= 2e-4 * abs(float(loss.detach()))
    for got, want in ((tr.da, a.grad), (tr.db, b.grad)):
        assert float((got.double().cpu() - want).abs().max()) <= 2e-3 * float(want.abs().max())
    # one step: the update is the formula on the gradients that the kernels made
    grad, before = tr.grads.double().clone(), bank.flat.double().clone()
    loss1 = tr.step(x, yd, index)
    assert torch.equal(tr.grads.double(), grad) and float(loss1) == float(tr.loss)
    norm = float(grad.norm())
    c = 1.0 if clip is None else min(1.0, clip / norm)
    if clip is not None:
        assert c < 1 and abs(float(tr.grad_norm) - norm) <= 1e-6 * norm
    p, m, v = _adam64(before, grad * c, torch.zeros_like(before), torch.zeros_like(before), 1, 1e-3)
    assert float((bank.flat.double() - p).abs().max()) <= 2e-6 * 1e-3 * 100 + 2.0 ** -24 * float(p.abs().max())
    assert not bool(bank.flat.isnan().any())
    again = AdapterTrainer(model, bank, lr=1e-3, global_clipnorm=clip)
    assert again.t == 0 and tr.t == 1


def test_adapters_train_apart():
    """An adapter that has no image in any step stays as it is (zero gradients from the first step on: zero moments)."""
    _, model, x, bank, _ = _setup()
    keep = bank.get(2)
    tr = AdapterTrainer(model, bank)
    yd = torch.from_numpy(_labels(N, 20, 9)).to(DEV)
    for _ in range(2):
        tr.step(x, yd, bank.index([0, 1, 0, -1, 1, 0]))
    got = bank.get(2)
    assert np.array_equal(got[0], keep[0]) and np.array_equal(got[1], keep[1])
    assert not np.array_equal(bank.get(0)[1], keep[1])
    with pytest.raises(ValueError, match='fp32'):
        AdapterTrainer(DeviceModel(P.make_random_params(seed=1), device=DEV, dtype='bf16'), bank)


def test_trainer_with_clipping():
    prm = P.make_random_params(seed=6, dense_init='glorot', bn='random')
    x = torch.rand((N, 448, 448, 3), generator=torch.Generator().manual_seed(3)).to(DEV)
    yd = torch.from_numpy(_labels(N, 20, 9)).to(DEV)
    probe = Trainer(DeviceModel(prm, device=DEV))
    probe.gradients(x, yd)
    norm = float(probe.bucket.grads.double().norm())
    for clip in (norm / 7, norm * 2):
        tr = Trainer(DeviceModel(prm, device=DEV), global_clipnorm=clip)
        before = tr.pflat.double().clone()
        tr.step(x, yd)
        grad = tr.bucket.grads.double()
        assert abs(float(tr.grad_norm) - norm) <= 1e-4 * norm
        p, _, _ = _adam64(before, grad * min(1.0, clip / float(grad.norm())), torch.zeros_like(before), torch.zeros_like(before), 1, 1e-3)
        assert float((tr.pflat.double() - p).abs().max()) <= 2e-7 + 2.0 ** -24 * float(p.abs().max())
    # the update in flight under the next backbone gives the serial step's bits.  (In the third step a predicted box has width 0:
    # the loss' gradient of sqrt(0) is NaN, in the oracle in float64 too, so the norm is and every weight becomes it: bits, not values.)
    for steps in (2, 3):
        runs = []
        for overlap in (True, False):
            tr = Trainer(DeviceModel(prm, device=DEV), overlap=overlap, global_clipnorm=norm / 7)
            for _ in range(steps):
                tr.step(x, yd, wait=not overlap)
            tr.join()
            torch.cuda.synchronize()
            runs.append((tr.pflat.clone(), tr.grad_norm.clone()))
        assert all(torch.equal(p.view(torch.int32), q.view(torch.int32)) for p, q in zip(*runs))
        assert bool(runs[0][0].isfinite().all()) == (steps == 2)
    with pytest.raises(ValueError, match='max_norm'):
        Trainer(DeviceModel(prm, device=DEV), global_clipnorm=0.0)


def test_facade_passes_the_norm_on():
    from yolo_amd.keras_facade import Model
    from yolo_amd.models.model_tiny_yolov1 import model_tiny_YOLOv1
    outputs, inputs = model_tiny_YOLOv1()
    m = Model(inputs=inputs, outputs=outputs)
    m.compile(optimizer=Adam(lr=1e-4, global_clipnorm=1.5))
    x = np.random.default_rng(0).random((2, 448, 448, 3), np.float32)
    loss = m.train_on_batch(x, _labels(2, 20, 1))
    assert np.isfinite(loss) and m._trainer.global_clipnorm == 1.5 and float(m._trainer.grad_norm) > 0
