"""GPU: images without an adapter keep the shared model's bits in a batch that also holds adapted images, whatever number of split-K
partials the Dense layer leaves: the kernels behind it sum partials in groups of four, so one more of them would change the order
of every row's sum where it fills a group (3 -> 4, 7 -> 8, 11 -> 12, 51 -> 52)."""
import pytest
import torch

from test_gpu_api import _labels
from yolo_amd import ops, params as P
from yolo_amd.adapters import AdapterBank
from yolo_amd.engine import AdapterTrainer, DeviceModel

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U32 = 2.0 ** -24


def _features(N, K, dtype, seed):
    x = torch.randn((N, K), generator=torch.Generator().manual_seed(seed))
    return torch.where(x > 0, x, 0.1 * x).to(torch.bfloat16 if dtype == 'bf16' else torch.float32).to(DEV)


def _bank(model, count=3, rank=8):
    bank = AdapterBank(model, count, rank, scale=0.75)
    bank.b.copy_(torch.randn(bank.b.shape, generator=torch.Generator().manual_seed(4)) * 0.1)
    bank.changed()
    return bank


# classes, type, images, splits of the Dense layer: every remainder modulo four, the group-filling ones first
@pytest.mark.parametrize('C, dtype, N, splits', [
    (20, 'f32', 65, 11), (20, 'bf16', 65, 11), (20, 'f32', 128, 11), (20, 'bf16', 128, 11), (20, 'f32', 129, 7), (20, 'f32', 321, 3),
    (1, 'f32', 1, 51), (1, 'f32', 8, 51), (1, 'f32', 257, 11), (1, 'bf16', 32, 49), (20, 'f32', 6, 21), (20, 'bf16', 33, 22), (1, 'f32', 33, 56)])
def test_rows_without_an_adapter(C, dtype, N, splits):
    model = DeviceModel(P.make_random_params(seed=5, C=C, dense_init='spread'), C=C, device=DEV, dtype=dtype)
    feats, bank = _features(N, model.K, dtype, N), _bank(model)
    which = [(0, -1, 2, None, 1)[n % 5] if N > 1 else -1 for n in range(N)]
    alone = [n for n, i in enumerate(which) if i in (-1, None)]
    adapted = [n for n in range(N) if n not in alone]
    index = bank.index(which)

    def tails(part, adapters=None, index=None):
        got = [model.head(feats, adapters=adapters, index=index)]
        got += ops.head_decode_nms(part, model.dense_b, model.S, model.B, model.C, model.img_size)
        if dtype == 'f32':
            y_true = torch.from_numpy(_labels(N, C, 9)).to(DEV)
            _, per, dz = ops.train_tail(part, model.dense_b, y_true, ops.round_up(model.units, 4), C=C)
            got += [per, dz]
        return [t.clone() for t in got]
    part = model.dense(feats)
    assert part.shape[0] == splits
    plain, plain64 = tails(part), part[:, :, :model.units].double().cpu()
    part = model.dense(feats, adapters=bank, index=index)
    mixed, mixed64 = tails(part, bank, index), part[:, :, :model.units].double().cpu()
    for p, q in zip(plain, mixed):
        # (as bits: a per-image loss may be NaN)
        p, q = p[alone].contiguous(), q[alone].contiguous()
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    assert all(not torch.equal(plain[0][n], mixed[0][n]) for n in adapted)
    # the adapted rows: their logits differ by the adapter's product; a nested sum of float32 products over K and R (8 sqrt(n) u of
    # the sum of absolute products each, four roundings) and one rounding of the partial that it is added to
    a, b = (t.double().cpu() for t in bank.weights(feats.dtype))
    f = feats.double().cpu()
    for n in adapted:
        i = which[n]
        delta = 0.75 * ((f[n] @ a[i].T) @ b[i])
        mag = 0.75 * ((f[n].abs() @ a[i].abs().T) @ b[i].abs())
        bound = (8 * (model.K ** 0.5 + bank.rank ** 0.5) + 4) * U32 * mag + U32 * (plain64[:, n].abs().max(0).values + delta.abs()) * 1.01
        err = (mixed64[:, n].sum(0) - plain64[:, n].sum(0) - delta).abs()
        assert bool((err <= bound).all()), (n, float((err / bound).max()))
    # once more without adapters: the buffers that both use hold nothing over
    part = model.dense(feats)
    for p, q in zip(plain, tails(part)):
        assert torch.equal(p.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))


def test_an_index_behind_the_bank_reaches_the_logits():
    model = DeviceModel(P.make_random_params(seed=5, dense_init='spread'), device=DEV)
    feats, bank = _features(65, model.K, 'f32', 1), _bank(model)
    index = torch.full((65,), -1, dtype=torch.int32, device=DEV)
    plain = model.head(feats).clone()
    index[7] = bank.count
    y = model.head(feats, adapters=bank, index=index)
    rest = [n for n in range(65) if n != 7]
    assert bool(y[7].isnan().all()) and torch.equal(y[rest], plain[rest])


@pytest.mark.parametrize('N', [6, 65])
def test_training_with_untrained_adapters_starts_from_the_shared_loss(N):
    """New adapters (b = 0) add zeros: loss, dz and so B's gradient are those of the shared model's own logits."""
    model = DeviceModel(P.make_random_params(seed=5), device=DEV)
    bank = AdapterBank(model, 3, 8)
    feats, y_true = _features(N, model.K, 'f32', 2), torch.from_numpy(_labels(N, 20, 9)).to(DEV)
    ldz = ops.round_up(model.units, 4)
    loss, _, dz = ops.train_tail(model.dense(feats), model.dense_b, y_true, ldz)
    loss, dz = loss.clone(), dz.clone()
    index = bank.index([n % 3 for n in range(N)])
    tr = AdapterTrainer(model, bank)
    got = tr.gradients_from_features(feats, y_true, index)
    assert torch.equal(got.view(torch.int32), loss.view(torch.int32))
    h = torch.empty((N, bank.rank), device=DEV)
    ops.adapter_forward(feats, bank.a, bank.b, index, bank.scale, h=h)
    da, db, _ = ops.adapter_backward(dz[:, :model.units], feats, bank.a, bank.b, index, bank.scale, h)
    assert int(da.count_nonzero()) == 0 and torch.equal(tr.da, da) and torch.equal(tr.db.view(torch.int32), db.view(torch.int32))
