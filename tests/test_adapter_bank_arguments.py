"""CPU: what an AdapterBank refuses, and that a refused call leaves the bank as it was."""
import types

import numpy as np
import pytest
import torch

from yolo_amd.adapters import AdapterBank


def _bank():
    return AdapterBank(types.SimpleNamespace(K=50, units=13, device=torch.device('cpu')), 3, 4)


@pytest.mark.parametrize('which', [[True, False], [0, False], np.array([True, False]), torch.tensor([False, True]), [np.True_, 0]])
def test_a_mask_is_not_a_list_of_adapters(which):
    with pytest.raises(ValueError, match='adapter'):
        _bank().index(which)


@pytest.mark.parametrize('i', [1.5, -0.5, True, '1', None, np.float32(1), torch.tensor(0.5)])
def test_an_adapter_number_is_whole(i):
    bank = _bank()
    with pytest.raises((TypeError, IndexError)):
        bank.get(i)
    with pytest.raises((TypeError, IndexError)):
        bank.set(i, np.ones((2, 50)), np.ones((2, 13)))


@pytest.mark.parametrize('i', [2, np.int64(2), np.int32(2), torch.tensor(2)])
def test_whole_numbers_of_any_kind(i):
    bank = _bank()
    bank.set(i, np.ones((2, 50)), np.ones((2, 13)))
    assert bool((bank.get(i)[1][:2] == 1).all()) and int(bank.b[:2].count_nonzero()) == 0
    assert bank.index([int(i), -1]).tolist() == [2, -1]


@pytest.mark.parametrize('scale', ['high', [1.0, 2.0], object()])
def test_a_refused_scale_leaves_the_adapter_as_it_was(scale):
    bank = _bank()
    bank.set(1, np.full((4, 50), 3.0), np.full((4, 13), 4.0), scale=0.5)
    with pytest.raises((TypeError, ValueError)):
        bank.set(1, np.ones((2, 50)), np.ones((2, 13)), scale=scale)
    a, b, s = bank.get(1)
    assert (a == 3).all() and (b == 4).all() and s == 0.5


def test_the_bf16_copy_is_made_on_the_banks_device(monkeypatch):
    """changed() while another GPU is the current one: the cast, and the wait for it, belong to the bank's device (recorded here
    without one)."""
    from yolo_amd import ops
    bank, at, seen = _bank(), ['cuda:0'], []
    bank.device, bank._bf16 = torch.device('cuda:1'), torch.zeros_like(bank.flat, dtype=torch.bfloat16)

    class Device:
        def __init__(self, device):
            self.device = str(device)

        def __enter__(self):
            at.append(self.device)

        def __exit__(self, *error):
            at.pop()

    def stream(device=None):
        device = at[-1] if device is None else str(device)
        return types.SimpleNamespace(synchronize=lambda: seen.append(('wait', device)))

    monkeypatch.setattr(torch.cuda, 'device', Device)
    monkeypatch.setattr(torch.cuda, 'current_stream', stream)
    monkeypatch.setattr(ops, 'cast_bf16', lambda x, out: seen.append(('cast', at[-1])))
    bank.changed()
    assert seen == [('cast', 'cuda:1'), ('wait', 'cuda:1')] and at == ['cuda:0']
