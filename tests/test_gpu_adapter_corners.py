"""GPU: corners of the adapter operators in whole numbers, where results must be EQUAL (see test_gpu_adapters.py): gradients of adapters
without rows whose operands hold NaN and infinities, batches whose sort goes through more rows a wave than it keeps in registers,
tall tiles in an expansion of fewer than eight column blocks, and a lopsided batch below the size at which pieces are always cut."""
import pytest
import torch

from test_gpu_adapters import DEV, _equal, _formula, _inputs
from yolo_amd import ops

pytestmark = pytest.mark.gpu


# found by ballots, sorted, sorted and in pieces (from 700 rows an adapter or 4096 rows on)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N, L', [(10, 6), (200, 6), (300, 6), (1500, 2), (4200, 6)])
def test_gradients_of_an_adapter_without_rows_are_zero(N, L, dtype):
    """Whatever its weights and its scale hold: neither 0 * NaN nor 0 * inf may reach the gradients."""
    K, U, R = 70, 40, 5
    empty = L - 1
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, dtype, N, whole=True)
    index = torch.where(index == empty, torch.zeros_like(index), index)
    a, b, scale = a.clone(), b.clone(), scale.clone()
    want, mag = _formula(x, a, b, index, scale, dz)
    assert max(float(m.max()) for m in mag.values()) < 2 ** 22
    h = torch.empty((N, R), device=DEV)
    ops.adapter_forward(x, a, b, index, scale, h=h)
    for bad in (float('nan'), float('inf')):
        a[empty], b[empty], scale[empty] = bad, -bad, bad
        for kept in (h, None):
            da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, kept, want_dx=True)
            assert int(da[empty].count_nonzero()) == 0 and int(db[empty].count_nonzero()) == 0       # (NaN counts as not zero)
            _equal(da, want['da'], 'da'); _equal(db, want['db'], 'db'); _equal(dx, want['dx'], 'dx')


@pytest.mark.parametrize('N, K, U, L, R, dtype', [
    (20000, 40, 900, 3, 20, torch.float32),         # 1280 rows a wave in the sort; 64-row tiles, 4 column blocks
    (12000, 600, 1470, 5, 40, torch.bfloat16),      # 768 rows a wave; 64-row tiles of 40 ranks, 6 column blocks
    (8000, 50, 1300, 2, 70, torch.float32),         # 32-row tiles of 70 ranks, 6 column blocks
    (2000, 20, 16, 4096, 3, torch.float32)])        # three waves in the sort
def test_long_sorts_and_tall_expansions(N, K, U, L, R, dtype):
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, dtype, N + U, whole=True, none=0.05)
    # one value in eight of x and dz, so that the longest sums stay below 2^24 quarters (the smallest scale): asserted
    g = torch.Generator().manual_seed(N)
    x, dz = x * (torch.rand(x.shape, generator=g) < 0.125).to(DEV), dz.sign() * (torch.rand(dz.shape, generator=g) < 0.125).to(DEV)
    want, mag = _formula(x, a, b, index, scale, dz)
    assert max(float(m.max()) for m in mag.values()) < 2 ** 24 * 0.25
    h = torch.empty((N, R), device=DEV)
    _equal(ops.adapter_forward(x, a, b, index, scale, h=h), want['out'], 'out')
    _equal(h, want['h'], 'h')
    for kept in (h, None):
        da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, kept, want_dx=True)
        _equal(da, want['da'], 'da'); _equal(db, want['db'], 'db'); _equal(dx, want['dx'], 'dx')


@pytest.mark.parametrize('N', [1500, 4095, 4096])
def test_lopsided_batches_on_both_sides_of_the_rule(N):
    """A fourth of the rows on one of 64 adapters: whole up to 4095 rows, in pieces from 4096 on."""
    K, U, L, R = 301, 70, 64, 12
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, 12, whole=True)
    lean = torch.rand(N, generator=torch.Generator().manual_seed(2)) < 0.25
    index = torch.where(lean.to(DEV), torch.full_like(index, 5), index)
    want, mag = _formula(x, a, b, index, scale, dz)
    assert max(float(m.max()) for m in mag.values()) < 2 ** 22
    da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
    _equal(da, want['da'], 'da'); _equal(db, want['db'], 'db'); _equal(dx, want['dx'], 'dx')


def test_accumulating_keeps_what_is_around():
    """accumulate into a slice of a wider buffer (the last partial of a Dense layer with padded rows): the padding, the rows without
    an adapter and the other slabs keep their bits."""
    for N in (37, 300):
        K, U, L, R = 203, 70, 4, 9
        x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, N, whole=True)
        want, _ = _formula(x, a, b, index, scale, dz)
        base = torch.randint(-9, 10, (3, N, U + 2), generator=torch.Generator().manual_seed(2)).float().to(DEV)
        part = base.clone()
        ops.adapter_forward(x, a, b, index, scale, out=part[-1][:, :U], accumulate=True)
        _equal(part[-1][:, :U], want['out'] + base[-1][:, :U].double().cpu(), 'accumulated')
        alone = index < 0
        assert torch.equal(part[:-1], base[:-1]) and torch.equal(part[-1][:, U:], base[-1][:, U:]) and torch.equal(part[-1][alone], base[-1][alone])
