"""GPU: low-rank adapters of many requests (ops.adapter_forward / adapter_backward) against the formula in float64.

Two kinds of comparison.  Inputs of small whole numbers (|x|, |a|, |b| <= 1, |dz| <= 2, scales that are powers of two): every
product and every partial sum is a whole number (times a power of two) below 2^24, so float32 holds all of them in any order of
summation and the results must be EQUAL.  Real-valued inputs: a sum of n float32 products, accumulated in any order in float32,
is off by at most lambda sqrt(n) u times the sum of the absolute products but for a chance of 2 n exp(-lambda^2 / 2) (u = 2^-24);
lambda = 8 makes that 1e-10 for the longest sum here, and the sums are nested twice (rank over features), so the bound is
8 (sqrt(n1) + sqrt(n2)) u plus four roundings (product with the scale, h and out stored, the join of partial sums)."""
import numpy as np
import pytest
import torch

from yolo_amd import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U32 = 2.0 ** -24


def _inputs(N, K, U, L, R, dtype, seed, whole, none=0.2, pad=0):
    """Inputs on the GPU with rows pad elements longer than needed (filled with NaN: nothing may read them)."""
    g = torch.Generator().manual_seed(seed)

    def values(*shape, spread=1.0):
        v = torch.randint(-1, 2, shape, generator=g).float() if whole else torch.randn(shape, generator=g) * spread
        v = torch.cat([v, torch.full(shape[:-1] + (pad,), float('nan'))], -1)
        return v.to(dtype).to(DEV)[..., :shape[-1]]
    x, a, b = values(N, K), values(L, R, K, spread=K ** -0.5), values(L, R, U, spread=0.3)
    scale = (2.0 ** torch.randint(-2, 2, (L,), generator=g)) if whole else 0.5 + torch.rand(L, generator=g)
    index = torch.randint(0, L, (N,), generator=g)
    index = torch.where(torch.rand(N, generator=g) < none, torch.full_like(index, -1), index)
    dz = (torch.randint(-2, 3, (N, U), generator=g).float() if whole else torch.randn((N, U), generator=g) * 0.1).to(DEV)
    return x, a, b, index.to(torch.int32).to(DEV), scale.float().to(DEV), dz


def _formula(x, a, b, index, scale, dz, h=None):
    """out, h, da, db, dx in float64 on the host, and the sums of absolute products behind each."""
    x, a, b, scale, dz = (t.double().cpu() for t in (x, a, b, scale, dz))
    i = index.long().cpu()
    N, U = dz.shape
    L, R, K = a.shape
    hh = torch.zeros((N, R), dtype=torch.float64)
    res = dict(out=torch.zeros((N, U), dtype=torch.float64), da=torch.zeros_like(a), db=torch.zeros_like(b), dx=torch.zeros_like(x))
    mag = {k: torch.zeros_like(v) for k, v in res.items()}
    hmag = torch.zeros_like(hh)
    for j in range(L):
        n = torch.nonzero(i == j).flatten()
        if n.numel() == 0:
            continue
        hh[n], hmag[n] = x[n] @ a[j].T, x[n].abs() @ a[j].abs().T
        hj = hh[n] if h is None else h.double().cpu()[n]
        g, gm = scale[j] * (dz[n] @ b[j].T), scale[j].abs() * (dz[n].abs() @ b[j].abs().T)
        res['out'][n], mag['out'][n] = scale[j] * (hh[n] @ b[j]), scale[j].abs() * (hmag[n] @ b[j].abs())
        res['da'][j], mag['da'][j] = g.T @ x[n], gm.T @ x[n].abs()
        res['db'][j], mag['db'][j] = scale[j] * (hj.T @ dz[n]), scale[j].abs() * (hmag[n].T @ dz[n].abs())
        res['dx'][n], mag['dx'][n] = g @ a[j], gm @ a[j].abs()
    res['h'], mag['h'] = hh, hmag
    for k in ('out', 'dx', 'h'):
        res[k][i >= L] = float('nan')
    return res, mag


def _equal(got, want, name):
    got, want = got.double().cpu(), want
    assert torch.equal(torch.nan_to_num(got, nan=-9e9), torch.nan_to_num(want, nan=-9e9)), \
        (name, int((got != want).sum()), got.flatten()[:4], want.flatten()[:4])


def _close(got, want, mag, n1, n2, name):
    bound = (8 * (n1 ** 0.5 + n2 ** 0.5) + 4) * U32 * mag + 1e-300
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), (name, float((err / bound).max()))


# N, K, U, L, R: one row, one feature, ranks on both sides of 16 / 32 / 64, odd sizes, many adapters, few rows, the detector's own
SHAPES = [(1, 12544, 1470, 4, 8), (1, 1, 1, 1, 1), (2, 7, 3, 1, 2), (5, 33, 17, 3, 5), (16, 64, 64, 1, 16), (17, 100, 65, 2, 17),
          (31, 129, 30, 40, 3), (64, 2304, 539, 16, 16), (63, 255, 100, 64, 32), (65, 1000, 257, 7, 33), (100, 4999, 41, 5, 11),
          (130, 512, 512, 1, 64), (200, 640, 300, 3, 65), (257, 96, 1470, 256, 4), (300, 300, 77, 2, 128), (1025, 260, 68, 9, 12),
          (700, 31, 129, 1000, 7), (2048, 128, 64, 16, 32), (32, 12544, 1470, 4, 16)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N, K, U, L, R', SHAPES)
def test_whole_numbers_exact(N, K, U, L, R, dtype):
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, dtype, N * 7 + R, whole=True)
    h = torch.full((N, R), 7.0, device=DEV)
    want, _ = _formula(x, a, b, index, scale, dz)
    _equal(ops.adapter_forward(x, a, b, index, scale, h=h), want['out'], 'out')
    _equal(h, want['h'], 'h')
    _equal(ops.adapter_forward(x, a, b, index, scale), want['out'], 'out without h')
    for kept in (h, None):
        da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, kept, want_dx=True)
        _equal(da, want['da'], 'da'); _equal(db, want['db'], 'db'); _equal(dx, want['dx'], 'dx')
    da2, db2, none = ops.adapter_backward(dz, x, a, b, index, scale, h)
    assert none is None and torch.equal(da2, da) and torch.equal(db2, db)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N, K, U, L, R', [(1, 12544, 1470, 4, 8), (64, 12544, 1470, 16, 16), (333, 4999, 539, 7, 11), (1000, 777, 100, 3, 64)])
def test_real_values_within_the_bound(N, K, U, L, R, dtype):
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, dtype, N + R, whole=False)
    h = torch.empty((N, R), device=DEV)
    out = ops.adapter_forward(x, a, b, index, scale, h=h)
    want, mag = _formula(x, a, b, index, scale, dz)
    _close(out, want['out'], mag['out'], K, R, 'out')
    _close(h, want['h'], mag['h'], K, 0, 'h')
    da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, h, want_dx=True)
    want, mag = _formula(x, a, b, index, scale, dz, h)
    _close(da, want['da'], mag['da'], U, N, 'da')
    _close(db, want['db'], mag['db'], N, 0, 'db')
    _close(dx, want['dx'], mag['dx'], U, R, 'dx')


# the variants that take long batches or long axes: contraction through LDS in its three type mixtures and all tile shapes, 64 and
# 32 rows a workgroup and several column blocks in the expansion, 128 ranks in halves, thousands of adapters
LONG = [(4000, 9001, 33, 2, 64, torch.float32), (2100, 9003, 20, 1, 100, torch.float32), (4000, 9001, 18, 3, 20, torch.float32),
        (4000, 9001, 35, 3, 9, torch.float32), (4000, 16500, 20, 2, 40, torch.bfloat16), (4000, 40, 9001, 2, 30, torch.bfloat16),
        (4000, 40, 9001, 2, 61, torch.bfloat16), (2100, 30, 9002, 1, 128, torch.bfloat16), (4000, 64, 4100, 2, 17, torch.float32),
        (40, 100, 50, 5, 100, torch.float32), (600, 20, 16, 4096, 3, torch.float32), (256, 40, 20, 4096, 2, torch.bfloat16),
        (257, 513, 1025, 1, 1, torch.float32), (2049, 303, 77, 700, 5, torch.float32),
        (701, 303, 77, 1, 16, torch.bfloat16), (5000, 130, 61, 1500, 18, torch.bfloat16)]


def test_one_adapter_with_most_of_the_rows():
    """Adapters of 0, 1, 256, 257, 512, 513 and the rest of 4200 rows: one piece, several, whole last ones and single rows."""
    N, K, U, L, R = 4200, 301, 70, 8, 12
    x, a, b, _, scale, dz = _inputs(N, K, U, L, R, torch.float32, 12, whole=True)
    counts = [0, 1, 256, 257, 512, 513, N - 1 - 256 - 257 - 512 - 513 - 40]
    index = torch.cat([torch.full((c,), i) for i, c in enumerate(counts)] + [torch.full((40,), -1)])
    index = index[torch.randperm(N, generator=torch.Generator().manual_seed(2))].to(torch.int32).to(DEV)
    want, mag = _formula(x, a, b, index, scale, dz)
    assert max(float(m.max()) for m in mag.values()) < 2 ** 22
    da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
    _equal(da, want['da'], 'da'); _equal(db, want['db'], 'db'); _equal(dx, want['dx'], 'dx')


@pytest.mark.parametrize('N, K, U, L, R, dtype', LONG)
def test_long_batches_exact(N, K, U, L, R, dtype):
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


def test_offsets_beyond_32_bits():
    """Rows, adapters and outputs 1.1e9 elements apart in buffers of 9 GB: element offsets above 2^31, byte offsets above 2^32."""
    far, N, K, U, L, R = 1_100_000_000, 3, 70, 40, 3, 5
    xs, as_, bs, index, scale, dzs = _inputs(N, K, U, L, R, torch.float32, 6, whole=True, none=0.0)
    index = torch.tensor([2, 0, 2], dtype=torch.int32, device=DEV)
    ins, outs = (torch.empty(2 * far + 4096, device=DEV) for _ in range(2))
    view = lambda buf, shape, at: buf.as_strided(shape, (far,) + ((shape[2],) if len(shape) == 3 else ()) + (1,), at)
    x, a, b, dz = view(ins, (N, K), 0), view(ins, (L, R, K), 100), view(ins, (L, R, U), 1000), view(ins, (N, U), 2000)
    for t, v in ((x, xs), (a, as_), (b, bs), (dz, dzs)):
        t.copy_(v)
    out, da, db, dx = view(outs, (N, U), 0), view(outs, (L, R, K), 100), view(outs, (L, R, U), 1000), view(outs, (N, K), 2000)
    want, _ = _formula(x, a, b, index, scale, dz)
    # (the spans of interleaved outputs overlap, which the call refuses: each gets what it can be given)
    _equal(ops.adapter_forward(x, a, b, index, scale, out=out), want['out'], 'out')
    got = ops.adapter_backward(dz, x, a, b, index, scale, da=da)
    _equal(da, want['da'], 'da'); _equal(got[1], want['db'], 'db')
    got = ops.adapter_backward(dz, x, a, b, index, scale, db=db)
    _equal(db, want['db'], 'db'); _equal(got[0], want['da'], 'da')
    got = ops.adapter_backward(dz, x, a, b, index, scale, dx=dx)
    _equal(dx, want['dx'], 'dx')


def test_gradients_against_differences():
    """dL of L = sum(dz * out) along random whole-number directions: out is bilinear, so the difference quotient of a whole step is
    exact (the operator's own forward in whole numbers), and equals the gradient's inner product."""
    N, K, U, L, R = 23, 57, 31, 3, 6
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, 5, whole=True)
    loss = lambda x, a, b: float((ops.adapter_forward(x, a, b, index, scale).double() * dz.double()).sum())
    da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
    g = torch.Generator().manual_seed(1)
    step = lambda t: torch.randint(-1, 2, t.shape, generator=g).float().to(DEV)
    for _ in range(3):
        sx, sa, sb = step(x), step(a), step(b)
        for plus, minus, grad, s in (((x + sx, a, b), (x - sx, a, b), dx, sx), ((x, a + sa, b), (x, a - sa, b), da, sa), ((x, a, b + sb), (x, a, b - sb), db, sb)):
            assert (loss(*plus) - loss(*minus)) / 2 == float((grad.double() * s.double()).sum())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('pad', [1, 2, 4, 8])
def test_strided_operands_and_outputs(pad, dtype):
    """Rows with padding (NaN behind them), operands at odd offsets, outputs as slices of larger buffers that keep what is around."""
    N, K, U, L, R = 37, 203, 70, 4, 9
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, dtype, pad, whole=True, pad=pad)
    want, _ = _formula(x, a, b, index, scale, dz)
    around = torch.full((N, U + 6), 3.0, device=DEV)
    h = torch.empty((N, R), device=DEV)
    out = ops.adapter_forward(x, a, b, index, scale, out=around[:, 3:3 + U], h=h)
    _equal(out, want['out'], 'out')
    assert out.data_ptr() == around[:, 3:].data_ptr() and bool((around[:, :3] == 3).all()) and bool((around[:, 3 + U:] == 3).all())
    dzp = torch.full((N, U + pad), float('nan'), device=DEV)
    dzp[:, :U] = dz
    da, db, dx = (torch.full(s, 5.0, device=DEV) for s in ((L, R + 1, K + pad), (L, R, U + pad), (N, K + pad)))
    ops.adapter_backward(dzp[:, :U], x, a, b, index, scale, h, da=da[:, :R, :K], db=db[:, :, :U], dx=dx[:, :K])
    _equal(da[:, :R, :K], want['da'], 'da'); _equal(db[:, :, :U], want['db'], 'db'); _equal(dx[:, :K], want['dx'], 'dx')
    assert bool((da[:, R] == 5).all()) and bool((da[:, :, K:] == 5).all()) and bool((db[:, :, U:] == 5).all()) and bool((dx[:, K:] == 5).all())


def test_unaligned_base_addresses():
    N, K, U, L, R = 20, 130, 33, 2, 5
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, 3, whole=True)
    want, _ = _formula(x, a, b, index, scale, dz)
    def shifted(t, by):
        flat = torch.full((t.numel() + by,), float('nan') if t.is_floating_point() else 1 << 20, dtype=t.dtype, device=DEV)
        flat[by:] = t.flatten()
        return flat[by:].view(t.shape)
    x, a, b, index, scale, dz = (shifted(t, by) for t, by in zip((x, a, b, index, scale, dz), (1, 2, 3, 1, 3, 1)))
    _equal(ops.adapter_forward(x, a, b, index, scale), want['out'], 'out')
    da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
    _equal(da, want['da'], 'da'); _equal(db, want['db'], 'db'); _equal(dx, want['dx'], 'dx')


def test_broadcast_rows_of_x():
    """One image against many adapters: x.expand, row stride 0."""
    L, R, K, U = 9, 4, 300, 50
    x, a, b, _, scale, dz = _inputs(L, K, U, L, R, torch.float32, 4, whole=True)
    x = x[:1].expand(L, K)
    index = torch.arange(L, dtype=torch.int32, device=DEV)
    want, _ = _formula(x, a, b, index, scale, dz)
    _equal(ops.adapter_forward(x, a, b, index, scale), want['out'], 'out')
    da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
    _equal(da, want['da'], 'da'); _equal(db, want['db'], 'db'); _equal(dx, want['dx'], 'dx')


@pytest.mark.parametrize('N', [3, 64, 65, 300])
def test_rows_without_an_adapter(N):
    """No adapter anywhere, accumulate, adapters without rows, an index behind the bank."""
    K, U, L, R = 70, 40, 6, 5
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, N, whole=True)
    nobody = torch.full((N,), -1, dtype=torch.int32, device=DEV)
    h = torch.ones((N, R), device=DEV)
    assert int(ops.adapter_forward(x, a, b, nobody, scale, h=h).count_nonzero()) == 0 and int(h.count_nonzero()) == 0
    base = torch.randint(-9, 10, (N, U), generator=torch.Generator().manual_seed(2)).float().to(DEV)
    assert torch.equal(ops.adapter_forward(x, a, b, nobody, scale, out=base.clone(), accumulate=True), base)
    for t in ops.adapter_backward(dz, x, a, b, nobody, scale, want_dx=True):
        assert int(t.count_nonzero()) == 0
    want, _ = _formula(x, a, b, index, scale, dz)
    _equal(ops.adapter_forward(x, a, b, index, scale, out=base.clone(), accumulate=True), want['out'] + base.double().cpu(), 'accumulated')
    # values of rows and adapters that take no part may be anything
    far = index.clone()
    far[1], far[2] = L, 2 ** 31 - 1
    far[0] = -2 ** 31
    x2 = x.clone()
    x2[0] = float('nan')
    a2, b2, scale2 = a.clone(), b.clone(), scale.clone()
    far = torch.where(far == 3, torch.full_like(far, 2), far)
    a2[3], b2[3], scale2[3] = float('nan'), float('inf'), float('nan')
    want, _ = _formula(x, a, b, far, scale, dz)
    out = ops.adapter_forward(x2, a2, b2, far, scale2)
    _equal(out, want['out'], 'out')
    assert bool(out[1:3].isnan().all())
    dz2 = dz.clone()
    dz2[0] = float('inf')
    da, db, dx = ops.adapter_backward(dz2, x2, a2, b2, far, scale2, want_dx=True)
    want['dx'][0] = 0
    keep = [i for i in range(L) if i != 3]
    _equal(da[keep], want['da'][keep], 'da'); _equal(db[keep], want['db'][keep], 'db'); _equal(dx, want['dx'], 'dx')
    assert int(torch.nan_to_num(da[3]).count_nonzero()) == 0


def test_a_row_of_infinities_stays_in_its_row():
    for N in (10, 100):
        K, U, L, R = 100, 36, 2, 6
        x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, 8, whole=True, none=0.0)
        want, _ = _formula(x, a, b, index, scale, dz)
        x[4, 7] = float('inf')
        out = ops.adapter_forward(x, a, b, index, scale)
        rest = [n for n in range(N) if n != 4]
        _equal(out[rest], want['out'][rest], 'out')
        assert not bool(out[4].isfinite().all())
        da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
        other = 1 - int(index[4])
        _equal(da[other], want['da'][other], 'da'); _equal(dx, want['dx'], 'dx')
        cols = [k for k in range(K) if k != 7]
        _equal(da[:, :, cols], want['da'][:, :, cols], 'da beside the column')
        g = dz[4].double().cpu() @ b[int(index[4])].double().cpu().T
        assert bool((da[int(index[4]), :, 7].cpu().isinf() == (g != 0)).all())


def test_nothing_to_do():
    x, a, b, index, scale, dz = _inputs(0, 20, 10, 3, 4, torch.float32, 1, whole=True)
    assert ops.adapter_forward(x, a, b, index, scale).shape == (0, 10)
    da, db, dx = ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
    assert int(da.count_nonzero()) == 0 and int(db.count_nonzero()) == 0 and dx.shape == (0, 20)


@pytest.mark.parametrize('N', [500, 2500, 4500])
def test_same_bits_every_time_and_apart_from_the_other_rows(N):
    """A run repeated gives the same bits; so does a row's result whatever rows stand beside it in the batch, as long as the
    batch takes the same variant (same N)."""
    K, U, L, R = 3000, 200, 6, 16
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, 77, whole=False)
    first = (ops.adapter_forward(x, a, b, index, scale),) + ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
    for _ in range(3):
        again = (ops.adapter_forward(x, a, b, index, scale),) + ops.adapter_backward(dz, x, a, b, index, scale, want_dx=True)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
    perm = torch.randperm(N, generator=torch.Generator().manual_seed(3)).to(DEV)
    out = ops.adapter_forward(x[perm], a, b, index[perm], scale)
    assert torch.equal(out, first[0][perm])


@pytest.mark.parametrize('N', [80, 700, 4200])
def test_on_a_side_stream_and_in_graphs(N):
    """Two graphs captured one after the other, replayed in turn with eager work between, and calls on two streams at once:
    every result is the eager one."""
    K, U, L, R = 1000, 300, 5, 16
    sets = [_inputs(N, K, U, L, R, torch.float32, s, whole=True) for s in (1, 2)]
    want = [(ops.adapter_forward(*s[:5]),) + ops.adapter_backward(s[5], *s[:5], want_dx=True) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for rep in range(4):
        for j, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[j] = (ops.adapter_forward(*sets[j][:5]),) + ops.adapter_backward(sets[j][5], *sets[j][:5], want_dx=True)
        torch.cuda.synchronize()
        for j in range(2):
            assert all(torch.equal(p, q) for p, q in zip(got[j], want[j]))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = (ops.adapter_forward(*s[:5]),) + ops.adapter_backward(s[5], *s[:5], want_dx=True)
        graphs.append((g, res))
    for rep in range(4):
        for g, res in graphs:
            for t in res:
                t.fill_(-1)
            g.replay()
        ops.adapter_forward(*sets[rep % 2][:5])
        torch.cuda.synchronize()
        for (g, res), w in zip(graphs, want):
            assert all(torch.equal(p, q) for p, q in zip(res, w))


def test_refusals():
    N, K, U, L, R = 6, 20, 10, 3, 4
    x, a, b, index, scale, dz = _inputs(N, K, U, L, R, torch.float32, 1, whole=True)
    fwd = lambda **kw: ops.adapter_forward(**{**dict(x=x, a=a, b=b, index=index, scale=scale), **kw})
    bwd = lambda **kw: ops.adapter_backward(**{**dict(dz=dz, x=x, a=a, b=b, index=index, scale=scale), **kw})
    for kw in (dict(x=x.half()), dict(x=x.double()), dict(a=a.bfloat16()), dict(b=b.cpu()), dict(index=index.long()), dict(index=index.cpu()), dict(scale=scale.double())):
        with pytest.raises(TypeError):
            fwd(**kw)
        with pytest.raises(TypeError):
            bwd(**kw)
    for kw in (dict(x=x[0]), dict(x=x[:, :-1]), dict(a=a[0]), dict(a=a[:2]), dict(b=b[:, :3]), dict(index=index[:5]), dict(scale=scale[:2]),
               dict(x=torch.zeros((K, N), device=DEV).t()), dict(a=torch.zeros((L, R, 2 * K), device=DEV)[:, :, ::2])):
        with pytest.raises(ValueError):
            fwd(**kw)
        with pytest.raises(ValueError):
            bwd(**kw)
    for name in ('a', 'b', 'index', 'scale'):
        with pytest.raises(TypeError, match=name):
            fwd(**{name: None})
    with pytest.raises(TypeError, match='h'):
        fwd(h=torch.zeros((N, R)))
    with pytest.raises(ValueError, match='rank'):
        ops.adapter_forward(x, torch.zeros((1, 129, K), device=DEV), torch.zeros((1, 129, U), device=DEV), index, scale[:1])
    for kw in (dict(accumulate=True), dict(out=torch.zeros((N, U + 1), device=DEV)), dict(h=torch.zeros((N, R + 1), device=DEV)), dict(h=torch.zeros((R, N), device=DEV).t()),
               dict(out=torch.zeros((1, U), device=DEV).expand(N, U)), dict(out=x[:, :U]), dict(out=x[:, 10:]), dict(h=x.flatten()[:N * R].view(N, R))):
        with pytest.raises(ValueError):
            fwd(**kw)
    with pytest.raises(TypeError):
        fwd(out=torch.zeros((N, U), dtype=torch.bfloat16, device=DEV))
    shared = torch.zeros((L, R, K + U), device=DEV)
    for kw in (dict(dz=dz[:, :-1]), dict(da=a), dict(dx=x), dict(dx=torch.zeros((N, K + 1), device=DEV)), dict(db=torch.zeros((1, R, U), device=DEV).expand(L, R, U)),
               dict(da=shared[:, :, :K], db=shared[:, :, U:][:, :, :U]), dict(h=torch.zeros((N, R + 1), device=DEV))):
        with pytest.raises(ValueError):
            bwd(**kw)
