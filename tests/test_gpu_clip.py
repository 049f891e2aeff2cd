"""GPU: the global norm over many tensors, clipping and the clipped Adam step against float64 on the host.

Bounds (u = 2^-24, half a step of float32 relative to the value; 2^-8 for bf16): the norm is summed in float64 and rounded once: u
plus n 2^-53.  A clipped value is one product in float64 with a coefficient off by a few 2^-53, rounded once: u, or 2^-8 for bf16
after a rounding to float32 in between (2^-8 + u).  The Adam step on g' = round(g c) (u): m is two products and a sum, v three
products and a sum - each term carries at most 3 u and 5 u, and beta and 1 - beta u each: 4 u and 6 u of the sum of absolute
terms; the step lr m / (sqrt(v) + eps) adds half of v's, the root's, the sum's, the rate's, eps', the product's and the
division's u: 4 + 3 + 6 = 13 u of the step made of absolute terms; p' takes u more."""
import numpy as np
import pytest
import torch

from yolo_amd import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U32 = 2.0 ** -24

LISTS = [[1], [0, 3], [5], [64], [1470], [4097, 1, 0, 3], [65536], [65537, 1023], [1, 2, 3, 4, 5, 6, 7, 8, 9], [17] * 200, [40000] * 3 + [1] * 62 + [7],
         [300001, 12], [1472 * 12544, 1470]]


def _tensors(sizes, kind, seed, offset=0):
    g = torch.Generator().manual_seed(seed)
    ts = []
    for i, n in enumerate(sizes):
        dt = torch.bfloat16 if kind == 'bf16' or (kind == 'mixed' and i % 2) else torch.float32
        buf = torch.full((n + 2 * offset,), float('nan'), dtype=dt, device=DEV)
        buf[offset:offset + n] = (torch.randn(n, generator=g) * 10.0 ** ((i % 5) - 3)).to(dt).to(DEV)
        ts.append(buf[offset:offset + n])
    return ts


def _norm64(ts):
    return float(np.sqrt(sum(float((t.double() ** 2).sum()) for t in ts)))


@pytest.mark.parametrize('offset', [0, 1, 3])
@pytest.mark.parametrize('kind', ['f32', 'bf16', 'mixed'])
@pytest.mark.parametrize('sizes', LISTS, ids=lambda s: f'{len(s)}x{max(s)}')
def test_norm_and_clipping(sizes, kind, offset):
    grads = _tensors(sizes, kind, len(sizes), offset)
    want = _norm64(grads)
    rel = U32 + sum(sizes) * 2.0 ** -53
    norm = ops.grad_norm(grads)
    assert norm.shape == (1,) and abs(float(norm) - want) <= rel * want
    before = [g.clone() for g in grads]
    # below the norm: scaled, into other buffers first and then in place with the same bits
    out = [torch.full_like(g, float('nan')) for g in grads]
    limit = 0.37 * want
    assert torch.equal(ops.clip_grad_norm(grads, limit, out=out), norm)
    for g, b, o in zip(grads, before, out):
        assert torch.equal(g, b)
        exact = b.double() * (limit / want)
        eps = (2.0 ** -8 + U32 if o.dtype == torch.bfloat16 else U32) + sum(sizes) * 2.0 ** -52
        assert bool(((o.double() - exact).abs() <= eps * exact.abs()).all())
    assert torch.equal(ops.clip_grad_norm(grads, limit), norm)
    assert all(torch.equal(g, o) for g, o in zip(grads, out))
    # at or above the norm: the same bits
    for g, b in zip(grads, before):
        g.copy_(b)
    for limit in (1.01 * want, float('inf')):
        assert torch.equal(ops.clip_grad_norm(grads, limit), norm)
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
        ops.clip_grad_norm(grads, limit, out=out)
        assert all(torch.equal(o, b) for o, b in zip(out, before))


def test_only_the_tensors_are_written():
    flat = torch.full((1000,), 2.0, device=DEV)
    ts = [flat[3:10], flat[11:500], flat[500:501], flat[700:999]]
    ops.clip_grad_norm(ts, 1.0)
    inside = torch.zeros(1000, dtype=torch.bool)
    for lo, hi in ((3, 10), (11, 500), (500, 501), (700, 999)):
        inside[lo:hi] = True
    assert bool((flat.cpu()[~inside] == 2).all()) and bool((flat.cpu()[inside] < 2).all())


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
def test_values_whose_squares_leave_float32(kind):
    dt = torch.float32 if kind == 'f32' else torch.bfloat16
    for v in (1e30, 1e-30, 3e38 if kind == 'f32' else 2.0 ** 127, 1e-40 if kind == 'f32' else 2.0 ** -130):
        g = [torch.full((1000,), v, device=DEV).to(dt), torch.zeros(7, device=DEV)]
        want = _norm64(g)
        norm = float(ops.grad_norm(g))
        assert abs(norm - want) <= 2 * U32 * want + 2.0 ** -149 or (np.isinf(norm) and want > 3.4e38)
        keep = g[0].clone()
        limit = float(min(want / 3, 1.0))
        ops.clip_grad_norm(g, limit)
        exact = keep.double() * (limit / want)
        step = 2.0 ** -149 if kind == 'f32' else 2.0 ** -133           # half a step below the normal range at the least
        assert bool(((g[0].double() - exact).abs() <= (2.0 ** -8 if kind == 'bf16' else U32) * 1.01 * exact.abs() + step).all()), v


def test_more_values_than_32_bits_count():
    n = 2 ** 31 + 5
    g = torch.full((n,), 0.5, device=DEV)
    small = torch.ones(3, device=DEV)
    want = np.sqrt(n * 0.25 + 3)
    assert abs(float(ops.clip_grad_norm([small, g], want / 4)) - want) <= 2 * U32 * want
    for t, v in ((g, 0.125), (small, 0.25)):
        lo, hi = t.aminmax()
        assert abs(float(lo) - v) <= U32 * v and float(hi) == float(lo)


def test_the_norm_may_not_lie_in_a_tensor():
    from yolo_amd._lib import Ty1Error
    g = torch.ones(100, device=DEV)
    with pytest.raises(Ty1Error, match='shares memory'):
        ops.clip_grad_norm(g, 1.0, norm=g[3:4])
    kept = torch.empty(1, device=DEV)
    assert ops.clip_grad_norm(g, 1.0, norm=kept) is kept and float(kept) == 10.0


def test_zeros_and_values_that_are_not_finite():
    z = [torch.zeros(100, device=DEV), torch.zeros(0, device=DEV)]
    assert float(ops.clip_grad_norm(z, 1.0)) == 0.0 and int(z[0].count_nonzero()) == 0
    assert float(ops.grad_norm([torch.zeros(0, device=DEV)])) == 0.0
    for bad in (float('inf'), float('nan'), -float('inf')):
        for n in (100, 300000):
            g = [torch.ones(n, device=DEV), torch.ones(5, device=DEV)]
            g[0][n // 2] = bad
            norm = float(ops.clip_grad_norm(g, 1.0))
            assert np.isnan(norm) if np.isnan(bad) else np.isinf(norm)
            assert all(bool(t.isnan().all()) for t in g)


def _adam64(p, g, m, v, t, c, lr=1e-3, b1=0.9, b2=0.999, eps=1e-7):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * c
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    mabs = (b1 * m).abs() + ((1 - b1) * g).abs()
    rate = lr * np.sqrt(1 - b2 ** t) / (1 - b1 ** t)
    return p - rate * m2 / (v2.sqrt() + eps), m2, v2, mabs, rate * mabs / (v2.sqrt() + eps)


@pytest.mark.parametrize('offset', [0, 1])
@pytest.mark.parametrize('limit', [0.1, 5.0, float('inf')])
@pytest.mark.parametrize('sizes', LISTS, ids=lambda s: f'{len(s)}x{max(s)}')
def test_clipped_adam_step(sizes, limit, offset):
    g = _tensors(sizes, 'f32', 1, offset)
    p, m = _tensors(sizes, 'f32', 2, offset), _tensors(sizes, 'f32', 3, offset)
    v = [x.square() for x in _tensors(sizes, 'f32', 4)]
    before = [[t.clone() for t in ts] for ts in (p, g, m, v)]
    norm = _norm64(g)
    t = 7
    c = min(1.0, limit * norm / norm) if np.isfinite(limit) else 1.0
    got = ops.adam_step_clipped(p, g, m, v, t, limit * norm)
    assert abs(float(got) - norm) <= (U32 + sum(sizes) * 2.0 ** -53) * norm
    for i in range(len(sizes)):
        p2, m2, v2, mabs, step = _adam64(*(x[i] for x in before), t, c)
        assert torch.equal(g[i], before[1][i])
        assert bool(((m[i].double() - m2).abs() <= 4 * U32 * mabs + 1e-44).all())
        assert bool(((v[i].double() - v2).abs() <= 6 * U32 * v2 + 1e-44).all())
        assert bool(((p[i].double() - p2).abs() <= 13.5 * U32 * step + 1.01 * U32 * p2.abs() + 1e-44).all())


def test_one_tensor_and_flat_buffers():
    flat = [torch.randn(5000, generator=torch.Generator().manual_seed(s)).to(DEV) for s in range(4)]
    flat[3].square_()
    views = [list(t.clone().split([1000, 1, 3999])) for t in flat]
    n1 = ops.adam_step_clipped(flat[0], flat[1], flat[2], flat[3], 3, 0.5)
    n2 = ops.adam_step_clipped(*views, 3, 0.5)
    assert torch.equal(n1, n2) or abs(float(n1) - float(n2)) <= 2 * U32 * float(n1)
    for t, vs in zip(flat, views):
        assert torch.allclose(t, torch.cat(vs), rtol=1e-6, atol=1e-12)
    assert float(ops.grad_norm(flat[1])) == float(ops.grad_norm([flat[1]]))


def test_same_bits_every_time_and_in_graphs():
    sizes = [100000, 33, 7000]
    g = _tensors(sizes, 'mixed', 1)
    out = [torch.empty_like(t) for t in g]
    norm = ops.clip_grad_norm(g, 1.0, out=out)
    want = [t.clone() for t in out]
    for _ in range(3):
        assert torch.equal(ops.clip_grad_norm(g, 1.0, out=out), norm) and all(torch.equal(a, b) for a, b in zip(out, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        o = [torch.empty_like(t) for t in g]
        with torch.cuda.graph(graph):
            n = ops.clip_grad_norm(g, 1.0, out=o)
        graphs.append((graph, o, n))
    for rep in range(4):
        for graph, o, n in graphs:
            for t in o:
                t.fill_(9)
            n.fill_(9)
            graph.replay()
        ops.grad_norm(out)
        torch.cuda.synchronize()
        for graph, o, n in graphs:
            assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(o, want))


def test_refusals():
    f = lambda n: torch.ones(n, device=DEV)
    with pytest.raises(TypeError):
        ops.grad_norm(f(4).half())
    with pytest.raises(TypeError):
        ops.grad_norm([f(4), torch.ones(4)])
    with pytest.raises(ValueError, match='contiguous'):
        ops.grad_norm(torch.ones((4, 4), device=DEV).t()[:3])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([f(4)], 1.0, out=[f(4), f(4)])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([f(4)], 1.0, out=[f(5)])
    with pytest.raises(TypeError):
        ops.clip_grad_norm([f(4)], 1.0, out=[f(4).bfloat16()])
    x = f(100)
    from yolo_amd._lib import Ty1Error
    with pytest.raises(Ty1Error, match='shares memory'):
        ops.clip_grad_norm([x, x], 1.0)
    with pytest.raises(Ty1Error, match='shares memory'):
        ops.clip_grad_norm([x[:60], x[50:]], 1.0)
    assert float(ops.grad_norm([x, x])) == np.float32(np.sqrt(200.0))            # reading a tensor twice is fine
    with pytest.raises(Ty1Error, match='shares memory'):
        ops.adam_step_clipped(x, x, f(100), f(100), 1, 1.0)
    with pytest.raises(ValueError):
        ops.adam_step_clipped(x, f(100), f(100), f(100), 0, 1.0)
    with pytest.raises(TypeError):
        ops.adam_step_clipped(*[f(4).bfloat16() for _ in range(4)], 1, 1.0)
    assert bool((x == 1).all())
