"""The adapter and gradient-clipping operators of yolo_amd.ops as a user's program calls them, beside their plain forms.

Four operators, in the shapes of this repository's detector: 12544 features per image, a Dense layer of 1470 units (20
classes) or 539 units (one class), and the 1472 x 12544 Dense weight with its bias as the trained tensors.

  adapter   delta[n] = scale[i] * (x[n] . A[i]^T) . B[i] for i = index[n]: the low-rank adapters of many requests (one per
            camera or customer) in one batch, beside the Dense layer that they share
  backward  gradients of that product for A, B and, where asked for, x
  clip      the global norm over many gradient tensors, and the tensors scaled down to a maximal norm
  adam      the optimiser step that clips by the global norm and updates parameters and moments of many tensors

`own` picks the side: False computes the operators with elementary torch operations, True calls the library's kernels.
"""
import math

import torch

own = False

FEATURES, UNITS_C20, UNITS_C1 = 12544, 1470, 539
DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases
def _adapter(name, n, l, r, dtype, k=FEATURES, u=UNITS_C20, none=0):
    return dict(name=name, op='adapter', n=n, l=l, r=r, k=k, u=u, dtype=dtype, none=none)


def _backward(name, n, l, r, dtype, k=FEATURES, u=UNITS_C20, none=0, dx=False):
    return dict(name=name, op='backward', n=n, l=l, r=r, k=k, u=u, dtype=dtype, none=none, dx=dx)


def listed():
    return [
        # one camera frame at a time, four adapters resident: latency
        _adapter('adapter_frame', 1, 4, 8, 'f32'),
        # a server's batch of 64 images from 16 cameras, a few requests on the shared weights alone
        _adapter('adapter_batch', 64, 16, 16, 'f32', none=8),
        # the bf16 network's batch of 128 images
        _adapter('adapter_batch_bf16', 128, 32, 16, 'bf16'),
        # odd everything: another image size's features cut to an odd width, the one-class head, an odd rank
        _adapter('adapter_odd', 333, 7, 11, 'f32', k=4999, u=UNITS_C1, none=5),
        # the one-class detector at 4096 images over 64 adapters of rank 64: throughput
        _adapter('adapter_4096', 4096, 64, 64, 'f32', u=UNITS_C1),
        # the training step of 32 images, four adapters in training, backbone frozen
        _backward('backward_step', 32, 4, 16, 'f32'),
        # a bf16 batch of 500 images, gradients in float32
        _backward('backward_bf16', 500, 8, 16, 'bf16', u=UNITS_C1, none=3),
        # a large batch with the gradient of the features too (a trained layer in front)
        _backward('backward_2048_dx', 2048, 16, 32, 'f32', dx=True),
        # the Dense layer's gradient bucket: one large tensor, one small one
        dict(name='clip_dense', op='clip', sizes='dense', count=2, dtype='f32', ratio=0.5),
        # the gradients of 31 adapters of rank 16 held one by one: 62 tensors of two sizes
        dict(name='clip_adapters', op='clip', sizes='adapters', count=62, dtype='mixed', ratio=0.25),
        # the optimiser step of the Dense layer
        dict(name='adam_dense', op='adam', sizes='dense', count=2, dtype='f32', ratio=0.5, t=3),
        # the optimiser step of a small bank: 4 adapters, 8 tensors
        dict(name='adam_adapters', op='adam', sizes='adapters', count=8, dtype='f32', ratio=2.0, t=100),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(['adapter', 'adapter', 'backward', 'backward', 'clip', 'adam'])
    if kind in ('adapter', 'backward'):
        back = kind == 'backward'
        n, l, r = _log_int(rng, 1, 2048 if back else 4096), _log_int(rng, 1, 16 if back else 64), _log_int(rng, 1, 32 if back else 64)
        k = FEATURES if rng.random() < 0.5 else _log_int(rng, 64, FEATURES)
        u = rng.choice([UNITS_C20 if back else UNITS_C1, UNITS_C1, _log_int(rng, 7, UNITS_C1)])
        case = dict(op=kind, n=n, l=l, r=r, k=k, u=u, dtype=rng.choice(['f32', 'bf16']),
                    none=rng.choice([0, 0, n // 8, n // 3]))
        if back:
            case['dx'] = rng.random() < 0.4
        return case
    case = dict(op=kind, sizes='ragged', count=_log_int(rng, 1, 200), largest=_log_int(rng, 1, 80000),
                dtype='f32' if kind == 'adam' else rng.choice(['f32', 'bf16', 'mixed']), ratio=rng.choice([0.01, 0.5, 0.9, 3.0]))
    if kind == 'adam':
        case['t'] = _log_int(rng, 1, 10000)
    return case


# --------------------------------------------------------------------------------------------------------------- inputs
def _sizes(case):
    if case['sizes'] == 'dense':
        return [1472 * FEATURES, UNITS_C20]
    if case['sizes'] == 'adapters':
        return [(FEATURES if i % 2 == 0 else UNITS_C20) * 16 for i in range(case['count'])]
    # ragged: from the largest downwards by a fixed stride through the range, odd sizes and ones among them
    top = case['largest']
    return [1 + (top - 1) * ((7919 * i) % 1009) // 1008 for i in range(1, case['count'] + 1)]


def _active(case):
    return case['n'] - case['none'], min(case['l'], case['n'] - case['none'])


def _index(case, gen):
    """One adapter per image: each used at least once where the images suffice, a few popular ones, -1 where none applies."""
    active, used = _active(case)
    first = torch.randperm(case['l'], generator=gen, device='cuda')[:used]
    popular = (torch.rand(active - used, generator=gen, device='cuda').square() * used).long().clamp(max=max(used - 1, 0))
    index = torch.cat([first, first[popular] if used else first, torch.full((case['none'],), -1, dtype=torch.long, device='cuda')])
    return index[torch.randperm(case['n'], generator=gen, device='cuda')].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device='cuda')
    if case['op'] in ('adapter', 'backward'):
        n, l, r, k, u = (case[c] for c in 'nlrku')
        dt = DTYPES[case['dtype']]
        x = randn(n, k)
        x = torch.where(x > 0, x, 0.1 * x).to(dt)                      # the backbone's features end in a LeakyReLU
        a = ((torch.rand((l, r, k), generator=gen, device='cuda') * 2 - 1) / math.sqrt(k)).to(dt)
        b = (randn(l, r, u) * 0.05).to(dt)
        scale = 0.5 + torch.rand(l, generator=gen, device='cuda')
        index = _index(case, gen)
        state = dict(op=case['op'], x=x, a=a, b=b, scale=scale, index=index)
        if case['op'] == 'backward':
            state['dz'] = randn(n, u) * randn(n, 1).square() * 0.01     # a few images carry most of the loss
            state['h'] = _hidden(x, a, index)                           # what the forward call kept
            state['dx'] = case['dx']
        return state
    sizes = _sizes(case)
    types = [torch.bfloat16 if case['dtype'] == 'bf16' or (case['dtype'] == 'mixed' and i % 4 == 3) else torch.float32
             for i in range(len(sizes))]
    grads, kept = _tensors(case, sizes, types)
    for i, g in enumerate(grads):
        g.copy_(randn(g.numel()) * (0.001 * 3.0 ** (i % 5)))
    # the expected norm of these values, times the ratio: below one the call clips, above it leaves the values as they are
    norm = math.sqrt(sum(m * (0.001 * 3.0 ** (i % 5)) ** 2 for i, m in enumerate(sizes)))
    state = dict(op=case['op'], grads=grads, max_norm=case['ratio'] * norm)
    if case['op'] == 'clip':
        state['out'], state['whole'] = _tensors(case, sizes, types)
    else:
        state['whole'] = []
        for name, values in (('p', lambda m: randn(m) * 0.02), ('m', lambda m: randn(m) * 0.0005), ('v', lambda m: randn(m).square() * 1e-6)):
            state[name], kept = _tensors(case, sizes, types)
            state['whole'] += kept
            for t in state[name]:
                t.copy_(values(t.numel()))
        state['t'] = case['t']
    return state


def _tensors(case, sizes, types):
    """Tensors of these sizes and the buffers they lie in: each one its own or, for the ragged sizes, one behind the other in
    a bucket for each type, at whatever offset that gives."""
    if case['sizes'] != 'ragged':
        own_each = [torch.zeros(m, dtype=t, device='cuda') for m, t in zip(sizes, types)]
        return own_each, own_each
    views, buckets = [None] * len(sizes), []
    for t in sorted(set(types), key=str):
        at = [i for i in range(len(sizes)) if types[i] == t]
        buckets.append(torch.zeros(sum(sizes[i] for i in at), dtype=t, device='cuda'))
        for i, view in zip(at, buckets[-1].split([sizes[i] for i in at])):
            views[i] = view
    return views, buckets


def _hidden(x, a, index):
    """h[n] = x[n] . A[index[n]]^T in float32, zero where no adapter applies."""
    l, r, k = a.shape
    every = (x.float() @ a.float().reshape(l * r, k).t()).view(-1, l, r)
    i = index.long()
    h = every[torch.arange(len(i), device=i.device), i.clamp(min=0)]
    return torch.where((i >= 0)[:, None], h, torch.zeros_like(h))


# ------------------------------------------------------------------------------------------------------- the plain forms
def _spread(rows, index, scale):
    """(N, R) -> (N, L * R): row n at its adapter's place, times the adapter's scale where one is given, zeros elsewhere."""
    l = scale.shape[0]
    mine = index[:, None] == torch.arange(l, device=index.device, dtype=index.dtype)[None]
    wide = rows[:, None, :] * scale[None, :, None]
    return torch.where(mine[:, :, None], wide, torch.zeros_like(wide)).reshape(rows.shape[0], -1)


def _plain_adapter(s):
    l, r, u = s['b'].shape
    h = _hidden(s['x'], s['a'], s['index'])
    return _spread(h, s['index'], s['scale']) @ s['b'].float().reshape(l * r, u)


def _plain_backward(s):
    x, a, b, dz, index, scale = s['x'].float(), s['a'].float(), s['b'].float(), s['dz'], s['index'], s['scale']
    l, r, k = a.shape
    g = _spread(_hidden(dz, b, index), index, scale)
    da = (g.t() @ x).view(l, r, k)
    db = (_spread(s['h'], index, scale).t() @ dz).view(l, r, -1)
    return [da, db] + ([g @ a.reshape(l * r, k)] if s['dx'] else [])


def _plain_coefficient(grads, max_norm):
    square = sum(g.float().square().sum(dtype=torch.float64) for g in grads)
    norm = square.sqrt()
    return norm.float().reshape(1), (max_norm / norm.clamp(min=max_norm)).float()


def _plain_clip(s):
    norm, c = _plain_coefficient(s['grads'], s['max_norm'])
    for g, out in zip(s['grads'], s['out']):
        out.copy_(g.float() * c)
    return [norm] + s['whole']


def _plain_adam(s, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-7):
    norm, c = _plain_coefficient(s['grads'], s['max_norm'])
    rate = lr * math.sqrt(1 - beta2 ** s['t']) / (1 - beta1 ** s['t'])
    for p, g, m, v in zip(s['p'], s['grads'], s['m'], s['v']):
        g = g * c
        m.copy_(beta1 * m + (1 - beta1) * g)
        v.copy_(beta2 * v + (1 - beta2) * g * g)
        p.sub_(rate * m / (v.sqrt() + eps))
    return [norm] + s['whole']


# ------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    s = state
    if not own:
        return {'adapter': _plain_adapter, 'backward': _plain_backward, 'clip': _plain_clip, 'adam': _plain_adam}[s['op']](s)
    from yolo_amd import ops
    if s['op'] == 'adapter':
        return ops.adapter_forward(s['x'], s['a'], s['b'], s['index'], s['scale'])
    if s['op'] == 'backward':
        da, db, dx = ops.adapter_backward(s['dz'], s['x'], s['a'], s['b'], s['index'], s['scale'], s['h'], want_dx=s['dx'])
        return [da, db, dx] if s['dx'] else [da, db]
    if s['op'] == 'clip':
        return [ops.clip_grad_norm(s['grads'], s['max_norm'], out=s['out'])] + s['whole']
    return [ops.adam_step_clipped(s['p'], s['grads'], s['m'], s['v'], s['t'], s['max_norm'])] + s['whole']


# ----------------------------------------------------------------------------------------------------- from the definition
def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] in ('adapter', 'backward'):
        n, l, r, k, u = (case[c] for c in 'nlrku')
        back = case['op'] == 'backward'
        out = torch.zeros((n, u), dtype=torch.float64, device='cuda')
        da, db = (torch.zeros(t.shape, dtype=torch.float64, device='cuda') for t in (s['a'], s['b']))
        dx = torch.zeros((n, k), dtype=torch.float64, device='cuda') if back and case['dx'] else None
        for i in range(l):
            rows = torch.nonzero(s['index'] == i).flatten()
            if rows.numel() == 0:
                continue
            x, a, b, c = s['x'][rows].double(), s['a'][i].double(), s['b'][i].double(), s['scale'][i].double()
            if not back:
                out[rows] = c * torch.matmul(torch.matmul(x, a.t()), b)
                continue
            dz, h = s['dz'][rows].double(), s['h'][rows].double()
            g = c * torch.matmul(dz, b.t())
            da[i] = torch.matmul(g.t(), x)
            db[i] = c * torch.matmul(h.t(), dz)
            if dx is not None:
                dx[rows] = torch.matmul(g, a)
        return ([da, db, dx] if dx is not None else [da, db]) if back else out
    total = torch.zeros((), dtype=torch.float64, device='cuda')
    for g in s['grads']:
        total = total + torch.dot(g.double(), g.double())
    norm = float(total.sqrt())
    c = min(1.0, s['max_norm'] / norm)
    first = torch.tensor([norm], dtype=torch.float64, device='cuda')
    if case['op'] == 'clip':
        return [first] + _laid_out(case, s['grads'], [g.double() * c for g in s['grads']])
    t, params, means, squares = case['t'], [], [], []
    for p, g, m, v in zip(s['p'], s['grads'], s['m'], s['v']):
        g = g.double() * c
        means.append(m.double() + (1 - 0.9) * (g - m.double()))
        squares.append(v.double() + (1 - 0.999) * (g.pow(2) - v.double()))
        unbiased = 1e-3 * (1 - 0.999 ** t) ** 0.5 / (1 - 0.9 ** t)
        params.append(p.double() - unbiased * means[-1] / (squares[-1].pow(0.5) + 1e-7))
    return [first] + [t for values in (params, means, squares) for t in _laid_out(case, s['grads'], values)]


def _laid_out(case, like, values):
    """The values as `_tensors` lays the tensors out: each its own, or one behind the other for each type."""
    if case['sizes'] != 'ragged':
        return values
    names = sorted({str(g.dtype) for g in like})
    return [torch.cat([v for g, v in zip(like, values) if str(g.dtype) == name]) for name in names]


# ------------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    if case['op'] in ('adapter', 'backward'):
        n, l, r, k, u = (case[c] for c in 'nlrku')
        active, used = _active(case)
        size = 2 if case['dtype'] == 'bf16' else 4
        if case['op'] == 'adapter':
            return dict(bytes=active * k * size + used * r * (k + u) * size + n * 4 + l * 4 + n * u * 4,
                        flops=2 * active * r * (k + u))
        nbytes = active * (k * size + u * 4 + r * 4) + used * r * u * size + l * r * (k + u) * 4 + n * 4 + l * 4
        flops = 2 * active * r * (k + 2 * u)
        if case['dx']:
            nbytes += used * r * k * size + n * k * 4
            flops += 2 * active * r * k
        return dict(bytes=nbytes, flops=flops)
    total = size = 0
    for i, m in enumerate(_sizes(case)):
        half = case['dtype'] == 'bf16' or (case['dtype'] == 'mixed' and i % 4 == 3)
        total += m
        size += m * (2 if half else 4)
    if case['op'] == 'clip':
        return dict(bytes=2 * size + 4, flops=3 * total)       # each value read once and written once
    return dict(bytes=size + 6 * 4 * total + 4, flops=16 * total)
