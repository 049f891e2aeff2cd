"""CPU: what the adapter and clipping entry points refuse before any GPU work, through the C ABI and through yolo_amd.ops."""
import ctypes

import pytest
import torch

from yolo_amd import _lib, ops

P = 0x10000          # an aligned address that no refused call reads


def _fwd(**kw):
    a = dict(x=P, a=P, b=P, index=P, scale=P, out=P, h=None, N=2, K=8, U=8, L=2, R=4, ldx=8, lda=8, sa=32, ldb=8, sb=32, ldo=8,
             accumulate=0, ws=P, ws_bytes=1 << 20, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


def _bwd(**kw):
    a = dict(dz=P, x=P, a=P, b=P, index=P, scale=P, h=None, da=P, db=P, dx=None, N=2, K=8, U=8, L=2, R=4, lddz=8, ldx=8, lda=8, sa=32,
             ldb=8, sb=32, ldda=8, sda=32, lddb=8, sdb=32, lddx=8, ws=P, ws_bytes=1 << 20, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


def _refused(name, args, text):
    L = _lib.lib()
    assert getattr(L, name)(*args) != 0
    assert text in L.ty1_last_error().decode(), L.ty1_last_error()


@pytest.mark.parametrize('suffix', ['f32', 'bf16'])
@pytest.mark.parametrize('kw, text', [
    (dict(N=-1), 'bad dimensions'), (dict(N=(1 << 30) + 1), 'bad dimensions'), (dict(K=0), 'bad dimensions'), (dict(U=0), 'bad dimensions'),
    (dict(L=0), '0 adapters'), (dict(L=4097), '4097 adapters'), (dict(R=0), 'rank 0'), (dict(R=129), 'rank 129'),
    (dict(x=None), 'null pointer'), (dict(b=None), 'null pointer'), (dict(index=None), 'null pointer'), (dict(scale=None), 'null pointer'),
    (dict(x=P + 1), 'not aligned'), (dict(scale=P + 2), 'not aligned'), (dict(ldx=-8), 'negative strides'), (dict(sb=-1), 'negative strides'),
    (dict(ws=None), 'workspace'), (dict(ws=P + 8), 'workspace'), (dict(ws_bytes=16), 'workspace')])
def test_adapter_calls_refused(suffix, kw, text):
    _refused(f'ty1_adapter_forward_{suffix}', _fwd(**kw), text)
    _refused(f'ty1_adapter_backward_{suffix}', _bwd(**kw), text)


def test_adapter_outputs_refused():
    _refused('ty1_adapter_forward_f32', _fwd(out=None), 'null pointer')
    _refused('ty1_adapter_forward_f32', _fwd(out=P + 2), 'not aligned')
    _refused('ty1_adapter_forward_f32', _fwd(ldo=7), 'overlap')
    for kw in (dict(da=None), dict(db=None), dict(dz=None)):
        _refused('ty1_adapter_backward_f32', _bwd(**kw), 'null pointer')
    for kw in (dict(ldda=7), dict(sda=31), dict(lddb=4), dict(sdb=8), dict(dx=P, lddx=7)):
        _refused('ty1_adapter_backward_f32', _bwd(**kw), 'overlap')
    assert _lib.lib().ty1_adapter_forward_f32(*_fwd(N=0, x=None, out=None, ws=None)) == 0          # nothing to do


def test_adapter_workspace_query():
    L, n = _lib.lib(), ctypes.c_size_t(0)
    for sizes in ((1, 12544, 1470, 4, 8), (4096, 12544, 539, 64, 64), (0, 1, 1, 1, 1), (300, 7, 5, 4096, 128)):
        assert L.ty1_adapter_workspace_bytes(*sizes, 0, ctypes.addressof(n)) == 0 and 0 <= n.value < 1 << 30
        assert L.ty1_adapter_workspace_bytes(*sizes, 1, ctypes.addressof(n)) == 0 and 0 < n.value < 1 << 30
    assert L.ty1_adapter_workspace_bytes(1, 8, 8, 1, 129, 0, ctypes.addressof(n)) != 0
    assert L.ty1_adapter_workspace_bytes(1, 8, 8, 1, 1, 0, None) != 0


def _ptrs(*a):
    return (ctypes.c_void_p * len(a))(*a)


def _i64s(*a):
    return (ctypes.c_int64 * len(a))(*a)


def test_clip_calls_refused():
    g, o, c = _ptrs(P, P + 4096), _ptrs(P + 8192, P + 16384), _i64s(1000, 8)
    big = (1 << 24, None)                       # workspace bytes, stream
    kinds = lambda *a: (ctypes.c_int * len(a))(*a)
    for args, text in (((g, c, None, 0, P, P, *big), 'no tensors'), ((None, c, None, 2, P, P, *big), 'null list'),
                       ((g, None, None, 2, P, P, *big), 'no tensors'), ((g, _i64s(5, -1), None, 2, P, P, *big), 'tensor 1 has -1'),
                       ((g, c, kinds(0, 2), 2, P, P, *big), 'tensor 1 has type 2'), ((_ptrs(P, None), c, None, 2, P, P, *big), 'tensor 1: null'),
                       ((_ptrs(P, P + 4098), c, None, 2, P, P, *big), 'misaligned'), ((g, c, None, 2, None, P, *big), 'null pointer'),
                       ((g, c, None, 2, P, None, *big), 'workspace'), ((g, c, None, 2, P, P, 8, None), 'workspace')):
        _refused('ty1_grad_norm', args, text)
    for args, text in (((g, o, c, None, 2, 0.0, P, P, *big), 'must be positive'), ((g, o, c, None, 2, -1.0, P, P, *big), 'must be positive'),
                       ((g, o, c, None, 2, float('nan'), P, P, *big), 'must be positive'), ((g, None, c, None, 2, 1.0, P, P, *big), 'null list'),
                       ((g, _ptrs(P + 4, P + 8192), c, None, 2, 1.0, 0x8000, P, *big), 'shares memory'),          # shifted onto itself
                       ((g, _ptrs(P + 8192, P + 8196), c, None, 2, 1.0, 0x8000, P, *big), 'shares memory'),       # outputs on one another
                       ((g, _ptrs(P + 4096, P), _i64s(8, 8), None, 2, 1.0, 0x8000, P, *big), 'shares memory'),    # crosswise
                       ((_ptrs(P, P), _ptrs(P, P), _i64s(8, 8), None, 2, 1.0, 0x8000, P, *big), 'shares memory'),  # one tensor twice
                       ((g, o, c, None, 2, 1.0, P, P, 8, None), 'workspace')):
        _refused('ty1_clip_grad_norm', args, text)


def test_clipped_adam_calls_refused():
    lists = [_ptrs(P + 65536 * l, P + 65536 * l + 8192) for l in range(4)]
    c = _i64s(1000, 8)
    tail = (1e-3, 0.9, 0.999, 1e-7, 1, 0x8000, P, 1 << 24, None)
    _refused('ty1_adam_step_clip_f32', (*lists, c, 0, 1.0, *tail), 'no tensors')
    _refused('ty1_adam_step_clip_f32', (*lists, c, 2, 0.0, *tail), 'must be positive')
    _refused('ty1_adam_step_clip_f32', (*lists, c, 2, 1.0, 1e-3, 0.9, 0.999, 1e-7, 0, P, P, 1 << 24, None), 'bad t=0')
    _refused('ty1_adam_step_clip_f32', (lists[0], lists[0], *lists[2:], c, 2, 1.0, *tail), 'shares memory')
    _refused('ty1_adam_step_clip_f32', (*lists[:3], lists[2], c, 2, 1.0, *tail), 'shares memory')
    _refused('ty1_adam_step_clip_f32', (*lists, c, 2, 1.0, 1e-3, 0.9, 0.999, 1e-7, 1, None, P, 1 << 24, None), 'null pointer')
    for betas in ((1.0, 0.999), (0.9, 1.0), (-0.1, 0.999), (0.9, float('nan'))):
        _refused('ty1_adam_step_clip_f32', (*lists, c, 2, 1.0, 1e-3, *betas, 1e-7, 1, 0x8000, P, 1 << 24, None), 'betas')
    _refused('ty1_adam_step_clip_f32', (*lists, c, 2, 1.0, 1e-3, 0.9, 0.999, 1e-7, 1, P + 3996, P, 1 << 24, None), 'shares memory')   # the norm in p


def test_ops_refuse_host_tensors():
    f = lambda *s: torch.zeros(s)
    with pytest.raises(TypeError, match='on the GPU'):
        ops.adapter_forward(f(2, 8), f(1, 4, 8), f(1, 4, 8), torch.zeros(2, dtype=torch.int32), f(1))
    with pytest.raises(TypeError, match='on the GPU'):
        ops.adapter_backward(f(2, 8), f(2, 8), f(1, 4, 8), f(1, 4, 8), torch.zeros(2, dtype=torch.int32), f(1))
    for call in (lambda: ops.grad_norm(f(3)), lambda: ops.clip_grad_norm([f(3)], 1.0), lambda: ops.adam_step_clipped(f(3), f(3), f(3), f(3), 1, 1.0)):
        with pytest.raises(TypeError, match='on the GPU'):
            call()
    for bad in (0, -1, float('nan')):
        with pytest.raises(ValueError, match='max_norm'):
            ops.clip_grad_norm([f(3)], bad)
    with pytest.raises(ValueError, match='no tensors'):
        ops.grad_norm([])
    with pytest.raises(TypeError, match='expected tensors'):
        ops.grad_norm([None])
