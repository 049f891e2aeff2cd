"""CPU: the norm and clipping entry points refuse a workspace or a norm that their float64 and float32 accesses cannot use, and a
workspace inside a tensor of the call (its partial sums would be written over values that are still to be read)."""
import ctypes

import pytest

from yolo_amd import _lib

P, NORM, WS = 0x100000, 0x8000, 0x900000          # aligned addresses that no refused call reads


def _array(kind, *a):
    return (kind * len(a))(*a)


def _call(name, norm=NORM, ws=WS, counts=(1000, 8), lists=None, dtypes=None):
    """A call with one list (norm), two (clip) or four (Adam) of two tensors; -> status, message."""
    n_lists = {'ty1_grad_norm': 1, 'ty1_clip_grad_norm': 2, 'ty1_adam_step_clip_f32': 4}[name]
    lists = lists or [(P + 0x10000 * l, P + 0x10000 * l + 0x2000) for l in range(n_lists)]
    ptrs = [_array(ctypes.c_void_p, *l) for l in lists]
    c, n = _array(ctypes.c_int64, *counts), len(counts)
    kinds = dtypes and _array(ctypes.c_int, *dtypes)
    size = 1 << 20
    args = {'ty1_grad_norm': lambda: (*ptrs, c, kinds, n, norm, ws, size, None),
            'ty1_clip_grad_norm': lambda: (*ptrs, c, kinds, n, 1.0, norm, ws, size, None),
            'ty1_adam_step_clip_f32': lambda: (*ptrs, c, n, 1.0, 1e-3, 0.9, 0.999, 1e-7, 1, norm, ws, size, None)}[name]()
    L = _lib.lib()
    return getattr(L, name)(*args), L.ty1_last_error().decode()


ENTRIES = ['ty1_grad_norm', 'ty1_clip_grad_norm', 'ty1_adam_step_clip_f32']


@pytest.mark.parametrize('name', ENTRIES)
@pytest.mark.parametrize('kw', [dict(ws=WS + 4), dict(ws=WS + 1), dict(norm=NORM + 2), dict(norm=NORM + 1)])
def test_misaligned(name, kw):
    rc, text = _call(name, **kw)
    assert rc != 0 and 'not aligned' in text, text


@pytest.mark.parametrize('name', ENTRIES)
def test_workspace_in_a_tensor(name):
    need = ctypes.c_size_t(0)
    assert _lib.lib().ty1_grad_norm_workspace_bytes(2, ctypes.addressof(need)) == 0
    size = need.value
    n_lists = {'ty1_grad_norm': 1, 'ty1_clip_grad_norm': 2, 'ty1_adam_step_clip_f32': 4}[name]
    for l in range(n_lists):
        first, second = P + 0x10000 * l, P + 0x10000 * l + 0x2000
        # at a tensor's start, at its last value, ending in its first, around the second (inside one buffer of gradients)
        for ws in (first, first + 3992, first - size + 8, second - 64):
            rc, text = _call(name, ws=ws)
            assert rc != 0 and 'shares memory' in text and 'workspace' in text, (hex(ws), text)
    for ws in (NORM - 8, NORM - size + 8, NORM):
        rc, text = _call(name, ws=ws)
        assert rc != 0 and 'shares memory' in text and 'workspace' in text, text


@pytest.mark.parametrize('name', ENTRIES[:2])
def test_a_bf16_tensor_counts_two_bytes_a_value(name):
    lists = [(P + 0x10000 * l, P + 0x10000 * l + 0x2000) for l in range(ENTRIES.index(name) + 1)]
    rc, text = _call(name, lists=lists, dtypes=(1, 0), ws=P + 1992)
    assert rc != 0 and 'shares memory' in text and 'workspace' in text, text
