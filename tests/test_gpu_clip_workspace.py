"""GPU: the norm through the C entry point with its workspace directly behind the tensors, as close as it is allowed to lie."""
import ctypes

import pytest
import torch

from yolo_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('n', [1000, 40000])
def test_workspace_right_behind_a_tensor(kind, n):
    size = ctypes.c_size_t(0)
    _lib.call('ty1_grad_norm_workspace_bytes', 1, ctypes.addressof(size))
    dt = torch.float32 if kind == 'f32' else torch.bfloat16
    held = n * dt.itemsize                                      # a multiple of 8
    buf = torch.zeros(held + size.value + 8, dtype=torch.uint8, device='cuda:0')
    g, norm = buf[:held].view(dt), buf[held + size.value:held + size.value + 4].view(torch.float32)
    g.copy_(torch.randint(-2, 3, (n,), generator=torch.Generator().manual_seed(n)))
    keep = g.clone()
    want = float((keep.double() ** 2).sum().sqrt())             # whole numbers: their squares and sums are exact
    _lib.call('ty1_grad_norm', (ctypes.c_void_p * 1)(g.data_ptr()), (ctypes.c_int64 * 1)(n), (ctypes.c_int * 1)(int(kind == 'bf16')), 1,
              norm.data_ptr(), buf.data_ptr() + held, size.value, _lib.current_stream())
    assert torch.equal(g, keep) and float(norm) == float(torch.tensor(want, dtype=torch.float32))
